"""Host side of ragged serving: the descriptor and the refusals of the calls (no kernel is launched)."""
import os
import re

import numpy as np
import pytest

import tl_hip as xp
from test_abi import HEADER, _Memory


def test_paged_desc_layout_matches_header():
    """The packed descriptor's format against tl_paged_desc, field for field."""
    body = re.search(r"typedef struct tl_paged_desc \{(.*?)\} tl_paged_desc;", open(HEADER).read(), re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    code = ""
    for decl in body.split(";"):
        decl = decl.strip()
        if decl:
            code += "P" if "*" in decl else {"int64_t": "q", "int32_t": "i"}[decl.split()[0]] * (decl.count(",") + 1)
    assert xp._PAGED_DESC.format == "@" + code + "0q"


def _t(shape, dt="bf16", pitch=None):
    return xp.DeviceTensor(shape, dt, pitch=pitch, buf=_Memory(1 << 30))


def _pages(**kw):
    d = dict(k_pages=_t((6, 2, 16, 64)), v_pages=_t((6, 2, 16, 64)), page_table=_t((3, 4), "int32"),
             q_start=_t((4,), "int32"), kv_len=_t((3,), "int32"))
    d.update(kw)
    return d


@pytest.mark.parametrize("change", [
    dict(k_pages=_t((6, 2, 16, 32))), dict(v_pages=_t((6, 2, 16, 64), "fp32")), dict(v_pages=_t((6, 2, 64))),
    dict(k_pages=_t((6, 2, 16, 64), pitch=72), v_pages=_t((6, 2, 16, 64), pitch=72)),
    dict(page_table=_t((2, 4), "int32")), dict(page_table=_t((3, 4), "int64")), dict(q_start=_t((3,), "int32")),
    dict(q_start=_t((4, 1), "int32", pitch=2)), dict(kv_len=_t((3,), "int64"))])
def test_batches_of_other_shapes_are_refused(change):
    with pytest.raises(ValueError):
        xp.paged_attention(_t((5, 256)), **_pages(**change), max_q=1, divisor=8.0)
    with pytest.raises(ValueError):
        xp.kv_append(_t((5, 512)), **_pages(**change), n_heads_q=4)


def test_rows_of_other_shapes_are_refused():
    for q in (_t((5, 250)), _t((5, 4, 64)), _t((5, 256), "fp32")):
        with pytest.raises(ValueError):
            xp.paged_attention(q, **_pages(), max_q=1, divisor=8.0)
    for out in (_t((5, 192)), _t((4, 256)), _t((5, 256), "fp32")):
        with pytest.raises(ValueError):
            xp.paged_attention(_t((5, 256)), **_pages(), max_q=1, divisor=8.0, out=out)
    rope = _t((2, 100, 32), "fp32")
    for kw in (dict(qkv=_t((5, 448))), dict(rope=_t((2, 100, 64), "fp32")), dict(rope=_t((2, 100, 32))),
               dict(rope=rope, out=_t((5, 192))), dict(out=_t((5, 256))), dict(rope=rope, out=_t((5, 256), "fp32"))):
        with pytest.raises(ValueError):
            xp.kv_append(**{**dict(qkv=_t((5, 512)), n_heads_q=4), **_pages(), **kw})


def test_i32_add_refuses_other_tensors():
    for t in (_t((3,), "int64"), _t((3, 1), "int32", pitch=2)):
        with pytest.raises(ValueError):
            xp.i32_add(t, 1)


class _FakeContext:
    """A context that hands out no memory: only the geometry of what is made is looked at."""
    handle, capture = 1, None


@pytest.fixture
def cache(monkeypatch):
    import layers

    class Host:
        def __init__(self, a):
            self.a = np.array(a)

    monkeypatch.setattr(layers.xp, "zeros", lambda shape, dtype: _t(shape, dtype))
    monkeypatch.setattr(layers.xp, "array", lambda a, dtype=None: Host(a))
    return layers.PagedKVCache(2, 12, 1, 64, "bf16", page_size=16)


def test_paged_cache_hands_out_and_takes_back_pages(cache):
    a, b = cache.add(), cache.add()
    one = cache.batch([a, b], [20, 1])
    assert [len(cache.pages[s]) for s in (a, b)] == [2, 1] and len(set(cache.pages[a] + cache.pages[b])) == 3
    assert one.q_start.a.tolist() == [0, 20, 21] and one.kv_len.a.tolist() == [20, 1] and one.page_table.a.shape == (2, 2)
    assert (one.rows, one.max_q, one.shared) == (21, 20, 0)
    assert one.last_rows().a.tolist() == [19, 20] and one.positions().a.tolist() == [*range(20), 0]
    two = cache.batch([b, a], [3, 0], reserve=12)
    assert two.kv_len.a.tolist() == [4, 20] and len(cache.pages[b]) == 1 and len(cache.pages[a]) == 2
    with pytest.raises(ValueError):
        two.last_rows()  # a has no row
    with pytest.raises(ValueError, match="full"):
        cache.batch([a, b], [16 * 11, 1])
    assert cache.lengths == {a: 20, b: 4}  # nothing was taken
    pages = set(cache.pages[a])
    cache.free(a)
    c = cache.add()
    cache.batch([c], [16 * 11])
    assert pages < set(cache.pages[c]) and not set(cache.pages[c]) & set(cache.pages[b])
    for args in (([b, b], [1, 1]), ([b], [1, 2]), ([b], [-1])):
        with pytest.raises(ValueError):
            cache.batch(*args)
    with pytest.raises(KeyError):
        cache.batch([a], [1])


def test_forked_sequences_share_whole_pages(cache):
    root = cache.add()
    cache.batch([root], [40])
    with pytest.raises(ValueError):
        cache.fork(root, 40)
    with pytest.raises(ValueError):
        cache.fork(root, 48)
    x, y = cache.fork(root, 32), cache.fork(root, 32)
    both = cache.batch([x, y], [5, 9])
    assert both.shared == 32 and cache.pages[x][:2] == cache.pages[y][:2] == cache.pages[root][:2]
    assert cache.pages[x][2] != cache.pages[y][2] and both.kv_len.a.tolist() == [37, 41]
    assert cache.batch([x, root], [1, 1]).shared == 32
    assert cache.batch([y], [1]).shared == 0
    z = cache.fork(x, 16)
    assert cache.batch([y, z], [1, 1]).shared == 16
    shared = cache.pages[root][:2]
    cache.free(root)
    cache.free(x)
    assert not set(shared) & set(cache._free)  # y still begins with them
    cache.free(y)
    cache.free(z)
    assert sorted(cache._free) == list(range(12))


def test_steps_advance_within_their_pages(cache, monkeypatch):
    import layers
    added = []
    monkeypatch.setattr(layers.xp, "i32_add", lambda t, n: added.append(n))
    s = cache.add()
    cache.batch([s], [14])
    step = cache.batch([s], [1], reserve=1)
    assert step.positions().a.tolist() == [14]
    step.advance()
    assert cache.lengths[s] == 16 and added == [1]
    with pytest.raises(ValueError):
        step.advance()
    assert added == [1]
    step._positions = None
    with pytest.raises(ValueError):
        step.positions()


def test_paged_cache_page_sizes():
    import layers
    for size in (0, 8, 24, 8192):
        with pytest.raises(ValueError):
            layers.PagedKVCache(0, 1, 1, 64, "bf16", page_size=size)
