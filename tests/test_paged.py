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
