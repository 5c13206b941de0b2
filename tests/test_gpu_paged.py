"""Ragged serving over a paged KV cache on the MI355X against float64: the append with its rotation,
and causal attention (whole prompts, pieces of prompts, single tokens; caps, windows, shared
prefixes). Tolerances are derived in paged_ref.Batch.tolerance and beside each test."""
import numpy as np
import pytest

from paged_ref import Batch, F32, rope64, rounded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def xp():
    import tl_hip
    tl_hip.ctx()
    return tl_hip


def _rows_tensor(xp, a, dt, extra=0, lead=0):
    """[N, cols] on the device, `extra` columns after and `lead` rows of NaN before it."""
    n, cols = a.shape
    host = np.full((n + lead, cols + extra), np.nan, F32)
    host[lead:, :cols] = a
    t = xp.array(host, dtype=dt)
    return xp.DeviceTensor((n, cols), dt, pitch=cols + extra, buf=t.buf,
                           offset=t.offset + lead * (cols + extra) * t.dtype.itemsize)


def _attend(xp, b, divisor=None, cap=0.0, window=0, shared=0, max_q=None, pitch=0, dev=None):
    """paged_attention of batch b with rows `pitch` columns apart; checked against float64, and that
    padding rows and the columns between rows stay as they were."""
    dev = dev or b.upload(xp)
    divisor = divisor or float(np.sqrt(b.d))
    n, w = b.n + b.pad, b.hq * b.d
    q = _rows_tensor(xp, b.q.reshape(n, w), b.dt, extra=pitch, lead=1 if pitch else 0)
    out = _rows_tensor(xp, np.full((n, w), 7.0, F32), b.dt, extra=2 * pitch, lead=0)
    xp.paged_attention(q, dev["k_pages"], dev["v_pages"], dev["page_table"], dev["q_start"], dev["kv_len"],
                       max_q=max_q or max(1, max(b.rows)), divisor=divisor, softcap=cap, window=window,
                       shared=shared, out=out)
    got = out.get().reshape(n, b.hq, b.d)
    want = b.want(divisor, cap, window)
    assert np.isfinite(got[:b.n]).all()
    err = np.abs(got[:b.n] - want) / b.tolerance(want)
    assert b.n == 0 or err.max() <= 1, (err.max(), np.unravel_index(err.argmax(), err.shape))
    assert (got[b.n:] == 7.0).all()
    if pitch:
        whole = xp.DeviceTensor((n * (w + 2 * pitch),), b.dt, buf=out.buf).get().reshape(n, -1)
        assert np.isnan(whole[:, w:]).all()
    return got


# ---- append ---------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("hq,hkv,d,page,lens,rows,pad", [
    (8, 1, 256, 64, [1, 70, 64, 2000], [1, 1, 1, 1], 0),
    (4, 4, 32, 16, [5, 40, 33, 16, 17], [5, 0, 33, 1, 17], 3),
    (10, 2, 64, 128, [300, 129], [301 - 1, 129], 2),
    (32, 4, 128, 32, list(range(1, 131)), [1 + i % 3 if i % 3 < i else 1 for i in range(130)], 0),
    (12, 12, 64, 16, [3], [3], 0)])
def test_append_rotates_and_writes_only_its_slots(xp, dt, hq, hkv, d, page, lens, rows, pad):
    rng = np.random.default_rng(d + page + len(lens))
    b = Batch(rng, lens, rows, hq, hkv, d, page, dt, pad=pad)
    n, w = b.n + pad, (hq + 2 * hkv) * d
    x = rounded(rng.standard_normal((n, w)), dt)
    x[b.n:] = np.nan
    # the cache before: what the sequences held without their new rows
    k0, v0 = b.k.copy(), b.v.copy()
    for s, (le, r) in enumerate(zip(lens, rows)):
        if r:
            at = b.slots(s, np.arange(le - r, le))
            k0[at] = v0[at] = np.nan
    dev = b.upload(xp)
    table = xp.rope_table(max(lens) + 1, d)
    for rope in (True, False):
        dev["k_pages"].set(k0)
        dev["v_pages"].set(v0)
        qkv = _rows_tensor(xp, x, dt, extra=16, lead=1)
        out = _rows_tensor(xp, np.full((n, hq * d), 7.0, F32), dt, extra=8) if rope else None
        q = xp.kv_append(qkv, **dev, n_heads_q=hq, rope=table if rope else None, out=out)
        q, k, v = q.get().reshape(n, hq, d), dev["k_pages"].get(), dev["v_pages"].get()
        want_k, want_v, want_q = k0.copy().astype(np.float64), v0.copy(), x[:, :hq * d].reshape(n, hq, d).astype(np.float64)
        for s, (le, r) in enumerate(zip(lens, rows)):
            if not r:
                continue
            i, pos = slice(b.start[s], b.start[s] + r), np.arange(le - r, le)
            xk = x[i, hq * d:(hq + hkv) * d].reshape(r, hkv, d)
            want_k[b.slots(s, pos)] = rope64(xk, pos) if rope else xk
            want_v[b.slots(s, pos)] = x[i, (hq + hkv) * d:].reshape(r, hkv, d)
            if rope:
                want_q[i] = rope64(want_q[i], pos)
        assert np.array_equal(v, want_v, equal_nan=True)
        if rope:
            # two products and a sum in fp32 with angles rounded to fp32 (4 roundings of values up to
            # |x1| + |x2| <= 12), then one rounding to bf16
            for got, want in ((k, want_k), (q[:b.n], want_q[:b.n])):
                assert np.array_equal(np.isnan(got), np.isnan(want))
                off = np.abs(got - want) - (2.0 ** -8 * np.abs(want) if dt == "bf16" else 0)
                assert np.nanmax(off) <= 12 * 4 * 2.0 ** -24
            assert (q[b.n:] == 7.0).all()
        else:
            assert np.array_equal(k, want_k.astype(F32), equal_nan=True)
            assert np.array_equal(q, x[:, :hq * d].reshape(n, hq, d), equal_nan=True)


def test_append_rows_without_a_place(xp):
    """Rows before position 0, past the table of angles, past the batch, or with a page that the cache
    lacks are not written, and all but the first are reported."""
    rng = np.random.default_rng(2)
    b = Batch(rng, [4, 20], [4, 3], 4, 2, 32, 16, "bf16")
    x = xp.array(rounded(rng.standard_normal((7, 8 * 32)), "bf16"), dtype="bf16")
    k0 = np.zeros_like(b.k)
    table = xp.rope_table(32, 32)

    def run(rope=table, **change):
        dev = b.upload(xp)
        dev["k_pages"].set(k0)
        dev["v_pages"].set(k0)
        for name, value in change.items():
            dev[name] = xp.array(np.asarray(value, np.int32))
        xp.kv_append(x, **dev, n_heads_q=4, rope=rope)
        return dev

    def written(dev):
        k = dev["k_pages"].get_raw()
        v = dev["v_pages"].get_raw()
        return (k != 0).any((1, 3)).sum(), (v != 0).any((1, 3)).sum()

    assert written(run()) == (7, 7)
    assert written(run(kv_len=[2, 20])) == (5, 5)  # two rows before the sequence's first position
    for change, n in ((dict(rope=xp.rope_table(18, 32)), 5), (dict(kv_len=[4, 1000]), 0 + 4),
                      (dict(kv_len=[-5, 20]), 3), (dict(q_start=[0, 4, 9]), 7), (dict(q_start=[0, 5, 4]), 4)):
        dev = run(**change)
        with pytest.raises(xp.BadInputError):
            xp.synchronize()
        assert written(dev)[0] <= max(n, 7)
    bad = b.table.copy()
    bad[0, 0] = b.n_pages
    dev = run(page_table=bad)
    with pytest.raises(xp.BadInputError, match="page"):
        xp.synchronize()
    assert written(dev) == (3, 3)
    bad[0, 0] = -1
    run(page_table=bad)
    with pytest.raises(xp.BadInputError, match="page"):
        xp.synchronize()


# ---- attention ------------------------------------------------------------------------
DIMS = [(4, 4, 32), (10, 2, 64), (12, 12, 64), (8, 2, 128), (32, 4, 128), (4, 1, 256), (8, 1, 256), (48, 2, 64), (3, 1, 32)]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("hq,hkv,d", DIMS)
def test_steps(xp, dt, hq, hkv, d):
    """Single tokens: lengths around pages and key blocks, sequences without a row."""
    for i, (page, lens, kw) in enumerate([
            (16, [1], {}), (16, [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 0, 129, 1000], {}),
            (64, [700, 64, 5], dict(cap=20.0)), (256, [1, 300, 513], dict(window=100)),
            (32, [40, 600, 1], dict(window=1, cap=5.0)), (4096, [5000, 31], {})]):
        rng = np.random.default_rng(d + i)
        rows = [1 if n and j % 5 != 3 else 0 for j, n in enumerate(lens)]
        b = Batch(rng, lens, rows, hq, hkv, d, page, dt, q_std=3.0, pad=i % 3)
        _attend(xp, b, pitch=16 * (i % 2), **kw)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("hq,hkv,d", DIMS)
def test_prompts(xp, dt, hq, hkv, d):
    """Whole prompts and pieces of prompts after a cached past, down to none and one row."""
    for i, (page, lens, rows, kw) in enumerate([
            (16, [1, 65, 17], [1, 65, 17], {}), (64, [300, 130, 3], [300, 2, 0], dict(cap=15.0)),
            (16, [129, 64, 200, 500], [128, 64, 33, 1], dict(window=50)), (128, [700], [250], {}),
            (32, [260, 90], [257, 90], dict(window=7, cap=30.0))]):
        rng = np.random.default_rng(d + 10 * i)
        b = Batch(rng, lens, rows, hq, hkv, d, page, dt, q_std=2.0, pad=2 * (i % 2))
        _attend(xp, b, pitch=8 * (i % 2), **kw)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("rows", [2, 4, 5, 16])
def test_a_few_rows_a_sequence(xp, dt, rows):
    """Between a step and a prompt: several rows of each sequence at once, and max_q larger than they are."""
    rng = np.random.default_rng(rows)
    lens = [rows, rows + 30, 400, 64, 65]
    b = Batch(rng, lens, [rows] * 4 + [1], 8, 2, 64, 16, dt)
    _attend(xp, b)
    _attend(xp, b, max_q=100)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("hq,hkv,d,page,shared,tails,rows", [
    (8, 1, 256, 64, 256, [1, 30, 64, 65, 100], 1), (12, 12, 64, 16, 1040, [5] * 9, 1),
    (32, 4, 128, 16, 64, [1 + i % 50 for i in range(70)], 1), (4, 4, 32, 128, 128, [200, 3], 2),
    (10, 2, 64, 32, 4064, [7, 40, 1], 1), (8, 2, 64, 16, 96, [90, 40, 64], 40)])
def test_shared_prefix(xp, dt, hq, hkv, d, page, shared, tails, rows):
    rng = np.random.default_rng(shared + d)
    n = [shared + t for t in tails]
    b = Batch(rng, n, [min(rows, t) for t in tails], hq, hkv, d, page, dt, shared=shared, q_std=2.0, pad=1)
    for cap in (0.0, 10.0):
        one = _attend(xp, b, shared=shared, cap=cap)
        two = _attend(xp, b, cap=cap)
        want = b.want(float(np.sqrt(d)), cap)
        assert (np.abs(one - two)[:b.n] <= 2 * b.tolerance(want)).all()


def test_shared_prefix_is_checked(xp):
    rng = np.random.default_rng(5)
    b = Batch(rng, [70, 80], [1, 1], 4, 2, 64, 16, "bf16", shared=64)
    dev = b.upload(xp)
    table = b.table.copy()
    table[1, 2] = table[1, 4]
    dev["page_table"] = xp.array(table)
    q = xp.array(b.q.reshape(2, -1), dtype="bf16")
    xp.paged_attention(q, *(dev[n] for n in ("k_pages", "v_pages", "page_table", "q_start", "kv_len")), max_q=1,
                       divisor=8.0, shared=64)
    with pytest.raises(xp.BadInputError, match="share"):
        xp.synchronize()
    dev = b.upload(xp)
    dev["kv_len"] = xp.array(np.array([70, 64], np.int32))  # the second row lies inside the prefix
    xp.paged_attention(q, *(dev[n] for n in ("k_pages", "v_pages", "page_table", "q_start", "kv_len")), max_q=1,
                       divisor=8.0, shared=64)
    with pytest.raises(xp.BadInputError):
        xp.synchronize()


@pytest.mark.parametrize("max_q", [1, 64])
def test_rows_before_the_first_position_give_zeros(xp, max_q):
    """A length shorter than its rows leaves the first ones nothing to see."""
    rng = np.random.default_rng(8)
    rows = [3, 1] if max_q == 64 else [1, 1]
    b = Batch(rng, [40, 9], rows, 4, 2, 64, 16, "bf16")
    dev = b.upload(xp)
    dev["kv_len"] = xp.array(np.array([1 if max_q == 64 else 0, 9], np.int32))
    q = xp.array(b.q.reshape(b.n, -1), dtype="bf16")
    out = xp.paged_attention(q, *(dev[n] for n in ("k_pages", "v_pages", "page_table", "q_start", "kv_len")),
                             max_q=max_q, divisor=8.0).get()
    k = rows[0] - (1 if max_q == 64 else 0)
    assert (out[:k] == 0).all() and np.isfinite(out).all() and (out[k:] != 0).any(-1).all()
    if max_q == 64:  # the third row sees position 0 alone
        assert np.array_equal(out[2].reshape(4, 64), np.repeat(b.values[0][0], 2, 0))


@pytest.mark.parametrize("rows,max_q", [(1, 1), (30, 30)])
def test_bad_bounds_and_pages_are_reported(xp, rows, max_q):
    rng = np.random.default_rng(9)
    b = Batch(rng, [100, 70], [rows, rows], 4, 2, 64, 16, "bf16")
    q = xp.array(b.q.reshape(b.n, -1), dtype="bf16")
    bad = b.table.copy()
    bad[1, 3] = -7
    for change in (dict(page_table=bad), dict(kv_len=[100, 100000]), dict(kv_len=[-3, 70]),
                   dict(q_start=[0, rows, 3 * rows]), dict(q_start=[0, rows, 0]), dict(q_start=[0, 2 * rows, 2 * rows])):
        dev = b.upload(xp)
        for name, value in change.items():
            dev[name] = xp.array(np.asarray(value, np.int32))
        xp.paged_attention(q, *(dev[n] for n in ("k_pages", "v_pages", "page_table", "q_start", "kv_len")),
                           max_q=max_q, divisor=8.0)
        with pytest.raises(xp.BadInputError):
            xp.synchronize()
    _attend(xp, b, max_q=max_q)  # and the next call is as before


def test_extreme_scores(xp):
    """Scores of +-1e4 and keys of the type's largest values leave finite results; an infinite score's
    row is NaN in a softmax and stays its own."""
    rng = np.random.default_rng(10)
    for rows in (1, 70):
        b = Batch(rng, [80, 75], [rows, rows], 4, 2, 64, 16, "bf16", q_std=1000.0)
        _attend(xp, b)
        _attend(xp, b, cap=50.0)
        b.q[0] = 0.0  # equal scores: the mean of the values
        _attend(xp, b)


def test_a_long_cache_past_32_bit_offsets(xp):
    """Pages whose elements lie past 2^31: the cache is larger than 4 GiB in each half."""
    rng = np.random.default_rng(11)
    page, hkv, d = 256, 4, 128
    n_pages = (1 << 31) // (page * hkv * d) + 64
    k = xp.empty((n_pages, hkv, page, d), "bf16")
    v = xp.empty((n_pages, hkv, page, d), "bf16")
    lens, rows = [300, 520], [1, 1]
    b = Batch(rng, lens, rows, 8, hkv, d, page, "bf16")
    where = n_pages - 1 - np.arange(b.n_pages)
    es = page * hkv * d * 2
    for i, p in enumerate(where):
        for t, host in ((k, b.k), (v, b.v)):
            xp.DeviceTensor((hkv, page, d), "bf16", buf=t.buf, offset=t.offset + int(p) * es).set(host[i])
    used = (b.table >= 0) & (b.table < b.n_pages)
    b.table[used] = where[b.table[used]]
    dev = dict(k_pages=k, v_pages=v, page_table=xp.array(b.table), q_start=xp.array(b.start),
               kv_len=xp.array(np.array(lens, np.int32)))
    _attend(xp, b, dev=dev)
    x = rounded(rng.standard_normal((2, (8 + 2 * hkv) * d)), "bf16")
    xp.kv_append(xp.array(x, dtype="bf16"), **dev, n_heads_q=8)
    for s, n in enumerate(lens):
        p, at = b.table[s, (n - 1) // page], (n - 1) % page
        got = xp.DeviceTensor((hkv, page, d), "bf16", buf=v.buf, offset=v.offset + int(p) * es).get()[:, at]
        assert np.array_equal(got, x[s, (8 + hkv) * d:].reshape(hkv, d))


def test_many_sequences(xp):
    """More sequences than one wave looks at in a round."""
    rng = np.random.default_rng(12)
    lens = [int(x) for x in rng.integers(1, 40, 300)]
    b = Batch(rng, lens, [1] * 300, 4, 1, 32, 16, "fp32")
    _attend(xp, b)
    lens = [int(x) for x in rng.integers(1, 40, 300)]
    rows = [int(rng.integers(0, n + 1)) for n in lens]
    b = Batch(rng, lens, rows, 4, 1, 32, 16, "bf16", pad=5)
    _attend(xp, b)


def test_empty_batches(xp):
    rng = np.random.default_rng(13)
    b = Batch(rng, [5, 3], [0, 0], 4, 2, 32, 16, "bf16", pad=2)
    got = _attend(xp, b)
    assert (got == 7.0).all()
    none = xp.empty((0, 128), "bf16")
    dev = b.upload(xp)
    pages = [dev[n] for n in ("k_pages", "v_pages", "page_table", "q_start", "kv_len")]
    assert xp.paged_attention(none, *pages, max_q=1, divisor=1.0).shape == (0, 128)
    assert xp.kv_append(xp.empty((0, 256), "bf16"), *pages, n_heads_q=4).shape == (0, 128)


@pytest.mark.parametrize("rows,shared", [(1, 0), (40, 0), (1, 64)])
def test_captured_calls_replay_at_new_lengths(xp, rows, shared):
    """A step captured once reads lengths, tables and rows of its replay's time; eager work and
    synchronisation in between."""
    rng = np.random.default_rng(14)
    lens = [100, 64 + rows, 200]
    b = Batch(rng, [n + 40 for n in lens], [rows] * 3, 8, 2, 64, 16, "bf16", shared=shared)
    full = b.upload(xp)
    pages = [full[n] for n in ("k_pages", "v_pages", "page_table", "q_start", "kv_len")]
    q = xp.array(b.q.reshape(b.n, -1), dtype="bf16")
    out = xp.empty(q.shape, "bf16")

    def call(dst):
        xp.paged_attention(q, *pages, max_q=rows, divisor=8.0, shared=shared, out=dst)

    pages[4].set(np.array(lens, np.int32))
    call(out)
    with xp.capture() as g:
        call(out)
        xp.i32_add(pages[4], 7)
    for step in range(4):
        now = [n + 7 * step for n in lens]
        g.launch()
        assert pages[4].get().tolist() == [n + 7 for n in now]
        got = out.get()
        pages[4].set(np.array(now, np.int32))
        eager = xp.empty(q.shape, "bf16")
        call(eager)
        assert np.array_equal(got, eager.get())
        xp.i32_add(pages[4], 7)
    g.destroy()


def test_repeated_calls_are_bit_equal(xp):
    rng = np.random.default_rng(15)
    for rows, shared in ((1, 0), (50, 0), (1, 64)):
        b = Batch(rng, [300, 90, 1000], [rows] * 3, 8, 2, 128, 16, "bf16", shared=shared)
        dev = b.upload(xp)
        first = _attend(xp, b, dev=dev, shared=shared)
        for _ in range(3):
            assert np.array_equal(first, _attend(xp, b, dev=dev, shared=shared))


def test_refusals(xp):
    """What the library itself refuses: each call fails with its reason and launches nothing."""
    rng = np.random.default_rng(16)
    b = Batch(rng, [100, 70], [1, 1], 4, 2, 64, 16, "bf16", shared=16)
    dev = b.upload(xp)
    pages = [dev[n] for n in ("k_pages", "v_pages", "page_table", "q_start", "kv_len")]
    q, out = xp.array(b.q.reshape(2, -1), dtype="bf16"), xp.zeros((2, 256), "bf16")

    def attend(match, q=q, pages=pages, out=out, status=xp.TL_ERR_INVALID, **kw):
        with pytest.raises(xp.TLError, match=match) as e:
            xp.paged_attention(q, *pages, **{**dict(max_q=1, divisor=8.0, out=out), **kw})
        assert e.value.status == status

    for bad in (0.0, -1.0, float("inf"), float("nan")):
        attend("divisor", divisor=bad)
    for bad in (-1.0, float("inf"), float("nan")):
        attend("softcap", softcap=bad)
    attend("max_q", max_q=0)
    attend("window", window=-1)
    attend("shared", shared=-16)
    attend("shared", shared=8)
    attend("shared", shared=16 * 100)
    attend("window", shared=16, window=5)

    def view(t, shape, at=0, pitch=None):
        return xp.DeviceTensor(shape, t.dtype, pitch=pitch, buf=t.buf, offset=at)

    big = xp.zeros((4096,), "bf16")
    attend("16-byte", q=view(big, (2, 256), at=2))
    attend("16-byte", out=view(big, (2, 256), at=8))
    attend("16-byte", q=view(big, (2, 256), pitch=260))
    attend("page_size", pages=[view(pages[0], (2, 2, 24, 64)), view(pages[1], (2, 2, 24, 64)), *pages[2:]])
    attend("page_size", pages=[view(pages[0], (2, 2, 8, 64)), view(pages[1], (2, 2, 8, 64)), *pages[2:]])
    attend("head config", pages=[view(pages[0], (2, 3, 16, 64)), view(pages[1], (2, 3, 16, 64)), *pages[2:]])
    attend("head_dim", q=view(big, (2, 192)), out=view(big, (2, 192)), status=xp.TL_ERR_UNSUPPORTED,
           pages=[view(pages[0], (2, 2, 16, 48)), view(pages[1], (2, 2, 16, 48)), *pages[2:]])
    attend("16-byte", pages=[view(pages[0], (2, 2, 16, 64), at=8), *[view(pages[1], (2, 2, 16, 64))], *pages[2:]])
    table = xp.rope_table(200, 64)
    qkv = view(big, (2, 512))
    for match, kw in (("overlap", dict(rope=table, out=view(big, (2, 256), at=512))),
                      ("16-byte", dict(rope=table, qkv=view(big, (2, 512), at=4))),
                      ("16-byte", dict(rope=table, out=view(big, (2, 256), at=2056)))):
        with pytest.raises(xp.TLError, match=match):
            xp.kv_append(**{**dict(qkv=qkv), **dev, **dict(n_heads_q=4), **kw})
    xp.synchronize()
    assert (out.get() == 0).all() and (big.get() == 0).all()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 1, 256), (8, 2, 128), (12, 12, 64), (4, 4, 32)])
def test_pieces_after_long_pasts(xp, dt, hq, hkv, d):
    """Blocks of rows that see so many keys that many workgroups share them, beside short ones; rows in
    blocks of 16 (a few a sequence) and in larger ones."""
    for i, (lens, rows, kw) in enumerate([([6000, 300], [140, 5], {}), ([5000, 2100, 64], [9, 1, 16], dict(cap=20.0)),
                                          ([4500], [200], dict(window=1000)), ([3100, 40], [33, 40], dict(cap=40.0))]):
        rng = np.random.default_rng(d + i)
        b = Batch(rng, lens, rows, hq, hkv, d, 64, dt, q_std=2.0)
        _attend(xp, b, **kw)


@pytest.mark.parametrize("d", [32, 256])
def test_long_steps(xp, d):
    """One sequence in more parts than are joined at a time, beside short ones and others without a row."""
    rng = np.random.default_rng(17)
    b = Batch(rng, [9000, 1, 500, 33, 70], [1, 1, 0, 1, 1], 8, 1, d, 128, "bf16", q_std=2.0)
    _attend(xp, b)
    _attend(xp, b, cap=10.0)
    _attend(xp, b, window=3000)


def test_very_many_sequences(xp):
    """More sequences than a workgroup looks at in a round, with one long enough that its keys are shared
    out; and more row blocks than the plan keeps at hand."""
    rng = np.random.default_rng(18)
    lens = [int(x) for x in rng.integers(1, 40, 700)]
    lens[350] = 1500
    b = Batch(rng, lens, [1] * 700, 4, 1, 32, 16, "bf16")
    _attend(xp, b)
    lens = [int(x) for x in rng.integers(0, 20, 4300)]
    rows = [min(n, int(rng.integers(0, 3))) for n in lens]
    lens[4000], rows[4000] = 300, 77
    b = Batch(rng, lens, rows, 4, 2, 32, 16, "bf16", pad=3)
    _attend(xp, b)


@pytest.mark.parametrize("rows,shared", [(1, 0), (90, 0), (1, 64), (20, 0)])
def test_outputs_in_the_queries_place(xp, rows, shared):
    rng = np.random.default_rng(19)
    b = Batch(rng, [400, 64 + rows, 200], [rows] * 3, 8, 2, 64, 16, "bf16", shared=shared)
    dev = b.upload(xp)
    pages = [dev[n] for n in ("k_pages", "v_pages", "page_table", "q_start", "kv_len")]
    q = xp.array(b.q.reshape(b.n, -1), dtype="bf16")
    want = xp.paged_attention(q, *pages, max_q=rows, divisor=8.0, shared=shared).get()
    xp.paged_attention(q, *pages, max_q=rows, divisor=8.0, shared=shared, out=q)
    assert np.array_equal(q.get(), want)


def test_queries_as_columns_of_the_qkv_rows(xp):
    """Without a rotation the queries are read where the product left them."""
    rng = np.random.default_rng(20)
    b = Batch(rng, [50, 20], [7, 20], 4, 2, 32, 16, "fp32")
    x = rounded(rng.standard_normal((27, 8 * 32)), "fp32")
    dev = b.upload(xp)
    q = xp.kv_append(xp.array(x), **dev, n_heads_q=4)
    assert q.pitch == 8 * 32
    b.q = x[:, :128].reshape(27, 4, 32)
    for s in range(2):
        i = slice(b.start[s], b.start[s + 1])
        r = b.rows[s]
        b.keys[s][-r:], b.values[s][-r:] = x[i, 128:192].reshape(r, 2, 32), x[i, 192:].reshape(r, 2, 32)
    out = xp.paged_attention(q, *(dev[n] for n in ("k_pages", "v_pages", "page_table", "q_start", "kv_len")), max_q=20,
                             divisor=float(np.sqrt(32)))
    want = b.want(float(np.sqrt(32)))
    assert (np.abs(out.get().reshape(27, 4, 32) - want) <= b.tolerance(want)).all()


def test_two_captured_batches_share_the_workspace(xp):
    """Two graphs of different batches and an eager call between their replays use one workspace in turn."""
    rng = np.random.default_rng(21)
    made = []
    for rows, lens in ((1, [900, 2000, 64]), (60, [700, 61, 1000])):
        b = Batch(rng, lens, [rows] * 3, 8, 2, 128, 16, "bf16")
        dev = b.upload(xp)
        pages = [dev[n] for n in ("k_pages", "v_pages", "page_table", "q_start", "kv_len")]
        q, out = xp.array(b.q.reshape(b.n, -1), dtype="bf16"), xp.empty((b.n, 8 * 128), "bf16")
        call = lambda q=q, pages=pages, rows=rows, out=out: xp.paged_attention(  # noqa: E731
            q, *pages, max_q=rows, divisor=11.0, out=out)
        call()
        made.append((call, out, out.get()))
    graphs = []
    for call, _, _ in made:
        with xp.capture() as g:
            call()
        graphs.append(g)
    for _ in range(3):
        for g, (_, out, want) in zip(graphs, made):
            out.fill(0)
            g.launch()
            made[0][0]()
        for _, out, want in made:
            assert np.array_equal(out.get(), want)
    for g in graphs:
        g.destroy()


def test_a_border_moved_to_the_end_of_a_heads_blocks(xp):
    """32 / 8 heads at D 128: on 256 CUs the blocks of 1300 rows (523 places a head) are cut into runs of 9, and
    the 58th border, at 522, moves to the end of the first head's. The batch before leaves a block in the workspace
    behind this one's last, which would lie across that place."""
    rng = np.random.default_rng(22)
    _attend(xp, Batch(rng, [640] * 41 + [3000], [1] * 41 + [60], 32, 8, 128, 64, "bf16", q_std=2.0))
    _attend(xp, Batch(rng, [1300], [1300], 32, 8, 128, 64, "bf16", q_std=2.0))


def test_caps_and_divisors_out_of_range_are_refused(xp):
    rng = np.random.default_rng(23)
    for dt in ("bf16", "fp32"):
        b = Batch(rng, [40, 9], [1, 1], 4, 2, 32, 16, dt, q_std=3.0)
        dev = b.upload(xp)
        q = xp.array(b.q.reshape(2, -1), dtype=dt)
        pages = [dev[n] for n in ("k_pages", "v_pages", "page_table", "q_start", "kv_len")]
        for kw in (dict(divisor=1e-39), dict(divisor=3.0, softcap=1e-39), dict(divisor=3.0, softcap=3e38),
                   dict(divisor=3e38, softcap=4e3), *([dict(divisor=3.0, softcap=5000.0)] if dt == "bf16" else [])):
            with pytest.raises(xp.TLError, match="softcap") as e:
                xp.paged_attention(q, *pages, max_q=1, **kw)
            assert e.value.status == xp.TL_ERR_INVALID
        _attend(xp, b, cap=4096.0)
        _attend(xp, b, cap=0.01)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 1, 256), (8, 2, 128), (12, 12, 64), (4, 4, 32)])
def test_values_that_some_rows_may_not_see(xp, dt, hq, hkv, d):
    """Infinite and NaN values (and keys) of the batch's own positions reach the rows that see them, and the
    others' results are those of finite ones: later positions, and with a window those before it."""
    rng = np.random.default_rng(d)
    for lens, rows, window, cap in (([300, 90], [300, 40], 0, 0.0), ([700, 2000], [150, 180], 64, 0.0),
                                    ([500, 60], [2, 9], 0, 20.0), ([500, 60], [2, 9], 33, 0.0), ([4000], [30], 0, 0.0)):
        b = Batch(rng, lens, rows, hq, hkv, d, 16, dt, q_std=2.0)
        hidden = np.zeros((b.n, b.hq), bool)
        for s, (n, r) in enumerate(zip(lens, rows)):
            pos = np.arange(n - r, n)
            for j, what, which in ((n - 1, np.inf, "v"), (n - r // 3 - 1, np.nan, "kv"), (n - r, -np.inf, "v")):
                if j == n - r and not window:
                    continue  # all rows would see it
                kv_at = [a[b.slots(s, [j])] for a in (b.k, b.v)]
                bad = np.full_like(kv_at[1], what)
                bad[..., 1::2] = kv_at[1][..., 1::2] if which == "v" else what
                b.v[b.slots(s, [j])] = bad
                if which == "kv":
                    b.k[b.slots(s, [j])] = what
                sees = (pos >= j) & ((pos < j + window) if window else True)
                hidden[b.start[s]:b.start[s] + r] |= sees[:, None]
        dev = b.upload(xp)
        q, out = xp.array(b.q.reshape(b.n, -1), dtype=dt), xp.empty((b.n, hq * d), dt)
        xp.paged_attention(q, dev["k_pages"], dev["v_pages"], dev["page_table"], dev["q_start"], dev["kv_len"],
                           max_q=max(rows), divisor=float(np.sqrt(d)), softcap=cap, window=window, out=out)
        got, want = out.get().reshape(b.n, hq, d), b.want(float(np.sqrt(d)), cap, window)
        ok = ~hidden
        assert ok.any() or window >= max(rows)  # (a window of all rows shows the first one's position to all)
        assert (np.abs(got - want)[ok] <= b.tolerance(want)[ok]).all()
        assert not np.isfinite(got[hidden]).all(-1).any()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("hq,hkv,d", [(71, 1, 64), (17, 1, 256), (15, 5, 32), (10, 2, 128), (3, 3, 256), (66, 2, 32)])
def test_odd_groups_of_heads(xp, dt, hq, hkv, d):
    """Query heads a kv head that are no power of two, or more than a block of 16 rows holds."""
    for i, (lens, rows, kw) in enumerate([([70, 1, 300], [1, 1, 1], {}), ([64 + 40, 64 + 3], [2, 1], dict(shared=64)),
                                          ([90, 33], [50, 7], dict(cap=30.0)), ([200, 17], [5, 17], dict(window=40))]):
        b = Batch(np.random.default_rng(i), lens, rows, hq, hkv, d, 32, dt, q_std=2.0, shared=kw.get("shared", 0))
        _attend(xp, b, **kw)
