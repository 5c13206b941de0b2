"""Models over a paged cache on the MI355X: ragged batches against the dense paths and the NumPy
oracle, capped and windowed layers, shared prefixes, and generation by replayed steps. fp32: max_rel
<= 1e-5, bf16: <= 2e-2, the bars of the same models over the dense cache."""
import numpy as np
import pytest

from oracle import numpy_ref as ref

pytestmark = pytest.mark.gpu
TINY = dict(vocab=97, ctx=160, layers=2, d=64, heads=4, kv_heads=1, head_dim=32, ffn=96)
WIDE = dict(vocab=101, ctx=256, layers=2, d=256, heads=8, kv_heads=2, head_dim=64, ffn=512)


@pytest.fixture(scope="module")
def tl():
    import tl_hip
    tl_hip.ctx()
    import backend
    import gemma
    import gpt
    import layers
    return dict(xp=tl_hip, backend=backend, gemma=gemma, gpt=gpt, layers=layers)


def _tol(dt):
    return 1e-5 if dt == "fp32" else 2e-2


def _bar(dt, P, cfg, ids):
    """bf16: 2e-2. fp32: 1e-5 as for the dense cache, or what large scores leave of it: kernel and oracle
    both hold a score s in fp32, rounded as a sum and again as its scaled form, 2^-24 |s| each, and an
    error of a score is the relative error of its probability. Two sides, two roundings and two layers
    make 8 2^-24 max |s|; the scores are the first layer's, whose rotation leaves |q| and |k| as they are."""
    if dt == "bf16":
        return 2e-2
    hq, hk, d = cfg["heads"], cfg["kv_heads"], cfg["head_dim"]
    x = ref.rmsnorm(P["table"][ids] * np.sqrt(np.float32(cfg["d"])), P["b0.g1"], np.float32(1e-6), 1.0) @ P["b0.wqkv"]
    q, k = x[:, :hq * d].reshape(-1, hq, d), x[:, hq * d:(hq + hk) * d].reshape(-1, hk, d)
    cos, sin = ref.rope_table(len(ids), d, cfg.get("rope_base", 10000.0), 0)
    q, k = (ref.rope(a.transpose(1, 0, 2), cos, sin) for a in (q, k))
    s = q @ np.repeat(k, hq // hk, 0).transpose(0, 2, 1) / d ** 0.5
    return max(1e-5, 8 * 2.0 ** -24 * np.abs(s).max())


def _gemma(tl, cfg, dt, seed):
    scale = 0.3 if dt == "fp32" else 0.05
    model = tl["gemma"].build_gemma(cfg, dt)
    tl["gemma"].seed_gemma(model, seed, scale)
    return model, ref.gemma_params(cfg, seed, scale, bf16=dt == "bf16")


def _ids(rng, cfg, lens):
    return [rng.integers(0, cfg["vocab"], n).tolist() for n in lens]


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("cfg", [TINY, WIDE, dict(TINY, softcap=2.0), dict(WIDE, window=[20, 0], softcap=3.0)])
def test_gemma_ragged_prompts_and_steps(tl, dt, cfg):
    """Prompts of unequal lengths as one batch, then a ragged second piece with single tokens among
    it, then a step: every sequence's last logits against the oracle's full forward."""
    xp = tl["xp"]
    model, P = _gemma(tl, cfg, dt, 31)
    rng = np.random.default_rng(32)
    seqs = _ids(rng, cfg, [90, 1, 33, 64])
    cuts = [(70, 85, 90), (1, 1, 1), (1, 30, 33), (63, 63, 64)]
    cache = model.new_paged_cache(16, page_size=16)
    ids = [cache.add() for _ in seqs]
    done = [0] * len(seqs)
    for turn in range(3):
        part = [(i, s) for i, s in enumerate(ids) if cuts[i][turn] > done[i]]
        counts = [cuts[i][turn] - done[i] for i, _ in part]
        batch = cache.batch([s for _, s in part], counts)
        rows = sum(([*seqs[i][done[i]:cuts[i][turn]]] for i, _ in part), [])
        got = model.forward_ragged(np.array([rows]), cache, batch).get()[0]
        for j, (i, _) in enumerate(part):
            done[i] = cuts[i][turn]
            want = ref.gemma_forward(np.array([seqs[i][:done[i]]]), P, cfg, bf16=dt == "bf16")[0, -1]
            assert ref.max_rel(got[j], want) <= _bar(dt, P, cfg, seqs[i][:done[i]]), (turn, i)
    xp.synchronize()


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("prefix", [0, 40, 64])
def test_gemma_generate_ragged(tl, dt, prefix):
    """Continuations of unequal prompts behind a common prefix: teacher-forced on the new ids, each id is
    the oracle's largest logit up to the bar; and the same ids again on a cache that was used before."""
    cfg = dict(WIDE, softcap=5.0)
    model, P = _gemma(tl, cfg, dt, 41)
    rng = np.random.default_rng(42)
    first = rng.integers(0, cfg["vocab"], prefix).tolist()
    prompts = _ids(rng, cfg, [30, 1, 17, 16, 5])
    cache = model.new_paged_cache(40, page_size=16)
    new = model.generate_ragged(prompts, 9, prefix=first, cache=cache)
    assert new.shape == (5, 9) and len(cache._free) == 40 and not cache.pages
    for p, n in zip(prompts, new):
        seq = np.array([first + p + n.tolist()])
        rows = ref.gemma_forward(seq[:, :-1], P, cfg, bf16=dt == "bf16")[0, -9:]
        short = rows.max(-1) - rows[np.arange(9), n]
        assert (short <= 2 * _bar(dt, P, cfg, seq[0, :-1]) * np.abs(rows).max()).all()
    assert np.array_equal(new, model.generate_ragged(prompts, 9, prefix=first, cache=cache))
    assert np.array_equal(new[:, :1], model.generate_ragged(prompts, 1, prefix=first))


def test_gemma_generate_ragged_refusals(tl):
    model, _ = _gemma(tl, TINY, "bf16", 51)
    assert model.generate_ragged([], 4).shape == (0, 4) and model.generate_ragged([[1]], 0).shape == (1, 0)
    with pytest.raises(ValueError):
        model.generate_ragged([[1], []], 4)
    with pytest.raises(ValueError):
        model.generate_ragged([[1] * 150], 12)
    cache = model.new_paged_cache(2, page_size=16)
    with pytest.raises(ValueError, match="full"):
        model.generate_ragged([[1] * 30], 12, cache=cache)
    assert len(cache._free) == 2
    # an empty prompt behind a prefix of whole pages computes the prefix's last page for each
    assert model.generate_ragged([[], [3]], 3, prefix=[5] * 16, page_size=16).shape == (2, 3)


def test_paged_layers_refuse_what_they_do_not_serve(tl):
    xp = tl["xp"]
    model, _ = _gemma(tl, dict(TINY, softcap=2.0), "bf16", 61)
    with pytest.raises(ValueError, match="PagedKVCache"):
        model.forward(np.array([[1, 2, 3]]))
    plain, _ = _gemma(tl, TINY, "bf16", 61)
    cache, other = plain.new_paged_cache(4, 16), plain.new_paged_cache(4, 16)
    s = cache.add()
    batch = cache.batch([s], [3])
    with pytest.raises(ValueError):
        plain.forward_ragged(np.array([[1, 2, 3]]), other, batch)
    with pytest.raises(ValueError):
        plain.forward_ragged(np.array([[1, 2]]), cache, batch)
    with pytest.raises(ValueError):
        plain.forward_ragged(np.array([[1, 2, 3]]), cache, 0)
    later = cache.batch([s], [3])
    with pytest.raises(ValueError, match="out of date"):
        plain.forward_ragged(np.array([[1, 2, 3]]), cache, batch)
    plain.forward_ragged(np.array([[1, 2, 3]]), cache, later)
    wrong = tl["layers"].PagedKVCache(2, 4, 2, 32, plain.dtype, 16)
    with pytest.raises(ValueError, match="heads"):
        plain.forward_ragged(np.array([[1]]), wrong, wrong.batch([wrong.add()], [1]))
    xp.synchronize()


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_gpt_ragged(tl, dt):
    """The learned-position GPT (biases, no rotation) over a paged cache: prompts of unequal lengths, then
    a step, against the oracle's probabilities."""
    cfg = dict(vocab=65, ctx=96, layers=2, d=128, heads=4, act="gelu")
    net, _ = tl["gpt"].build_gpt(cfg, dt)
    tl["gpt"].seed_parameters(net, 7, 0.1)
    P = ref.gpt_params(cfg, 7, 0.1, bf16=dt == "bf16")
    rng = np.random.default_rng(8)
    seqs = _ids(rng, cfg, [50, 17, 96])
    cache = tl["layers"].PagedKVCache(2, 14, 4, 32, dt, 16)
    ids = [cache.add() for _ in seqs]
    for rows in ([s[:-1] for s in seqs], [s[-1:] for s in seqs]):
        batch = cache.batch(ids, [len(r) for r in rows])
        got = tl["gpt"].forward_ragged(net, np.array([sum(rows, [])]), cache, batch).get()[0]
        for j, s in enumerate(seqs):
            n = cache.lengths[ids[j]]
            want = ref.gpt_forward(np.array([s[:n]]), P, cfg, bf16=dt == "bf16")[0, -1]
            assert ref.max_rel(got[j], want) <= _tol(dt)
    with pytest.raises(ValueError):
        tl["gpt"].forward_ragged(net, np.array([[1]]), cache, cache.batch([ids[2]], [1]))


def test_a_sequence_without_a_row_has_no_answer(tl):
    model, _ = _gemma(tl, TINY, "bf16", 53)
    cache = model.new_paged_cache(4, page_size=16)
    seqs = [cache.add(), cache.add()]
    for counts in ([1, 0], [2, 0]):
        ids = tl["xp"].array(np.ones((1, sum(counts)), np.int64))
        with pytest.raises(ValueError, match="no row"):
            model.forward_ragged(ids, cache, cache.batch(seqs, counts))
