"""Ragged batches over a paged KV cache for the tests: random ones, and their results in 64 bits."""
import numpy as np

from oracle import numpy_ref as ref

F32 = np.float32


def rounded(a, dt):
    a = np.asarray(a, F32)
    return ref.round_bf16(a) if dt == "bf16" else a


def rope64(x, pos, base=10000.0):
    """Rotate-half RoPE of x [rows, heads, D] at positions pos [rows], in float64."""
    half = x.shape[-1] // 2
    ang = np.asarray(pos, np.float64)[:, None] * base ** (-2.0 * np.arange(half) / x.shape[-1])
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = x[..., :half].astype(np.float64), x[..., half:].astype(np.float64)
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


class Batch:
    """Sequences of `lens` positions of which the last `rows` are the batch's, in shuffled pages.
    Whatever no row may see is NaN: other pages, slots past a sequence's end; table entries that no
    position needs are far out of range. `pad` rows follow the last sequence."""

    def __init__(self, rng, lens, rows, hq, hkv, d, page, dt, pad=0, shared=0, q_std=1.0, spare=3):
        self.lens, self.rows, self.hq, self.hkv, self.d, self.page, self.dt = lens, rows, hq, hkv, d, page, dt
        self.shared, self.n, self.pad = shared, sum(rows), pad
        alike = shared // page
        need = [max(0, -(-n // page) - alike) for n in lens]
        perm = rng.permutation(alike + sum(need) + spare).astype(np.int32)
        self.n_pages = len(perm)
        self.table = np.full((len(lens), max([1] + [alike + n for n in need]) + 1), 1 << 29, np.int32)
        self.table[1::2] *= -1
        at = alike
        for s, n in enumerate(need):
            self.table[s, :alike] = perm[:alike]
            self.table[s, alike:alike + n] = perm[at:at + n]
            at += n
        self.start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.k = np.full((self.n_pages, hkv, page, d), np.nan, F32)
        self.v = self.k.copy()
        first = rounded(rng.standard_normal((2, shared, hkv, d)), dt)
        self.keys, self.values = [], []
        for s, n in enumerate(lens):
            kv = rounded(rng.standard_normal((2, n, hkv, d)), dt)
            kv[:, :min(n, shared)] = first[:, :min(n, shared)]
            self.keys.append(kv[0])
            self.values.append(kv[1])
            self.put(s, kv[0], kv[1])
        self.q = rounded(rng.standard_normal((self.n + pad, hq, d)) * q_std, dt)
        self.q[self.n:] = np.nan

    def slots(self, s, pos):
        pos = np.asarray(pos)
        return self.table[s, pos // self.page], slice(None), pos % self.page

    def put(self, s, k, v, pos0=0):
        if len(k):
            at = self.slots(s, np.arange(pos0, pos0 + len(k)))
            self.k[at], self.v[at] = k, v

    def want(self, divisor, cap=0.0, window=0):
        """[n, hq, d] in float64."""
        out = np.zeros((self.n, self.hq, self.d))
        for s, (n, r) in enumerate(zip(self.lens, self.rows)):
            q = self.q[self.start[s]:self.start[s] + r].astype(np.float64)
            pos = np.arange(n - r, n)[:, None]
            j = np.arange(n)[None]
            see = (j <= pos) & (j > pos - window if window else True)
            for h in range(self.hq):
                hk = h // (self.hq // self.hkv)
                x = q[:, h] @ self.keys[s][:, hk].T.astype(np.float64) / divisor
                if cap:
                    x = cap * np.tanh(x / cap)
                x = np.where(see, x, -np.inf)
                m = x.max(-1, keepdims=True, initial=-np.inf)
                e = np.where(see, np.exp(x - np.where(np.isfinite(m), m, 0)), 0.0)
                l = e.sum(-1, keepdims=True)
                out[self.start[s]:self.start[s] + r, h] = np.where(l > 0, e @ self.values[s][:, hk] / np.where(l > 0, l, 1), 0)
        return out

    def tolerance(self, want):
        """bf16: the probabilities and the output are rounded, each by at most 2^-8 of its value, so
        by 2^-8 (max |v| + |out|); fp32: the parity bar of the other fp32 outputs, 1e-5 of the largest
        value. A few fp32 roundings (2^-24 each) of scores, sums and weights come on top in bf16."""
        vmax = max([np.abs(v).max() for v in self.values if v.size] + [0.0])
        if self.dt == "fp32":
            return np.full(want.shape, 1e-5 * max(vmax, 1e-30))
        return 2.0 ** -8 * (vmax + np.abs(want)) + 1e-4 * vmax

    # -- on the device
    def upload(self, xp):
        up = lambda a, t: xp.array(a, dtype=t)  # noqa: E731
        return dict(k_pages=up(self.k, self.dt), v_pages=up(self.v, self.dt), page_table=up(self.table, "int32"),
                    q_start=up(self.start, "int32"), kv_len=up(np.array(self.lens, np.int32), "int32"))
