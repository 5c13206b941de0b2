"""Operators of ragged serving over a paged KV cache: sequences of unequal lengths in one batch, their
keys and values in pages that a table per sequence lists.

  append   the rows of a QKV product, [Q | K | V]: queries and keys rotated by their positions, keys
           and values written into the pages of their sequences
  attend   causal attention of the batch's queries over those pages: whole prompts, pieces of
           prompts after a cached past, single tokens; optionally with scores capped by a tanh and
           with a sliding window
  shared   single tokens of sequences that begin with the same long prefix, whose pages they share

`run` takes the plain form of each from torch, or, where `own` is true, makes the framework's calls.
"""
import math
import os
import sys

import torch

own = False  # whether run() makes the framework's calls

# the package's modules import each other by bare name; they come from the tree that this process runs in
_PKG = os.path.join(os.getcwd(), "torchless-nn_amd")
_BASE = 10000.0

# (query heads, key/value heads, head dim): the multi-query decoder, its half and a grouped one, the
# GPT-2-small-shaped model, the character model, and generic grouped ones
_SHAPES = [(8, 1, 256), (4, 1, 256), (8, 2, 128), (12, 12, 64), (4, 4, 32), (32, 4, 128), (10, 2, 64)]


def _case(name, op, dtype, shape, seqs, q, kv, page, rope=True, cap=0.0, window=0, shared=0):
    """q, kv: the shortest and longest of the batch's new rows and of its lengths with them."""
    c = dict(op=op, dtype=dtype, heads=shape[0], kv_heads=shape[1], head_dim=shape[2], seqs=seqs, q_min=q[0],
             q_max=q[1], kv_min=kv[0], kv_max=kv[1], page=page)
    c.update(dict(rope=rope) if op == "append" else dict(cap=cap, window=window, shared=shared))
    return dict(c, name=name) if name else c


def listed():
    return [
        # one step of a server: a token each of 32 sequences, all latency
        _case("append_step_bf16", "append", "bf16", (8, 1, 256), 32, (1, 1), (1, 2048), 64),
        # a batch of prompts of unequal lengths for the 2B-class multi-query decoder
        _case("append_prompts_bf16", "append", "bf16", (8, 1, 256), 7, (300, 2000), (300, 2000), 64),
        # the GPT-2-small-shaped model in the default FLOAT_TYPE, whose positions are learned: nothing to rotate
        _case("append_gpt_f32", "append", "fp32", (12, 12, 64), 5, (99, 1000), (99, 1000), 16, rope=False),
        # the multi-query decoder's four long prompts
        _case("prompts_mqa_bf16", "attend", "bf16", (8, 1, 256), 4, (2048, 2048), (2048, 2048), 64),
        # large pieces of long prompts after a cached past, scores capped
        _case("prompts_long_capped_bf16", "attend", "bf16", (32, 4, 128), 3, (1000, 4000), (4000, 8001), 128, cap=30.0),
        # a ragged batch of prompts in a layer that looks back 512 positions
        _case("prompts_window_bf16", "attend", "bf16", (8, 2, 128), 9, (17, 1500), (17, 1500), 16, window=512),
        # prompts of the GPT-2-small-shaped model in the default FLOAT_TYPE
        _case("prompts_gpt_f32", "attend", "fp32", (12, 12, 64), 5, (99, 1000), (99, 1000), 16),
        # one token of the character model: the smallest call, all latency
        _case("step_char_f32", "attend", "fp32", (4, 4, 32), 1, (1, 1), (65, 65), 16),
        # a batched server's step with the multi-query decoder, sequences of all ages
        _case("step_mqa_b48_bf16", "attend", "bf16", (8, 1, 256), 48, (1, 1), (500, 2048), 64),
        # a few sequences with very long pasts
        _case("step_long_bf16", "attend", "bf16", (32, 4, 128), 6, (1, 1), (20001, 60000), 128),
        # 64 answers to one long prompt in the multi-query decoder
        _case("shared_mqa_b64_bf16", "shared", "bf16", (8, 1, 256), 64, (1, 1), (2049, 2350), 64, shared=2048),
        # a server whose requests all begin with the same long instructions
        _case("shared_b150_bf16", "shared", "bf16", (32, 4, 128), 150, (1, 1), (8193, 8700), 16, shared=8192),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["append", "prompts", "prompts", "step", "step", "shared"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    shape = rng.choice(_SHAPES)
    page = rng.choice([16, 32, 64, 128, 256])
    cap = rng.choice([0.0, 0.0, 30.0, 50.0])
    window = rng.choice([0, 0, 0, 1]) and _log(rng, 64, 4096)
    # rows of keys that a case may hold in all: about 250 MB of them at most
    most = 250_000_000 // (2 * shape[1] * shape[2] * (2 if dtype == "bf16" else 4))
    if op == "append":
        hi = _log(rng, 1, 2000)
        seqs = _log(rng, 1, max(1, min(128, 7000 // hi)))
        return _case(None, op, dtype, shape, seqs, (max(1, hi // 7), hi), (hi, _log(rng, hi, 4000)), page,
                     rope=rng.random() < 0.7)
    if op == "prompts":
        hi = _log(rng, 3, 2500)
        seqs = _log(rng, 1, max(1, min(16, 8000 // hi)))
        kv = _log(rng, hi, max(hi, min(8000, 20000 // seqs)))
        return _case(None, "attend", dtype, shape, seqs, (max(1, hi // 9), hi), (hi, kv), page, cap=cap, window=window)
    if op == "step":
        hi = _log(rng, 10, 60000)
        seqs = _log(rng, 1, max(1, min(128, most // hi)))
        return _case(None, "attend", dtype, shape, seqs, (1, 1), (max(1, hi // 6), hi), page, cap=cap, window=window)
    shared = page * _log(rng, max(1, 256 // page), 8192 // page)
    tail = _log(rng, 1, 800)
    seqs = _log(rng, 2, max(2, min(150, (most - shared) // tail)))
    return _case(None, op, dtype, shape, seqs, (1, 1), (shared + 1, shared + tail), page, cap=cap, shared=shared)


# ---- the batch ------------------------------------------------------------------------
def _lengths(c):
    """(new rows, length with them) of each sequence, spread over their ranges."""
    def spread(lo, hi, step):
        return [hi - round((hi - lo) * ((i * step) % 1.0)) for i in range(c["seqs"])]

    q = spread(c["q_min"], c["q_max"], 0.754877666)
    return q, [max(n, r) for n, r in zip(spread(c["kv_min"], c["kv_max"], 0.618033989), q)]


def _dtype(c):
    return torch.bfloat16 if c["dtype"] == "bf16" else torch.float32


def _inputs(c, seed):
    """What the call is given, as torch tensors on the GPU."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt = _dtype(c)
    hq, hk, d, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    q, kv = _lengths(c)
    rows = sum(q)

    def normal(*shape, std=1.0):
        return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(0.0, std, generator=g).to(dt)

    # pages in no order, as a server that has run for a while hands them out, a few of them unused; the
    # prefix's pages are the same for all
    alike = c.get("shared", 0) // page
    needed = [-(-n // page) - alike for n in kv]
    pages = torch.randperm(alike + sum(needed) + 3, device="cuda", generator=g).to(torch.int32)
    table = torch.full((c["seqs"], alike + max(needed)), -1, device="cuda", dtype=torch.int32)
    table[:, :alike] = pages[:alike]
    listed_pages = torch.arange(max(needed), device="cuda") < torch.tensor(needed, device="cuda")[:, None]
    table[:, alike:][listed_pages] = pages[alike:-3]
    s = dict(table=table, k=normal(len(pages), hk, page, d), v=normal(len(pages), hk, page, d),
             start=torch.tensor([sum(q[:i]) for i in range(len(q) + 1)], device="cuda", dtype=torch.int32),
             length=torch.tensor(kv, device="cuda", dtype=torch.int32))
    if c["op"] == "append":
        s["qkv"] = normal(rows, (hq + 2 * hk) * d)
        s["q"] = torch.zeros(rows, hq * d, device="cuda", dtype=dt)
        if c["rope"]:  # cosines and sines of every position that the model serves
            s["rope"] = _angles(torch.arange(c["kv_max"], device="cuda"), d)
    else:
        # scores of a few units, as trained heads have them; a capping layer's reach into the bend
        s["q"] = normal(rows, hq * d, std=8.0 if c["cap"] else 2.0)
        s["out"] = torch.zeros(rows, hq * d, device="cuda", dtype=dt)
    return s


def _angles(pos, d):
    inv = _BASE ** (-2.0 * torch.arange(d // 2, device="cuda", dtype=torch.float64) / d)
    a = pos.double()[:, None] * inv
    return torch.stack([a.cos(), a.sin()]).float()


class _Memory:
    """A framework tensor's memory for torch.as_tensor; it keeps the tensor alive."""

    def __init__(self, t):
        typestr = {"float32": "<f4", "bfloat16": "<i2", "int32": "<i4"}[t.dtype.name]
        self.tensor = t
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": typestr, "data": (t.ptr, False), "version": 2}


def prepare(case, seed):
    c = case
    s = dict(_inputs(c, seed), case=c, max_q=max(_lengths(c)[0]))
    if own:
        # the same tensors in the framework's memory, where its user's program has them, and torch's view of
        # what the call writes
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        os.environ.setdefault("XP_RUNTIME", "MI355X")
        import tl_hip as xp
        s["xp"] = xp
        for name in ("table", "k", "v", "start", "length", "qkv", "q", "out", "rope"):
            if name in s:
                t = xp.empty(tuple(s[name].shape), str(s[name].dtype).replace("torch.", ""))
                view = torch.as_tensor(_Memory(t), device="cuda")
                view = view.view(torch.bfloat16) if s[name].dtype == torch.bfloat16 else view
                view.copy_(s[name])
                s[name], s[name + "_seen"] = t, view
    torch.cuda.synchronize()
    return s


# ---- the plain forms --------------------------------------------------------------------
def _rows_of(start, length, rows):
    """The sequence of each of the batch's rows, its index there and its position."""
    r = torch.arange(rows, device="cuda")
    seq = torch.bucketize(r, start[1:].long(), right=True)
    i = r - start[seq]
    return seq, i, i + length[seq] - (start[seq + 1] - start[seq])


def _append(c, s):
    hq, hk, d, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    seq, _, pos = _rows_of(s["start"], s["length"], s["qkv"].shape[0])
    q, k, v = s["qkv"].split([hq * d, hk * d, hk * d], 1)
    k, v = k.reshape(-1, hk, d), v.reshape(-1, hk, d)
    at = s["table"][seq, pos // page].long()
    if c["rope"]:
        cos, sin = s["rope"][0][pos][:, None], s["rope"][1][pos][:, None]
        x = torch.cat([q.reshape(-1, hq, d), k], 1).float()
        a, b = x[..., :d // 2], x[..., d // 2:]
        x = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(q.dtype)
        s["q"].copy_(x[:, :hq].reshape(-1, hq * d))
        k = x[:, hq:]
    s["k"][at, :, pos % page] = k
    s["v"][at, :, pos % page] = v
    return (s["q"], s["k"], s["v"]) if c["rope"] else (s["k"], s["v"])


def _gather(pages, table, n):
    """The first n positions that each row of `table` lists: [sequences, heads, n, head dim], 32 bits."""
    x = pages[table.clamp(min=0).long()].permute(0, 2, 1, 3, 4)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[4])[:, :, :n].float().contiguous()


def _scores(q, k, cap):
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(q.shape[-1])
    return torch.tanh(s / cap) * cap if cap else s


def _softmax(s):
    e = torch.exp(s - s.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _attend(c, s):
    hq, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    n, most = c["kv_max"], s["max_q"]
    seq, i, pos = _rows_of(s["start"], s["length"], s["q"].shape[0])
    q = torch.zeros(c["seqs"], most, hk, hq // hk, d, device="cuda")
    q[seq, i] = s["q"].float().reshape(-1, hk, hq // hk, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(c["seqs"], hk, -1, d)
    at = torch.zeros(c["seqs"], most, device="cuda", dtype=torch.int64)
    at[seq, i] = pos.long()
    j = torch.arange(n, device="cuda")
    keep = j <= at[..., None]
    if c["window"]:
        keep &= j > at[..., None] - c["window"]
    keep = keep[:, None, None]
    a = _scores(q, _gather(s["k"], s["table"], n), c["cap"]).reshape(c["seqs"], hk, hq // hk, most, n)
    p = _softmax(a.masked_fill(~keep, float("-inf"))).reshape(c["seqs"], hk, -1, n)
    o = torch.matmul(p, _gather(s["v"], s["table"], n))
    o = o.reshape(c["seqs"], hk, hq // hk, most, d).permute(0, 3, 1, 2, 4)[seq, i]
    s["out"].copy_(o.reshape(-1, hq * d))
    return s["out"]


def _attend_shared(c, s):
    hq, hk, d, n = c["heads"], c["kv_heads"], c["head_dim"], c["shared"]
    b, g, rest = c["seqs"], c["heads"] // c["kv_heads"], c["kv_max"] - c["shared"]
    q = s["q"].float().reshape(b, hk, g, d)
    alike, tail = s["table"][:1, :n // c["page"]], s["table"][:, n // c["page"]:]
    # the prefix for all sequences' queries at once, the rest of each by itself
    together = q.transpose(0, 1).reshape(hk, b * g, d)
    first = _scores(together, _gather(s["k"], alike, n)[0], c["cap"]).reshape(hk, b, g, n).transpose(0, 1)
    then = _scores(q, _gather(s["k"], tail, rest), c["cap"])
    keep = torch.arange(rest, device="cuda") < (s["length"][:, None] - n)
    p = _softmax(torch.cat([first, then.masked_fill(~keep[:, None, None], float("-inf"))], -1))
    first = p[..., :n].transpose(0, 1).reshape(hk, b * g, n)
    o = torch.matmul(first, _gather(s["v"], alike, n)[0]).reshape(hk, b, g, d).transpose(0, 1)
    o = o + torch.matmul(p[..., n:].contiguous(), _gather(s["v"], tail, rest))
    s["out"].copy_(o.reshape(b, hq * d))
    return s["out"]


def run(state):
    s, c = state, state["case"]
    if own:
        xp = s["xp"]
        pages = (s["k"], s["v"], s["table"], s["start"], s["length"])
        if c["op"] == "append":
            xp.kv_append(s["qkv"], *pages, n_heads_q=c["heads"], rope=s.get("rope"), out=s["q"] if c["rope"] else None)
            return (s["q_seen"], s["k_seen"], s["v_seen"]) if c["rope"] else (s["k_seen"], s["v_seen"])
        xp.paged_attention(s["q"], *pages, max_q=s["max_q"], divisor=math.sqrt(c["head_dim"]), softcap=c["cap"],
                           window=c["window"], shared=c["shared"], out=s["out"])
        return s["out_seen"]
    if c["op"] == "append":
        return _append(c, s)
    return _attend_shared(c, s) if c["op"] == "shared" else _attend(c, s)


# ---- what a pass cannot do without ------------------------------------------------------
def work(case):
    c = case
    es = 2 if c["dtype"] == "bf16" else 4
    hq, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    q, kv = _lengths(c)
    if c["op"] == "append":
        # without a rotation the queries stay where they are
        moved = sum(q) * ((hq if c["rope"] else 0) + 2 * hk) * d
        angles = 4 * d * min(sum(q), max(kv)) if c["rope"] else 0
        return {"bytes": 2.0 * es * moved + angles, "flops": 3.0 * sum(q) * (hq + hk) * d if c["rope"] else 0.0}
    span = c["window"] or max(kv)
    # the keys that any of a sequence's rows sees, and those that each row sees
    keys = sum(min(n, r - 1 + span) for r, n in zip(q, kv)) - c["shared"] * (c["seqs"] - 1)
    pairs = sum(sum(min(span, n - r + i + 1) for i in range(r)) for r, n in zip(q, kv))
    return {"bytes": es * (2.0 * sum(q) * hq * d + 2.0 * keys * hk * d), "flops": 4.0 * pairs * hq * d}


# ---- the same in 64 bits ----------------------------------------------------------------
def _turned(x, pos):
    """Rotate-half RoPE of one sequence's x [rows, heads, d] at positions pos, as complex numbers."""
    half = x.shape[-1] // 2
    freq = torch.tensor([_BASE ** (-i / half) for i in range(half)], device="cuda", dtype=torch.float64)
    z = torch.complex(x[..., :half], x[..., half:]) * torch.exp(1j * (pos.double()[:, None] * freq))[:, None]
    return torch.cat([z.real, z.imag], -1)


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    hq, hk, d, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    q_len, kv_len = _lengths(c)
    first = 0
    if c["op"] == "append":
        x = s["qkv"].double().reshape(-1, hq + 2 * hk, d)
        q, k, v = x[:, :hq].clone(), s["k"].double(), s["v"].double()
        for i, (r, n) in enumerate(zip(q_len, kv_len)):
            rows = x[first:first + r]
            pos = torch.arange(n - r, n, device="cuda")
            turn = rows[:, :hq + hk]
            if c["rope"]:
                turn = _turned(turn, pos)
                q[first:first + r] = turn[:, :hq]
            where = (s["table"][i][pos // page].long(), slice(None), pos % page)
            k[where] = turn[:, hq:]
            v[where] = rows[:, hq + hk:]
            first += r
        return (q.reshape(-1, hq * d), k, v) if c["rope"] else (k, v)
    out = torch.empty(sum(q_len), hq, d, device="cuda", dtype=torch.float64)
    for i, (r, n) in enumerate(zip(q_len, kv_len)):
        ids = s["table"][i, :-(-n // page)].long()
        pos = torch.arange(n - r, n, device="cuda")[:, None]
        at = torch.arange(n, device="cuda")[None, :]
        hidden = (at > pos) | (at <= pos - c["window"]) if c["window"] else at > pos
        for h in range(hk):
            k = s["k"][ids, h].reshape(-1, d)[:n].double()
            v = s["v"][ids, h].reshape(-1, d)[:n].double()
            for e in range(h * (hq // hk), (h + 1) * (hq // hk)):
                w = s["q"][first:first + r, e * d:(e + 1) * d].double() @ k.T * d ** -0.5
                if c["cap"]:
                    w = c["cap"] * torch.tanh(w / c["cap"])
                w = w.masked_fill(hidden, -math.inf)
                out[first:first + r, e] = torch.softmax(w, -1) @ v
        first += r
    return out.reshape(-1, hq * d)
