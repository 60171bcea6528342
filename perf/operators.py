"""Cases of the operators for speculative decoding over a bounded KV cache.

Four operators work on the engine's ggml-typed cache rows (a row is one position, every KV head, head size 64):

  tree    attention for a tree of drafted tokens over the committed cache and the drafted rows beside it
  commit  the accepted drafts' rows of every layer copied to the end of the cache
  scores  the attention weight that each cached position received, added up per KV head
  evict   per layer, sequence and KV head: the positions to keep, and kept rows moved into the freed slots

With ``own`` false, ``run`` computes them from elementary torch operations in 32 bits; with ``own`` true it calls the
engine's entry points.  ``exact`` computes them in 64 bits from their definitions.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

D = 64
TYPE_IDS = {"f32": 0, "f16": 1, "q4_0": 2, "q4_1": 3, "q5_0": 6, "q5_1": 7, "q8_0": 8}
BLOCK_BYTES = {"q4_0": 18, "q4_1": 20, "q5_0": 22, "q5_1": 24, "q8_0": 34}


def row_bytes(t, heads):
    if t in BLOCK_BYTES:
        return heads * D // 32 * BLOCK_BYTES[t]
    return heads * D * (4 if t == "f32" else 2)


# ------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one utterance, a short prompt, four drafts of a small head: the latency of a single verification
        {"name": "tree 1x4 over 300", "op": "tree", "k": "q8_0", "v": "q8_0", "seqs": 1, "len": 300, "nodes": 4, "hq": 14, "hkv": 2,
         "mixed": False, "chain": False},
        # the serving mix: 64 sequences of 128 to 2048 positions, chains of eight drafts from a lookup
        {"name": "tree 64x8 mixed 2048", "op": "tree", "k": "q8_0", "v": "q4_0", "seqs": 64, "len": 2048, "nodes": 8, "hq": 14, "hkv": 2,
         "mixed": True, "chain": True},
        # wide trees of a trained draft head over long contexts in an f16 cache
        {"name": "tree 16x64 over 4096", "op": "tree", "k": "f16", "v": "f16", "seqs": 16, "len": 4096, "nodes": 64, "hq": 14, "hkv": 2,
         "mixed": False, "chain": False},
        # odd sizes, one KV head for each query head, a cache with block minima
        {"name": "tree 3x27 over 777", "op": "tree", "k": "q5_1", "v": "q4_1", "seqs": 3, "len": 777, "nodes": 27, "hq": 16, "hkv": 16,
         "mixed": True, "chain": False},
        # one very long context, few drafts: the axis of the keys has to be split
        {"name": "tree 1x16 over 65536", "op": "tree", "k": "q8_0", "v": "q8_0", "seqs": 1, "len": 65536, "nodes": 16, "hq": 14, "hkv": 2,
         "mixed": False, "chain": False},
        # one utterance's accepted path, every layer of the model
        {"name": "commit 1x4", "op": "commit", "k": "q8_0", "v": "q8_0", "seqs": 1, "len": 600, "nodes": 8, "layers": 24, "hkv": 2},
        # a full batch with an asymmetric cache
        {"name": "commit 64x16", "op": "commit", "k": "q8_0", "v": "q4_0", "seqs": 64, "len": 512, "nodes": 16, "layers": 24, "hkv": 2},
        # the weights of one decoded token of one utterance
        {"name": "scores 1x1 over 500", "op": "scores", "k": "q8_0", "seqs": 1, "len": 500, "rows": 1, "hq": 14, "hkv": 2, "mixed": False,
         "picked": False},
        # a batch after a commit: the accepted tokens' weights, a few of the drafted rows picked
        {"name": "scores 64x4 mixed 4096", "op": "scores", "k": "q8_0", "seqs": 64, "len": 4096, "rows": 4, "hq": 14, "hkv": 2, "mixed": True,
         "picked": True},
        # the last 64 tokens of prompts as the observation window of a first eviction
        {"name": "scores 8x64 over 8192", "op": "scores", "k": "f16", "seqs": 8, "len": 8192, "rows": 64, "hq": 14, "hkv": 2, "mixed": False,
         "picked": False},
        # one utterance back to 512 positions after 64 new ones, every layer
        {"name": "evict 1x576 to 512", "op": "evict", "k": "q8_0", "v": "q8_0", "seqs": 1, "len": 576, "budget": 512, "layers": 24, "hkv": 2,
         "mixed": False},
        # a batch of long contexts cut to an eighth
        {"name": "evict 16x8192 to 1024", "op": "evict", "k": "q8_0", "v": "q4_0", "seqs": 16, "len": 8192, "budget": 1024, "layers": 6, "hkv": 2,
         "mixed": True},
    ]


def _between(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("tree", "tree", "commit", "scores", "evict"))
    types = sorted(TYPE_IDS)
    most = [work(c) for c in listed() if c["op"] == op]
    while True:
        hq, hkv = rng.choice(((14, 2), (14, 2), (16, 16), (8, 2), (12, 4)))
        c = {"op": op, "k": rng.choice(types), "seqs": _between(rng, 1, 64), "hkv": hkv}
        if op == "tree":
            c |= {"v": rng.choice(types), "len": _between(rng, 1, 65536), "nodes": _between(rng, 1, 128), "hq": hq, "mixed": rng.random() < 0.5,
                  "chain": rng.random() < 0.3}
        elif op == "commit":
            c |= {"v": rng.choice(types), "len": _between(rng, 32, 2048), "nodes": _between(rng, 1, 64), "layers": _between(rng, 1, 24)}
        elif op == "scores":
            c |= {"len": _between(rng, 1, 32768), "rows": _between(rng, 1, 128), "hq": hq, "mixed": rng.random() < 0.5, "picked": rng.random() < 0.5}
        else:
            c |= {"v": rng.choice(types), "len": _between(rng, 128, 32768), "layers": _between(rng, 1, 24), "mixed": rng.random() < 0.5}
            c["budget"] = max(96, int(c["len"] * rng.uniform(0.1, 0.95)))
        if 3072 in c.values():
            continue
        w = work(c)
        whole = c["seqs"] * c.get("layers", 1) * (_capacity(c) * sum(row_bytes(c[x], hkv) for x in "kv" if x in c))
        pairs = c["seqs"] * c.get("nodes", c.get("rows", 0)) * c.get("hq", 0) * c["len"]
        if whole <= 400e6 and pairs <= 60e6 and all(w[m] <= max(x[m] for x in most) for m in w):
            return c


def _lengths(c):
    """Committed positions of each sequence: all of them "len", or spread between a sixteenth of it and the whole."""
    if not c.get("mixed"):
        return [c["len"]] * c["seqs"]
    r = random.Random(c["len"] * 131 + c["seqs"])
    return [c["len"]] + [r.randint(max(1, c["len"] // 16), c["len"]) for _ in range(c["seqs"] - 1)]


def _counts(c, most):
    """Drafted, accepted or observed tokens of each sequence."""
    if not c.get("mixed") and c["op"] != "commit":
        return [most] * c["seqs"]
    r = random.Random(most * 977 + c["seqs"])
    return [most] + [r.randint(1, most) for _ in range(c["seqs"] - 1)]


def _capacity(c):
    return c["len"] + (c["nodes"] if c["op"] == "commit" else c["rows"] if c["op"] == "scores" else 0)


def _window(c):
    """(first tokens, last tokens) that an eviction never takes."""
    return min(4, c["budget"] // 8), min(64, c["budget"] // 4)


def work(case):
    c, L = case, _lengths(case)
    rk = row_bytes(c["k"], c["hkv"])
    rv = row_bytes(c["v"], c["hkv"]) if "v" in c else 0
    if c["op"] == "tree":
        n = _counts(c, c["nodes"])
        rows = c["seqs"] * c["nodes"] * c["hq"]
        pairs = sum(a * (b + a) for a, b in zip(n, L))
        return {"bytes": sum(a + b for a, b in zip(n, L)) * (rk + rv) + sum(n) * c["hq"] * D * 4 + rows * (D * 4 + 4)
                + c["seqs"] * c["nodes"] * ((c["nodes"] + 31) // 32) * 4 * (not c["chain"]), "flops": 4 * D * c["hq"] * pairs}
    if c["op"] == "commit":
        return {"bytes": 2 * sum(_counts(c, c["nodes"])) * c["layers"] * (rk + rv), "flops": 0}
    if c["op"] == "scores":
        n = [min(a, b) for a, b in zip(_counts(c, c["rows"]), L)]
        pairs = sum(a * b for a, b in zip(n, L))
        return {"bytes": sum(L) * (rk + 8 * c["hkv"]) + sum(n) * c["hq"] * (D * 4 + 4), "flops": 2 * D * c["hq"] * pairs}
    sink, recent = _window(c)
    size = 0
    for n in L:
        m = (n - c["budget"]) * (c["budget"] - sink) / (n - sink - recent) if n > c["budget"] else 0
        size += c["layers"] * (c["hkv"] * (16 * n + 16 * m) + 2 * m * (rk + rv))
    return {"bytes": int(size), "flops": 0}


# -------------------------------------------------------------------------------------------------------- cache rows

def _encode(t, x):
    """f32 [..., n] to the bytes of ggml rows."""
    if t == "f32":
        return x.contiguous().view(torch.uint8)
    if t == "f16":
        return x.half().contiguous().view(torch.uint8)
    b = x.reshape(*x.shape[:-1], -1, 32)
    two = lambda v: v.half().contiguous().view(torch.uint8)  # noqa: E731
    if t == "q8_0":
        d = b.abs().amax(-1, keepdim=True) / 127
        q = torch.round(b / d.clamp_min(1e-30)).clamp(-127, 127).to(torch.int8)
        return torch.cat((two(d), q.view(torch.uint8)), -1).flatten(-2)
    five, low = t.startswith("q5"), t.endswith("_1")
    top = 31 if five else 15
    if low:
        base = b.amin(-1, keepdim=True)
        d = (b.amax(-1, keepdim=True) - base) / top
        q = torch.round((b - base) / d.clamp_min(1e-30))
        head = [two(d), two(base)]
    else:
        far = b.gather(-1, b.abs().argmax(-1, keepdim=True))
        d = far / -(16 if five else 8)
        q = torch.trunc(b / torch.where(d == 0, torch.ones_like(d), d) + (16.5 if five else 8.5))
        head = [two(d)]
    q = q.clamp(0, top).to(torch.int32)
    if five:
        bits = ((q >> 4) << torch.arange(32, device=x.device, dtype=torch.int32)).sum(-1, keepdim=True, dtype=torch.int32)
        head.append(bits.contiguous().view(torch.uint8))
    return torch.cat(head + [((q[..., :16] & 15) | ((q[..., 16:] & 15) << 4)).to(torch.uint8)], -1).flatten(-2)


def _decode(t, raw, heads):
    """Bytes [..., row] to f32 [..., heads, 64]."""
    if t == "f32":
        return raw.view(torch.float32).unflatten(-1, (heads, D))
    if t == "f16":
        return raw.view(torch.float16).float().unflatten(-1, (heads, D))
    b = raw.unflatten(-1, (-1, BLOCK_BYTES[t]))
    d = b[..., 0:2].contiguous().view(torch.float16).float()
    if t == "q8_0":
        return (d * b[..., 2:].contiguous().view(torch.int8).float()).flatten(-2).unflatten(-1, (heads, D))
    nib = b[..., -16:]
    q = torch.cat((nib & 15, nib >> 4), -1).float()
    if t.startswith("q5"):
        at = 4 if t == "q5_1" else 2
        j = torch.arange(32, device=raw.device)
        q = q + 16.0 * ((b[..., at:at + 4][..., j // 8] >> (j % 8).to(torch.uint8)) & 1).float()
    if t.endswith("_1"):
        x = d * q + b[..., 2:4].contiguous().view(torch.float16).float()
    else:
        x = d * (q - (16 if t == "q5_0" else 8))
    return x.flatten(-2).unflatten(-1, (heads, D))


def _rows(g, t, shape, heads, spread=1.0):
    """Random cache rows of `shape`: keys and values of unit size with a few channels that stand out, as rotated keys have."""
    size = 1 + 3 * (torch.rand(heads * D, generator=g, device="cuda") < 0.04)
    out = torch.empty((*shape, row_bytes(t, heads)), dtype=torch.uint8, device="cuda")
    flat = out.view(-1, out.shape[-1])
    for i in range(0, flat.shape[0], 1 << 18):
        part = flat[i:i + (1 << 18)]
        part.copy_(_encode(t, torch.randn((part.shape[0], heads * D), generator=g, device="cuda") * size * spread))
    return out


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# --------------------------------------------------------------------------------------------------------- the inputs

def _tree_bits(rng, seqs, nodes):
    """Ancestors-and-self matrices [seqs, nodes, nodes] of random trees: a node hangs below one of the few before it, or at the root."""
    sees = np.zeros((seqs, nodes, nodes), dtype=bool)
    every = np.arange(seqs)
    for i in range(nodes):
        parent = i - 1 - rng.integers(0, 4, seqs)
        has = parent >= 0
        sees[every[has], i] = sees[every[has], parent[has]]
        sees[:, i, i] = True
    return sees


def _pack(bits):
    n = bits.shape[-1]
    wide = np.zeros((*bits.shape[:-1], (n + 31) // 32 * 32), dtype=bool)
    wide[..., :n] = bits
    return torch.from_numpy(np.packbits(wide, axis=-1, bitorder="little").view(np.int32).copy()).cuda()


def _log_sums(q, k, L, n, scale):
    """The log-sum-exp of each observed row, as the attention that came before gave it (row i of n sees L - n + i + 1 keys)."""
    S, R, hq, _ = q.shape
    hkv, cap = k.shape[2], k.shape[1]
    j, i = torch.arange(cap, device="cuda"), torch.arange(R, device="cuda")
    out = torch.zeros((S, R, hq), device="cuda")
    for s in range(S):
        x = torch.einsum("nhgd,lhd->nhgl", q[s].view(R, hkv, hq // hkv, D), k[s]) * scale
        sees = j[None] < (L[s] - n[s] + i + 1)[:, None]
        x = x.masked_fill(~sees[:, None, None], -math.inf).logsumexp(-1)
        out[s] = x.reshape(R, hq)
    return out


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    S, hkv, L = c["seqs"], c["hkv"], _lengths(c)
    cap = _capacity(c)
    s = {"case": c, "seed": seed}
    if c["op"] == "tree":
        n, hq = c["nodes"], c["hq"]
        s |= {"k": _rows(g, c["k"], (S, cap), hkv), "v": _rows(g, c["v"], (S, cap), hkv),
              "k_draft": _rows(g, c["k"], (S, n), hkv), "v_draft": _rows(g, c["v"], (S, n), hkv),
              "q": torch.randn((S, n, hq, D), generator=g, device="cuda"), "kv_len": _ints(L), "n_nodes": _ints(_counts(c, n)),
              "mask": None if c["chain"] else _pack(_tree_bits(rng, S, n)),
              "out": torch.empty((S, n, hq, D), device="cuda"), "lse": torch.empty((S, n, hq), device="cuda")}
    elif c["op"] == "commit":
        n, count = c["nodes"], _counts(c, c["nodes"])
        path = np.zeros((S, n), dtype=np.int32)
        for i, m in enumerate(count):  # an accepted path: nodes in the order of their depth
            path[i, :m] = np.sort(rng.permutation(n)[:m])
        s |= {"k": _rows(g, c["k"], (c["layers"], S, cap), hkv), "v": _rows(g, c["v"], (c["layers"], S, cap), hkv),
              "k_draft": _rows(g, c["k"], (c["layers"], S, n), hkv), "v_draft": _rows(g, c["v"], (c["layers"], S, n), hkv),
              "path": torch.from_numpy(path).cuda(), "count": _ints(count),
              "kv_len": _ints(rng.integers(c["len"] // 2, c["len"] + 1, S).tolist()), "kv_len_out": torch.zeros(S, dtype=torch.int32, device="cuda")}
    elif c["op"] == "scores":
        R, hq = c["rows"], c["hq"]
        count = [min(a, b) for a, b in zip(_counts(c, R), L)]
        pool = 2 * R if c["picked"] else R  # the drafted rows that the accepted ones were picked from
        k = _rows(g, c["k"], (S, cap), hkv)
        q = torch.randn((S, pool, hq, D), generator=g, device="cuda")
        pick = np.sort(np.stack([rng.permutation(pool)[:R] for _ in range(S)]), axis=1).astype(np.int32)
        pick = torch.from_numpy(pick).cuda()
        at = pick.long()[:, :, None].expand(S, R, hq)
        lse = torch.zeros((S, pool, hq), device="cuda")
        seen = q.gather(1, at[..., None].expand(S, R, hq, D))
        found = torch.cat([_log_sums(seen[i:i + 1], _decode(c["k"], k[i:i + 1], hkv), L[i:i + 1], count[i:i + 1], D ** -0.5) for i in range(S)])
        lse.scatter_(1, at, found)
        old = torch.rand((S, hkv, cap), generator=g, device="cuda") ** 4
        s |= {"k": k, "q": q, "lse": lse, "rows": pick if c["picked"] else None, "n_rows": _ints(count), "kv_len": _ints(L),
              "scores": old * (torch.arange(cap, device="cuda") < _ints(L)[:, None])[:, None], "out": torch.zeros((S, hkv, cap), device="cuda")}
    else:
        shape = (c["layers"], S, hkv, cap)
        kept = [min(a, c["budget"] - c["budget"] // 8) for a in L]
        j = torch.arange(cap, device="cuda")
        old = torch.rand(shape, generator=g, device="cuda") ** 4
        old = old * (0.5 < torch.rand(shape, generator=g, device="cuda"))  # many positions never got any weight to speak of
        # after an earlier eviction the kept slots hold any of the past tokens, each once
        total = [n + n // 2 for n in L]
        past = torch.rand((*shape[:3], cap + cap // 2), generator=g, device="cuda")
        first = _ints(total) - _ints(L) + _ints(kept)  # tokens that the kept slots were taken from
        past = past.masked_fill(torch.arange(past.shape[-1], device="cuda") >= first[:, None, None], 2.0)
        pos = past.argsort(-1)[..., :cap].int()
        s |= {"k": _rows(g, c["k"], (c["layers"], S, cap), hkv), "v": _rows(g, c["v"], (c["layers"], S, cap), hkv),
              "scores": old * (j < _ints(L)[:, None, None]), "pos": pos, "kv_len": _ints(L), "kept": _ints(kept), "total": _ints(total),
              "scores_out": torch.zeros(shape, device="cuda"), "pos_out": torch.zeros(shape, dtype=torch.int32, device="cuda"),
              "kv_len_out": torch.zeros(S, dtype=torch.int32, device="cuda")}
    return s


# ------------------------------------------------------------------------------------------------------- plain forms

def _plain_tree(s, c):
    S, n, hq, _ = s["q"].shape
    hkv, cap = c["hkv"], s["k"].shape[1]
    k = torch.cat((_decode(c["k"], s["k"], hkv), _decode(c["k"], s["k_draft"], hkv)), 1)
    v = torch.cat((_decode(c["v"], s["v"], hkv), _decode(c["v"], s["v_draft"], hkv)), 1)
    j, i = torch.arange(cap, device="cuda"), torch.arange(n, device="cuda")
    if s["mask"] is None:
        drafts = (i[None] <= i[:, None]).expand(S, n, n)
    else:
        drafts = ((s["mask"][..., i // 32] >> (i % 32).int()) & 1).bool()
    real = i[None] < s["n_nodes"][:, None]
    sees = torch.cat(((j[None] < s["kv_len"][:, None])[:, None].expand(S, n, cap), drafts & real[:, None]), -1) & real[..., None]
    x = torch.einsum("snhgd,slhd->shgnl", s["q"].view(S, n, hkv, hq // hkv, D), k) * D ** -0.5
    x = torch.where(sees[:, None, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.einsum("shgnl,slhd->snhgd", p, v) / torch.where(total == 0, 1.0, total).permute(0, 3, 1, 2, 4)
    lse = (top + torch.log(total)).squeeze(-1)
    return out.reshape(S, n, hq, D), lse.permute(0, 3, 1, 2).reshape(S, n, hq)


def _plain_commit(s, c):
    S, n = s["path"].shape
    i = torch.arange(n, device="cuda")
    seq, step = (i[None] < s["count"][:, None]).nonzero(as_tuple=True)
    node, slot = s["path"][seq, step].long(), (s["kv_len"][seq] + step).long()
    s["k"][:, seq, slot] = s["k_draft"][:, seq, node]
    s["v"][:, seq, slot] = s["v_draft"][:, seq, node]
    return s["k"], s["v"], s["kv_len"] + s["count"]


def _plain_scores(s, c):
    hkv, R = c["hkv"], c["rows"]
    q, lse = s["q"], s["lse"]
    S, _, hq, _ = q.shape
    if s["rows"] is not None:
        at = s["rows"].long()[:, :, None].expand(S, R, hq)
        q, lse = q.gather(1, at[..., None].expand(S, R, hq, D)), lse.gather(1, at)
    k = _decode(c["k"], s["k"], hkv)
    j, i = torch.arange(k.shape[1], device="cuda"), torch.arange(R, device="cuda")
    sees = j[None, None] <= (s["kv_len"] - s["n_rows"])[:, None, None] + i[None, :, None]
    sees = sees & (i[None] < s["n_rows"][:, None])[..., None]
    x = torch.einsum("snhgd,slhd->shgnl", q.view(S, R, hkv, hq // hkv, D), k) * D ** -0.5
    x = x - lse.view(S, R, hkv, hq // hkv).permute(0, 2, 3, 1)[..., None]
    got = torch.where(sees[:, None, None], torch.exp(x), 0.0).sum((2, 3))
    return torch.where((j[None] < s["kv_len"][:, None])[:, None], DECAY * s["scores"] + got, 0.0)


DECAY = 0.98


def _plain_evict(s, c):
    Ly, S, H, cap = s["scores"].shape
    budget, (sink, recent) = c["budget"], _window(c)
    L, total, kept = (s[x][None, :, None, None] for x in ("kv_len", "total", "kept"))
    j = torch.arange(cap, device="cuda")
    token = torch.where(j < kept, s["pos"], (total - L + j).int())
    real = j < L
    rank = torch.where(real, torch.where((token < sink) | (token >= total - recent), 0, 1), 2).expand(Ly, S, H, cap)
    by_score = s["scores"].argsort(dim=-1, descending=True, stable=True)
    order = by_score.gather(-1, rank.gather(-1, by_score).argsort(dim=-1, stable=True))
    place = torch.empty_like(order).scatter_(-1, order, j.expand(Ly, S, H, cap))
    keep = real & (place < budget)
    hole, mover = real & ~keep & (j < budget), keep & (j >= budget)
    # the i-th free slot below the budget takes the i-th kept row above it
    sources = torch.where(mover, j, cap).sort(-1).values
    source = torch.where(hole, sources.gather(-1, (hole.cumsum(-1) - 1).clamp_min(0)), j)
    left = torch.minimum(L, torch.full_like(L, budget))
    scores = torch.where(j < left, s["scores"].gather(-1, source), 0.0)
    pos = torch.where(j < left, token.gather(-1, source), 0)
    a, b, h, to = hole.nonzero(as_tuple=True)
    by = source[a, b, h, to]
    for name in ("k", "v"):
        x = s[name].view(Ly, S, cap, H, -1)
        x[a, b, to, h] = x[a, b, by, h]
    return {"k": s["k"], "v": s["v"], "scores": scores, "pos": pos.int(), "kv_len": left.flatten().int()}


# -------------------------------------------------------------------------------------------------- the engine's calls

_engine = {}


def _cv():
    """The engine and one context of this process."""
    if not _engine:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cosyvoice.cpp_b200"))
        import cvattn
        _engine["cv"], _engine["ctx"] = cvattn, cvattn.Context(0)
    return _engine["cv"], _engine["ctx"]


def _tensors(cv, s, c, name, which):
    """Descriptors of the layers of a cache buffer [layers, seqs, positions, row] or of one layer's [seqs, positions, row]."""
    b = s[name] if s[name].dim() == 4 else s[name][None]
    return [cv.kv_tensor(b[i], TYPE_IDS[c[which]], c["hkv"], D, b.shape[2], b.shape[1]) for i in range(b.shape[0])]


def _plan(s, c):
    """The launcher that a program builds once over its buffers and calls at every step."""
    cv, ctx = _cv()
    of = lambda name, which: _tensors(cv, s, c, name, which)  # noqa: E731
    if c["op"] == "tree":
        return cv.TreeDecoder(ctx, of("k", "k")[0], of("v", "v")[0], of("k_draft", "k")[0], of("v_draft", "v")[0], s["q"], s["out"], s["kv_len"],
                              max_kv_len=c["len"], lse=s["lse"], mask=s["mask"], n_nodes=s["n_nodes"])
    if c["op"] == "commit":
        return cv.TreeCommitter(ctx, of("k", "k") + of("v", "v"), of("k_draft", "k") + of("v_draft", "v"), s["path"], s["count"], s["kv_len"],
                                s["kv_len_out"])
    if c["op"] == "scores":
        return cv.KVScorer(ctx, of("k", "k")[0], s["q"], s["lse"], s["kv_len"], s["scores"], s["out"], max_kv_len=c["len"], decay=DECAY,
                           rows=s["rows"], n_rows=s["n_rows"])
    sink, recent = _window(c)
    return cv.KVEvictor(ctx, of("k", "k"), of("v", "v"), s["scores"], s["pos"], s["kv_len"], s["kept"], s["total"], c["budget"], s["scores_out"],
                        s["pos_out"], s["kv_len_out"], max_kv_len=c["len"], n_sink=sink, n_recent=recent)


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"tree": _plain_tree, "commit": _plain_commit, "scores": _plain_scores, "evict": _plain_evict}[c["op"]](s, c)
    if "plan" not in s:
        s["plan"] = _plan(s, c)
    s["plan"]()
    if c["op"] == "tree":
        return s["out"], s["lse"]
    if c["op"] == "commit":
        return s["k"], s["v"], s["kv_len_out"]
    if c["op"] == "scores":
        return s["out"]
    return {"k": s["k"], "v": s["v"], "scores": s["scores_out"], "pos": s["pos_out"], "kv_len": s["kv_len_out"]}


# ------------------------------------------------------------------------------------------------------------- exact

def _exact_rows(t, raw, heads):
    """Bytes [positions, row] to f64 [positions, heads, 64], block by block as the formats define them."""
    n = raw.shape[0]
    if t in ("f32", "f16"):
        return raw.contiguous().view(torch.float32 if t == "f32" else torch.float16).double().reshape(n, heads, D)
    b = raw.reshape(-1, BLOCK_BYTES[t]).long()
    half = lambda at: (b[:, at] + 256 * b[:, at + 1]).to(torch.int32).to(torch.int16).view(torch.float16).double()[:, None]  # noqa: E731
    if t == "q8_0":
        w = b[:, 2:]
        return (half(0) * (w - 256 * (w > 127)).double()).reshape(n, heads, D)
    first = {"q4_0": 2, "q4_1": 4, "q5_0": 6, "q5_1": 8}[t]
    w = torch.zeros((b.shape[0], 32), dtype=torch.long, device=raw.device)
    w[:, :16] = b[:, first:] % 16
    w[:, 16:] = b[:, first:] // 16
    if first in (6, 8):
        for e in range(32):
            w[:, e] += 16 * ((b[:, first - 4 + e // 8] >> (e % 8)) % 2)
    if first in (4, 8):
        return (half(0) * w.double() + half(2)).reshape(n, heads, D)
    return (half(0) * (w - (8 if first == 2 else 16)).double()).reshape(n, heads, D)


def exact(case, seed):
    s, c = prepare(case, seed), dict(case)
    S, hkv = c["seqs"], c["hkv"]
    if c["op"] == "tree":
        hq, n = c["hq"], c["nodes"]
        out = torch.zeros((S, n, hq, D), dtype=torch.float64, device="cuda")
        lse = torch.full((S, n, hq), -math.inf, dtype=torch.float64, device="cuda")
        for i in range(S):
            L, m = int(s["kv_len"][i]), int(s["n_nodes"][i])
            k = torch.cat((_exact_rows(c["k"], s["k"][i, :L], hkv), _exact_rows(c["k"], s["k_draft"][i, :m], hkv)))
            v = torch.cat((_exact_rows(c["v"], s["v"][i, :L], hkv), _exact_rows(c["v"], s["v_draft"][i, :m], hkv)))
            sees = torch.zeros((m, L + m), dtype=torch.bool)
            sees[:, :L] = True
            words = None if s["mask"] is None else s["mask"][i].cpu().numpy().view(np.uint32)
            for a in range(m):
                for b in range(m):
                    sees[a, L + b] = b <= a if words is None else bool((int(words[a, b // 32]) >> (b % 32)) & 1)
            sees = sees.cuda()
            for h in range(hq):
                x = (s["q"][i, :m, h].double() @ k[:, h // (hq // hkv)].T) / 8.0
                x[~sees] = -math.inf
                lse[i, :m, h] = torch.logsumexp(x, 1)
                out[i, :m, h] = torch.softmax(x, 1) @ v[:, h // (hq // hkv)]
        return out, lse
    if c["op"] == "commit":
        k, v = s["k"].clone(), s["v"].clone()
        for i in range(S):
            for a in range(int(s["count"][i])):
                node, slot = int(s["path"][i, a]), int(s["kv_len"][i]) + a
                k[:, i, slot] = s["k_draft"][:, i, node]
                v[:, i, slot] = s["v_draft"][:, i, node]
        return k, v, s["kv_len"] + s["count"]
    if c["op"] == "scores":
        hq = c["hq"]
        out = torch.zeros(s["scores"].shape, dtype=torch.float64, device="cuda")
        for i in range(S):
            L, m = int(s["kv_len"][i]), int(s["n_rows"][i])
            k = _exact_rows(c["k"], s["k"][i, :L], hkv)
            out[i, :, :L] = DECAY * s["scores"][i, :, :L].double()
            for a in range(m):
                at = a if s["rows"] is None else int(s["rows"][i, a])
                far = L - m + a + 1
                x = torch.einsum("hgd,lhd->hgl", s["q"][i, at].double().view(hkv, hq // hkv, D), k[:far]) / 8.0
                out[i, :, :far] += torch.exp(x - s["lse"][i, at].double().view(hkv, hq // hkv, 1)).sum(1)
        return out
    if c["layers"] * S * hkv > 4000:
        return None
    budget, (sink, recent) = c["budget"], _window(c)
    k, v = s["k"].cpu().numpy().copy(), s["v"].cpu().numpy().copy()
    old, pos, lens, kept, total = (s[x].cpu().numpy() for x in ("scores", "pos", "kv_len", "kept", "total"))
    scores, where = np.zeros(old.shape), np.zeros_like(pos)
    for layer in range(c["layers"]):
        for i in range(S):
            n = int(lens[i])
            for h in range(hkv):
                token = pos[layer, i, h, :n].astype(np.int64)
                token[kept[i]:] = np.arange(kept[i], n) + total[i] - n
                slot = np.arange(n)
                if n > budget:
                    safe = (token < sink) | (token >= total[i] - recent)
                    order = np.lexsort((slot, -old[layer, i, h, :n].astype(np.float64), ~safe))
                    best = np.sort(order[:budget])
                    slot = np.arange(budget)
                    free = np.setdiff1d(slot, best)
                    slot[free] = best[best >= budget]
                    for x in (k, v):
                        w = x.shape[-1] // hkv
                        x[layer, i, free, h * w:(h + 1) * w] = x[layer, i, slot[free], h * w:(h + 1) * w]
                scores[layer, i, h, :len(slot)] = old[layer, i, h, slot]
                where[layer, i, h, :len(slot)] = token[slot]
    return {"k": k, "v": v, "scores": scores, "pos": where, "kv_len": np.minimum(lens, budget)}
