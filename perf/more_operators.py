"""Cases of the operators for serving from a paged 8-bit KV cache, and of the verification of drafted tokens.

Four operators.  A page holds `page` positions (a multiple of 16) of one layer's keys or values, head by head, in blocks of
16 positions x 64 values with one f32 scale each; a table lists each sequence's pages in order.

  attend  attention of each sequence's last tokens over its pages
  append  new keys and values rounded into the pages, and the rows of the touched blocks read back
  assign  tables forked, cut back and grown, shared tail pages copied;  compact  pages moved to the pool's front
  verify  drafted tokens checked against the target's logits with given random numbers

With ``own`` false, ``run`` computes them from elementary torch operations, in 32 bits (verification in 64: a sum over a
vocabulary next to a border decides a token); with ``own`` true it calls the engine's entry points.  ``exact`` computes them
in 64 bits from their definitions.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

D = 64
BLOCK = 16
FORMATS = ("i8", "e4m3")
MOST_CODE = {"i8": 127.0, "e4m3": 448.0}


# ------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one utterance after a short prompt, one token: the latency of a single layer's attention
        {"name": "attend 1x1 over 300", "op": "attend", "format": "i8", "seqs": 1, "len": 300, "rows": 1, "hq": 14, "hkv": 2, "page": 16,
         "mixed": False},
        # a batch of utterances of all lengths, a token each
        {"name": "attend 64x1 mixed 4096", "op": "attend", "format": "e4m3", "seqs": 64, "len": 4096, "rows": 1, "hq": 14, "hkv": 2,
         "page": 64, "mixed": True},
        # chains of drafts verified over long contexts
        {"name": "attend 16x16 over 8192", "op": "attend", "format": "i8", "seqs": 16, "len": 8192, "rows": 16, "hq": 14, "hkv": 2,
         "page": 32, "mixed": False},
        # pieces of long prompts, an odd length, one KV head for each query head
        {"name": "attend 4x512 of 2501", "op": "attend", "format": "e4m3", "seqs": 4, "len": 2501, "rows": 512, "hq": 16, "hkv": 16,
         "page": 128, "mixed": True},
        # the step's token of a batch: most blocks have rows already, some scales grow
        {"name": "append 64x1 at 700", "op": "append", "format": "i8", "seqs": 64, "len": 700, "rows": 1, "hkv": 2, "page": 32, "mixed": True},
        # prompts of several utterances at once
        {"name": "append 16x1500", "op": "append", "format": "e4m3", "seqs": 16, "len": 5, "rows": 1500, "hkv": 2, "page": 64, "mixed": True},
        # a decode step's room for one more token: a page for a few, nothing to copy
        {"name": "assign 64 step", "op": "assign", "seqs": 64, "len": 1024, "page": 16, "hkv": 2, "layers": 24, "fan": 1, "more": 1,
         "mixed": True},
        # sixteen utterances forked to four candidates each: three copies of every partly filled page in every layer
        {"name": "assign 16 to 64", "op": "assign", "seqs": 64, "len": 1000, "page": 64, "hkv": 2, "layers": 24, "fan": 4, "more": 8,
         "mixed": True},
        # a pool of which two thirds are free, scattered: live pages to the front
        {"name": "compact 32 of 1500", "op": "compact", "seqs": 32, "len": 1500, "page": 32, "hkv": 2, "layers": 12, "mixed": True},
        # one utterance over a vocabulary of speech tokens, drafts from a lookup, checked as a tree
        {"name": "verify 1x7 tree of 6563", "op": "verify", "type": "f32", "seqs": 1, "nodes": 7, "vocab": 6563, "chain": False,
         "probs": False, "heat": 0.8},
        # a batch with chains of a draft model over a vocabulary of speech tokens
        {"name": "verify 64x5 of 6563", "op": "verify", "type": "f32", "seqs": 64, "nodes": 5, "vocab": 6563, "chain": True, "probs": True,
         "heat": 1.0},
        # a batch over a large text vocabulary, 16-bit logits
        {"name": "verify 32x8 of 151937", "op": "verify", "type": "bf16", "seqs": 32, "nodes": 8, "vocab": 151937, "chain": True,
         "probs": True, "heat": 0.7},
    ]


def _between(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("attend", "attend", "append", "assign", "compact", "verify"))
    most = [work(c) for c in listed() if c["op"] == op]
    while True:
        c = {"op": op, "seqs": _between(rng, 1, 64)}
        hq, hkv = rng.choice(((14, 2), (14, 2), (16, 16), (8, 2), (12, 4), (5, 5), (8, 1)))
        if op != "verify":
            c |= {"len": _between(rng, 1, 65536 if op == "attend" else 4096), "hkv": hkv, "page": rng.choice((16, 32, 64, 128)),
                  "mixed": rng.random() < 0.5}
        if op == "attend":
            c |= {"format": rng.choice(FORMATS), "rows": _between(rng, 1, 512), "hq": hq}
        elif op == "append":
            c |= {"format": rng.choice(FORMATS), "rows": _between(rng, 1, 1500)}
        elif op == "assign":
            c |= {"layers": _between(rng, 1, 24), "fan": rng.choice((1, 2, 3, 4, 8)), "more": _between(rng, 1, 100)}
        elif op == "compact":
            c |= {"layers": _between(rng, 1, 24)}
        else:
            c |= {"type": rng.choice(("f32", "f16", "bf16")), "nodes": _between(rng, 1, 32), "vocab": _between(rng, 100, 160000),
                  "chain": rng.random() < 0.6, "probs": rng.random() < 0.5, "heat": rng.choice((0.0, 0.7, 1.0, 1.3))}
        w = work(c)
        pairs = c["seqs"] * c.get("rows", 0) * c.get("hq", 0) * c.get("len", 0)
        held = c["seqs"] * (c.get("len", 0) + c.get("rows", 0)) * hkv * D * 2 * c.get("layers", 1)
        if c.get("nodes", 0) * c["seqs"] * c.get("vocab", 0) > 45e6:
            continue
        if held <= 400e6 and pairs <= 100e6 and all(w[m] <= max(x[m] for x in most) for m in w):
            return c


def _spread(c, most, salt):
    """A number for each sequence: `most`, or spread between a sixteenth of it and the whole, the first one whole."""
    if not c.get("mixed"):
        return [most] * c["seqs"]
    r = random.Random(most * 131 + c["seqs"] + salt)
    return [most] + [r.randint(max(1, most // 16), most) for _ in range(c["seqs"] - 1)]


def _lengths(c):
    """(positions of each sequence, its own rows): for append the positions before it, for attend the whole, rows included."""
    L = _spread(c, c["len"], 0)
    if "rows" not in c:
        return L, None
    n = _spread(c, c["rows"], 7)
    return L, [min(a, b) for a, b in zip(n, L)] if c["op"] == "attend" else n


def _kept(c):
    """Positions that each sequence of an assignment starts from: groups of `fan` fork the same one."""
    L = _spread(c, c["len"], 0)
    return [L[s // c["fan"]] for s in range(c["seqs"])]


#: How often a draft is taken, about: what it says of the rows that a verification cannot do without.
TAKEN = 0.7


def work(case):
    c = case
    if c["op"] == "verify":
        # the logits of the nodes on the accepted path, and one row of probabilities where a draft was refused
        size = {"f32": 4, "f16": 2, "bf16": 2}[c["type"]]
        deep = c["nodes"] if c["chain"] else 1 + c["nodes"] // 3
        rows = sum(TAKEN ** i for i in range(deep))
        row = c["vocab"] * (rows * size + 4 * (1 - TAKEN ** deep) * c["probs"])
        return {"bytes": int(c["seqs"] * (row + 20 * c["nodes"] + 12)), "flops": int(c["seqs"] * rows * c["vocab"] * 2)}
    P, hkv = c["page"], c["hkv"]
    pages = lambda n: -(-n // P)  # noqa: E731
    page_bytes = 2 * hkv * (P * D + P // BLOCK * 4)
    if c["op"] == "assign":
        kept = _kept(c)
        whole = sum(pages(n + c["more"]) for n in kept)
        copies = sum(kept[g] % P != 0 for g in range(0, c["seqs"], c["fan"]) for _ in range(min(c["fan"], c["seqs"] - g) - 1))
        return {"bytes": 8 * whole + 4 * _pool_pages(c) + 2 * copies * page_bytes * c["layers"], "flops": 0}
    L, n = _lengths(c)
    if c["op"] == "compact":
        live = sum(pages(x) for x in L)
        moved = live * (1 - live / _pool_pages(c))
        return {"bytes": int(8 * live + 4 * _pool_pages(c) + 2 * moved * page_bytes * c["layers"]), "flops": 0}
    if c["op"] == "append":
        touched = sum(x % BLOCK + y for x, y in zip(L, n))
        return {"bytes": 2 * hkv * D * (4 * sum(n) + 2 * touched + 4 * touched) + 2 * hkv * 8 * touched // BLOCK, "flops": 0}
    pairs = sum(a * b - a * (a - 1) // 2 for a, b in zip(n, L))
    rows = c["seqs"] * c["rows"] * c["hq"]
    return {"bytes": sum(L) * hkv * (2 * D + 8 // BLOCK) + sum(n) * c["hq"] * D * 4 + rows * (D * 4 + 4) + 4 * sum(pages(x) for x in L),
            "flops": 4 * D * c["hq"] * pairs}


# ------------------------------------------------------------------------------------------------------------- pages

def _pack(x, values):
    """Codes uint8 [..., 16, 64] of blocks, position by position, as they lie in a page's K or (values) V."""
    if not values:
        return x.flatten(-2)
    y = x.unflatten(-1, (2, 4, 8)).unflatten(-4, (4, 4))  # position: quarter, step; value: half, tile, lane
    n = y.dim()
    return y.permute(*range(n - 5), n - 3, n - 1, n - 5, n - 2, n - 4).flatten(-5)


def _unpack(x, values):
    """The inverse: uint8 [..., 1024] to [..., 16, 64]."""
    if not values:
        return x.unflatten(-1, (BLOCK, D))
    y = x.unflatten(-1, (2, 8, 4, 4, 4))  # half, lane, quarter, tile, step
    n = y.dim()
    return y.permute(*range(n - 5), n - 3, n - 1, n - 5, n - 2, n - 4).flatten(-3).flatten(-3, -2)


def _values(fmt, codes):
    """What codes stand for, in units of their block's scale."""
    if fmt == "i8":
        return codes.float() - 128.0
    return codes.view(torch.float8_e4m3fn).float()


def _codes(fmt, x):
    """Codes of the nearest values to x (f64, so that next to a border between two the nearer one is found), ties to even."""
    x = x.clamp(-MOST_CODE[fmt], MOST_CODE[fmt])
    if fmt == "i8":
        return (torch.round(x) + 128.0).to(torch.uint8)
    step = torch.ldexp(torch.ones_like(x), torch.frexp(x).exponent.clamp_min(-5) - 4)
    return (torch.round(x / step) * step).to(torch.float8_e4m3fn).view(torch.uint8)


def _scales(fmt, x):
    """Scales of blocks [..., 16, 64]: the largest finite value over the format's largest; none that is not a normal number."""
    a = torch.where(torch.isfinite(x), x.abs(), 0.0).amax((-2, -1))
    a = a / torch.full_like(a, MOST_CODE[fmt])  # (a tensor: by a number torch multiplies by its rounded inverse)
    return torch.where(a < torch.finfo(torch.float32).tiny, 0.0, a)


def _encode(fmt, x, scale):
    """Codes of x [..., 16, 64] under their blocks' scales."""
    scale = scale[..., None, None].double()
    return _codes(fmt, torch.where(torch.isnan(x) | (scale == 0), 0.0, x / torch.where(scale > 0, scale, 1.0)))


def _pool_pages(c):
    """Pages of a pool: room for the sequences and a quarter more, thrice as many for one that is to be compacted."""
    P = c["page"]
    if c["op"] == "assign":
        need = sum(-(-(n + c["more"]) // P) for n in _kept(c)) + c["seqs"]
    else:
        L, n = _lengths(c)
        need = sum(-(-(a + (b if c["op"] == "append" else 0)) // P) for a, b in zip(L, n or L))
    return 3 * need + 2 if c["op"] == "compact" else need + need // 4 + 1


def _fill_pool(g, c, pages, values):
    """One layer's K or V: keys of unit size with a few channels that stand out, as rotated keys have; blocks of differing size."""
    fmt, hkv, P = c["format"], c["hkv"], c["page"]
    size = 1 + 3 * (torch.rand((hkv, 1, 1, D), generator=g, device="cuda") < 0.04)
    codes = torch.empty((pages, hkv, P * D), dtype=torch.uint8, device="cuda")
    scales = torch.empty((pages, hkv, P // BLOCK), device="cuda")
    step = max(1, (1 << 24) // (hkv * P * D))
    for i in range(0, pages, step):
        m = min(step, pages - i)
        x = torch.randn((m, hkv, P // BLOCK, BLOCK, D), generator=g, device="cuda") * size
        x *= 0.5 + torch.rand((m, hkv, P // BLOCK, 1, 1), generator=g, device="cuda")
        scales[i:i + m] = _scales(fmt, x)
        codes[i:i + m] = _pack(_encode(fmt, x, scales[i:i + m]), values).flatten(-2)
    return codes, scales


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _table(rng, c, counts, width, pages):
    """Tables of scattered pages: counts[s] entries for sequence s, the rest -1."""
    order = rng.permutation(pages)
    t = np.full((len(counts), width), -1, dtype=np.int32)
    at = 0
    for s, m in enumerate(counts):
        t[s, :m] = order[at:at + m]
        at += m
    return torch.from_numpy(t).cuda()


# --------------------------------------------------------------------------------------------------------- the inputs

def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    S, s = c["seqs"], {"case": c, "seed": seed}
    if c["op"] == "verify":
        return s | _prepare_verify(c, g, rng)
    P, hkv, pages = c["page"], c["hkv"], _pool_pages(c)
    if c["op"] in ("attend", "append"):
        L, n = _lengths(c)
        ends = [a + (b if c["op"] == "append" else 0) for a, b in zip(L, n)]
        s |= {"table": _table(rng, c, [-(-x // P) for x in ends], -(-max(ends) // P), pages), "kv_len": _ints(L), "n": _ints(n)}
        for name, values in (("k", False), ("v", True)):
            s[name], s[name + "_scale"] = _fill_pool(g, c, pages, values)
        if c["op"] == "attend":
            shape = (S, c["rows"], c["hq"], D)
            s |= {"q": torch.randn(shape, generator=g, device="cuda"), "out": torch.empty(shape, device="cuda"),
                  "lse": torch.empty(shape[:3], device="cuda")}
        else:
            m = c["rows"]
            for name in ("k_new", "v_new"):
                size = 0.25 + torch.rand((S, m, 1), generator=g, device="cuda") * 1.75
                s[name] = torch.randn((S, m, hkv * D), generator=g, device="cuda") * size
                s[name + "_back"] = torch.empty((S, m + BLOCK - 1, hkv * D), device="cuda")
            s |= {"first": _ints([x // BLOCK * BLOCK for x in L]), "touched": _ints([x % BLOCK + y for x, y in zip(L, n)])}
        return s
    layers = c["layers"]
    for name, width, dtype in (("k", P * D, torch.uint8), ("v", P * D, torch.uint8), ("k_scale", P // BLOCK, torch.float32),
                               ("v_scale", P // BLOCK, torch.float32)):
        shape = (layers, pages, hkv, width)
        s[name] = (torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8) if dtype == torch.uint8
                   else torch.rand(shape, generator=g, device="cuda"))
    if c["op"] == "assign":
        kept = _kept(c)
        # the rows of the table that the forked ones get were empty
        held = [kept[i] if i % c["fan"] == 0 else 0 for i in range(S)]
        s["table"] = _table(rng, c, [-(-x // P) for x in held], -(-(max(kept) + c["more"]) // P), pages)
        s |= {"src": _ints([i // c["fan"] * c["fan"] for i in range(S)]), "keep": _ints(kept), "need": _ints([x + c["more"] for x in kept]),
              "room": _ints([0] * S)}
    else:
        L, _ = _lengths(c)
        s["table"] = _table(rng, c, [-(-x // P) for x in L], -(-max(L) // P), pages)
        s["n_live"] = _ints([0])
    s |= {"table_out": torch.empty_like(s["table"]), "refs": torch.empty(pages, dtype=torch.int32, device="cuda")}
    return s


DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _prepare_verify(c, g, rng):
    """Logits with the spread that language models have, a draft model that is near them, and drafts drawn from it."""
    S, n, V = c["seqs"], c["nodes"], c["vocab"]
    sigma = math.sqrt(2 * math.log(V / 20)) if V > 40 else 1.0  # about twenty likely tokens
    logits = torch.randn((S, n, V), generator=g, device="cuda").mul_(sigma)
    parents = np.arange(-1, n - 1, dtype=np.int32)[None].repeat(S, 0)
    if not c["chain"]:
        for i in range(1, n):
            parents[:, i] = np.maximum(0, i - 1 - rng.integers(0, 4, S))
    above = torch.from_numpy(np.maximum(parents, 0)).cuda().long()
    probs = torch.empty((S, n, V), device="cuda")
    for i in range(S):
        near = logits[i] + torch.randn((n, V), generator=g, device="cuda") * 0.4
        probs[i] = torch.softmax(near if c["probs"] else near * 2, -1)
    drawn = torch.stack([torch.multinomial(probs[i, above[i]], 1, generator=g)[:, 0] for i in range(S)]).int()
    every = torch.arange(S * n, device="cuda").view(S, n)
    s = {"logits": logits.to(DTYPES[c["type"]]), "tokens": drawn, "probs": probs if c["probs"] else None,
         "parents": None if c["chain"] else torch.from_numpy(parents).cuda(),
         "accept_u": torch.rand((S, n), generator=g, device="cuda"), "sample_u": torch.rand(S, generator=g, device="cuda"),
         "heat": torch.full((S,), c["heat"], device="cuda"), "accepted": torch.empty_like(every, dtype=torch.int32)}
    return s | {"count": torch.empty(S, dtype=torch.int32, device="cuda"), "token": torch.empty(S, dtype=torch.int32, device="cuda"),
                "log_probs": torch.empty((S, n), device="cuda")}


# ---------------------------------------------------------------------------------------------------- the plain forms

def _gather(s, c, name, values):
    """f32 [S, positions, Hkv, 64] of every page of the tables (-1: page 0)."""
    at = s["table"].clamp_min(0).long()
    x = _values(c["format"], _unpack(s[name][at].unflatten(-1, (-1, BLOCK * D)), values))  # [S, pages, H, blocks, 16, 64]
    x = x * s[name + "_scale"][at][..., None, None]
    return x.transpose(2, 3).transpose(3, 4).flatten(1, 3)


def _plain_attend(s, c):
    S, n, hq, hkv = c["seqs"], c["rows"], c["hq"], c["hkv"]
    k, v = _gather(s, c, "k", False), _gather(s, c, "v", True)
    j, i = torch.arange(k.shape[1], device="cuda"), torch.arange(n, device="cuda")
    sees = j < (s["kv_len"] - s["n"])[:, None, None] + i[:, None] + 1
    sees = sees & (i[:, None] < s["n"][:, None, None])
    x = torch.einsum("snhgd,slhd->shgnl", s["q"].view(S, n, hkv, hq // hkv, D), k) * D ** -0.5
    x = torch.where(sees[:, None, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.einsum("shgnl,slhd->snhgd", p, v) / torch.where(total == 0, 1.0, total).permute(0, 3, 1, 2, 4)
    lse = (top + torch.log(total)).squeeze(-1)
    return out.reshape(S, n, hq, D), lse.permute(0, 3, 1, 2).reshape(S, n, hq)


def _plain_append(s, c):
    fmt, P, hkv, S = c["format"], c["page"], c["hkv"], c["seqs"]
    m = s["k_new"].shape[1]
    blocks = (m + 2 * BLOCK - 2) // BLOCK
    b = s["first"][:, None] // BLOCK + torch.arange(blocks, device="cuda")
    real = b * BLOCK < (s["kv_len"] + s["n"])[:, None]
    seq, which = real.nonzero(as_tuple=True)
    b = b[seq, which].long()
    page, part = s["table"][seq, b * BLOCK // P].long(), b % (P // BLOCK)
    at = b[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")  # positions of the touched blocks
    L, n = s["kv_len"][seq][:, None], s["n"][seq][:, None]
    old, new = (at < L)[:, None, :, None], ((at >= L) & (at < L + n))[:, None, :, None]
    for name, values in (("k", False), ("v", True)):
        pool, scales = s[name].unflatten(-1, (-1, BLOCK * D)), s[name + "_scale"]
        was = _unpack(pool[page, :, part], values)  # [touched, H, 16, 64]
        x = s[name + "_new"][seq[:, None], (at - L).clamp(0, m - 1)].unflatten(-1, (hkv, D)).transpose(1, 2)
        x = torch.where(new, x, 0.0)
        before = torch.where(old.any(2).expand(-1, hkv, -1)[..., 0], scales[page, :, part], 0.0)
        scale = torch.maximum(before, _scales(fmt, x))
        grows, by = (scale > before)[..., None, None], torch.where(scale > 0, scale, 1.0).double()[..., None, None]
        kept = torch.where(grows, _codes(fmt, _values(fmt, was) * before[..., None, None].double() / by), was)
        pool[page, :, part] = _pack(torch.where(new, _encode(fmt, x, scale), torch.where(old, kept, was)), values)
        scales[page, :, part] = scale
    # the rows of the touched blocks as they stand now
    i = torch.arange(m + BLOCK - 1, device="cuda")
    at = (s["first"][:, None] + i).long()
    there = i < s["touched"][:, None]
    page = s["table"].gather(1, torch.where(there, at // P, 0)).long()
    part, row = at % P // BLOCK, at % BLOCK
    back = []
    for name, values in (("k", False), ("v", True)):
        x = _values(fmt, _unpack(s[name].unflatten(-1, (-1, BLOCK * D))[page, :, part], values))  # [S, rows, H, 16, 64]
        x = x.gather(3, row[:, :, None, None, None].expand(-1, -1, hkv, 1, D))[:, :, :, 0] * s[name + "_scale"][page, :, part][..., None]
        back.append(torch.where(there[..., None, None], x, 0.0).reshape(S, -1, hkv * D))
    return tuple(back)


def _plain_assign(s, c):
    P, pages, width = c["page"], s["refs"].shape[0], s["table"].shape[1]
    j, every = torch.arange(width, device="cuda"), torch.arange(c["seqs"], device="cuda")
    keep, need = s["keep"].long(), s["need"].long()
    kept = (keep + P - 1) // P
    table = torch.where(j < kept[:, None], s["table"][s["src"].long()], -1).long()
    count = lambda x: torch.zeros(pages, dtype=torch.int64, device="cuda").scatter_add_(0, x, torch.ones_like(x))  # noqa: E731
    refs = count(table[table >= 0])
    # who writes into a partly filled page that others hold copies it, but for the first where only writers hold it
    writes = (need > keep) & (keep % P != 0)
    tail = torch.where(writes, table.gather(1, (keep // P).clamp_max(width - 1)[:, None])[:, 0], 0)
    writers = torch.zeros(pages, dtype=torch.int64, device="cuda").scatter_add_(0, tail, writes.long())
    lowest = torch.full((pages,), c["seqs"], device="cuda").scatter_reduce_(0, tail, torch.where(writes, every, c["seqs"]), "amin")
    copies = writes & (refs[tail] > 1) & ~((writers[tail] == refs[tail]) & (lowest[tail] == every))
    fresh = ((need + P - 1) // P - kept).clamp_min(0) + copies
    end = fresh.cumsum(0)
    free = (refs == 0).nonzero()[:, 0]
    granted = end <= free.shape[0]
    first = kept - copies.long()  # the first entry that gets a page of its own
    rank = (end - fresh)[:, None] + j - first[:, None]
    takes = granted[:, None] & (j >= first[:, None]) & (j < (first + fresh)[:, None])
    copied = copies & granted
    source, target = tail[copied], free[(end - fresh)[copied]]
    table = torch.where(takes, free[rank.clamp(0, free.shape[0] - 1)], table)
    for name in ("k", "v", "k_scale", "v_scale"):
        s[name][:, target] = s[name][:, source]
    refs = count(table[table >= 0])
    room = torch.where(granted, torch.maximum(need, keep), keep)
    return {"table": table.int(), "refs": refs.int(), "room": room.int(), **{x: s[x] for x in ("k", "v", "k_scale", "v_scale")}}


def _plain_compact(s, c):
    pages = s["refs"].shape[0]
    table = s["table"].long()
    refs = torch.zeros(pages, dtype=torch.int64, device="cuda").scatter_add_(0, table[table >= 0], torch.ones_like(table[table >= 0]))
    page = torch.arange(pages, device="cuda")
    live = (refs > 0).sum()
    source, target = ((refs > 0) & (page >= live)).nonzero()[:, 0], ((refs == 0) & (page < live)).nonzero()[:, 0]
    to = page.clone()
    to[source] = target
    for name in ("k", "v", "k_scale", "v_scale"):
        s[name][:, target] = s[name][:, source]
    refs = torch.zeros_like(refs).scatter_(0, to[refs > 0], refs[refs > 0])
    table = torch.where(table >= 0, to[table.clamp_min(0)], -1)
    return {"table": table.int(), "refs": refs.int(), "n_live": live.int().view(1), **{x: s[x] for x in ("k", "v", "k_scale", "v_scale")}}


def _target(s, node):
    """f64 [S, V]: the target's probabilities at one node of each sequence."""
    every = torch.arange(node.shape[0], device="cuda")
    x = s["logits"][every, node].double()
    hot = x.argmax(-1, keepdim=True)
    heat = s["heat"].double()[:, None]
    x = (x - x.gather(1, hot)) / torch.where(heat > 0, heat, 1.0)
    w = torch.where(heat > 0, torch.exp(x), torch.zeros_like(x).scatter_(1, hot, 1.0))
    return w / w.sum(-1, keepdim=True)


def _plain_verify(s, c):
    S, n, _ = s["logits"].shape
    every = torch.arange(S, device="cuda")
    at, count = torch.zeros(S, dtype=torch.int64, device="cuda"), torch.ones(S, dtype=torch.int64, device="cuda")
    path = torch.full((S, n), -1, dtype=torch.int64, device="cuda")
    path[:, 0] = 0
    log_probs = torch.zeros((S, n), dtype=torch.float64, device="cuda")
    first = p = _target(s, at)  # of the node that a sequence is at, and what refused drafts have left of it
    for i in range(1, n):  # a node comes after its parent, siblings in order: each sequence walks down its tree
        here = s["parents"][:, i] == at if s["parents"] is not None else at == i - 1
        t = s["tokens"][:, i:i + 1].long()
        q = s["probs"][every, at].double() if s["probs"] is not None else torch.zeros_like(p).scatter_(1, t, 1.0)
        u = s["accept_u"][:, i].double()
        takes = here & (u * q.gather(1, t)[:, 0] < p.gather(1, t)[:, 0])
        if s["probs"] is not None:
            left = (p - q).clamp_min(0.0)
        else:
            left = p.scatter(1, t, 0.0)
        total = left.sum(-1, keepdim=True)
        left = torch.where(total > 0, left / torch.where(total > 0, total, 1.0), p)
        p = torch.where((here & ~takes)[:, None], left, p)
        at = torch.where(takes, i, at)
        path[every, count.clamp_max(n - 1)] = torch.where(takes, i, path[every, count.clamp_max(n - 1)])
        log_probs[every, count - 1] = torch.where(takes, torch.log(first.gather(1, t)[:, 0]), 0.0)
        count = count + takes.long()
        after = _target(s, at)
        first, p = after, torch.where(takes[:, None], after, p)
    sums = p.cumsum(-1)
    token = (sums > (s["sample_u"].double() * sums[:, -1])[:, None]).int().argmax(-1)
    log_probs[every, count - 1] = torch.log(first.gather(1, token[:, None])[:, 0])
    return {"accepted": path.int(), "count": count.int(), "token": token.int(), "log_probs": log_probs.float()}


# -------------------------------------------------------------------------------------------------- the engine's calls

_engine = {}


def _cv():
    """The engine and one context of this process."""
    if not _engine:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cosyvoice.cpp_b200"))
        import cvattn
        _engine["cv"], _engine["ctx"] = cvattn, cvattn.Context(0)
    return _engine["cv"], _engine["ctx"]


def _plan(s, c):
    """The launchers that a program builds once over its buffers and calls at every step."""
    cv, ctx = _cv()
    if c["op"] == "verify":
        return [cv.DraftVerifier(ctx, s["logits"], s["tokens"], s["accept_u"], s["sample_u"], s["accepted"], s["count"], s["token"],
                                 parents=s["parents"], draft_probs=s["probs"], temperature=s["heat"], log_probs=s["log_probs"])]
    if c["op"] in ("assign", "compact"):
        pools = [cv.PagePool(s["k"][i], s["v"][i], s["k_scale"][i], s["v_scale"][i], cv.PAGE_I8) for i in range(c["layers"])]
        if c["op"] == "assign":
            return [cv.PageAssigner(ctx, pools, s["table"], s["keep"], s["need"], src=s["src"], table_out=s["table_out"], refs=s["refs"],
                                    room=s["room"])]
        return [cv.PageCompactor(ctx, pools, s["table"], s["n_live"], table_out=s["table_out"], refs=s["refs"])]
    pool = cv.PagePool(s["k"], s["v"], s["k_scale"], s["v_scale"], cv.PAGE_I8 if c["format"] == "i8" else cv.PAGE_E4M3)
    if c["op"] == "attend":
        return [cv.PagedAttention(ctx, pool, s["q"], s["out"], s["table"], s["kv_len"], max_kv_len=c["len"], lse=s["lse"], n_q=s["n"])]
    return [cv.PageAppender(ctx, pool, s["k_new"], s["v_new"], s["table"], s["kv_len"], n_new=s["n"]),
            cv.PageReader(ctx, pool, s["k_new_back"], s["v_new_back"], s["table"], first=s["first"], n_rows=s["touched"])]


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"attend": _plain_attend, "append": _plain_append, "assign": _plain_assign, "compact": _plain_compact,
                "verify": _plain_verify}[c["op"]](s, c)
    if "plan" not in s:
        s["plan"] = _plan(s, c)
    for call in s["plan"]:
        call()
    if c["op"] == "attend":
        return s["out"], s["lse"]
    if c["op"] == "append":
        return s["k_new_back"], s["v_new_back"]
    if c["op"] == "verify":
        return {x: s[x] for x in ("accepted", "count", "token", "log_probs")}
    pools = {x: s[x] for x in ("k", "v", "k_scale", "v_scale")}
    if c["op"] == "assign":
        return {"table": s["table_out"], "refs": s["refs"], "room": s["room"], **pools}
    return {"table": s["table_out"], "refs": s["refs"], "n_live": s["n_live"], **pools}


# ------------------------------------------------------------------------------------------------------------- exact

def _exact_values(fmt, codes):
    """f64 values of codes, bit by bit as the formats define them."""
    b = codes.long()
    if fmt == "i8":
        return (b - 128).double()
    e, m = (b >> 3) & 15, (b & 7).double()
    x = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2((e - 10).double()))
    return torch.where(b >= 128, -x, x)


def _exact_rows(s, c, name, seq, n):
    """f64 [n, Hkv, 64]: positions 0 .. n - 1 of a sequence."""
    P, hkv = c["page"], c["hkv"]
    at = s["table"][seq, :-(-n // P)].long()
    codes = s[name][at].view(len(at), hkv, P // BLOCK, BLOCK * D)
    t, d = torch.arange(BLOCK, device="cuda")[:, None], torch.arange(D, device="cuda")[None]
    place = t * D + d if name == "k" else d // 32 * 512 + (d % 8 * 4 + t // 4) * 16 + d // 8 % 4 * 4 + t % 4
    x = _exact_values(c["format"], codes[..., place]) * s[name + "_scale"][at].double()[..., None, None]
    return x.permute(0, 2, 3, 1, 4).reshape(-1, hkv, D)[:n]


def _nearest(fmt, x):
    """f64 x to the format's nearest value."""
    if fmt == "i8":
        return torch.round(x).clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def exact(case, seed):
    s, c = prepare(case, seed), dict(case)
    if c["op"] in ("assign", "compact"):
        return _exact_pages(s, c)
    if c["op"] == "verify":
        return _exact_verify(s, c)
    S, hkv = c["seqs"], c["hkv"]
    if c["op"] == "attend":
        hq, n = c["hq"], c["rows"]
        out = torch.zeros((S, n, hq, D), dtype=torch.float64, device="cuda")
        lse = torch.full((S, n, hq), -math.inf, dtype=torch.float64, device="cuda")
        for i in range(S):
            L, m = int(s["kv_len"][i]), int(s["n"][i])
            k, v = _exact_rows(s, c, "k", i, L), _exact_rows(s, c, "v", i, L)
            hidden = torch.arange(L, device="cuda")[None] > torch.arange(L - m, L, device="cuda")[:, None]
            for h in range(hq):
                x = (s["q"][i, :m, h].double() @ k[:, h // (hq // hkv)].T) / 8.0
                x[hidden] = -math.inf
                lse[i, :m, h] = torch.logsumexp(x, 1)
                out[i, :m, h] = torch.softmax(x, 1) @ v[:, h // (hq // hkv)]
        return out, lse
    fmt, M = c["format"], MOST_CODE[c["format"]]
    if sum(-(-(int(b) + BLOCK) // BLOCK) for b in s["n"]) > 4000:
        return None
    back = []
    for name in ("k", "v"):
        got = torch.zeros(s[name + "_new_back"].shape, dtype=torch.float64, device="cuda")
        for i in range(S):
            L, n = int(s["kv_len"][i]), int(s["n"][i])
            before = _exact_rows(s, c, name, i, L)
            x = s[name + "_new"][i, :n].double().view(n, hkv, D)
            first = L // BLOCK * BLOCK
            for at in range(first, L + n, BLOCK):
                fresh = x[max(at - L, 0):at + BLOCK - L]
                old = before[at:L]
                scale = (fresh.abs().amax((0, 2)) / M).float().double()  # per head, as it is held
                if len(old):
                    page = int(s["table"][i, at // c["page"]])
                    stored = s[name + "_scale"][page, :, at % c["page"] // BLOCK].double()
                    scale = torch.maximum(scale, stored)
                rows = torch.cat((old, fresh)) / scale[:, None]
                if len(old):
                    rows = torch.where((scale == stored)[:, None] & (torch.arange(len(rows), device="cuda") < len(old))[:, None, None],
                                       rows, _nearest(fmt, rows))
                else:
                    rows = _nearest(fmt, rows)
                got[i, at - first:at - first + len(rows)] = (rows * scale[:, None]).reshape(len(rows), -1)
        back.append(got)
    return tuple(back)


def _exact_pages(s, c):
    """Page by page, as a host would keep its books."""
    P, pages = c["page"], s["refs"].shape[0]
    table = s["table"].cpu().numpy()
    moves = []
    if c["op"] == "assign":
        src, keep, need = (s[x].cpu().numpy() for x in ("src", "keep", "need"))
        lists = [list(table[src[i], :-(-keep[i] // P)]) for i in range(c["seqs"])]
        refs = np.bincount([p for x in lists for p in x], minlength=pages)
        room, free = keep.copy(), [p for p in range(pages) if refs[p] == 0]
        writes = [need[i] > keep[i] and keep[i] % P != 0 for i in range(c["seqs"])]
        by = {}
        for i in range(c["seqs"]):
            if writes[i]:
                by.setdefault(lists[i][-1], []).append(i)
        asked = taken = 0
        for i in range(c["seqs"]):
            copy = writes[i] and refs[lists[i][-1]] > 1 and not (len(by[lists[i][-1]]) == refs[lists[i][-1]] and by[lists[i][-1]][0] == i)
            more = max(0, -(-need[i] // P) - len(lists[i]))
            asked += more + copy
            if asked > len(free):
                continue
            if copy:
                moves.append((lists[i][-1], free[taken]))
                lists[i][-1] = free[taken]
            lists[i] += free[taken + copy:taken + copy + more]
            taken += copy + more
            room[i] = max(need[i], keep[i])
        new = np.full_like(table, -1)
        for i, x in enumerate(lists):
            new[i, :len(x)] = x
        said = {"room": room}
    else:
        live = sorted({int(p) for p in table.ravel() if p >= 0})
        free = sorted(set(range(len(live))) - set(live))
        moves = list(zip([p for p in live if p >= len(live)], free))
        to = dict(moves)
        new = np.vectorize(lambda p: to.get(int(p), int(p)), otypes=[np.int32])(table)
        said = {"n_live": np.array([len(live)], dtype=np.int32)}
    pools = {x: s[x].clone() for x in ("k", "v", "k_scale", "v_scale")}
    for a, b in moves:
        for x in pools:
            pools[x][:, b] = s[x][:, a]
    return {"table": new, "refs": np.bincount(new[new >= 0], minlength=pages).astype(np.int32), **said, **pools}


def _exact_verify(s, c):
    """Sequence by sequence, down the tree, in numpy."""
    S, n, V = s["logits"].shape
    tokens, u, last = s["tokens"].cpu().numpy(), s["accept_u"].double().cpu().numpy(), s["sample_u"].double().cpu().numpy()
    heat = s["heat"].double().cpu().numpy()
    parents = None if s["parents"] is None else s["parents"].cpu().numpy()
    paths, counts, ends = np.full((S, n), -1, np.int32), np.zeros(S, np.int32), np.zeros(S, np.int32)
    said = np.zeros((S, n))
    for i in range(S):
        at, path, tried = 0, [0], 0
        while True:
            x = s["logits"][i, at].double().cpu().numpy()
            if heat[i] > 0:
                w = np.exp((x - x.max()) / heat[i])
            else:
                w = np.zeros(V)
                w[int(np.argmax(x))] = 1.0
            p, q, logs = w / w.sum(), None, (x - x.max()) / (heat[i] or 1.0) - math.log(w.sum())
            down = None
            for child in range(tried + 1, n):
                if (child - 1 if parents is None else parents[i, child]) != at:
                    continue
                t = int(tokens[i, child])
                if s["probs"] is None:
                    takes, left = u[i, child] < p[t], p.copy()
                    left[t] = 0.0
                else:
                    q = s["probs"][i, at].double().cpu().numpy() if q is None else q
                    takes, left = u[i, child] * q[t] < p[t], np.maximum(p - q, 0.0)
                if takes:
                    down = child
                    break
                if left.sum() > 0:
                    p = left / left.sum()
            if down is None:
                break
            said[i, len(path) - 1] = logs[tokens[i, down]]
            at = tried = down
            path.append(down)
        sums = np.cumsum(p)
        paths[i, :len(path)], counts[i] = path, len(path)
        ends[i] = int(np.argmax(sums > last[i] * sums[-1]))
        said[i, len(path) - 1] = logs[ends[i]]
    return {"accepted": paths, "count": counts, "token": ends, "log_probs": said}
