"""GPU: attention for a tree of drafted tokens and the commit of accepted drafts.

The kernels keep cached quants exact and split the queries and weights into two
f16 parts (or compute in f32), so the bar is the decode's: rel-L2 1e-5 and
max-abs 2e-3 against attention in 64 bits over the dequantized rows.  A log-sum
is off by at most about the error of its largest scores: |q.k| scale <= 30 here
times 2^-20 of the split products and sums, 3e-5.
"""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

D = 64
REL_L2, MAX_ABS, LSE_ABS = 1e-5, 2e-3, 3e-5
ALL = ["f32", "f16", "q8_0", "q5_1", "q5_0", "q4_1", "q4_0"]


def rel_l2(a, b):
    return float(np.linalg.norm((a - b).ravel()) / max(np.linalg.norm(b.ravel()), 1e-30))


def ancestors(parents):
    S, n = parents.shape
    sees = np.zeros((S, n, n), dtype=bool)
    for s in range(S):
        for i in range(n):
            j = i
            while j >= 0:
                sees[s, i, j] = True
                j = parents[s, j]
    return sees


def random_parents(rng, S, n):
    return np.array([[-1 if i == 0 else int(rng.integers(-1, i)) for i in range(n)] for _ in range(S)]).reshape(S, n)


def pack(sees):
    S, n, _ = sees.shape
    w = (n + 31) // 32
    wide = np.zeros((S, n, w * 32), dtype=bool)
    wide[..., :n] = sees
    return np.packbits(wide, axis=-1, bitorder="little").view(np.int32).reshape(S, n, w)


class Rows:
    """Cache rows [n_seq, cap] of one type on the device, with optional padding between rows and a byte offset."""

    def __init__(self, cv, torch, oracle, t, x, heads, pad=0, offset=0):
        self.t, self.heads = t, heads
        S, cap, _ = x.shape
        raw = oracle.quantize(t, x)
        rb = raw.shape[-1]
        host = np.full((S, cap, rb + pad), 0xA5, dtype=np.uint8)
        host[..., :rb] = raw
        self.buf = torch.full((offset + host.size,), 0x5A, dtype=torch.uint8, device="cuda")
        self.buf[offset:] = torch.tensor(host.reshape(-1), device="cuda")
        self.desc = cv.kv_tensor(self.buf, t, heads, D, cap, S, nb1=rb + pad, byte_offset=offset)
        self.offset, self.shape, self.rb = offset, host.shape, rb
        self.f = oracle.dequantize(t, raw, heads * D).reshape(S, cap, heads, D).astype(np.float64)

    def raw(self):
        return self.buf[self.offset:].view(*self.shape).cpu().numpy()[..., :self.rb]


def reference(q, k, v, kd, vd, lens, counts, sees, scale):
    """64 bits; kd, vd None: no drafted rows."""
    S, n, Hq, _ = q.shape
    Hkv = k.shape[2]
    out, lse = np.zeros(q.shape), np.full((S, n, Hq), -np.inf)
    for s in range(S):
        L, m = lens[s], counts[s]
        keys = k[s, :L] if kd is None else np.concatenate([k[s, :L], kd[s, :m]])
        vals = v[s, :L] if kd is None else np.concatenate([v[s, :L], vd[s, :m]])
        for i in range(m):
            ok = np.ones(len(keys), dtype=bool)
            ok[L:] = sees[s, i, :m] if kd is not None else True
            if not ok.any():
                continue
            for h in range(Hq):
                g = h // (Hq // Hkv)
                x = keys[ok, g] @ q[s, i, h].astype(np.float64) * scale
                top = x.max()
                p = np.exp(x - top)
                lse[s, i, h] = top + np.log(p.sum())
                out[s, i, h] = p @ vals[ok, g] / p.sum()
    return out, lse


def run_case(ctx, cv, torch, oracle, kname, vname, Hq, Hkv, lens, n, counts=None, sees=None, seed=0, cap=None, pads=(0, 0, 0, 0),
             offsets=(0, 0, 0, 0), scale=0.125, q_extra=0, drafts=True, shared_mask=False, seq_ptrs=False, size=1.0, rows_at=None):
    rng = np.random.default_rng(seed)
    kt, vt = cv.TYPE_BY_NAME[kname], cv.TYPE_BY_NAME[vname]
    S = len(lens)
    cap = cap or max(max(lens), 1)
    mk = lambda t, m, i: Rows(cv, torch, oracle, t, (rng.standard_normal((S, m, Hkv * D)) * size).astype(np.float32), Hkv, pads[i], offsets[i])  # noqa: E731
    k, v, kd, vd = mk(kt, cap, 0), mk(vt, cap, 1), mk(kt, n, 2), mk(vt, n, 3)
    q = rng.standard_normal((S, n, Hq, D)).astype(np.float32)
    qbuf = torch.zeros((S, n + 1, Hq * D + q_extra), device="cuda")
    qt = qbuf[:, :n, :Hq * D].unflatten(-1, (Hq, D))
    qt.copy_(torch.tensor(q, device="cuda"))
    obuf = torch.full((S, n + 1, Hq * D + q_extra), 7.0, device="cuda")
    out = obuf[:, :n, :Hq * D].unflatten(-1, (Hq, D))
    lse = torch.full((S, n, Hq), 7.0, device="cuda")
    chain = np.tril(np.ones((n, n), dtype=bool))[None].repeat(S, 0)
    mask = None if sees is None else torch.tensor(pack(sees[:1] if shared_mask else sees), device="cuda")
    counts = counts or [n] * S
    kw = {}
    if seq_ptrs:
        rows = k.desc.nb2, v.desc.nb2
        order = rng.permutation(S)
        kw = {"k_seq_ptrs": torch.tensor([k.desc.data + int(i) * rows[0] for i in order], dtype=torch.int64, device="cuda"),
              "v_seq_ptrs": torch.tensor([v.desc.data + int(i) * rows[1] for i in order], dtype=torch.int64, device="cuda")}
        kf, vf = k.f[order], v.f[order]
    else:
        kf, vf = k.f, v.f
    cv.TreeDecoder(ctx, k.desc, v.desc, kd.desc if drafts else None, vd.desc if drafts else None, qt, out,
                   torch.tensor(lens, dtype=torch.int32, device="cuda"), max_kv_len=max(lens), lse=lse, mask=mask,
                   n_nodes=torch.tensor(counts, dtype=torch.int32, device="cuda"), scale=scale, **kw)()
    got, got_lse = out.cpu().numpy(), lse.cpu().numpy()
    want, want_lse = reference(q, kf, vf, kd.f if drafts else None, vd.f if drafts else None, lens, counts,
                               chain if sees is None else (sees[:1].repeat(S, 0) if shared_mask else sees), scale)
    assert rel_l2(got, want) <= REL_L2 and np.abs(got - want).max() <= MAX_ABS, rel_l2(got, want)
    empty = np.isneginf(want_lse)
    assert np.array_equal(empty, np.isneginf(got_lse))
    assert not got[empty].any()
    assert np.abs(got_lse[~empty] - want_lse[~empty]).max(initial=0.0) <= LSE_ABS
    assert bool((obuf[:, n:] == 7.0).all()) and bool((obuf[..., Hq * D:] == 7.0).all())  # nothing past the rows
    return got


@pytest.mark.parametrize("kname", ALL)
@pytest.mark.parametrize("vname", ALL)
def test_type_pairs(ctx, cv, cuda, oracle, kname, vname):
    rng = np.random.default_rng(5)
    sees = ancestors(random_parents(rng, 3, 11))
    run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, [1, 130, 257], 11, counts=[11, 5, 1], sees=sees)


@pytest.mark.parametrize("Hq,Hkv", [(14, 2), (2, 2), (16, 16), (3, 1), (8, 1), (12, 4), (15, 3)])
@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("f16", "f16"), ("q4_1", "f32")])
def test_head_layouts(ctx, cv, cuda, oracle, Hq, Hkv, kname, vname):
    run_case(ctx, cv, cuda, oracle, kname, vname, Hq, Hkv, [70, 3], 6)


@pytest.mark.parametrize("n", [1, 2, 3, 31, 32, 33, 63, 64, 65, 129, 256])
@pytest.mark.parametrize("kname,vname", [("q8_0", "q8_0"), ("f16", "q5_0"), ("f32", "f32")])
def test_tree_sizes(ctx, cv, cuda, oracle, n, kname, vname):
    rng = np.random.default_rng(n)
    sees = ancestors(random_parents(rng, 2, n))
    run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, [100, 63], n, counts=[n, max(1, n // 2)], sees=sees)


@pytest.mark.parametrize("L", [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 1000, 4097])
@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("f16", "f16"), ("q5_1", "q5_1"), ("f32", "q8_0")])
def test_cache_lengths(ctx, cv, cuda, oracle, L, kname, vname):
    run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, [L], 5)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q8_0"), ("f16", "f16"), ("f32", "f32")])
def test_long_context_is_split(ctx, cv, cuda, oracle, kname, vname):
    run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, [20011], 3, seed=3)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("f16", "f16"), ("f32", "f32")])
def test_many_ragged_sequences(ctx, cv, cuda, oracle, kname, vname):
    rng = np.random.default_rng(1)
    lens = rng.integers(0, 700, 64).tolist()
    counts = rng.integers(0, 9, 64).tolist()
    sees = ancestors(random_parents(rng, 64, 8))
    run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, lens, 8, counts=counts, sees=sees)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q5_1"), ("f16", "f16"), ("f32", "f32")])
def test_rows_that_see_nothing(ctx, cv, cuda, oracle, kname, vname):
    sees = np.zeros((2, 70, 70), dtype=bool)
    sees[0, 3, 69] = True   # one lone draft of the second tile, no committed key
    sees[0, 5, :] = True
    sees[1, ::2] = np.eye(70, dtype=bool)[::2]
    run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, [0, 0], 70, sees=sees)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("f16", "f16"), ("q5_0", "q4_1"), ("f32", "f32")])
def test_masks_beyond_ancestors_and_one_mask_for_all(ctx, cv, cuda, oracle, kname, vname):
    rng = np.random.default_rng(8)
    sees = rng.random((3, 40, 40)) < 0.3
    run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, [5, 64, 90], 40, sees=sees)
    run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, [5, 64, 90], 40, sees=sees, shared_mask=True)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("f16", "f16"), ("q5_1", "q5_0"), ("f32", "q4_1")])
@pytest.mark.parametrize("pads,offsets", [((2, 6, 10, 14), (2, 2, 2, 2)), ((16, 32, 48, 64), (0, 0, 0, 0)), ((4, 8, 12, 4), (4, 12, 8, 4))])
def test_strides_and_alignment(ctx, cv, cuda, oracle, kname, vname, pads, offsets):
    if "f32" in (kname, vname):  # an f32 row starts at a multiple of its elements
        pads, offsets = tuple(p // 4 * 4 for p in pads), tuple(o // 4 * 4 for o in offsets)
    run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, [130, 77], 9, pads=pads, offsets=offsets, q_extra=8)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q8_0"), ("f16", "f16"), ("f32", "f32")])
def test_sequences_by_address(ctx, cv, cuda, oracle, kname, vname):
    run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, [130, 77, 300, 5], 9, cap=300, seq_ptrs=True)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q8_0"), ("f16", "f16"), ("q4_1", "q5_1"), ("f32", "f32")])
def test_queries_over_the_cache_alone(ctx, cv, cuda, oracle, kname, vname):
    run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, [130, 0], 4, drafts=False)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q8_0"), ("f16", "f16"), ("q4_1", "q5_1"), ("f32", "f32")])
@pytest.mark.parametrize("size", [1e-3, 20.0])
def test_small_and_large_rows(ctx, cv, cuda, oracle, kname, vname, size):
    # sizes whose scores stay below 30: the scale takes up the large keys
    run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, [600], 7, size=size, scale=0.125 / max(1.0, size))


@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("f16", "f16"), ("q5_1", "q4_1"), ("f32", "f32")])
def test_a_draft_that_is_not_seen_may_hold_anything(ctx, cv, cuda, oracle, kname, vname):
    """Infinities and NaN in a drafted row reach only the rows that see it."""
    torch = cuda
    kt, vt = cv.TYPE_BY_NAME[kname], cv.TYPE_BY_NAME[vname]
    rng = np.random.default_rng(2)
    n, L, bad = 12, 40, 4
    k = Rows(cv, torch, oracle, kt, rng.standard_normal((1, L, 128)).astype(np.float32), 2)
    v = Rows(cv, torch, oracle, vt, rng.standard_normal((1, L, 128)).astype(np.float32), 2)
    kd = Rows(cv, torch, oracle, kt, rng.standard_normal((1, n, 128)).astype(np.float32), 2)
    vd = Rows(cv, torch, oracle, vt, rng.standard_normal((1, n, 128)).astype(np.float32), 2)
    sees = ancestors(np.array([[-1, 0, 0, 1, 1, 2, 4, 5, 6, 0, 9, 9]]))
    q = rng.standard_normal((1, n, 14, D)).astype(np.float32)
    want, _ = reference(q, k.f, v.f, kd.f, vd.f, [L], [n], sees, 0.125)
    nan16, inf16 = np.array([0x00, 0x7E], np.uint8), np.array([0x00, 0x7C], np.uint8)
    for rows, what in ((kd, nan16), (vd, inf16)):
        raw = rows.raw().copy()
        if rows.t == cv.F32:
            raw[0, bad] = np.full(128, np.nan if rows is kd else np.inf, np.float32).view(np.uint8)
        elif rows.t == cv.F16:
            raw[0, bad] = np.tile(what, 128)
        else:
            for b in range(4):
                raw[0, bad, b * rows.rb // 4:b * rows.rb // 4 + 2] = what
        rows.buf.copy_(torch.tensor(raw.reshape(-1), device="cuda"))
    out = cv.tree_decode(ctx, torch.tensor(q, device="cuda"), k.desc, v.desc, kd.desc, vd.desc,
                         torch.tensor([L], dtype=torch.int32, device="cuda"), L, mask=torch.tensor(pack(sees), device="cuda")).cpu().numpy()
    blind = ~sees[0, :, bad]
    assert np.isfinite(out[0, blind]).all()
    assert rel_l2(out[0, blind], want[0, blind]) <= REL_L2
    assert not np.isfinite(out[0, ~blind]).all(axis=(1, 2)).any()


def test_equals_decode_for_one_query_without_drafts(ctx, cv, cuda, oracle):
    torch = cuda
    rng = np.random.default_rng(4)
    lens = [1, 200, 513]
    k = Rows(cv, torch, oracle, cv.Q8_0, rng.standard_normal((3, 513, 128)).astype(np.float32), 2)
    v = Rows(cv, torch, oracle, cv.Q4_0, rng.standard_normal((3, 513, 128)).astype(np.float32), 2)
    q = torch.tensor(rng.standard_normal((3, 14, D)).astype(np.float32), device="cuda")
    kl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    a = cv.decode(ctx, q, k.desc, v.desc, kl, 513).cpu().numpy()
    b = cv.tree_decode(ctx, q[:, None].contiguous(), k.desc, v.desc, None, None, kl, 513)[:, 0].cpu().numpy()
    assert rel_l2(b, a) <= 2 * REL_L2


def test_results_do_not_depend_on_the_run_or_the_stream(ctx, cv, cuda, oracle):
    torch = cuda
    rng = np.random.default_rng(6)
    k = Rows(cv, torch, oracle, cv.Q8_0, rng.standard_normal((2, 3000, 128)).astype(np.float32), 2)
    kd = Rows(cv, torch, oracle, cv.Q8_0, rng.standard_normal((2, 9, 128)).astype(np.float32), 2)
    q = torch.tensor(rng.standard_normal((2, 9, 14, D)).astype(np.float32), device="cuda")
    kl = torch.tensor([3000, 1700], dtype=torch.int32, device="cuda")
    a = cv.tree_decode(ctx, q, k.desc, k.desc, kd.desc, kd.desc, kl, 3000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(q)
    plan = cv.TreeDecoder(ctx, k.desc, k.desc, kd.desc, kd.desc, q, out, kl, 3000)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        plan(side)
    side.synchronize()
    assert torch.equal(a, out)


def test_captured_in_a_graph_with_lengths_that_grow(ctx, cv, cuda, oracle):
    torch = cuda
    rng = np.random.default_rng(7)
    k = Rows(cv, torch, oracle, cv.Q8_0, rng.standard_normal((2, 800, 128)).astype(np.float32), 2)
    kd = Rows(cv, torch, oracle, cv.Q8_0, rng.standard_normal((2, 4, 128)).astype(np.float32), 2)
    q = torch.tensor(rng.standard_normal((2, 4, 14, D)).astype(np.float32), device="cuda")
    kl = torch.tensor([10, 20], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    plan = cv.TreeDecoder(ctx, k.desc, k.desc, kd.desc, kd.desc, q, out, kl, 800)
    plan()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan()
    for lens in ([10, 20], [500, 0], [800, 799]):
        kl.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        chain = np.tril(np.ones((4, 4), dtype=bool))[None].repeat(2, 0)
        want, _ = reference(q.cpu().numpy(), k.f, k.f, kd.f, kd.f, lens, [4, 4], chain, 0.125)
        assert rel_l2(out.cpu().numpy(), want) <= REL_L2


def test_bad_lengths_are_recorded_and_give_empty_rows(ctx, cv, cuda, oracle):
    torch = cuda
    rng = np.random.default_rng(9)
    k = Rows(cv, torch, oracle, cv.Q8_0, rng.standard_normal((3, 64, 128)).astype(np.float32), 2)
    q = torch.tensor(rng.standard_normal((3, 4, 14, D)).astype(np.float32), device="cuda")
    for lens, counts in (([10, 65, 20], [4, 4, 4]), ([10, -1, 20], [4, 4, 4]), ([10, 20, 20], [4, 5, 4]), ([10, 20, 20], [4, -3, 4])):
        out = torch.full_like(q, 3.0)
        lse = torch.full((3, 4, 14), 3.0, device="cuda")
        cv.tree_decode(ctx, q, k.desc, k.desc, k.desc, k.desc, torch.tensor(lens, dtype=torch.int32, device="cuda"), 64, out=out, lse=lse,
                       n_nodes=torch.tensor(counts, dtype=torch.int32, device="cuda"))
        st, detail = ctx.sync_status()
        assert (st, detail) == (6, 2)
        assert not bool(out[1].any()) and bool(torch.isneginf(lse[1]).all())
        assert bool(out[0].any()) and bool(out[2].any())


def test_refusals(ctx, cv, cuda):
    torch = cuda
    lib, ct = cv.lib, __import__("ctypes")
    buf, k = cv.alloc_kv(cv.Q8_0, 2, D, 640, 2)
    fbuf, f = cv.alloc_kv(cv.F32, 2, D, 640, 2)
    dbuf, d = cv.alloc_kv(cv.Q8_0, 2, D, 8, 2)
    q = torch.zeros((2, 8, 14, D), device="cuda")
    out = torch.zeros_like(q)
    kl = torch.zeros(2, dtype=torch.int32, device="cuda")
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")  # enough for every type
    plan = lambda: cv.TreeDecoder(ctx, k, k, d, d, q, out, kl, 640, workspace=ws)  # noqa: E731

    def status(**kw):
        p = plan().params
        for name, v in kw.items():
            obj = p
            *path, last = name.split("__")
            for part in path:
                obj = getattr(obj, part)
            setattr(obj, last, v)
        return lib.cvattn_tree_decode(ctx.handle, 0, ct.byref(p))

    assert status() == 0
    assert status(n_seq=0) == 0 and status(max_nodes=0) == 0
    assert lib.cvattn_tree_decode(None, 0, ct.byref(plan().params)) == 1
    assert lib.cvattn_tree_decode(ctx.handle, 0, None) == 1
    for bad in ({"q": None}, {"out": None}, {"kv_len": None}, {"n_seq": -1}, {"max_nodes": -1}, {"n_q_heads": 0}, {"flags": 1},
                {"q": q.data_ptr() + 4}, {"q_nb_node": 14 * D - 4}, {"out_nb_node": 14 * D + 2}, {"out_nb_seq": 0}, {"out_nb_seq": 64 * D},
                {"k__data": None}, {"k__nb1": 135}, {"k__ne2": 1}, {"k_draft__type": cv.Q4_0}, {"k_draft__data": None},
                {"k_draft__ne2": 1}, {"v__n_heads": 1}, {"mask": q.data_ptr(), "mask_nb_seq": 7}, {"mask": q.data_ptr(), "mask_nb_seq": -8},
                {"mask": q.data_ptr(), "k_draft__data": None, "v_draft__data": None}, {"workspace": None}, {"workspace_size": 15}):
        assert status(**bad) == 1, bad
    # an f32 cache starts at a multiple of four bytes
    assert status(k=f, k_draft__data=None, v_draft__data=None) == 0
    for name in ("data", "nb1", "nb2"):
        assert status(k=f, k_draft__data=None, v_draft__data=None, **{"k__" + name: getattr(f, name) + 2}) == 1
    for bad in ({"n_q_heads": 13}, {"n_q_heads": 18}, {"max_nodes": 257, "k_draft__ne1": 257, "v_draft__ne1": 257, "out_nb_seq": 1 << 20}):
        assert status(**bad) == 2, bad
    for bad in ({"max_kv_len": 641}, {"max_nodes": 9, "out_nb_seq": 1 << 20}):
        assert status(**bad) == 3, bad
    assert cv.tree_decode_workspace_size(cv.Q8_0, cv.Q8_0, 2, 64, 257, 14, 2) == 0
    assert cv.tree_decode_workspace_size(cv.Q8_0, cv.Q8_0, 2, 64, 8, 13, 2) == 0
    with pytest.raises(ValueError):
        cv.TreeDecoder(ctx, k, k, d, d, q.half(), out, kl, 640)
    with pytest.raises(ValueError):
        cv.TreeDecoder(ctx, k, k, d, d, q, out[:1], kl, 640)
    with pytest.raises(ValueError):
        cv.TreeDecoder(ctx, k, k, d, d, q, out, kl.long(), 640)
    with pytest.raises(ValueError):
        cv.TreeDecoder(ctx, k, k, d, d, q, out, kl, 640, mask=torch.zeros((2, 8, 2), dtype=torch.int32, device="cuda"))
    with pytest.raises(cv.CvattnError):
        cv.TreeDecoder(ctx, k, k, d, d, q, out, kl, 641)()


# ---------------------------------------------------------------------------------------------------------------- commit

@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("f16", "f32"), ("q5_1", "q5_0"), ("q4_1", "q8_0")])
@pytest.mark.parametrize("Hkv", [1, 2, 16])
@pytest.mark.parametrize("pad,offset", [(0, 0), (2, 2), (12, 4), (16, 16)])
def test_commit(ctx, cv, cuda, oracle, kname, vname, Hkv, pad, offset):
    torch = cuda
    if "f32" in (kname, vname):
        pad, offset = pad // 4 * 4, offset // 4 * 4
    rng = np.random.default_rng(Hkv)
    lens, counts, n, cap, layers = [0, 3, 17, 28], [4, 0, 6, 1], 9, 29, 2
    path = np.stack([rng.permutation(n)[:6] for _ in lens]).astype(np.int32)
    mk = lambda t, m, p, o: Rows(cv, torch, oracle, t, rng.standard_normal((4, m, Hkv * D)).astype(np.float32), Hkv, p, o)  # noqa: E731
    caches = [mk(cv.TYPE_BY_NAME[t], cap, pad, offset) for _ in range(layers) for t in (kname, vname)]
    drafts = [mk(cv.TYPE_BY_NAME[t], n, 0, 0) for _ in range(layers) for t in (kname, vname)]
    want = [c.raw().copy() for c in caches]
    for w, d in zip(want, drafts):
        raw = d.raw()
        for s, (L, m) in enumerate(zip(lens, counts)):
            w[s, L:L + m] = raw[s, path[s, :m]]
    kl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    nl = torch.zeros_like(kl)
    args = (ctx, [c.desc for c in caches], [d.desc for d in drafts], torch.tensor(path, device="cuda"),
            torch.tensor(counts, dtype=torch.int32, device="cuda"), kl)
    whole = [c.buf.clone() for c in caches]
    cv.tree_commit(*args, nl)
    for c, w, before in zip(caches, want, whole):
        assert np.array_equal(c.raw(), w)
        changed = (c.buf != before).sum().item()
        assert changed <= sum(counts) * c.rb  # padding and other rows as they were
    assert nl.tolist() == [a + b for a, b in zip(lens, counts)] and kl.tolist() == lens
    cv.tree_commit(*args)  # in place
    assert kl.tolist() == [a + b for a, b in zip(lens, counts)]


def test_commit_of_more_tensors_than_one_launch_takes(ctx, cv, cuda, oracle):
    torch = cuda
    rng = np.random.default_rng(1)
    mk = lambda m: Rows(cv, torch, oracle, cv.Q8_0, rng.standard_normal((1, m, 128)).astype(np.float32), 2)  # noqa: E731
    caches, drafts = [mk(8) for _ in range(101)], [mk(3) for _ in range(101)]
    kl = torch.tensor([5], dtype=torch.int32, device="cuda")
    cv.tree_commit(ctx, [c.desc for c in caches], [d.desc for d in drafts], torch.tensor([[2, 0]], dtype=torch.int32, device="cuda"),
                   torch.tensor([2], dtype=torch.int32, device="cuda"), kl)
    for c, d in zip(caches, drafts):
        assert np.array_equal(c.raw()[0, 5:7], d.raw()[0, [2, 0]])
    assert kl.tolist() == [7]


def test_commit_skips_what_does_not_fit(ctx, cv, cuda, oracle):
    torch = cuda
    rng = np.random.default_rng(1)
    mk = lambda m: Rows(cv, torch, oracle, cv.Q8_0, rng.standard_normal((5, m, 128)).astype(np.float32), 2)  # noqa: E731
    c, d = mk(8), mk(3)
    before = c.raw().copy()
    lens, counts = [7, -1, 2, 2, 2], [2, 1, 3, 1, 2]
    path = np.array([[0, 1], [0, 1], [0, 1], [3, 0], [1, 2]], dtype=np.int32)
    for out in (torch.zeros(5, dtype=torch.int32, device="cuda"), None):
        kl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        got = cv.tree_commit(ctx, [c.desc], [d.desc], torch.tensor(path, device="cuda"), torch.tensor(counts, dtype=torch.int32, device="cuda"),
                             kl, out)
        assert ctx.sync_status() == (6, 1)
        assert got.tolist() == [7, -1, 2, 2, 4]
        assert np.array_equal(c.raw()[:4], before[:4]) and np.array_equal(c.raw()[4, 2:4], d.raw()[4, 1:3])


def test_commit_refusals(ctx, cv, cuda):
    torch = cuda
    lib, ct = cv.lib, __import__("ctypes")
    buf, c = cv.alloc_kv(cv.Q8_0, 2, D, 16, 2)
    dbuf, d = cv.alloc_kv(cv.Q8_0, 2, D, 4, 2)
    ebuf, e = cv.alloc_kv(cv.Q4_0, 2, D, 4, 2)
    path = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    lens = torch.zeros((8,), dtype=torch.int32, device="cuda")
    count, kl, out = lens[:2], lens[2:4], lens[4:6]
    plan = lambda a=c, b=d: cv.TreeCommitter(ctx, [a], [b], path, count, kl, out).params  # noqa: E731

    def status(**kw):
        p = plan()
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.cvattn_tree_commit(ctx.handle, 0, ct.byref(p))

    assert status() == 0 and status(n_seq=0) == 0
    for bad in ({"n_seq": -1}, {"n_tensors": 0}, {"n_tensors": -1}, {"accepted": None}, {"n_accepted": None}, {"kv_len": None},
                {"kv_len_out": None}, {"max_accepted": -1}, {"accepted_stride": 3}, {"n_seq": 3}, {"kv_len_out": kl.data_ptr() + 4},
                {"kv_len_out": count.data_ptr()}):
        assert status(**bad) == 1, bad
    for a, b in ((c, e), (c, c), (e, d)):
        keep = cv.TreeCommitter(ctx, [a], [b], path, count, kl, out)
        assert lib.cvattn_tree_commit(ctx.handle, 0, ct.byref(keep.params)) == 1
    with pytest.raises(ValueError):
        cv.TreeCommitter(ctx, [c], [], path, count, kl, out)
    with pytest.raises(ValueError):
        cv.TreeCommitter(ctx, [c], [d], path.long(), count, kl, out)
