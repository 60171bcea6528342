"""GPU: tree attention, scores, commit and eviction where work is cut across the device: long lists of key tiles that CTAs
share, row counts around the limits of each kernel, more sequences than a table holds, rows past 32-bit offsets.

The bars are those of test_gpu_tree.py and test_gpu_bounded_cache.py.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_bounded_cache import run_scores, scores_reference, true_lse
from test_gpu_bounded_cache import REL_L2 as SCORES_REL_L2
from test_gpu_tree import D, LSE_ABS, MAX_ABS, REL_L2, ancestors, random_parents, reference, rel_l2, run_case

pytestmark = pytest.mark.gpu

TYPES = ["f16", "q8_0", "q5_1", "q5_0", "q4_1", "q4_0"]


def ragged(seed, S, most):
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, most, S)
    lens[rng.integers(0, S, 3)] = 0
    lens[1], lens[2] = most, 128
    return rng, lens.tolist()


@pytest.mark.parametrize("kname", TYPES)
@pytest.mark.parametrize("shift", range(3))
def test_tree_list_of_tiles_is_shared(ctx, cv, cuda, oracle, kname, shift):
    """More tiles than SMs, whole units next to parts; 63 rows: half a tile of rows is padding."""
    vname = TYPES[(TYPES.index(kname) + 2 * shift) % 6]
    rng, lens = ragged(shift, 24, 1300)
    counts = rng.integers(0, 10, 24).tolist()
    run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, lens, 9, counts=counts, sees=ancestors(random_parents(rng, 24, 9)), seed=shift)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("f16", "q8_0"), ("q5_1", "f16")])
def test_tree_drafts_after_long_contexts(ctx, cv, cuda, oracle, kname, vname):
    """K tiles run ahead of V tiles; whether a draft's values are finite must not be asked before its V tile is there."""
    lens = np.random.default_rng(5).integers(128, 2049, 64).tolist()
    for _ in range(2):
        run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, lens, 8)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q8_0"), ("f16", "f16"), ("q4_1", "f16"), ("f16", "q5_1")])
@pytest.mark.parametrize("pads,offsets", [((2, 6, 10, 14), (2, 2, 2, 2)), ((4, 8, 12, 4), (4, 12, 8, 4))])
def test_tree_shared_list_strides_and_addresses(ctx, cv, cuda, oracle, kname, vname, pads, offsets):
    _, lens = ragged(7, 20, 1100)
    run_case(ctx, cv, cuda, oracle, kname, vname, 14, 2, lens, 12, pads=pads, offsets=offsets, seq_ptrs=True, q_extra=12)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("f16", "f16")])
@pytest.mark.parametrize("G,n", [(8, 4), (1, 32), (1, 33), (8, 16), (8, 17), (1, 128), (1, 129), (4, 256)])
def test_tree_rows_around_the_tiles(ctx, cv, cuda, oracle, kname, vname, G, n):
    run_case(ctx, cv, cuda, oracle, kname, vname, 2 * G, 2, [300, 1, 129], n, counts=[n, 1, max(n - 1, 0)])


@pytest.mark.parametrize("kname", ["q8_0", "f16", "q5_1", "f32"])
@pytest.mark.parametrize("n", [2, 9, 20])
def test_tree_negative_scale(ctx, cv, cuda, oracle, kname, n):
    run_case(ctx, cv, cuda, oracle, kname, kname, 14, 2, [400, 20], n, scale=-0.125)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("f16", "f16")])
def test_tree_more_sequences_than_the_table_holds(ctx, cv, cuda, oracle, kname, vname):
    rng = np.random.default_rng(0)
    lens = rng.integers(0, 40, 1030).tolist()
    run_case(ctx, cv, cuda, oracle, kname, vname, 6, 1, lens, 6, counts=rng.integers(0, 7, 1030).tolist())


@pytest.mark.parametrize("kname", TYPES)
@pytest.mark.parametrize("Hq,Hkv,n", [(14, 2, 1), (16, 16, 5), (16, 16, 20), (14, 2, 20)])
def test_scores_list_of_tiles_is_shared(ctx, cv, cuda, oracle, kname, Hq, Hkv, n):
    rng, lens = ragged(n, 20, 1000 if Hkv == 16 else 2000)
    counts = [int(rng.integers(0, min(L, n) + 1)) for L in lens]
    run_scores(ctx, cv, cuda, oracle, kname, Hq, Hkv, lens, n, counts=counts, picked=n == 5, in_place=n == 1)


@pytest.mark.parametrize("kname", ["q8_0", "f16", "q4_1"])
@pytest.mark.parametrize("n", [63, 64, 65])
def test_scores_rows_around_the_limit(ctx, cv, cuda, oracle, kname, n):
    """8 rows a node: 512 rows fit the tensor cores' kernel, 520 take the other."""
    run_scores(ctx, cv, cuda, oracle, kname, 16, 2, [4000] * 8 + [1, 64, 3900], n)


@pytest.mark.parametrize("kname", ["q8_0", "f16", "q5_0"])
@pytest.mark.parametrize("pad,offset", [(2, 2), (12, 4)])
def test_scores_shared_list_strides_and_addresses(ctx, cv, cuda, oracle, kname, pad, offset):
    _, lens = ragged(5, 24, 2000)
    run_scores(ctx, cv, cuda, oracle, kname, 14, 2, lens, 8, pad=pad, offset=offset, seq_ptrs=True, extra=7)


@pytest.mark.parametrize("kname", ["q8_0", "f16", "q4_1"])
@pytest.mark.parametrize("size", [1e-3, 20.0])
def test_scores_shared_list_small_and_large_rows(ctx, cv, cuda, oracle, kname, size):
    run_scores(ctx, cv, cuda, oracle, kname, 14, 2, [1700] * 24, 8, size=size)


@pytest.mark.parametrize("kname", ["q8_0", "f16"])
def test_scores_more_sequences_than_the_table_holds(ctx, cv, cuda, oracle, kname):
    lens = np.random.default_rng(0).integers(0, 40, 1030).tolist()
    run_scores(ctx, cv, cuda, oracle, kname, 2, 1, lens, 2)


@pytest.mark.parametrize("lens", [[300] * 2, [2000] * 24], ids=["few", "many"])
@pytest.mark.parametrize("kname", ["q8_0", "f16", "q5_1"])
def test_scores_negative_scale_and_rows_without_keys(ctx, cv, cuda, oracle, lens, kname):
    torch = cuda
    from test_gpu_tree import Rows

    rng = np.random.default_rng(2)
    S, n = len(lens), 7
    k = Rows(cv, torch, oracle, cv.TYPE_BY_NAME[kname], rng.standard_normal((S, max(lens), 128)).astype(np.float32), 2)
    q = rng.standard_normal((S, n, 14, D)).astype(np.float32)
    lse = true_lse(q, k.f, lens, [n] * S, scale=-0.125)
    lse[:, 1, ::3] = -np.inf  # these rows saw nothing: no weight
    old = torch.rand((S, 2, max(lens)), device="cuda")
    want = scores_reference(q, lse, k.f, lens, [n] * S, old.cpu().numpy(), 0.5, scale=-0.125)
    out = torch.empty_like(old)
    cv.kv_scores(ctx, k.desc, torch.tensor(q, device="cuda"), torch.tensor(lse, device="cuda"),
                 torch.tensor(lens, dtype=torch.int32, device="cuda"), old, out, max_kv_len=max(lens), decay=0.5, scale=-0.125)
    assert rel_l2(out.cpu().numpy(), want) <= SCORES_REL_L2


class FarRows:
    """One sequence whose rows lie 2^20 bytes apart: its last ones are past 2^32 bytes (only the rows are ever touched)."""

    def __init__(self, cv, torch, oracle, t, x, heads):
        L = x.shape[0]
        raw = oracle.quantize(t, x[None])[0]
        self.nb1, self.rb = 1 << 20, raw.shape[-1]
        self.buf = torch.empty((L, self.nb1), dtype=torch.uint8, device="cuda")
        self.buf[:, :self.rb] = torch.tensor(raw, device="cuda")
        self.desc = cv.kv_tensor(self.buf, t, heads, D, L, 1, nb1=self.nb1)
        self.f = oracle.dequantize(t, raw[None], heads * D).reshape(1, L, heads, D).astype(np.float64)

    def raw(self):
        return self.buf[:, :self.rb].cpu().numpy()


@pytest.mark.parametrize("kname,n", [("q8_0", 1), ("q8_0", 8), ("f16", 8), ("f32", 1)])
def test_rows_past_32_bit_offsets(ctx, cv, cuda, oracle, kname, n):
    """5000 rows of a cache whose row stride is 2^20: attention, weights, eviction and a commit reach bytes past 2^32."""
    torch = cuda
    rng = np.random.default_rng(4)
    L, cap, t = 4990, 5000, cv.TYPE_BY_NAME[kname]
    k, v = (FarRows(cv, torch, oracle, t, rng.standard_normal((cap, 128)).astype(np.float32), 2) for _ in range(2))
    from test_gpu_tree import Rows

    kd, vd = (Rows(cv, torch, oracle, t, rng.standard_normal((1, n, 128)).astype(np.float32), 2) for _ in range(2))
    q = rng.standard_normal((1, n, 14, D)).astype(np.float32)
    qt = torch.tensor(q, device="cuda")
    out, lse = torch.empty_like(qt), torch.empty((1, n, 14), device="cuda")
    kl = torch.tensor([L], dtype=torch.int32, device="cuda")
    cv.TreeDecoder(ctx, k.desc, v.desc, kd.desc, vd.desc, qt, out, kl, max_kv_len=cap, lse=lse)()
    want, want_lse = reference(q, k.f, v.f, kd.f, vd.f, [L], [n], np.tril(np.ones((1, n, n), dtype=bool)), 0.125)
    got = out.cpu().numpy()
    assert rel_l2(got, want) <= REL_L2 and np.abs(got - want).max() <= MAX_ABS
    assert np.abs(lse.cpu().numpy() - want_lse).max() <= LSE_ABS

    path = torch.arange(n, dtype=torch.int32, device="cuda")[None].contiguous()
    cv.tree_commit(ctx, [k.desc, v.desc], [kd.desc, vd.desc], path, torch.tensor([n], dtype=torch.int32, device="cuda"), kl)
    assert kl.tolist() == [L + n]
    for c, d in ((k, kd), (v, vd)):
        assert np.array_equal(c.raw()[L:L + n], d.raw()[0])
        c.f[0, L:L + n] = d.f[0]

    lens = [L + n]
    weights = true_lse(q, k.f, lens, [n])
    scores = torch.zeros((1, 2, cap), device="cuda")
    want_scores = scores_reference(q, weights, k.f, lens, [n], scores.cpu().numpy(), 1.0)
    cv.kv_scores(ctx, k.desc, qt, torch.tensor(weights, device="cuda"), kl, scores, scores, max_kv_len=cap, decay=1.0)
    assert rel_l2(scores.cpu().numpy(), want_scores) <= SCORES_REL_L2

    budget = 4500  # the rows from there on move down into holes
    scores = torch.arange(cap, device="cuda", dtype=torch.float32).repeat(1, 1, 2, 1).contiguous()
    pos = torch.zeros((1, 1, 2, cap), dtype=torch.int32, device="cuda")
    before = k.raw(), v.raw()
    cv.kv_evict(ctx, [k.desc], [v.desc], scores, pos, kl, None, kl.clone(), budget, max_kv_len=cap)
    first = L + n - budget  # the lowest scores go
    for c, b in zip((k, v), before):
        a = c.raw()
        assert np.array_equal(a[first:budget], b[first:budget])
        assert np.array_equal(a[:first], b[budget:L + n])
    assert kl.tolist() == [budget]


@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("f16", "f16"), ("q5_1", "q4_1"), ("f16", "q5_0")])
def test_tree_shared_list_with_drafts_that_are_not_finite(ctx, cv, cuda, oracle, kname, vname):
    """NaN in a drafted key and infinity in a drafted value, other ones in each sequence, reach only the rows that see them."""
    torch = cuda
    from test_gpu_tree import Rows, pack

    rng = np.random.default_rng(2)
    S, n, L = 40, 12, 600
    kt, vt = cv.TYPE_BY_NAME[kname], cv.TYPE_BY_NAME[vname]
    mk = lambda t, m: Rows(cv, torch, oracle, t, rng.standard_normal((S, m, 128)).astype(np.float32), 2)  # noqa: E731
    k, v, kd, vd = mk(kt, L), mk(vt, L), mk(kt, n), mk(vt, n)
    sees = ancestors(random_parents(rng, S, n))
    q = rng.standard_normal((S, n, 14, D)).astype(np.float32)
    lens = rng.integers(0, L + 1, S).tolist()
    want, _ = reference(q, k.f, v.f, kd.f, vd.f, lens, [n] * S, sees, 0.125)
    bad = {id(kd): rng.integers(0, n, S), id(vd): rng.integers(0, n, S)}
    hit = np.zeros((S, n), dtype=bool)
    for rows, half in ((kd, [0x00, 0x7E]), (vd, [0x00, 0x7C])):
        raw = rows.raw().copy()
        for s, at in enumerate(bad[id(rows)]):
            if s % 4 == 0:
                continue  # a sequence without any
            step = 2 if rows.t == cv.F16 else rows.rb // 4
            for b in range(0, rows.rb, step):
                raw[s, at, b:b + 2] = half
            hit[s] |= sees[s, :, at]
        rows.buf.copy_(torch.tensor(raw.reshape(-1), device="cuda"))
    out = cv.tree_decode(ctx, torch.tensor(q, device="cuda"), k.desc, v.desc, kd.desc, vd.desc,
                         torch.tensor(lens, dtype=torch.int32, device="cuda"), L, mask=torch.tensor(pack(sees), device="cuda")).cpu().numpy()
    assert np.isfinite(out[~hit]).all()
    assert rel_l2(out[~hit], want[~hit]) <= REL_L2
    assert not np.isfinite(out[hit]).all(axis=(1, 2)).any()
