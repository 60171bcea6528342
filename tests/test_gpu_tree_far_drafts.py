"""GPU: drafted rows of any finite size beside ordinary ones.

A draft that a row does not see may hold anything, so the rows that do not see it
are held to the bars of test_gpu_tree.py: rel-L2 1e-5 against 64 bits, and 3e-5
for a log-sum.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_tree import D, LSE_ABS, REL_L2, Rows, ancestors, pack, random_parents, reference, rel_l2

pytestmark = pytest.mark.gpu

TYPES = ["q8_0", "q5_1", "q5_0", "q4_1", "q4_0", "f16"]


def with_far_rows(rows, torch, at, half):
    """The same rows with the scale of every block (every value of f16) of node at[s] replaced by the f16 of these bits."""
    raw = rows.raw().copy()
    step = 2 if rows.t == 1 else rows.rb // (2 * rows.heads)
    for s, j in enumerate(at):
        for b in range(0, rows.rb, step):
            raw[s, j, b:b + 2] = half
    rows.buf.copy_(torch.tensor(raw.reshape(-1), device="cuda"))


def run_far(ctx, cv, torch, oracle, kname, vname, lens, n, size, half, seed=0, broken=False, Hq=14, Hkv=2, sign=1.0):
    rng = np.random.default_rng(seed)
    S, cap = len(lens), max(max(lens), 1)
    kt, vt = cv.TYPE_BY_NAME[kname], cv.TYPE_BY_NAME[vname]
    mk = lambda t, m: Rows(cv, torch, oracle, t, (rng.standard_normal((S, m, Hkv * D)) * size).astype(np.float32), Hkv)  # noqa: E731
    k, v, kd, vd = mk(kt, cap), mk(vt, cap), mk(kt, n), mk(vt, n)
    sees = ancestors(random_parents(rng, S, n))
    q = rng.standard_normal((S, n, Hq, D)).astype(np.float32)
    scale = sign * 0.125 / size
    want, want_lse = reference(q, k.f, v.f, kd.f, vd.f, lens, [n] * S, sees, scale)
    at = [rng.integers(1, n, S), rng.integers(1, n, S)]
    with_far_rows(kd, torch, at[0], half)
    with_far_rows(vd, torch, at[1], half)
    if broken:  # and others that are not finite
        at += [rng.integers(1, n, S), rng.integers(1, n, S)]
        with_far_rows(kd, torch, at[2], [0x00, 0x7E])
        with_far_rows(vd, torch, at[3], [0x00, 0x7C])
    hit, blown = np.zeros((S, n), dtype=bool), np.zeros((S, n), dtype=bool)
    for s in range(S):
        for j in at:
            hit[s] |= sees[s, :, j[s]]
        for j in at[2:]:
            blown[s] |= sees[s, :, j[s]]
    lse = torch.empty((S, n, Hq), device="cuda")
    out = cv.tree_decode(ctx, torch.tensor(q, device="cuda"), k.desc, v.desc, kd.desc, vd.desc,
                         torch.tensor(lens, dtype=torch.int32, device="cuda"), cap, mask=torch.tensor(pack(sees), device="cuda"), lse=lse,
                         scale=scale).cpu().numpy()
    assert (~hit).sum() > S and hit.sum() >= S
    worst = max(rel_l2(out[s, i], want[s, i]) for s in range(S) for i in range(n) if not hit[s, i])
    assert worst <= REL_L2, worst
    assert np.abs(lse.cpu().numpy()[~hit] - want_lse[~hit]).max() <= LSE_ABS
    assert not np.isfinite(out[blown]).all(axis=(1, 2)).any()


LARGE, SMALL = [0xFF, 0x7B], [0x01, 0x00]  # 65504 and the least f16 above 0


@pytest.mark.parametrize("kname", TYPES)
@pytest.mark.parametrize("vname", TYPES)
@pytest.mark.parametrize("half", [LARGE, SMALL], ids=["large", "small"])
def test_far_drafts_little_work(ctx, cv, cuda, oracle, kname, vname, half):
    run_far(ctx, cv, cuda, oracle, kname, vname, [60, 0], 11, 1.0, half)


@pytest.mark.parametrize("size", [0.05, 30.0])
@pytest.mark.parametrize("kname,vname", [("q8_0", "q8_0"), ("q4_1", "q5_0"), ("q5_1", "f16")])
@pytest.mark.parametrize("lens,n", [([60, 0], 11), ([0, 130, 400], 60), ([200] * 40, 20), ([5], 200)])
def test_far_drafts_of_other_sizes(ctx, cv, cuda, oracle, kname, vname, lens, n, size):
    run_far(ctx, cv, cuda, oracle, kname, vname, lens, n, size, LARGE)


@pytest.mark.parametrize("kname", TYPES)
@pytest.mark.parametrize("vname", TYPES)
@pytest.mark.parametrize("half", [LARGE, SMALL], ids=["large", "small"])
def test_far_drafts_on_the_persistent_kernel(ctx, cv, cuda, oracle, kname, vname, half):
    """More than 128 rows of a KV head; the second sequence has drafts alone, in two tiles."""
    run_far(ctx, cv, cuda, oracle, kname, vname, [60, 0], 140, 1.0, half)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("q5_1", "q8_0"), ("f16", "q5_0")])
@pytest.mark.parametrize("Hq,Hkv,n", [(16, 16, 140), (3, 1, 70), (16, 2, 30), (6, 2, 5)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_far_drafts_head_layouts(ctx, cv, cuda, oracle, kname, vname, Hq, Hkv, n, sign):
    run_far(ctx, cv, cuda, oracle, kname, vname, [130, 0], n, 1.0, LARGE, seed=n, Hq=Hq, Hkv=Hkv, sign=sign)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("q4_1", "f16")])
def test_far_drafts_after_long_contexts(ctx, cv, cuda, oracle, kname, vname):
    """Parts of a sequence on many CTAs, the drafts on one of them."""
    run_far(ctx, cv, cuda, oracle, kname, vname, [9001, 300, 128], 20, 1.0, LARGE)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("q5_1", "q5_0"), ("f16", "q8_0"), ("q4_1", "f16"), ("f16", "f16")])
@pytest.mark.parametrize("lens,n", [([60, 0], 30), ([300] * 20, 12), ([0, 90], 200)])
def test_far_drafts_beside_ones_that_are_not_finite(ctx, cv, cuda, oracle, kname, vname, lens, n):
    run_far(ctx, cv, cuda, oracle, kname, vname, lens, n, 1.0, LARGE, seed=7, broken=True)


@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("q5_0", "q5_1"), ("f16", "q8_0"), ("q4_0", "f16")])
def test_rows_that_see_a_far_draft(ctx, cv, cuda, oracle, kname, vname):
    """A far value alone: rows that see it are right relative to their own size, on either kernel."""
    torch = cuda
    for lens, n in (([60, 3], 11), ([200] * 40, 20), ([5, 90], 140)):
        rng = np.random.default_rng(n)
        S, cap = len(lens), max(lens)
        kt, vt = cv.TYPE_BY_NAME[kname], cv.TYPE_BY_NAME[vname]
        mk = lambda t, m: Rows(cv, torch, oracle, t, rng.standard_normal((S, m, 128)).astype(np.float32), 2)  # noqa: E731
        k, v, kd, vd = mk(kt, cap), mk(vt, cap), mk(kt, n), mk(vt, n)
        with_far_rows(vd, torch, rng.integers(0, n, S), LARGE)
        raw = vd.raw()
        vd.f = oracle.dequantize(vt, np.ascontiguousarray(raw), 128).reshape(S, n, 2, D).astype(np.float64)
        sees = ancestors(random_parents(rng, S, n))
        q = rng.standard_normal((S, n, 14, D)).astype(np.float32)
        want, _ = reference(q, k.f, v.f, kd.f, vd.f, lens, [n] * S, sees, 0.125)
        out = cv.tree_decode(ctx, torch.tensor(q, device="cuda"), k.desc, v.desc, kd.desc, vd.desc,
                             torch.tensor(lens, dtype=torch.int32, device="cuda"), cap, mask=torch.tensor(pack(sees), device="cuda")).cpu().numpy()
        worst = max(rel_l2(out[s, i], want[s, i]) for s in range(S) for i in range(n))
        assert worst <= REL_L2, worst
