"""GPU: attention weight per cached position, eviction by it, and the loop that uses both with drafted tokens.

Scores: sums of exp(score - lse) over rows, each term relative to 2^-20 of the
scores (see test_gpu_tree.py), so rel-L2 1e-5 against 64 bits; a sum of n weights
in f32 adds n 2^-24 at most.  Eviction is exact: whole numbers and moved bytes.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_tree import ALL, D, Rows, ancestors, pack, rel_l2

pytestmark = pytest.mark.gpu

REL_L2 = 1e-5


def scores_reference(q, lse, kf, lens, counts, old, decay, rows=None, scale=0.125):
    S, Hkv, cap = old.shape
    Hq = q.shape[2]
    G = Hq // Hkv
    want = old.astype(np.float64).copy()
    for s in range(S):
        L, m = lens[s], counts[s]
        want[s, :, :L] *= decay
        for i in range(m):
            at = i if rows is None else rows[s, i]
            far = L - m + i + 1
            for h in range(Hq):
                if np.isneginf(lse[s, at, h]):
                    continue
                x = kf[s, :far, h // G] @ q[s, at, h].astype(np.float64) * scale
                want[s, h // G, :far] += np.exp(x - float(lse[s, at, h]))
    return want


def true_lse(q, kf, lens, counts, rows=None, scale=0.125):
    S, n, Hq, _ = q.shape
    G = Hq // kf.shape[2]
    lse = np.zeros((S, n, Hq), dtype=np.float32)
    for s in range(S):
        for i in range(counts[s]):
            at = i if rows is None else rows[s, i]
            far = lens[s] - counts[s] + i + 1
            for h in range(Hq):
                x = kf[s, :far, h // G] @ q[s, at, h].astype(np.float64) * scale
                lse[s, at, h] = np.log(np.exp(x - x.max()).sum()) + x.max()
    return lse


def run_scores(ctx, cv, torch, oracle, kname, Hq, Hkv, lens, n, counts=None, picked=False, decay=0.9, pad=0, offset=0, seed=0,
               in_place=False, extra=0, seq_ptrs=False, size=1.0):
    rng = np.random.default_rng(seed)
    S, cap = len(lens), max(max(lens), 1)
    counts = counts or [min(n, L) for L in lens]
    k = Rows(cv, torch, oracle, cv.TYPE_BY_NAME[kname], (rng.standard_normal((S, cap, Hkv * D)) * size).astype(np.float32), Hkv, pad, offset)
    pool = 2 * n + 1 if picked else n
    q = rng.standard_normal((S, pool, Hq, D)).astype(np.float32)
    rows = np.stack([rng.permutation(pool)[:n] for _ in range(S)]).astype(np.int32) if picked else None
    kw, kf = {}, k.f
    if seq_ptrs:
        order = rng.permutation(S)
        kw["k_seq_ptrs"] = torch.tensor([k.desc.data + int(i) * k.desc.nb2 for i in order], dtype=torch.int64, device="cuda")
        kf = k.f[order]
    scale = 0.125 / max(1.0, size)
    lse = true_lse(q, kf, lens, counts, rows, scale)
    buf = torch.rand((S, Hkv, cap + 3 + extra), device="cuda")
    scores = buf[..., 3:3 + cap]
    old = scores.cpu().numpy()
    want = scores_reference(q, lse, kf, lens, counts, old, decay, rows, scale)
    out = scores if in_place else buf.clone()[..., 3:3 + cap]
    cv.kv_scores(ctx, k.desc, torch.tensor(q, device="cuda"), torch.tensor(lse, device="cuda"),
                 torch.tensor(lens, dtype=torch.int32, device="cuda"), scores, out, max_kv_len=max(lens), decay=decay,
                 rows=None if rows is None else torch.tensor(rows, device="cuda"),
                 n_rows=torch.tensor(counts, dtype=torch.int32, device="cuda"), scale=scale, **kw)
    got = out.cpu().numpy()
    for s, L in enumerate(lens):
        assert np.array_equal(got[s, :, L:], old[s, :, L:])  # not written
    gain = np.concatenate([(got[s, :, :L] - decay * old[s, :, :L]).ravel() for s, L in enumerate(lens)])
    assert rel_l2(got, want) <= REL_L2
    # each row's weights add up to one over the keys that it sees
    assert abs(gain.sum() - sum(counts) * Hq) <= 1e-5 * (sum(counts) * Hq + np.abs(old).sum())
    return got


@pytest.mark.parametrize("kname", ALL)
@pytest.mark.parametrize("picked", [False, True])
def test_scores_types(ctx, cv, cuda, oracle, kname, picked):
    run_scores(ctx, cv, cuda, oracle, kname, 14, 2, [1, 130, 257], 5, picked=picked)


@pytest.mark.parametrize("kname", ["q8_0", "f16", "q4_1", "f32"])
@pytest.mark.parametrize("L", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 4097])
def test_scores_lengths(ctx, cv, cuda, oracle, kname, L):
    run_scores(ctx, cv, cuda, oracle, kname, 14, 2, [L], 3)


@pytest.mark.parametrize("kname", ["q8_0", "f16", "q5_0", "f32"])
@pytest.mark.parametrize("n", [1, 2, 3, 9, 16, 17, 64, 129])
def test_scores_rows(ctx, cv, cuda, oracle, kname, n):
    run_scores(ctx, cv, cuda, oracle, kname, 14, 2, [200, 150], n, seed=n)


@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (16, 16), (3, 1), (8, 1), (12, 4), (15, 3)])
@pytest.mark.parametrize("kname", ["q8_0", "f16", "f32"])
def test_scores_head_layouts(ctx, cv, cuda, oracle, Hq, Hkv, kname):
    run_scores(ctx, cv, cuda, oracle, kname, Hq, Hkv, [70, 5], 4)


@pytest.mark.parametrize("kname", ["q8_0", "f16", "q5_1", "f32"])
def test_scores_ragged_in_place_and_by_address(ctx, cv, cuda, oracle, kname):
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 500, 40).tolist()
    counts = [int(rng.integers(0, min(L, 6) + 1)) for L in lens]
    run_scores(ctx, cv, cuda, oracle, kname, 14, 2, lens, 6, counts=counts, in_place=True, extra=5, seq_ptrs=True, picked=True)


@pytest.mark.parametrize("kname", ["q8_0", "f16", "q4_0", "f32"])
@pytest.mark.parametrize("pad,offset", [(2, 2), (12, 4), (16, 16)])
def test_scores_strides(ctx, cv, cuda, oracle, kname, pad, offset):
    if kname == "f32":
        pad, offset = pad // 4 * 4, offset // 4 * 4
    run_scores(ctx, cv, cuda, oracle, kname, 14, 2, [130, 77], 4, pad=pad, offset=offset)


@pytest.mark.parametrize("kname", ["q8_0", "f16", "q4_1", "f32"])
@pytest.mark.parametrize("size", [1e-3, 20.0])
def test_scores_small_and_large_rows(ctx, cv, cuda, oracle, kname, size):
    run_scores(ctx, cv, cuda, oracle, kname, 14, 2, [300], 4, size=size)


def test_scores_follow_the_attention_that_gave_the_log_sums(ctx, cv, cuda, oracle):
    """Empty rows (lse -inf) add nothing; bad lengths and rows are recorded and left out."""
    torch = cuda
    rng = np.random.default_rng(3)
    k = Rows(cv, torch, oracle, cv.Q8_0, rng.standard_normal((4, 90, 128)).astype(np.float32), 2)
    q = rng.standard_normal((4, 6, 14, D)).astype(np.float32)
    lens, counts = [90, 91, 50, 3], [4, 4, 7, 4]
    rows = np.array([[0, 6, 2, 5], [0, 1, 2, 3], [0, 1, 2, 3], [0, 1, 2, 3]], dtype=np.int32)
    lse = np.full((4, 6, 14), 3.0, dtype=np.float32)
    lse[0, 2] = -np.inf
    old = rng.random((4, 2, 90)).astype(np.float32)
    for bad, want_code in (((0,), 1), ((1, 2, 3), 2)):
        out = torch.tensor(old, device="cuda")
        ln, cn, rw = list(lens), list(counts), rows.copy()
        if bad == (0,):
            ln[1], cn[2], cn[3] = 80, 4, 3
        else:
            rw[0, 1] = 1
        cv.kv_scores(ctx, k.desc, torch.tensor(q, device="cuda"), torch.tensor(lse, device="cuda"), torch.tensor(ln, dtype=torch.int32, device="cuda"),
                     out, rows=torch.tensor(rw, device="cuda"), n_rows=torch.tensor(cn, dtype=torch.int32, device="cuda"), max_kv_len=90)
        assert ctx.sync_status() == (6, want_code)
        got = out.cpu().numpy()
        if bad == (0,):
            l2 = lse.copy()
            fixed = np.where(rw > 5, 2, rw)  # row 2 adds nothing: what a left-out row does
            want = scores_reference(q, l2, k.f, ln, cn, old, 1.0, fixed)
            assert rel_l2(got, want) <= REL_L2
        else:
            assert np.array_equal(got[1:], old[1:])


def test_scores_repeat_bit_for_bit(ctx, cv, cuda, oracle):
    a = run_scores(ctx, cv, cuda, oracle, "q8_0", 14, 2, [700], 20, seed=5)
    del a
    torch = cuda
    rng = np.random.default_rng(5)
    k = Rows(cv, torch, oracle, cv.Q8_0, rng.standard_normal((2, 900, 128)).astype(np.float32), 2)
    q = torch.tensor(rng.standard_normal((2, 20, 14, D)).astype(np.float32), device="cuda")
    lse = torch.full((2, 20, 14), 5.0, device="cuda")
    kl = torch.tensor([900, 333], dtype=torch.int32, device="cuda")
    outs = []
    for _ in range(3):
        sc = torch.zeros((2, 2, 900), device="cuda")
        outs.append(cv.kv_scores(ctx, k.desc, q, lse, kl, sc))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_scores_refusals(ctx, cv, cuda):
    torch = cuda
    lib, ct = cv.lib, __import__("ctypes")
    buf, k = cv.alloc_kv(cv.Q8_0, 2, D, 64, 2)
    q = torch.zeros((2, 8, 14, D), device="cuda")
    lse = torch.zeros((2, 8, 14), device="cuda")
    kl = torch.zeros(2, dtype=torch.int32, device="cuda")
    sc = torch.zeros((2, 2, 64), device="cuda")
    n0 = torch.zeros(2, dtype=torch.int32, device="cuda")
    plan = cv.KVScorer(ctx, k, q, lse, kl, sc, n_rows=n0)

    def status(**kw):
        p = cv.KVScoresParams.from_buffer_copy(plan.params)
        for name, v in kw.items():
            obj = p
            *path, last = name.split("__")
            for part in path:
                obj = getattr(obj, part)
            setattr(obj, last, v)
        return lib.cvattn_kv_scores(ctx.handle, 0, ct.byref(p))

    assert status() == 0 and status(n_seq=0) == 0 and status(max_kv_len=0) == 0
    for bad in ({"q": None}, {"lse": None}, {"kv_len": None}, {"scores": None}, {"scores_out": None}, {"n_seq": -1}, {"max_rows": -1},
                {"max_rows": 9}, {"n_q_heads": 0}, {"q": q.data_ptr() + 8}, {"q_nb_node": 14 * D - 4}, {"q_nb_seq": -4}, {"k__data": None},
                {"k__ne2": 1}, {"scores_nb_head": 63}, {"scores_nb_seq": 127}, {"reserved": 1}):
        assert status(**bad) == 1, bad
    assert status(n_q_heads=13) == 2 and status(n_q_heads=18) == 2
    assert status(max_kv_len=65, scores_nb_head=100, scores_nb_seq=200) == 3
    with pytest.raises(ValueError):
        cv.KVScorer(ctx, k, q, lse[:1], kl, sc)
    with pytest.raises(ValueError):
        cv.KVScorer(ctx, k, q, lse, kl, sc[:, :1])
    with pytest.raises(ValueError):
        cv.KVScorer(ctx, k, q, lse, kl, sc, max_kv_len=65)


# -------------------------------------------------------------------------------------------------------------- eviction

def evict_reference(scores, pos, lens, kept, total, budget, sink, recent, caches):
    """caches: arrays [layers, S, cap, Hkv, bytes], changed in place.  Returns scores, pos (of slots below kv_len), lengths."""
    Ly, S, H, cap = scores.shape
    scores, pos = scores.copy(), pos.copy()
    for y in range(Ly):
        for s in range(S):
            L = lens[s]
            for h in range(H):
                tok = [int(pos[y, s, h, j]) if j < kept[s] else total[s] - L + j for j in range(L)]
                sc = scores[y, s, h].copy()
                if L > budget:
                    def rank(j):
                        v = sc[j]
                        safe = tok[j] < sink or tok[j] >= total[s] - recent
                        return (0 if safe else 1, 0.0 if safe else (np.inf if np.isnan(v) else -float(v)), j)
                    stay = sorted(sorted(range(L), key=rank)[:budget])
                    free = [j for j in range(budget) if j not in set(stay)]
                    late = [j for j in stay if j >= budget]
                    assert len(free) == len(late)
                    for a, b in zip(free, late):
                        tok[a], scores[y, s, h, a] = tok[b], sc[b]
                        for c in caches:
                            c[y, s, a, h] = c[y, s, b, h]
                    scores[y, s, h, budget:L] = 0
                pos[y, s, h, :min(L, budget)] = tok[:min(L, budget)]
    return scores, pos, [min(L, budget) for L in lens]


def run_evict(ctx, cv, torch, oracle, kname, vname, Hkv, lens, budget, kept=None, layers=2, sink=0, recent=0, make=None, seed=0, cap=None,
              in_place=False, pad=0, offset=0, total=None):
    rng = np.random.default_rng(seed)
    S, cap = len(lens), cap or max(max(lens), 1)
    kept = kept if kept is not None else [min(L, budget) * 3 // 4 for L in lens]
    total = total if total is not None else [L + 11 for L in lens]
    ks = [Rows(cv, torch, oracle, cv.TYPE_BY_NAME[kname], rng.standard_normal((S, cap, Hkv * D)).astype(np.float32), Hkv, pad, offset) for _ in range(layers)]
    vs = [Rows(cv, torch, oracle, cv.TYPE_BY_NAME[vname], rng.standard_normal((S, cap, Hkv * D)).astype(np.float32), Hkv, pad, offset) for _ in range(layers)]
    scores = (make(rng, (layers, S, Hkv, cap)) if make else rng.random((layers, S, Hkv, cap))).astype(np.float32)
    pos = np.zeros((layers, S, Hkv, cap), dtype=np.int32)
    for y in range(layers):
        for s in range(S):
            for h in range(Hkv):
                past = max(total[s] - lens[s] + kept[s], kept[s])
                pos[y, s, h, :kept[s]] = rng.permutation(past)[:kept[s]]
    raws = [np.stack([r.raw() for r in side]).reshape(layers, S, cap, Hkv, -1).copy() for side in (ks, vs)]
    want_s, want_p, want_l = evict_reference(scores, pos, lens, kept, total, budget, sink, recent, raws)
    cu = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    ts, tp, kl = torch.tensor(scores, device="cuda"), torch.tensor(pos, device="cuda"), cu(lens)
    so, po, lo = (ts, tp, kl) if in_place else (torch.full_like(ts, 5.0), torch.full_like(tp, -9), torch.full_like(kl, -9))
    cv.kv_evict(ctx, [r.desc for r in ks], [r.desc for r in vs], ts, tp, kl, cu(kept), cu(total), budget, scores_out=so, pos_out=po,
                kv_len_out=lo, max_kv_len=max(lens), n_sink=sink, n_recent=recent)
    assert lo.tolist() == want_l
    got_s, got_p = so.cpu().numpy(), po.cpu().numpy()
    for s, L in enumerate(lens):
        m = min(L, budget)
        assert np.array_equal(got_p[:, s, :, :m], want_p[:, s, :, :m])
        a, b = got_s[:, s, :, :L], want_s[:, s, :, :L]
        assert np.array_equal(a.view(np.int32), b.view(np.int32))
        if not in_place:
            assert (got_s[:, s, :, L:] == 5.0).all() and (got_p[:, s, :, m:] == -9).all()
    for side, want in zip((ks, vs), raws):
        for r, w in zip(side, want):
            assert np.array_equal(r.raw(), w.reshape(r.raw().shape))
            assert bool((r.buf[:offset] == 0x5A).all())
            if pad:
                assert bool((r.buf[offset:].view(*r.shape)[..., r.rb:] == 0xA5).all())


@pytest.mark.parametrize("kname,vname", [("f32", "f32"), ("f16", "q8_0"), ("q8_0", "q4_0"), ("q5_1", "q5_0"), ("q4_1", "f16")])
@pytest.mark.parametrize("Hkv", [1, 2, 16])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_types_and_heads(ctx, cv, cuda, oracle, kname, vname, Hkv, in_place):
    run_evict(ctx, cv, cuda, oracle, kname, vname, Hkv, [300, 100, 129], 100, sink=3, recent=17, in_place=in_place, layers=2)


@pytest.mark.parametrize("L,budget", [(1, 1), (2, 1), (33, 32), (32, 33), (64, 1), (65, 64), (1000, 999), (1000, 1), (1000, 500), (1025, 31), (3000, 2500),
                                      (9000, 700)])
def test_evict_sizes(ctx, cv, cuda, oracle, L, budget):
    run_evict(ctx, cv, cuda, oracle, "q8_0", "q4_0", 2, [L], budget, layers=1)


@pytest.mark.parametrize("sink,recent", [(0, 64), (64, 0), (32, 32), (0, 0), (1, 0), (0, 1)])
def test_evict_protects_first_and_last_tokens(ctx, cv, cuda, oracle, sink, recent):
    run_evict(ctx, cv, cuda, oracle, "q8_0", "q8_0", 2, [200, 64, 65], 64, sink=sink, recent=recent)


@pytest.mark.parametrize("what", ["zeros", "ties", "few levels", "signs", "tiny", "extremes"])
def test_evict_orders_scores(ctx, cv, cuda, oracle, what):
    def make(rng, shape):
        if what == "zeros":
            return np.zeros(shape)
        if what == "ties":
            return np.where(rng.random(shape) < 0.5, 1.5, 1.5)
        if what == "few levels":
            return rng.integers(0, 3, shape) * 0.25
        if what == "signs":
            return np.where(rng.random(shape) < 0.3, -0.0, rng.standard_normal(shape))
        if what == "tiny":
            return rng.integers(0, 50, shape) * np.float32(1e-45)
        x = rng.standard_normal(shape)
        pick = rng.integers(0, 8, shape)
        for i, v in enumerate((np.inf, -np.inf, np.nan, 3.4e38, -3.4e38)):
            x[pick == i] = v
        return x
    run_evict(ctx, cv, cuda, oracle, "q4_0", "q8_0", 2, [500, 190], 180, sink=2, recent=9, make=make)


def test_evict_lengths_zero_and_within_the_budget(ctx, cv, cuda, oracle):
    run_evict(ctx, cv, cuda, oracle, "q8_0", "q8_0", 2, [0, 1, 50, 51, 200], 50, sink=4, recent=10)


def test_evict_strides(ctx, cv, cuda, oracle):
    for pad, offset in ((2, 2), (6, 4), (4, 0), (16, 32)):
        run_evict(ctx, cv, cuda, oracle, "q8_0", "q5_0", 2, [150, 149], 70, pad=pad, offset=offset, cap=160)


def test_evict_more_layers_than_one_launch_takes(ctx, cv, cuda, oracle):
    run_evict(ctx, cv, cuda, oracle, "q4_0", "q4_0", 1, [40, 9], 20, layers=67, in_place=True)


def test_evict_without_positions_and_records_bad_lengths(ctx, cv, cuda, oracle):
    torch = cuda
    rng = np.random.default_rng(0)
    k = Rows(cv, torch, oracle, cv.Q8_0, rng.standard_normal((4, 64, 128)).astype(np.float32), 2)
    before = k.raw().copy()
    sc = torch.rand((1, 4, 2, 64), device="cuda")
    pos = torch.full((1, 4, 2, 64), 77, dtype=torch.int32, device="cuda")
    kl = torch.tensor([60, 65, -1, 40], dtype=torch.int32, device="cuda")
    kept = torch.tensor([0, 0, 0, 41], dtype=torch.int32, device="cuda")
    old = sc.clone()
    for kp in (kept, None):
        kl = torch.tensor([60, 65, -1, 40 if kp is not None else 20], dtype=torch.int32, device="cuda")
        cv.kv_evict(ctx, [k.desc], [k.desc], sc, pos, kl, kp, None, 32, max_kv_len=64, n_recent=32)
        assert ctx.sync_status() == (6, 2)
        assert kl.tolist() == [32, 65, -1, 40 if kp is not None else 20]
        # no tokens were evicted before: the last 32 of 60 stay, in ascending order in the freed slots
        want = sorted(range(28, 32)) + list(range(32, 60))
        assert sorted(pos[0, 0, 0, :32].tolist()) == want
        assert torch.equal(sc[0, 1:3], old[0, 1:3]) and np.array_equal(k.raw()[1:], before[1:])
        sc.copy_(old)
        pos.fill_(77)
        k.buf.copy_(torch.tensor(before.reshape(-1), device="cuda"))


def test_evict_refusals(ctx, cv, cuda):
    torch = cuda
    lib, ct = cv.lib, __import__("ctypes")
    buf, k = cv.alloc_kv(cv.Q8_0, 2, D, 64, 2)
    vbuf, v = cv.alloc_kv(cv.Q4_0, 2, D, 64, 2)
    sc = torch.zeros((1, 2, 2, 64), device="cuda")
    pos = torch.zeros((1, 2, 2, 64), dtype=torch.int32, device="cuda")
    lens = torch.zeros(10, dtype=torch.int32, device="cuda")
    kl, kept, tot, lo = lens[:2], lens[2:4], lens[4:6], lens[6:8]
    plan = cv.KVEvictor(ctx, [k], [v], sc, pos, kl, kept, tot, 32, kv_len_out=lo, n_sink=1, n_recent=2)

    def status(**kw):
        p = cv.KVEvictParams.from_buffer_copy(plan.params)
        for name, val in kw.items():
            setattr(p, name, val)
        return lib.cvattn_kv_evict(ctx.handle, 0, ct.byref(p))

    assert status() == 0 and status(n_seq=0) == 0 and status(n_layers=0) == 0
    other = (cv.Tensor * 1)(v)
    wide = (cv.Tensor * 1)(cv.kv_tensor(buf, cv.Q8_0, 1, D, 64, 2))
    for bad in ({"k": None}, {"scores": None}, {"scores_out": None}, {"pos": None}, {"pos_out": None}, {"kv_len": None}, {"kv_len_out": None},
                {"n_seq": 3}, {"n_seq": -1}, {"n_layers": -1}, {"budget": 0}, {"n_sink": -1}, {"n_recent": -1}, {"n_recent": 32}, {"nb_head": 63},
                {"nb_seq": 127}, {"workspace": None}, {"workspace_size": 8}, {"kv_len_out": kl.data_ptr() + 4}, {"kv_len_out": tot.data_ptr()}):
        assert status(**bad) == 1, bad
    assert status(k=wide) == 2
    assert status(max_kv_len=65, nb_head=100, nb_seq=200) == 3
    assert status(k=other) == 0  # any two types
    with pytest.raises(ValueError):
        cv.KVEvictor(ctx, [k], [], sc, pos, kl, kept, tot, 32)
    with pytest.raises(ValueError):
        cv.KVEvictor(ctx, [k], [v], sc, pos.long(), kl, kept, tot, 32)
    with pytest.raises(ValueError):
        cv.KVEvictor(ctx, [k], [v], sc, pos, kl, kept, tot, 32, max_kv_len=65)


# ------------------------------------------------------------------------------------------------------------- together

def test_draft_verify_commit_score_evict(ctx, cv, cuda, oracle):
    """A few steps of speculative decoding in a cache of 96 positions kept to 64, against the same steps in 64 bits."""
    torch = cuda
    rng = np.random.default_rng(12)
    S, n, Hq, Hkv, cap, budget = 3, 7, 14, 2, 96, 64
    row = Hkv * D
    start = [60, 33, 50]
    k = Rows(cv, torch, oracle, cv.Q8_0, rng.standard_normal((S, cap, row)).astype(np.float32), Hkv)
    v = Rows(cv, torch, oracle, cv.Q4_0, rng.standard_normal((S, cap, row)).astype(np.float32), Hkv)
    kd, vd = (Rows(cv, torch, oracle, t, np.zeros((S, n, row), np.float32), Hkv) for t in (cv.Q8_0, cv.Q4_0))
    parents = np.array([[-1, 0, 0, 1, 1, 3, 4]] * S)
    sees = ancestors(parents)
    mask = cv.pack_tree_mask(parents).cuda()
    assert np.array_equal(mask.cpu().numpy(), pack(sees))
    kl = torch.tensor(start, dtype=torch.int32, device="cuda")
    total = kl.clone()
    kept = torch.zeros_like(kl)
    scores = torch.zeros((1, S, Hkv, cap), device="cuda")
    pos = torch.zeros((1, S, Hkv, cap), dtype=torch.int32, device="cuda")
    q, out = torch.empty((S, n, Hq, D), device="cuda"), torch.empty((S, n, Hq, D), device="cuda")
    lse = torch.empty((S, n, Hq), device="cuda")
    path, count = torch.zeros((S, 4), dtype=torch.int32, device="cuda"), torch.zeros(S, dtype=torch.int32, device="cuda")
    verify = cv.TreeDecoder(ctx, k.desc, v.desc, kd.desc, vd.desc, q, out, kl, cap, lse=lse, mask=mask)
    commit = cv.TreeCommitter(ctx, [k.desc, v.desc], [kd.desc, vd.desc], path, count, kl, kl)
    weigh = cv.KVScorer(ctx, k.desc, q, lse, kl, scores[0], rows=path, n_rows=count, decay=0.95)
    shrink = cv.KVEvictor(ctx, [k.desc], [v.desc], scores, pos, kl, kept, total, budget, kv_len_out=kl, n_sink=2, n_recent=16)
    node = torch.arange(n, dtype=torch.int32, device="cuda")
    # the same in 64 bits: per (sequence, head) lists of (token, key, value, score)
    heads = [[[[j, k.f[s, j, h], v.f[s, j, h], 0.0] for j in range(start[s])] for h in range(Hkv)] for s in range(S)]
    seen = list(start)
    for step in range(14):
        kn, vn = (rng.standard_normal((S, n, row)).astype(np.float32) for _ in range(2))
        kf = oracle.dequantize(cv.Q8_0, oracle.quantize(cv.Q8_0, kn), row).reshape(S, n, Hkv, D).astype(np.float64)
        vf = oracle.dequantize(cv.Q4_0, oracle.quantize(cv.Q4_0, vn), row).reshape(S, n, Hkv, D).astype(np.float64)
        cv.kv_append(ctx, kd.desc, torch.tensor(kn, device="cuda"), node)
        cv.kv_append(ctx, vd.desc, torch.tensor(vn, device="cuda"), node)
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(step)))
        qf = q.cpu().numpy().astype(np.float64)
        verify()
        want = np.zeros((S, n, Hq, D))
        tops = np.zeros((S, n, Hq))
        for s in range(S):
            for i in range(n):
                for h in range(Hq):
                    g = h // (Hq // Hkv)
                    ks = np.array([e[1] for e in heads[s][g]] + [kf[s, j, g] for j in range(n) if sees[s, i, j]])
                    vs = np.array([e[2] for e in heads[s][g]] + [vf[s, j, g] for j in range(n) if sees[s, i, j]])
                    x = ks @ qf[s, i, h] / 8
                    tops[s, i, h] = np.log(np.exp(x - x.max()).sum()) + x.max()
                    want[s, i, h] = np.exp(x - tops[s, i, h]) @ vs
        assert rel_l2(out.cpu().numpy(), want) <= REL_L2, step
        take = [int(rng.integers(1, 5)) for _ in range(S)]
        paths = [[0, 1, 3, 5], [0, 2, 0, 0], [0, 1, 4, 6]]
        take[1] = min(take[1], 2)
        path.copy_(torch.tensor(paths, dtype=torch.int32))
        count.copy_(torch.tensor(take, dtype=torch.int32))
        commit()
        total += count
        weigh()
        for s in range(S):
            for g in range(Hkv):
                have = heads[s][g]
                for e in have:
                    e[3] *= 0.95
                for i in range(take[s]):
                    have.append([seen[s] + i, kf[s, paths[s][i], g], vf[s, paths[s][i], g], 0.0])
                base = len(have) - take[s]
                for i in range(take[s]):
                    for h in range(g * 7, g * 7 + 7):
                        for e in have[:base + i + 1]:
                            e[3] += np.exp(e[1] @ qf[s, paths[s][i], h] / 8 - tops[s, paths[s][i], h])
            seen[s] += take[s]
        got = scores[0].cpu().numpy()
        for s in range(S):
            for g in range(Hkv):
                assert rel_l2(got[s, g, :len(heads[s][g])], np.array([e[3] for e in heads[s][g]])) <= 2 * REL_L2
        if step % 5 == 4:
            shrink()
            kept.copy_(kl)
            for s in range(S):
                for g in range(Hkv):
                    have = heads[s][g]
                    if len(have) <= budget:
                        continue
                    order = sorted(range(len(have)), key=lambda j: (not (have[j][0] < 2 or have[j][0] >= seen[s] - 16), -have[j][3], j))
                    stay = sorted(order[:budget], key=lambda j: j)
                    late = [j for j in stay if j >= budget]
                    for j in [j for j in range(budget) if j not in set(stay)]:
                        have[j] = have[late.pop(0)]
                    del have[budget:]
            tokens = pos[0].cpu().numpy()
            for s in range(S):
                for g in range(Hkv):
                    assert tokens[s, g, :len(heads[s][g])].tolist() == [e[0] for e in heads[s][g]]
        assert kl.tolist() == [len(heads[s][0]) for s in range(S)]
