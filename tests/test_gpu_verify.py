"""GPU: verification of drafted tokens, against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from paged_reference import verify

pytestmark = pytest.mark.gpu

DTYPES = ("float32", "float16", "bfloat16")


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


def trees(rng, S, n, chain):
    p = np.arange(-1, n - 1)[None].repeat(S, 0)
    if not chain:
        for i in range(1, n):
            p[:, i] = np.maximum(0, i - 1 - rng.integers(0, 4, S))
    return p.astype(np.int32)


def check(cv, ctx, torch, logits, tokens, parents, u, last, heat=None, probs=None, n=None, one_tree=False, chain=False, plan_only=False,
          logits_view=None, probs_view=None):
    S, N, V = logits.shape
    dev = lambda a, t: torch.tensor(np.asarray(a), dtype=t, device="cuda")  # noqa: E731
    lg = logits_view if logits_view is not None else logits
    i32, f32 = torch.int32, torch.float32
    accepted, count, token = (torch.full(s, 77, dtype=i32, device="cuda") for s in ((S, N), (S,), (S,)))
    logs = torch.full((S, N), 77.0, device="cuda")
    pv = probs_view if probs_view is not None else None if probs is None else dev(probs, f32)
    plan = cv.DraftVerifier(ctx, lg, dev(tokens, i32), dev(u, f32), dev(last, f32), accepted, count, token,
                            parents=None if chain else dev(parents[:1] if one_tree else parents, i32), n_nodes=None if n is None else dev(n, i32),
                            draft_probs=pv, temperature=None if heat is None else dev(heat, f32), log_probs=logs)
    plan()
    host = logits.float().cpu().numpy()
    got = [x.cpu().numpy() for x in (accepted, count, token, logs)]
    u, last = np.asarray(u, np.float32), np.asarray(last, np.float32)
    for s in range(S):
        m = N if n is None else n[s]
        path, end, said = verify(host[s], tokens[s], parents[s], m, u[s].astype(np.float64), np.float64(last[s]),
                                 1.0 if heat is None else np.float32(heat[s]), None if probs is None else np.asarray(probs[s], np.float32))
        assert got[1][s] == len(path), s
        assert got[0][s].tolist() == path + [-1] * (N - len(path)), s
        assert got[2][s] == end, s
        # f32 of a logarithm whose argument is good to a few 2^-24 (its sum is of f32 exponentials in 64 bits)
        want = np.array(said + [0.0] * (N - len(said)))
        assert np.all(np.abs(got[3][s] - want) <= 2.0 ** -23 * np.abs(want) + 2.0 ** -21 * (want != 0)), (s, got[3][s], want)
    return plan


def case(rng, torch, S, N, V, dtype, chain, with_probs, sigma=3.0):
    logits = torch.tensor(rng.standard_normal((S, N, V)) * sigma, dtype=getattr(torch, dtype), device="cuda")
    host = logits.float().cpu().numpy().astype(np.float64)
    parents = trees(rng, S, N, chain)
    probs = softmax(host + rng.standard_normal(host.shape) * 0.4).astype(np.float32)
    tokens = np.zeros((S, N), np.int32)
    for s in range(S):
        for i in range(N):
            tokens[s, i] = rng.choice(V, p=probs[s, max(parents[s, i], 0)].astype(np.float64) / probs[s, max(parents[s, i], 0)].astype(np.float64).sum())
    return logits, tokens, parents, rng.random((S, N)), rng.random(S), probs if with_probs else None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("chain", [True, False])
@pytest.mark.parametrize("with_probs", [True, False])
@pytest.mark.parametrize("S,N,V", [(5, 1, 1), (9, 4, 2), (40, 9, 33), (17, 6, 1000), (3, 8, 6563), (2, 3, 50001)])
def test_verify(ctx, cv, cuda, dtype, chain, with_probs, S, N, V):
    rng = np.random.default_rng(S * N + V)
    logits, tokens, parents, u, last, probs = case(rng, cuda, S, N, V, dtype, chain, with_probs)
    heat = rng.choice([0.0, 0.5, 1.0, 1.7], S)
    n = rng.integers(0, N + 1, S)
    check(cv, ctx, cuda, logits, tokens, parents, u, last, heat, probs, chain=chain)
    check(cv, ctx, cuda, logits, tokens, parents, u, last, None, probs, n=n, chain=chain)


def test_verify_of_a_large_vocabulary(ctx, cv, cuda):
    """Flat and peaked rows over more tokens than any cluster of blocks keeps on its chips."""
    rng = np.random.default_rng(2)
    for V, sigma, probs in ((151937, 3.0, True), (300007, 0.01, True), (300007, 5.0, False)):
        logits, tokens, parents, u, last, q = case(rng, cuda, 3, 3, V, "float32", True, probs, sigma)
        check(cv, ctx, cuda, logits, tokens, parents, u, last, None, q, chain=True)


def test_wide_trees(ctx, cv, cuda):
    """Many siblings, the same token twice among them, one tree for all; 256 nodes."""
    rng = np.random.default_rng(4)
    S, N, V = 12, 256, 64
    logits, tokens, parents, u, last, probs = case(rng, cuda, S, N, V, "float32", False, True)
    parents[:] = np.where(np.arange(N) == 0, -1, np.maximum(0, (np.arange(N) - 1) // 20))[None]
    for q in (probs, None):
        check(cv, ctx, cuda, logits, tokens, parents, u, last, None, q, one_tree=True)
        check(cv, ctx, cuda, logits, tokens, parents, np.full((S, N), 0.999), last, None, q, one_tree=True)
        check(cv, ctx, cuda, logits, tokens, parents, np.zeros((S, N)), last, None, q, one_tree=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan(ctx, cv, cuda, dtype):
    torch, rng = cuda, np.random.default_rng(6)
    S, N, V = 8, 4, 700
    logits, tokens, parents, u, last, probs = case(rng, torch, S, N, V, dtype, True, True)
    logits[0, 0, 100:] = -np.inf
    logits[1, 0, ::2] = np.nan
    logits[2, 0, [5, 600]] = np.inf
    logits[3, 1] = -np.inf           # nothing left at a node that may be reached
    logits[4, 0] = np.nan            # or at the first
    logits[5, :, :] = -np.inf
    logits[5, :, 699] = -3.0         # a single token
    logits[6] = torch.finfo(logits.dtype).min
    logits[7, 0] = torch.finfo(logits.dtype).min
    logits[7, 0, 3] = torch.finfo(logits.dtype).max
    probs[0, 0, ::3], probs[2, 0, ::5] = np.nan, -1.0
    u[3] = 0.0
    for heat in (1.0, 0.0, 0.3):
        for q in (probs, None):
            check(cv, ctx, torch, logits, tokens, parents, u, last, np.full(S, heat), q, chain=True)


def test_temperatures_that_leave_a_single_token(ctx, cv, cuda):
    """Temperatures so low, and logits so large, that neighbouring numbers are far more than all weights apart."""
    torch, rng = cuda, np.random.default_rng(7)
    S, N, V = 12, 3, 300
    logits, tokens, parents, u, last, probs = case(rng, torch, S, N, V, "float32", True, True)
    logits[:, :, 7] = 9.0
    logits[:, :, 250] = float(np.nextafter(np.float32(9), np.float32(8)))
    logits[4] *= 1e10
    logits[5] *= 1e30
    logits[6] = torch.finfo(torch.float32).min
    logits[6:8, :, ::3] = -np.inf
    logits[8, :, 20:] = torch.finfo(torch.float32).min
    heat = np.array([1e-9, 3e-9, 1e-8, 1e-6, 1.0, 0.5, 2.0, 1e-7, 1e-30, 1e-42, 3e38, 1e-9], np.float32)
    tokens[::2, 1] = 7
    for q in (probs, None):
        for numbers in (u, np.zeros((S, N)), np.full((S, N), 0.9999)):
            check(cv, ctx, torch, logits, tokens, parents, numbers, last, heat, q, chain=True)
            check(cv, ctx, torch, logits, tokens, parents, numbers, np.full(S, 1 - 2.0 ** -24), heat, q, chain=True)


def test_nothing_left_stays_as_it_was(ctx, cv, cuda):
    """Draft and target alike: a refusal cannot happen by the rule, but with numbers at 1 it is asked for."""
    torch, rng = cuda, np.random.default_rng(8)
    logits = torch.tensor(np.log([[[0.5, 0.25, 0.25]] * 3] * 4), dtype=torch.float32, device="cuda")
    probs = np.array([[[0.5, 0.25, 0.25]] * 3] * 4, np.float32) * 1.25  # above the target everywhere
    tokens = np.array([[0, 0, 1]] * 4, np.int32)
    parents = np.array([[-1, 0, 0]] * 4, np.int32)
    check(cv, ctx, torch, logits, tokens, parents, np.full((4, 3), 0.99), [0.1, 0.4, 0.6, 0.9], None, probs)


def test_ties_and_borders(ctx, cv, cuda):
    """Equal logits: the lowest token when greedy; random numbers at 0 and just below 1; tokens of no weight never follow."""
    torch = cuda
    S, N, V = 6, 1, 5000
    logits = torch.zeros((S, N, V), device="cuda")
    logits[1, 0, :7] = -np.inf
    logits[2, 0, 4000:] = -np.inf
    logits[3, 0, 1:] = -200.0
    logits[4, 0, :4999] = -np.inf
    zeros, none = np.zeros((S, N), np.int32), np.full((S, N), -1, np.int32)
    for last in (0.0, np.nextafter(np.float32(1), np.float32(0)), 0.5):
        for heat in (None, np.zeros(S)):
            check(cv, ctx, torch, logits, zeros, none, np.zeros((S, N)), np.full(S, last), heat)


def test_strided_and_shared_rows(ctx, cv, cuda):
    """Logits and draft probabilities as parts of wider tensors, at any alignment."""
    torch, rng = cuda, np.random.default_rng(10)
    S, N, V = 4, 5, 1003
    for dtype in DTYPES:
        logits, tokens, parents, u, last, probs = case(rng, torch, S, N, V, dtype, True, True)
        wide = torch.full((S, N + 1, V + 13), 50.0, dtype=logits.dtype, device="cuda")
        view = wide[:, 1:, 7:7 + V]
        view.copy_(logits)
        pw = torch.full((S, N, V + 6), 0.5, device="cuda")
        pv = pw[..., 3:3 + V]
        pv.copy_(torch.from_numpy(probs))
        check(cv, ctx, torch, logits, tokens, parents, u, last, None, probs, chain=True, logits_view=view, probs_view=pv)


def test_bad_sequences_are_recorded(ctx, cv, cuda):
    """Counts, temperatures, tokens and parents out of range: nothing is accepted there; the others go on."""
    torch, rng = cuda, np.random.default_rng(12)
    S, N, V = 8, 4, 100
    logits, tokens, parents, u, last, _ = case(rng, torch, S, N, V, "float32", False, False)
    n, heat = np.full(S, N), np.ones(S, np.float32)
    n[0], n[1], heat[2], heat[3], tokens[4, 2], tokens[5, 1], parents[6, 2] = -1, N + 1, -1.0, np.nan, V, -1, 2
    dev = lambda a, t: torch.tensor(np.asarray(a), dtype=t, device="cuda")  # noqa: E731
    accepted, count, token = (torch.full(s, 77, dtype=torch.int32, device="cuda") for s in ((S, N), (S,), (S,)))
    logs = torch.full((S, N), 7.0, device="cuda")
    cv.DraftVerifier(ctx, logits, dev(tokens, torch.int32), dev(u, torch.float32), dev(last, torch.float32), accepted, count, token,
                     parents=dev(parents, torch.int32), n_nodes=dev(n, torch.int32), temperature=dev(heat, torch.float32), log_probs=logs)()
    assert ctx.sync_status() == (6, 6)
    assert count[:7].tolist() == [0] * 7 and token[:7].tolist() == [-1] * 7
    assert bool((accepted[:7] == -1).all()) and not logs[:7].any()
    path, end, _ = verify(logits[7].cpu().numpy(), tokens[7], parents[7], N, u[7].astype(np.float32).astype(np.float64), np.float64(np.float32(last[7])), 1.0)
    assert int(count[7]) == len(path) and int(token[7]) == end
    # a tree for all: the first tokens are whatever
    tokens[:] = 5
    tokens[:, 0] = -3
    check(cv, ctx, torch, logits, tokens, trees(rng, 1, N, False).repeat(S, 0), u, last, one_tree=True)


def test_verify_replays(ctx, cv, cuda):
    torch, rng = cuda, np.random.default_rng(14)
    S, N, V = 7, 5, 6563
    first = case(rng, torch, S, N, V, "bfloat16", True, True)
    plan = check(cv, ctx, torch, first[0], *first[1:5], None, first[5], chain=True)
    logits, tokens, u, last, accepted, count, token, probs = (plan._keep[i] for i in (0, 1, 2, 3, 4, 5, 6, 9))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan()
        plan()
    for seed in range(3):
        rng = np.random.default_rng(seed)
        c = case(rng, torch, S, N, V, "bfloat16", True, True)
        for t, x in ((logits, c[0]), (tokens, torch.from_numpy(c[1])), (u, torch.tensor(c[3])), (last, torch.tensor(c[4])), (probs, torch.from_numpy(c[5]))):
            t.copy_(x)
        graph.replay()
        got = [x.clone() for x in (accepted, count, token)]
        plan()
        assert all(torch.equal(a, b) for a, b in zip(got, (accepted, count, token)))


def test_verify_of_the_largest_vocabulary(ctx, cv, cuda):
    """As many tokens as a call takes: drafts with probabilities, one refused."""
    torch, rng = cuda, np.random.default_rng(16)
    V = 2 ** 21
    logits = torch.randn(1, 2, V, device="cuda") * 2
    probs = torch.softmax(logits + 0.5 * torch.randn(1, 2, V, device="cuda"), -1)
    host, q = logits.cpu().numpy(), probs.cpu().numpy()
    worse = int(np.argmax(q[0, 0] - softmax(host[0, 0].astype(np.float64))))
    for u, last in ((0.0, 0.3), (0.999, 0.7)):
        check(cv, ctx, torch, logits, np.array([[0, worse]]), np.array([[-1, 0]]), np.array([[0.0, u]]), [last], None, q, chain=True)
    with pytest.raises(cv.CvattnError, match="UNSUPPORTED"):
        big = torch.zeros(1, 1, V + 1, device="cuda")
        one = [torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((1, 1), (1, 1), (1,), (1,))]
        cv.DraftVerifier(ctx, big, one[0], torch.zeros(1, 1, device="cuda"), torch.zeros(1, device="cuda"), *one[1:])()
