"""GPU: verification by clusters of CTAs, where some sequences end before the first exchange between CTAs."""
from __future__ import annotations

import numpy as np
import pytest

from paged_reference import verify
from test_gpu_verify import case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S,V,dtype", [(18, 17000, "float32"), (18, 40000, "bfloat16"), (30, 9000, "float32"), (60, 5000, "float32"), (4, 17000, "float16")])
@pytest.mark.parametrize("with_probs", [True, False])
def test_sequences_that_end_at_once_beside_others(ctx, cv, cuda, S, V, dtype, with_probs):
    """Clusters of 8, 4 and 2 CTAs to a sequence: no nodes, counts, temperatures and tokens out of range, a first node without any
    weight; the others are verified, many times over with the same outcome."""
    torch, rng = cuda, np.random.default_rng(S + V)
    N = 4
    logits, tokens, parents, u, last, probs = case(rng, torch, S, N, V, dtype, True, with_probs)
    n, heat = np.full(S, N), np.ones(S, np.float32)
    n[0], n[1], n[2], heat[3 % S] = 0, -1, N + 1, 0.0
    if S > 4:
        heat[4], heat[5], tokens[6, 2], n[7] = np.nan, -1.0, V, 1
        logits[8] = -np.inf
    bad = [s for s in range(S) if s in (1, 2) or S > 4 and s in (4, 5, 6)]
    dev = lambda a, t: torch.tensor(np.asarray(a), dtype=t, device="cuda")  # noqa: E731
    accepted, count, token = (torch.empty(s, dtype=torch.int32, device="cuda") for s in ((S, N), (S,), (S,)))
    plan = cv.DraftVerifier(ctx, logits, dev(tokens, torch.int32), dev(u, torch.float32), dev(last, torch.float32), accepted, count, token,
                            n_nodes=dev(n, torch.int32), temperature=dev(heat, torch.float32),
                            draft_probs=None if probs is None else dev(probs, torch.float32))
    host, want = logits.float().cpu().numpy(), []
    for s in range(S):
        path, end, _ = ([], -1, []) if s in bad else verify(host[s], tokens[s], parents[s], n[s], u[s].astype(np.float32).astype(np.float64),
                                                            np.float64(np.float32(last[s])), heat[s], None if probs is None else probs[s])
        want.append((path + [-1] * (N - len(path)), len(path), end))
    for _ in range(20):
        accepted.fill_(77), count.fill_(77), token.fill_(77)
        plan()
        for s in range(S):
            assert (accepted[s].tolist(), int(count[s]), int(token[s])) == want[s], s
    assert ctx.sync_status() == (6, 6)
