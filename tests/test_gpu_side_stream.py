"""GPU: one-shot calls of tree attention and eviction on another stream than the current one.

Their scratch memory must not be handed out on the current stream while they run: what is allocated and filled there
right after the call, which is still waiting on its stream, keeps its contents.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_bounded_cache import evict_reference
from test_gpu_tree import D, REL_L2, Rows, reference, rel_l2

pytestmark = pytest.mark.gpu


def waiting_stream(torch):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # some 10 ms
    return side


@pytest.mark.parametrize("handle", [False, True])
@pytest.mark.parametrize("kname", ["q8_0", "f32"])
def test_tree_decode(ctx, cv, cuda, oracle, kname, handle):
    torch = cuda
    rng = np.random.default_rng(0)
    t, L, n = cv.TYPE_BY_NAME[kname], 3000, 8
    k = Rows(cv, torch, oracle, t, rng.standard_normal((1, L, 128)).astype(np.float32), 2)
    kd = Rows(cv, torch, oracle, t, rng.standard_normal((1, n, 128)).astype(np.float32), 2)
    q = torch.tensor(rng.standard_normal((1, n, 14, D)).astype(np.float32), device="cuda")
    kl = torch.tensor([L], dtype=torch.int32, device="cuda")
    need = cv.tree_decode_workspace_size(t, t, 1, L, n, 14, 2)
    assert need
    torch.cuda.synchronize()
    side = waiting_stream(torch)
    out = cv.tree_decode(ctx, q, k.desc, k.desc, kd.desc, kd.desc, kl, L, stream=side.cuda_stream if handle else side)
    others = [torch.full((size,), 0x55, dtype=torch.uint8, device="cuda") for size in (need, need, q.numel() * 4, q.numel() * 4)]
    torch.cuda.synchronize()
    for x in others:
        assert bool((x == 0x55).all())
    want, _ = reference(q.cpu().numpy(), k.f, k.f, kd.f, kd.f, [L], [n], np.tril(np.ones((1, n, n), dtype=bool)), 0.125)
    assert rel_l2(out.cpu().numpy(), want) <= REL_L2


@pytest.mark.parametrize("L,budget", [(300, 200), (2000, 900)])
def test_kv_evict(ctx, cv, cuda, oracle, L, budget):
    torch = cuda
    rng = np.random.default_rng(1)
    k = Rows(cv, torch, oracle, cv.Q8_0, rng.standard_normal((1, L, 128)).astype(np.float32), 2)
    raw = k.raw().reshape(1, 1, L, 2, -1).copy()
    scores = rng.random((1, 1, 2, L)).astype(np.float32)
    pos = np.zeros((1, 1, 2, L), dtype=np.int32)
    want_s, want_p, want_l = evict_reference(scores, pos, [L], [0], [L], budget, 0, 8, [raw])
    ts, tp = torch.tensor(scores, device="cuda"), torch.tensor(pos, device="cuda")
    kl, total = (torch.tensor([L], dtype=torch.int32, device="cuda") for _ in range(2))
    need = int(cv.lib.cvattn_kv_evict_workspace_size(1, 1, 2, L, budget))
    torch.cuda.synchronize()
    side = waiting_stream(torch)
    cv.kv_evict(ctx, [k.desc], [k.desc], ts, tp, kl, None, total, budget, stream=side, n_recent=8)
    others = [torch.full((need,), 0x55, dtype=torch.uint8, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for x in others:
        assert bool((x == 0x55).all())
    assert kl.tolist() == want_l
    assert np.array_equal(tp.cpu().numpy()[..., :budget], want_p[..., :budget])
    assert np.array_equal(ts.cpu().numpy(), want_s)
    assert np.array_equal(k.raw().reshape(raw.shape), raw)
