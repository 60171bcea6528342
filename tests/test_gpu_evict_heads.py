"""GPU: eviction at every head size that the entry takes (whole blocks of 32).

Whole numbers and moved bytes: exact.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_bounded_cache import evict_reference

pytestmark = pytest.mark.gpu


def moved(ctx, cv, torch, oracle, kname, vname, Hkv, head_dim, L, budget, offset=0, pad=0):
    rng = np.random.default_rng(head_dim + Hkv)
    layers, S = 2, 2
    lens, total = [L, L - 1], [L + 5, L - 1]
    raws, descs, bufs = [], [], []
    for name in (kname, vname):
        t = cv.TYPE_BY_NAME[name]
        raw = np.stack([oracle.quantize(t, rng.standard_normal((S, L, Hkv * head_dim)).astype(np.float32)) for _ in range(layers)])
        rb = raw.shape[-1]
        side, mem = [], []
        for y in range(layers):
            host = np.full((S, L, rb + pad), 0xA5, dtype=np.uint8)
            host[..., :rb] = raw[y]
            buf = torch.zeros(offset + host.size, dtype=torch.uint8, device="cuda")
            buf[offset:] = torch.tensor(host.reshape(-1), device="cuda")
            side.append(cv.kv_tensor(buf, t, Hkv, head_dim, L, S, nb1=rb + pad, byte_offset=offset))
            mem.append(buf)
        raws.append(raw.reshape(layers, S, L, Hkv, rb // Hkv).copy())
        descs.append(side)
        bufs.append((mem, rb))
    scores = rng.random((layers, S, Hkv, L)).astype(np.float32)
    pos = np.zeros((layers, S, Hkv, L), dtype=np.int32)
    want_s, want_p, want_l = evict_reference(scores, pos, lens, [0, 0], total, budget, 2, 9, raws)
    cu = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    ts, tp, kl = torch.tensor(scores, device="cuda"), torch.tensor(pos, device="cuda"), cu(lens)
    cv.kv_evict(ctx, *descs, ts, tp, kl, cu([0, 0]), cu(total), budget, n_sink=2, n_recent=9)
    assert kl.tolist() == want_l
    for s in range(S):
        assert np.array_equal(tp.cpu().numpy()[:, s, :, :budget], want_p[:, s, :, :budget])
        assert np.array_equal(ts.cpu().numpy()[:, s, :, :lens[s]], want_s[:, s, :, :lens[s]])
    for (mem, rb), want in zip(bufs, raws):
        for y, buf in enumerate(mem):
            got = buf[offset:].view(S, L, rb + pad).cpu().numpy()
            assert np.array_equal(got[..., :rb], want[y].reshape(S, L, rb))
            assert (got[..., rb:] == 0xA5).all()


@pytest.mark.parametrize("head_dim", [32, 64, 96, 160])
@pytest.mark.parametrize("kname,vname", [("q8_0", "q4_0"), ("q5_0", "q8_0"), ("q4_0", "q5_0"), ("q4_1", "q8_0"), ("q5_1", "q4_1"), ("f16", "q4_0"), ("q8_0", "f32")])
@pytest.mark.parametrize("Hkv", [1, 2, 3])
def test_evict_head_sizes(ctx, cv, cuda, oracle, head_dim, kname, vname, Hkv):
    """A head's slice of a row may be an odd number of 2-byte units although rows and addresses are multiples of 4."""
    moved(ctx, cv, cuda, oracle, kname, vname, Hkv, head_dim, 90, 60)


@pytest.mark.parametrize("head_dim", [32, 96])
@pytest.mark.parametrize("kname,vname", [("q8_0", "q8_0"), ("q4_0", "q5_0")])
@pytest.mark.parametrize("offset,pad", [(0, 0), (2, 2), (4, 8)])
def test_evict_head_sizes_with_many_moves(ctx, cv, cuda, oracle, head_dim, kname, vname, offset, pad):
    """More than 256 rows of a head move: a launch of their own."""
    moved(ctx, cv, cuda, oracle, kname, vname, 2, head_dim, 640, 320, offset=offset, pad=pad)
