"""GPU: what the tests of paged attention ask for with many rows, at sizes that the tcgen05 kernel takes (each asserts that it does)."""
from __future__ import annotations

import numpy as np
import pytest

from paged_reference import D, Pool, attention
from test_gpu_paged_cache import check_attention, filled, ints, rows_of
from test_gpu_paged_precision import on_tcgen05

pytestmark = pytest.mark.gpu


def check(cv, ctx, torch, rng, host, table, L, n, Hq, max_q, max_kv_len=None, **kw):
    bound = table.shape[1] * host.size if max_kv_len is None else max_kv_len
    assert on_tcgen05(cv, len(L), max_q, bound, Hq, host.heads)
    return check_attention(cv, ctx, torch, rng, host, table, L, n, Hq, max_q, max_kv_len=max_kv_len, **kw)


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("size", [16, 32, 64, 128])
def test_strided_memory(ctx, cv, cuda, fmt, size):
    """Pages and query rows that lie apart, a table wider than it has to be, scales of one's own, a bound above the lengths."""
    rng = np.random.default_rng(size + fmt)
    lens, max_q = [70, 1, 333, 0], 100
    host, table = filled(rng, fmt, lens, size, 2)
    table = np.concatenate([table, np.full((4, 400 // size), -1, np.int32)], 1)
    n = [max_q, 1, max_q, max_q]
    check(cv, ctx, cuda, rng, host, table, lens, n, 14, max_q, apart=5, q_apart=12, max_kv_len=400, scale=0.3)
    check(cv, ctx, cuda, rng, host, table, lens, n, 14, max_q, max_kv_len=390, scale=-0.2)
    check(cv, ctx, cuda, rng, host, table, lens, n, 14, max_q, max_kv_len=385, scale=0.0)


@pytest.mark.parametrize("fmt", [0, 1])
def test_blocks_of_differing_size(ctx, cv, cuda, fmt):
    """Neighbouring blocks whose scales are far apart, and blocks of zeros."""
    rng = np.random.default_rng(fmt)
    lens = [400, 130, 17, 256]
    host, table = filled(rng, fmt, lens, 64, 2)
    for s, n in enumerate(lens):
        for b in range(-(-n // 16)):
            page, part = table[s, b // 4], b % 4
            host.scales["v"][page, :, part] *= (1.0, 1e-3, 1e3, 0.0, 1e-6)[b % 5]
            host.scales["k"][page, :, part] *= (1.0, 0.1, 0.0, 3.0)[b % 4]
    check(cv, ctx, cuda, rng, host, table, lens, [100, 100, 30, 64], 14, 100)


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("zeros", [1.0, 0.0])
def test_values_of_zero_first(ctx, cv, cuda, fmt, zeros):
    """Whole tiles whose values are all zero, before, between and behind others, and a sequence of nothing else."""
    rng = np.random.default_rng(fmt)
    lens = [500, 300, 384, 300]
    host, table = filled(rng, fmt, lens, 128, 2)
    for s, tiles in enumerate(([0, 2], [1], [0, 1], [0, 1, 2])):
        for t in tiles:
            host.scales["v"][table[s, t]] = 0.0
            host.scales["k"][table[s, t]] *= zeros
    check(cv, ctx, cuda, rng, host, table, lens, [100, 100, 70, 100], 14, 100)


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("size", [16, 128])
def test_pages_out_of_range_are_left_out(ctx, cv, cuda, fmt, size):
    """Blocks of a tile, whole tiles, the first and the last of a sequence, all of one; what the slots held before does not show."""
    rng = np.random.default_rng(size + fmt)
    lens = [200, 100, 64, 500, 500, 500, 260, 130] if size == 16 else [200, 100, 64, 512, 700, 500, 260, 130]
    host, table = filled(rng, fmt, lens, size, 2)
    most = table.shape[1]
    for s, holes in ((0, [0, 3, 7, 12]), (2, range(4)), (3, range(8, 24)), (4, range(0, 32, 2)), (5, [most - 2, most - 1, 31]), (6, [8, 16]), (7, [1])):
        for j in holes:
            if j < most:
                table[s, j] = rng.choice([-1, host.pages, 2 ** 30, -5])
    check(cv, ctx, cuda, rng, host, table, lens, [100, 100, 64, 100, 33, 100, 1, 100], 14, 100)
    assert ctx.sync_status() == (6, 4)


def test_lengths_out_of_range_give_empty_rows(ctx, cv, cuda):
    torch, rng, max_q = cuda, np.random.default_rng(0), 100
    lens = [300] * 6
    host, table = filled(rng, 0, lens, 16, 2)
    pool, q = host.device(torch, cv), torch.randn(6, max_q, 14, D, device="cuda")
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:3], 7.0, device="cuda")
    given, n = [-1, 311, 300, 300, 300, 0], [max_q, max_q, max_q + 1, -1, max_q, max_q]
    assert on_tcgen05(cv, 6, max_q, 310, 14, 2)
    cv.PagedAttention(ctx, pool, q, out, ints(torch, table), ints(torch, given), 310, lse=lse, n_q=ints(torch, n))()
    assert ctx.sync_status() == (6, 2)
    for s in (0, 1, 2, 3, 5):
        assert not out[s].any() and bool((lse[s] == -np.inf).all())
    want, _ = attention(q[4].cpu().numpy(), host.rows("k", table[4], 300), host.rows("v", table[4], 300), max_q, D ** -0.5)
    assert np.abs(out[4].cpu().numpy() - want).max() < 1e-4


def test_offsets_past_32_bits(ctx, cv, cuda):
    """Pages that lie 2^31 bytes apart, which many sequences share."""
    torch, rng, S, max_q = cuda, np.random.default_rng(0), 60, 73
    host = Pool(0, 3, 64, 2)
    for x in "kv":
        host.append(x, [0, 2], 0, rows_of(rng, 100, 2, 0.7))
    small, far = host.device(torch, cv), 1 << 31
    k, v = (torch.zeros(2 * far + 8192, dtype=torch.uint8, device="cuda") for _ in "kv")
    big = [t.as_strided(small.k.shape, (far, 4096, 1)) for t in (k, v)]
    big[0].copy_(small.k), big[1].copy_(small.v)
    pool = cv.PagePool(*big, small.k_scale, small.v_scale, 0)
    table, lens = ints(torch, [[0, 2]] * S), ints(torch, 30 + np.arange(S))
    assert on_tcgen05(cv, S, max_q, 128, 14, 2)
    q = torch.randn(S, max_q, 14, D, device="cuda")
    out, want = torch.empty_like(q), torch.empty_like(q)
    cv.PagedAttention(ctx, pool, q, out, table, lens)()
    cv.PagedAttention(ctx, small, q, want, table, lens)()
    assert torch.equal(out, want)
    host_out, _ = attention(q[59].cpu().numpy(), host.rows("k", [0, 2], 89), host.rows("v", [0, 2], 89), max_q, D ** -0.5)
    assert np.abs(out[59].cpu().numpy() - host_out).max() < 1e-4


def test_two_streams_at_once(ctx, cv, cuda):
    """Two batches with launchers of their own, under way together, many times over with the same bits."""
    torch, rng = cuda, np.random.default_rng(0)
    made, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for fmt in range(2):
        lens = [384, 100, 700, 256]
        host, table = filled(rng, fmt, lens, 32, 2)
        q = torch.randn(4, 100, 14, D, device="cuda")
        assert on_tcgen05(cv, 4, 100, table.shape[1] * 32, 14, 2)
        made.append(cv.PagedAttention(ctx, host.device(torch, cv), q, torch.empty_like(q), ints(torch, table), ints(torch, lens)))
    for plan in made:
        plan()
    torch.cuda.synchronize()
    want = [plan._keep[2].clone() for plan in made]
    for _ in range(20):
        for plan, stream in zip(made, streams):
            plan._keep[2].fill_(7.0)
            stream.wait_stream(torch.cuda.current_stream())
            plan(stream)
        torch.cuda.synchronize()
        for plan, w in zip(made, want):
            assert torch.equal(plan._keep[2], w)


def test_a_replayed_graph_reads_the_lengths_of_its_time(ctx, cv, cuda):
    torch, rng = cuda, np.random.default_rng(3)
    lens = [900, 333, 64, 700]
    host, table = filled(rng, 1, lens, 64, 2)
    t, L, n = ints(torch, table), ints(torch, lens), ints(torch, [100] * 4)
    q = torch.randn(4, 100, 14, D, device="cuda")
    assert on_tcgen05(cv, 4, 100, table.shape[1] * 64, 14, 2)
    make = lambda: cv.PagedAttention(ctx, host_pool, q, torch.empty_like(q), t, L, lse=torch.empty(q.shape[:3], device="cuda"), n_q=n)  # noqa: E731
    host_pool = host.device(torch, cv)
    a, b = make(), make()
    a()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b()
    for given, rows in ((lens, [100] * 4), ([0, 128, 64, 129], [100, 1, 0, 99]), ([900, 0, 0, 0], [3, 0, 0, 0]), ([1, 1, 1, 1], [1, 1, 1, 1])):
        L.copy_(ints(torch, given)), n.copy_(ints(torch, rows))
        graph.replay()
        a()
        assert torch.equal(a._keep[2], b._keep[2]) and torch.equal(a._keep[3], b._keep[3])
        for s in range(4):
            assert not a._keep[2][s, rows[s]:].any()
            want, _ = attention(q[s].cpu().numpy(), host.rows("k", table[s], given[s]), host.rows("v", table[s], given[s]), rows[s], D ** -0.5)
            assert np.abs(a._keep[2][s].cpu().numpy() - want).max(initial=0.0) < 1e-4
