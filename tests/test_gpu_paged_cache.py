"""GPU: append to, reading of and attention over a paged 8-bit cache against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from paged_reference import D, Pool, attention

pytestmark = pytest.mark.gpu


def tables(rng, counts, pages, width):
    order = rng.permutation(pages)
    t, at = np.full((len(counts), width), -1, np.int32), 0
    for s, m in enumerate(counts):
        t[s, :m] = order[at:at + m]
        at += m
    return t


def ints(torch, v):
    return torch.tensor(np.asarray(v, np.int32), device="cuda")


def rows_of(rng, n, heads, spread=2.0):
    return (rng.standard_normal((n, heads, D)) * np.exp(rng.uniform(-spread, spread, (n, 1, 1)))).astype(np.float32)


def filled(rng, fmt, lens, size, heads, extra=3, stale=True):
    """A host pool that holds the sequences, whatever elsewhere, and their table."""
    counts = [-(-x // size) for x in lens]
    pool = Pool(fmt, sum(counts) + extra, size, heads, rng if stale else None)
    table = tables(rng, counts, pool.pages, max(counts + [1]) + 1)
    for s, n in enumerate(lens):
        for x in "kv":
            pool.append(x, table[s], 0, rows_of(rng, n, heads, 0.7))
    return pool, table


# -------------------------------------------------------------------------------------------------------------- append

@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("size,heads,apart", [(16, 2, 0), (32, 1, 0), (64, 5, 3), (128, 2, 0)])
def test_append_and_read(ctx, cv, cuda, fmt, size, heads, apart):
    torch, rng = cuda, np.random.default_rng(size + fmt)
    L = [0, 1, 15, 16, 17, 31, 100, 7, 128, 40]
    n = [1, 16, 17, 40, 0, 33, 1, 25, 130, 9]
    most = max(n) + 2
    counts = [-(-(a + b) // size) for a, b in zip(L, n)]
    host = Pool(fmt, sum(counts) + 2, size, heads, rng)
    table = tables(rng, counts, host.pages, max(counts) + 1)
    for s, a in enumerate(L):
        for x in "kv":
            host.append(x, table[s], 0, rows_of(rng, a, heads))
    pool = host.device(torch, cv, apart)
    new = {x: np.stack([rows_of(rng, most, heads) for _ in L]) for x in "kv"}
    for x in "kv":  # what the formats cannot hold
        new[x][3, 5, 0, 7], new[x][3, 6, 0, 9], new[x][3, 7, 0, 11] = np.inf, -np.inf, np.nan
        new[x][1, :, 0] = 0.0
        new[x][5, :16, 0] *= 1e-39
        new[x][7, 2] = np.nan
        new[x][8, 3] *= 1e30
        for s, a in enumerate(L):
            host.append(x, table[s], a, new[x][s, :n[s]])
    wide = torch.zeros((len(L), most, 2, heads * D + 4), device="cuda")  # rows apart
    for i, x in enumerate("kv"):
        wide[:, :, i, :heads * D] = torch.from_numpy(new[x].reshape(len(L), most, -1)).cuda()
    k, v = wide[:, :, 0, :heads * D], wide[:, :, 1, :heads * D]
    cv.PageAppender(ctx, pool, k, v, ints(torch, table), ints(torch, L), n_new=ints(torch, n))()
    host.same(pool)
    # read back: whole sequences, and from odd places
    for first in ([0] * len(L), [a // 3 for a in L]):
        ends = [a + b for a, b in zip(L, n)]
        count = [e - f for e, f in zip(ends, first)]
        got = torch.full((2, len(L), max(count) + 1, heads * D), 9.0, device="cuda")
        cv.PageReader(ctx, pool, got[0], got[1], ints(torch, table), first=ints(torch, first), n_rows=ints(torch, count))()
        for i, x in enumerate("kv"):
            for s in range(len(L)):
                want = host.rows(x, table[s], ends[s])[first[s]:].reshape(count[s], -1).astype(np.float32)
                assert np.array_equal(got[i, s, :count[s]].cpu().numpy(), want), (x, s)
                assert not got[i, s, count[s]:].any()


@pytest.mark.parametrize("fmt", [0, 1])
def test_append_token_by_token(ctx, cv, cuda, fmt):
    """Scales grow on the way: every earlier row is rounded anew each time."""
    torch, rng = cuda, np.random.default_rng(5 + fmt)
    heads, size, S = 2, 32, 3
    host = Pool(fmt, 8, size, heads, rng)
    table = tables(rng, [2] * S, 8, 2)
    pool, at = host.device(torch, cv), np.array([0, 3, 14])
    for s in range(S):
        for x in "kv":
            host.append(x, table[s], 0, rows_of(rng, at[s], heads))
    pool = host.device(torch, cv)
    for _ in range(40):
        new = {x: np.stack([rows_of(rng, 1, heads, 3.0) for _ in range(S)]) for x in "kv"}
        cv.PageAppender(ctx, pool, *(torch.from_numpy(new[x].reshape(S, 1, -1)).cuda() for x in "kv"), ints(torch, table), ints(torch, at))()
        for s in range(S):
            for x in "kv":
                host.append(x, table[s], at[s], new[x][s])
        at += 1
    host.same(pool)


@pytest.mark.parametrize("fmt", [0, 1])
def test_append_next_to_borders(ctx, cv, cuda, fmt):
    """Values one rounding away from the middle between two codes, under scales that are no powers of two."""
    torch, rng = cuda, np.random.default_rng(9 + fmt)
    heads, size, S = 4, 128, 4
    host = Pool(fmt, 4, size, heads, rng)
    table = tables(rng, [1] * S, 4, 1)
    grid = np.arange(127.0) if fmt == 0 else np.unique(np.abs(host_values(fmt)))
    new = {}
    for x in "kv":
        top = np.exp(rng.uniform(-3, 3, (S, size // 16, 1, heads, 1))).astype(np.float32)
        scale = (top / np.float32(127 if fmt == 0 else 448)).astype(np.float64)
        i = rng.integers(0, len(grid) - 1, (S, size // 16, 16, heads, D))
        mid = ((grid[i] + grid[i + 1]) / 2 * scale).astype(np.float32)
        step = rng.integers(-1, 2, mid.shape)
        mid = np.where(step < 0, np.nextafter(mid, np.float32(0)), np.where(step > 0, np.nextafter(mid, np.float32(np.inf)), mid))
        mid *= rng.choice([-1, 1], mid.shape).astype(np.float32)
        mid[:, :, 3, :, 5] = top[:, :, 0, :, 0]  # the block's largest
        new[x] = mid.reshape(S, size, heads, D).astype(np.float32)
        for s in range(S):
            host.append(x, table[s], 0, new[x][s])
    pool = Pool(fmt, 4, size, heads, rng).device(torch, cv)
    cv.PageAppender(ctx, pool, *(torch.from_numpy(new[x].reshape(S, size, -1)).cuda() for x in "kv"), ints(torch, table), ints(torch, [0] * S))()
    host.same(pool)


def host_values(fmt):
    from paged_reference import VALUES
    return VALUES[fmt][np.arange(127)]


def test_append_refuses_what_it_cannot_place(ctx, cv, cuda):
    """Sequences out of range, pages out of range and shared pages are skipped and recorded; the others go in."""
    torch, rng = cuda, np.random.default_rng(3)
    heads, size, S = 2, 16, 6
    host = Pool(0, 12, size, heads, rng)
    table = tables(rng, [2] * S, 12, 2)
    L, n = [0, 30, -1, 0, 20, 5], [3, 3, 1, -2, 2, 40]
    table[4, 1] = 12  # out of range
    new = {x: np.stack([rows_of(rng, 41, heads) for _ in range(S)]) for x in "kv"}
    pool = host.device(torch, cv)
    args = [torch.from_numpy(new[x].reshape(S, 41, -1)).cuda() for x in "kv"]
    with pytest.raises(cv.CvattnError, match="LENGTH"):
        cv.PageAppender(ctx, pool, *args, ints(torch, table), ints(torch, L), n_new=ints(torch, n))()
    wide = np.concatenate([table, np.full((S, 1), -1, np.int32)], 1)
    cv.PageAppender(ctx, pool, *args, ints(torch, wide), ints(torch, L), n_new=ints(torch, n))()
    assert ctx.sync_status()[0] == 6
    for x in "kv":
        host.append(x, table[0], 0, new[x][0, :3])
        host.append(x, list(table[1]) + [0], 30, new[x][1, :2])  # its third row has no page
        host.append(x, table[5], 5, new[x][5, :27])              # what lies on its two pages
    host.same(pool)
    refs = np.ones(12, np.int32)
    refs[table[0, 0]] = 2
    cv.PageAppender(ctx, pool, *args, ints(torch, wide), ints(torch, [3] * S), n_new=ints(torch, [1, 1, 0, 0, 0, 0]), refs=ints(torch, refs))()
    assert ctx.sync_status() == (6, 5)
    for x in "kv":
        host.append(x, table[1], 3, new[x][1, :1])
    host.same(pool)


# ----------------------------------------------------------------------------------------------------------- attention

def check_attention(cv, ctx, torch, rng, host, table, L, n, Hq, max_q, apart=0, q_apart=0, max_kv_len=None, scale=None):
    S = len(L)
    q = rng.standard_normal((S, max_q, Hq, D)).astype(np.float32)
    pool = host.device(torch, cv, apart)
    qd = torch.zeros((S, max_q, Hq * D + q_apart), device="cuda")
    qd[..., :Hq * D] = torch.from_numpy(q.reshape(S, max_q, -1)).cuda()
    qd = qd[..., :Hq * D].unflatten(-1, (Hq, D)) if q_apart else qd.view(S, max_q, Hq, D)
    out, lse = torch.full((S, max_q, Hq, D), 7.0, device="cuda"), torch.full((S, max_q, Hq), 7.0, device="cuda")
    plan = cv.PagedAttention(ctx, pool, qd, out, ints(torch, table), ints(torch, L), max_kv_len, lse=lse, n_q=ints(torch, n), scale=scale)
    plan()
    out, lse = out.cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64)
    c = D ** -0.5 if scale is None else scale
    for s in range(S):
        k, v = host.rows("k", table[s], L[s]), host.rows("v", table[s], L[s])
        want, wl = attention(q[s], k, v, n[s], c)
        # Scores are sums of 64 products, formed in f32 with truncating adds: off by 2^-21 of the sum of magnitudes, in which
        # the exponential's argument and ex2 (2^-22) have room too.  A weight is off by that much, the weighted mean by twice,
        # and the joins of parts round a few times more: 2^-19 (1 + magnitudes) of the largest value.
        size = abs(c) * np.einsum("nhd,lhd->nhl", np.abs(q[s]), np.repeat(np.nan_to_num(np.abs(k)), Hq // host.heads, 1)).max(initial=0.0)
        far = 2.0 ** -19 * (1 + size)
        assert np.array_equal(np.isinf(lse[s]), np.isinf(wl)), s
        assert np.all(np.abs(out[s] - want) <= far * np.nan_to_num(np.abs(v)).max(initial=1e-30)), (s, np.abs(out[s] - want).max())
        assert not out[s][np.isinf(wl)].any()
        fine = np.isfinite(wl)
        assert np.all(np.abs(lse[s][fine] - wl[fine]) <= far + 2.0 ** -22 * np.abs(wl[fine])), s
    return plan


LENS = [0, 1, 2, 15, 16, 17, 33, 64, 127, 128, 129, 200, 300, 511]


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("Hq,heads", [(14, 2), (8, 1), (5, 5), (6, 2)])
@pytest.mark.parametrize("max_q", [1, 2, 3])
def test_attention_of_few_rows(ctx, cv, cuda, fmt, Hq, heads, max_q):
    rng = np.random.default_rng(Hq + 10 * max_q + fmt)
    host, table = filled(rng, fmt, LENS, (16, 32, 64, 128)[(Hq + max_q) % 4], heads)
    n = [max_q - s % (max_q + 1) if max_q > 1 else int(s != 7) for s in range(len(LENS))]
    check_attention(cv, ctx, cuda, rng, host, table, LENS, n, Hq, max_q)


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("Hq,heads,max_q", [(14, 2, 5), (14, 2, 16), (16, 16, 20), (8, 1, 40), (14, 2, 70), (5, 5, 260)])
def test_attention_of_many_rows(ctx, cv, cuda, fmt, Hq, heads, max_q):
    rng = np.random.default_rng(Hq * max_q + fmt)
    lens = [300, 0, 129, 17, 640, 128]
    host, table = filled(rng, fmt, lens, (16, 32, 64, 128)[max_q % 4], heads)
    n = [max_q, max_q, max_q - 1, max_q, max_q // 2, 0]  # (more rows than positions: the first see nothing)
    check_attention(cv, ctx, cuda, rng, host, table, lens, n, Hq, max_q)


@pytest.mark.parametrize("fmt,size,max_q", [(0, 16, 1), (1, 128, 1), (0, 64, 9), (1, 32, 33)])
def test_attention_of_long_contexts(ctx, cv, cuda, fmt, size, max_q):
    rng = np.random.default_rng(size)
    lens = [5003, 4096]
    host, table = filled(rng, fmt, lens, size, 2, stale=False)
    check_attention(cv, ctx, cuda, rng, host, table, lens, [max_q] * 2, 14, max_q)


@pytest.mark.parametrize("fmt", [0, 1])
def test_attention_of_a_long_prompt(ctx, cv, cuda, fmt):
    """Many tiles of rows per sequence, behind positions of their own and without."""
    rng = np.random.default_rng(fmt)
    lens = [700, 131, 900]
    host, table = filled(rng, fmt, lens, 64, 2)
    check_attention(cv, ctx, cuda, rng, host, table, lens, [700, 131, 650], 14, 700)


@pytest.mark.parametrize("fmt", [0, 1])
def test_attention_of_many_short_sequences(ctx, cv, cuda, fmt):
    """A dozen sequences' heads, one or two tiles each, follow one another on an SM; empty ones among them."""
    rng = np.random.default_rng(fmt)
    lens = rng.integers(0, 300, 100)
    lens[::9] = 0
    host, table = filled(rng, fmt, lens.tolist(), 32, 16)
    check_attention(cv, ctx, cuda, rng, host, table, lens, np.minimum(lens, rng.integers(0, 101, 100)), 16, 100)


@pytest.mark.parametrize("fmt", [0, 1])
def test_attention_of_more_sequences_than_one_list_holds(ctx, cv, cuda, fmt):
    rng = np.random.default_rng(fmt)
    lens = rng.integers(0, 90, 1030)
    host, table = filled(rng, fmt, lens.tolist(), 16, 1)
    check_attention(cv, ctx, cuda, rng, host, table, lens, np.minimum(lens, rng.integers(0, 13, 1030)), 8, 12)


@pytest.mark.parametrize("max_q", [1, 40])
def test_attention_over_nothing(ctx, cv, cuda, max_q):
    """A bound of no positions at all."""
    rng = np.random.default_rng(0)
    host, table = filled(rng, 0, [0, 0], 16, 2)
    check_attention(cv, ctx, cuda, rng, host, table, [0, 0], [max_q, 0], 14, max_q, max_kv_len=0)


@pytest.mark.parametrize("max_q", [1, 12, 40])
def test_attention_over_strided_memory(ctx, cv, cuda, max_q):
    """Pages and query rows that lie apart, a table wider than it has to be, a scale of one's own, a bound above the lengths."""
    rng = np.random.default_rng(max_q)
    lens = [70, 1, 333]
    host, table = filled(rng, 1, lens, 32, 2)
    table = np.concatenate([table, np.full((3, 5), -1, np.int32)], 1)
    n = [max_q, 1, max_q]
    check_attention(cv, ctx, cuda, rng, host, table, lens, n, 14, max_q, apart=5, q_apart=12, max_kv_len=400, scale=0.3)
    check_attention(cv, ctx, cuda, rng, host, table, lens, n, 14, max_q, scale=-0.2)
    check_attention(cv, ctx, cuda, rng, host, table, lens, n, 14, max_q, scale=0.0)


@pytest.mark.parametrize("max_q", [1, 3, 12, 40])
@pytest.mark.parametrize("fmt", [0, 1])
def test_attention_over_blocks_of_differing_size(ctx, cv, cuda, fmt, max_q):
    """Neighbouring blocks whose scales are far apart, and blocks of zeros."""
    rng = np.random.default_rng(max_q)
    lens = [400, 130]
    host, table = filled(rng, fmt, lens, 64, 2)
    for s, n in enumerate(lens):
        for b in range(-(-n // 16)):
            page, part = table[s, b // 4], b % 4
            host.scales["v"][page, :, part] *= (1.0, 1e-3, 1e3, 0.0, 1e-6)[b % 5]
            host.scales["k"][page, :, part] *= (1.0, 0.1, 0.0, 3.0)[b % 4]
    check_attention(cv, ctx, cuda, rng, host, table, lens, [max_q] * 2, 14, max_q)


@pytest.mark.parametrize("max_q", [1, 12, 40])
def test_pages_out_of_range_are_left_out(ctx, cv, cuda, max_q):
    rng = np.random.default_rng(max_q)
    lens = [200, 100, 64]
    host, table = filled(rng, 0, lens, 16, 2)
    table[0, 3], table[0, 7], table[0, 12] = -1, host.pages, 2 ** 30
    table[2, :4] = -5
    check_attention(cv, ctx, cuda, rng, host, table, lens, [max_q] * 3, 14, max_q)
    assert ctx.sync_status() == (6, 4)


@pytest.mark.parametrize("max_q", [1, 12, 40])
def test_lengths_out_of_range_give_empty_rows(ctx, cv, cuda, max_q):
    torch, rng = cuda, np.random.default_rng(max_q)
    lens = [70, 70, 70, 70, 70]
    host, table = filled(rng, 0, lens, 16, 2)
    pool, q = host.device(torch, cv), torch.randn(5, max_q, 14, D, device="cuda")
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:3], 7.0, device="cuda")
    given, n = [-1, 81, 70, 70, 70], [max_q, max_q, max_q + 1, -1, max_q]
    cv.PagedAttention(ctx, pool, q, out, ints(torch, table), ints(torch, given), 80, lse=lse, n_q=ints(torch, n))()
    assert ctx.sync_status() == (6, 2)
    assert not out[:4].any() and bool((lse[:4] == -np.inf).all())
    want, wl = attention(q[4].cpu().numpy(), host.rows("k", table[4], 70), host.rows("v", table[4], 70), max_q, D ** -0.5)
    assert np.abs(out[4].cpu().numpy() - want).max() < 1e-4


@pytest.mark.parametrize("max_q", [1, 40])
def test_offsets_past_32_bits(ctx, cv, cuda, max_q):
    """Pages that lie 2^31 bytes apart."""
    torch, rng = cuda, np.random.default_rng(max_q)
    lens = [100]
    host, table = filled(rng, 0, lens, 64, 2, extra=1)
    table[0, :2] = [0, 2]
    host = Pool(0, 3, 64, 2)
    for x in "kv":
        host.append(x, table[0], 0, rows_of(rng, 100, 2, 0.7))
    small = host.device(torch, cv)
    far = 1 << 31
    k, v = (torch.empty(2 * far + 8192, dtype=torch.uint8, device="cuda") for _ in "kv")
    big = [t.as_strided(small.k.shape, (far, 4096, 1)) for t in (k, v)]
    pool = cv.PagePool(*big, torch.full_like(small.k_scale, np.nan), torch.full_like(small.v_scale, np.nan), 0)
    rows = [torch.from_numpy(host.rows(x, table[0], 100).astype(np.float32).reshape(1, 100, -1)).cuda() for x in "kv"]
    cv.PageAppender(ctx, pool, *rows, ints(torch, table), ints(torch, [0]))()
    back = torch.empty((2, 1, 100, 128), device="cuda")
    cv.PageReader(ctx, pool, back[0], back[1], ints(torch, table))()
    # rounded once more under a scale that was rounded itself: at most a step of 1/127 of a block's largest
    for got, want in zip(back, rows):
        assert float((got - want).abs().max()) <= float(want.abs().max()) / 127
    q = torch.randn(1, max_q, 14, D, device="cuda")
    out, want = torch.empty_like(q), torch.empty_like(q)
    near = cv.PagePool(*(t.contiguous() for t in big), pool.k_scale, pool.v_scale, 0)
    cv.PagedAttention(ctx, pool, q, out, ints(torch, table), ints(torch, [100]))()
    cv.PagedAttention(ctx, near, q, want, ints(torch, table), ints(torch, [100]))()
    assert torch.equal(out, want) and bool(out.any())


@pytest.mark.parametrize("max_q", [1, 12, 64])
def test_attention_repeats_itself_and_replays(ctx, cv, cuda, max_q):
    """The same bits every time, in a graph and on another stream too; a replayed graph reads the lengths of its time."""
    torch, rng = cuda, np.random.default_rng(max_q)
    lens = [900, 333, 64, 1500]
    host, table = filled(rng, 1, lens, 64, 2)
    pool, q = host.device(torch, cv), torch.randn(4, max_q, 14, D, device="cuda")
    t, L = ints(torch, table), ints(torch, lens)
    make = lambda: cv.PagedAttention(ctx, pool, q, torch.empty_like(q), t, L, lse=torch.empty(q.shape[:3], device="cuda"))  # noqa: E731
    a, b, c = make(), make(), make()
    a()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    b(side)
    a()
    torch.cuda.synchronize()
    out = lambda x: x._keep[2]  # noqa: E731
    assert torch.equal(out(a), out(b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c()
        c()
    graph.replay()
    assert torch.equal(out(a), out(c))
    L.copy_(ints(torch, [64, 64, 64, 100]))
    graph.replay()
    a()
    assert torch.equal(out(a), out(c))
