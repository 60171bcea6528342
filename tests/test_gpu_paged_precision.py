"""GPU: paged attention where value scales and scores are far apart, held to each row's own sums of p |v|.

Bounds, M being the largest code (127 or 448), s_j the scale of a position's values, size the largest sum |scale| |q| |k| of a row:
  scores   sums of 64 products with truncating adds, 2^-21 size; ex2 2^-22: a weight is off by 2^-21 (1 + size), the mean by twice
  sums     16 truncating adds in a tile of 128 (2^-23 each), tiles and joins in f32: 2^-19
           together below 2^-18 (1 + size) of the row's sum of p |v|, dim by dim
  tcgen05  p s is kept in f16 hi + lo under a power of two: 2^-22 of itself (counted above) or 2^-27.5 of the row's largest, anew for
           each change of that power inside a tile, three at most, times a code of up to M: 2^-25 M max(p s) for each position
  mma.sync p is kept so: 2^-22 of itself or 2^-32 of the row's largest, times s_j and a code of up to M: 2^-31 M max(p) sum(s_j)
"""
from __future__ import annotations

import numpy as np
import pytest

from paged_reference import D, Pool
from test_gpu_paged_cache import filled, ints

pytestmark = pytest.mark.gpu

MOST = {0: 127.0, 1: 448.0}


def on_tcgen05(cv, S, max_q, max_kv_len, Hq, heads):
    """Which kernel a call takes: the tcgen05 kernel's workspace has two parts of 128 rows for each of its CTAs."""
    row_tiles = -(-max_q * (Hq // heads) // 128)
    units, tiles = S * heads * row_tiles, S * heads * row_tiles * -(-max_kv_len // 128)
    own = -(-(S + 1) * 4 // 256) * 256 + 2 * min(148, tiles + 4 * units) * 128 * 66 * 4
    return cv.paged_attention_workspace_size(S, max_q, max_kv_len, Hq, heads) == own


def sums(q, k, v, s, see, scale):
    """out, sum p |v|, max p s, max p x sum s, size of rows q [n, Hq, D] of which row i sees see[i] positions; k, v [L, H, D], s [L, H]."""
    n, Hq = q.shape[:2]
    G = Hq // k.shape[1]
    out, most = np.zeros((n, Hq, D)), np.zeros((n, Hq, D))
    top, all_s, size = np.zeros((n, Hq)), np.zeros((n, Hq)), np.zeros((n, Hq))
    for h in range(Hq):
        x = scale * (q[:, h].astype(np.float64) @ k[:, h // G].T)
        x[np.arange(len(k))[None] >= np.asarray(see)[:, None]] = -np.inf
        seen = np.isfinite(x)
        x = np.exp(x - np.where(seen.any(1), x.max(1, initial=-np.inf), 0.0)[:, None])
        p = x / np.maximum(x.sum(1), 1e-300)[:, None]
        out[:, h], most[:, h] = p @ v[:, h // G], p @ np.abs(v[:, h // G])
        top[:, h] = (p * s[None, :, h // G]).max(1, initial=0.0)
        all_s[:, h] = p.max(1, initial=0.0) * (seen * s[None, :, h // G]).sum(1)
        size[:, h] = (abs(scale) * (np.abs(q[:, h].astype(np.float64)) @ np.abs(k[:, h // G]).T) * seen).max(1, initial=0.0)
    return out, most, top, all_s, size


def scales_of(host, table, L):
    """[L, heads]: the scale of each position's values."""
    j = np.arange(L)
    return np.stack([host.scales["v"][table[i // host.size], :, i % host.size // 16] for i in j]).astype(np.float64)


def hold(cv, ctx, torch, host, table, lens, q, scale, tcgen05):
    """Every row of every sequence (all max_q of them) within its bound."""
    S, n, Hq = q.shape[:3]
    assert on_tcgen05(cv, S, n, max(lens), Hq, host.heads) == tcgen05
    out = torch.empty(q.shape, device="cuda")
    cv.PagedAttention(ctx, host.device(torch, cv), torch.from_numpy(q).cuda(), out, ints(torch, table), ints(torch, lens), max(lens), scale=scale)()
    out = out.cpu().numpy().astype(np.float64)
    worst = 0.0
    for s, L in enumerate(lens):
        see = np.clip(L - n + np.arange(n) + 1, 0, L)
        want, most, top, all_s, size = sums(q[s], host.rows("k", table[s], L), host.rows("v", table[s], L), scales_of(host, table[s], L), see, scale)
        floor = MOST[host.fmt] * (L * 2.0 ** -25 * top if tcgen05 else 2.0 ** -31 * all_s)
        far = 2.0 ** -18 * (1 + size[..., None]) * most + floor[..., None]
        off = np.abs(out[s] - want)
        assert np.isfinite(out[s]).all(), s
        worst = max(worst, (off / np.maximum(far, 1e-300)).max())
    assert worst <= 1.0, worst


# (sequences, rows of each, query heads, KV heads, tcgen05)
SHAPES = [(3, 4, 14, 2, False), (2, 20, 8, 1, False), (1, 17, 5, 5, False), (24, 54, 14, 2, True), (16, 120, 16, 16, True)]


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("S,n,Hq,heads,tcgen05", SHAPES)
@pytest.mark.parametrize("r", [20, 40, 90])
def test_what_a_row_does_not_see_costs_it_nothing(ctx, cv, cuda, fmt, S, n, Hq, heads, tcgen05, r):
    """Values 2^r larger than all before them, in the block of a sequence's last positions: rows before it keep their precision."""
    rng = np.random.default_rng(n + r)
    lens = [int(x) for x in rng.integers(n, 250, S)]
    lens[0], lens[-1] = 250 if S > 1 else 129, max(n, 129)
    host, table = filled(rng, fmt, lens, 32, heads)
    for s, L in enumerate(lens):
        b = (L - 1) // 16
        host.scales["v"][table[s, b // 2], :, b % 2] *= np.float32(2.0 ** r)
    q = rng.standard_normal((S, n, Hq, D)).astype(np.float32)
    hold(cv, ctx, cuda, host, table, lens, q, 0.125, tcgen05)


def steered(rng, fmt, lens, heads, Hq, n, level, spread=0.0):
    """A pool and queries whose scores are level[s][j] (natural units), about: keys along one direction, queries along the same."""
    most = max(lens)
    host = Pool(fmt, sum(-(-x // 32) for x in lens) + 1, 32, heads, rng)
    order, table, at = rng.permutation(host.pages), np.full((len(lens), -(-most // 32)), -1, np.int32), 0
    way = rng.choice([-1.0, 1.0], (heads, D))
    for s, L in enumerate(lens):
        m = -(-L // 32)
        table[s, :m] = order[at:at + m]
        at += m
        # blocks hold one level each, so that a key's direction is rounded alike
        k = level[s][:L, None, None] * way[None] / D + spread * rng.standard_normal((L, heads, D))
        host.append("k", table[s], 0, k.astype(np.float32))
        host.append("v", table[s], 0, rng.standard_normal((L, heads, D)).astype(np.float32))
    q = np.repeat(way, Hq // heads, 0)[None, None] * (1 + 0.01 * rng.standard_normal((len(lens), n, Hq, 1)))
    return host, table, q.astype(np.float32)


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("S,n,Hq,heads,tcgen05", SHAPES)
@pytest.mark.parametrize("r", [-28, 12, 20, 28])
def test_low_scores_over_large_values(ctx, cv, cuda, fmt, S, n, Hq, heads, tcgen05, r):
    """Blocks whose weights are 2^-r of the largest and whose values are 2^r larger weigh as much as the others (r < 0: the other way
    round, the first of them are followed by far higher scores over far smaller values)."""
    rng = np.random.default_rng(n + r + 100)
    lens = [int(x) for x in rng.integers(n + 1, 300, S)]
    block = np.arange(320) // 16
    kind = [rng.integers(0, 2, 20) if r > 0 else np.sort(rng.integers(0, 2, 20)) for _ in lens]
    for x in kind:
        x[:2] = [0, 1] if r > 0 else [0, 0]
    gap = abs(r) * np.log(2.0)
    level = [np.where(x[block] == (1 if r > 0 else 0), -gap, 0.0) + 0.2 for x in kind]
    host, table, q = steered(rng, fmt, lens, heads, Hq, n, level)
    for s, L in enumerate(lens):
        for b in range(-(-L // 16)):
            if kind[s][b] == (1 if r > 0 else 0):
                host.scales["v"][table[s, b // 2], :, b % 2] *= np.float32(2.0 ** abs(r))
    hold(cv, ctx, cuda, host, table, lens, q, 1.0, tcgen05)


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("S,n,Hq,heads,tcgen05", [(3, 2, 14, 2, False), (2, 20, 8, 1, False), (40, 128, 16, 16, True)])
@pytest.mark.parametrize("r", [102, -100])
def test_values_near_the_ends_of_f32(ctx, cv, cuda, fmt, S, n, Hq, heads, tcgen05, r):
    """Scales near 2^r, and one position whose weight is 2^7.5 times that of the others: sums stay finite and as precise as any."""
    rng = np.random.default_rng(n)
    lens = [48] * S
    level = [np.zeros(48) for _ in lens]
    for x in level:
        x[rng.integers(32, 48 - min(n, 8))] = 7.5 * np.log(2.0)
    host, table, q = steered(rng, fmt, lens, heads, Hq, n, level)
    for x in host.scales.values():
        x[np.isnan(x)] = 0.0
    host.scales["v"] *= np.float32(2.0 ** r) / np.exp2(np.floor(np.log2(host.scales["v"].max())))
    # weights up to 2^15 times values below 2^(r + 1) M, and 47 more of 2^7.5: below 2^(r + 1) M 2^15.3
    assert (2.0 ** (r + 1)) * MOST[fmt] * 2.0 ** 15.3 < 2.0 ** 128
    hold(cv, ctx, cuda, host, table, lens, q, 1.0, tcgen05)


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("S,n,Hq,heads,tcgen05", SHAPES)
@pytest.mark.parametrize("r", [117, 112, -112])
def test_queries_near_the_ends_of_f32(ctx, cv, cuda, fmt, S, n, Hq, heads, tcgen05, r):
    """Queries 2^r larger over keys 2^r smaller give what they give at ordinary sizes."""
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(n, 250, S)]
    lens[0] = max(lens[0], 129)
    host, table = filled(rng, fmt, lens, 32, heads)
    host.scales["k"] *= np.float32(2.0 ** -r)
    assert np.nanmin(np.where(host.scales["k"] > 0, host.scales["k"], np.nan)) >= 2.0 ** -126
    q = rng.standard_normal((S, n, Hq, D)).astype(np.float32)
    q[:, :, 0] *= np.float32(2.0 ** -6)  # (a row whose largest value is smaller)
    hold(cv, ctx, cuda, host, table, lens, q * np.float32(2.0 ** r), 0.125, tcgen05)
