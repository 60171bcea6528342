"""GPU: assignment and compaction whose books take more than one CTA's shared memory (about 12800 pages, or as many entries)."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_pages import check, ints, parts, pools, random_state

pytestmark = pytest.mark.gpu

# sequences, entries of each, pages: clusters of 2, 4 and 8 CTAs (4096 pages or entries each)
SIZES = [(8192, 1, 8000), (2600, 3, 14000), (500, 40, 20000), (60, 30, 60000)]


@pytest.mark.parametrize("S,width,pages", SIZES)
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(ctx, cv, cuda, S, width, pages, in_place):
    """Shared pages, entries out of range, empty sequences."""
    torch, rng = cuda, np.random.default_rng(S)
    table, _, held = random_state(rng, S, 16, pages, width, True)
    table[::7, -1] = pages + 5  # out of range: dropped
    made = pools(torch, cv, 2, pages, 16, heads=1)
    before = [[t.clone() for t in parts(x)] for x in made]
    t = ints(torch, table)
    out = t if in_place else torch.empty_like(t)
    refs = torch.empty(pages, dtype=torch.int32, device="cuda")
    c = cv.PageCompactor(ctx, made, t, table_out=out, refs=refs)
    c()
    live = np.unique(table[(table >= 0) & (table < pages)])
    n = len(live)
    to = np.arange(pages)
    gone = live[live >= n]
    to[gone] = np.setdiff1d(np.arange(n), live)
    want = np.where((table >= 0) & (table < pages), to[table.clip(0, pages - 1)], -1)
    assert len(gone) > 100 and int(c.n_live) == n
    assert np.array_equal(out.cpu().numpy(), want)
    assert np.array_equal(refs.cpu().numpy(), np.bincount(want[want >= 0], minlength=pages))
    a, b = ints(torch, gone).long(), ints(torch, to[gone]).long()
    for x, old in zip(made, before):
        for now, was in zip(parts(x), old):
            was[b] = was[a]
            assert torch.equal(now, was)


@pytest.mark.parametrize("S,width,pages", SIZES)
def test_assign(ctx, cv, cuda, S, width, pages):
    rng = np.random.default_rng(S + 1)
    table, L, _ = random_state(rng, S, 16, pages, width, True)
    src = rng.integers(0, S, S)
    keep = np.array([int(rng.integers(0, L[x] + 1)) if rng.random() < 0.4 else int(L[x]) for x in src])
    need = np.minimum(keep + rng.integers(-5, 30, S), width * 16).clip(0)
    check(cv, ctx, cuda, table, src, keep, need, 16, pages, layers=1, heads=1, in_place=bool(S % 3))
