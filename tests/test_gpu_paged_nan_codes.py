"""GPU: pages that a caller has filled with all 256 bytes of OCP e4m3, of which 0x7f and 0xff are NaN."""
from __future__ import annotations

import numpy as np
import pytest

from paged_reference import BLOCK, D, PLACE

pytestmark = pytest.mark.gpu


def every_code(torch, x):
    """[BLOCK, D] codes, all 256 of them in each of four groups of rows, and a block's bytes in their order."""
    codes = (np.arange(BLOCK * D) % 256).astype(np.uint8).reshape(BLOCK, D)
    block = np.empty(BLOCK * D, np.uint8)
    block[PLACE[x]] = codes
    return codes, torch.from_numpy(block).cuda()


def test_read_gives_what_the_bytes_stand_for(ctx, cv, cuda):
    torch = cuda
    pool = cv.alloc_pages(cv.PAGE_E4M3, 2, 16, 1)
    pool.k_scale.fill_(0.375), pool.v_scale.fill_(3.0)
    want = {}
    for x in "kv":
        codes, block = every_code(torch, x)
        getattr(pool, x)[1, 0] = block
        want[x] = torch.from_numpy(codes).view(torch.float8_e4m3fn).float() * (0.375 if x == "k" else 3.0)
    table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    k, v = (torch.empty(1, BLOCK, D, device="cuda") for _ in "kv")
    cv.PageReader(ctx, pool, k, v, table)()
    for got, x in ((k, "k"), (v, "v")):
        assert int(want[x].isnan().sum()) == 8
        torch.testing.assert_close(got[0].cpu(), want[x], rtol=0, atol=0, equal_nan=True)


def test_append_leaves_them_what_they_are(ctx, cv, cuda):
    """A larger row makes the block's scale grow by 8: codes are rounded anew to an eighth (exact but for the smallest), NaN stays NaN."""
    torch = cuda
    pool = cv.alloc_pages(cv.PAGE_E4M3, 1, 16, 1)
    want = {}
    for x in "kv":
        codes, block = every_code(torch, x)
        getattr(pool, x)[0, 0] = block
        getattr(pool, x + "_scale").fill_(1.0)
        want[x] = torch.from_numpy(codes).view(torch.float8_e4m3fn).float()
    table, at = torch.tensor([[0]], dtype=torch.int32, device="cuda"), torch.tensor([15], dtype=torch.int32, device="cuda")
    row = torch.full((1, 1, D), 448.0 * 8, device="cuda")
    cv.PageAppender(ctx, pool, row, row, table, at)()
    k, v = (torch.empty(1, BLOCK, D, device="cuda") for _ in "kv")
    cv.PageReader(ctx, pool, k, v, table)()
    for got, x in ((k, "k"), (v, "v")):
        assert float(getattr(pool, x + "_scale")) == 8.0
        again = (want[x] / 8).to(torch.float8_e4m3fn).float() * 8
        again[15] = 448.0 * 8
        torch.testing.assert_close(got[0].cpu(), again, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("n,S", [(1, 2), (4, 2), (40, 60)])
@pytest.mark.parametrize("x", ["k", "v"])
@pytest.mark.parametrize("where", [0, 94])
def test_attention_passes_them_on(ctx, cv, cuda, n, S, x, where):
    """Both kernels.  A NaN key reaches the rows that see it; a NaN value those at least, in its own dim alone; a sequence that ends
    before it nobody."""
    torch = cuda
    pool = cv.alloc_pages(cv.PAGE_E4M3, 6, 16, 2)
    rows = torch.randn(1, 96, 2 * D, device="cuda")
    table = torch.arange(6, dtype=torch.int32, device="cuda").view(1, 6)
    cv.PageAppender(ctx, pool, rows, rows, table, torch.zeros(1, dtype=torch.int32, device="cuda"))()
    getattr(pool, x)[where // 16, :, int(PLACE[x][where % 16, 5])] = 0xff
    lens = torch.full((S,), 96, dtype=torch.int32, device="cuda")
    lens[1::2] = 94
    q = torch.randn(S, n, 14, D, device="cuda")
    out = cv.paged_attention(ctx, pool, q, table.repeat(S, 1), lens)
    sees = lens[:, None] - n + torch.arange(n, device="cuda") >= where
    got = out.isnan()
    if x == "k":
        assert bool((got.all(-1) == sees[..., None]).all()) and bool((got.any(-1) == sees[..., None]).all())
    else:
        assert bool(got[..., 5][sees].all()) and not got[..., :5].any() and not got[..., 6:].any()
    if where:
        assert not got[1::2].any()
