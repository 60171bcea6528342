"""GPU: what a commit of drafts refuses before it launches anything."""
from __future__ import annotations

import pytest

from test_gpu_tree import D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shift", [0, 1, 5, -1])
def test_lengths_are_not_written_over_the_accepted_nodes(ctx, cv, cuda, shift):
    """Nodes index the drafts: a length in the place of one would be a row far outside of them."""
    torch = cuda
    (_, c), (_, d) = cv.alloc_kv(cv.Q8_0, 2, D, 64, 2), cv.alloc_kv(cv.Q8_0, 2, D, 4, 2)
    mem = torch.zeros(24, dtype=torch.int32, device="cuda")
    path, count, kl = mem[4:10].view(2, 3), mem[12:14], mem[14:16]
    for at, status in ((4 + shift, 1), (16, 0), (2, 0), (10, 0)):
        plan = cv.TreeCommitter(ctx, [c], [d], path, count, kl, mem[at:at + 2])
        if status:
            with pytest.raises(cv.CvattnError):
                plan()
        else:
            plan()
    assert not bool(mem.any())
