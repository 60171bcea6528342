"""CPU: which of its two kernels paged attention takes, by the size of the workspace that it asks for."""
from __future__ import annotations

import cvattn as cv
from test_gpu_paged_precision import on_tcgen05


def test_which_kernel():
    """One token a sequence and little work: mma.sync; a change of the rule shows here, beside the sizes that it was made for."""
    few = [(64, 1, 4096, 14, 2), (1, 1, 65536, 14, 2), (16, 2, 8192, 14, 2), (3, 40, 400, 14, 2), (1, 700, 100, 14, 2), (1030, 100, 90, 8, 1)]
    many = [(16, 16, 8192, 14, 2), (4, 512, 2501, 16, 16), (3, 100, 400, 14, 2), (8, 100, 224, 14, 2), (60, 73, 128, 14, 2), (100, 100, 320, 16, 16)]
    assert not any(on_tcgen05(cv, *x) for x in few) and all(on_tcgen05(cv, *x) for x in many)
