"""GPU: which positions an eviction keeps where the scores leave it to the slots, and in lists longer than a CTA keeps keys of."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_bounded_cache import run_evict

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [0, 1])
@pytest.mark.parametrize("in_place", [False, True])
def test_nan_counts_as_minus_infinity(ctx, cv, cuda, oracle, first, in_place):
    """They tie, in either order of the slots: the lower slots stay, whichever of the two they hold."""
    def alternate(rng, shape):
        x = np.where(np.arange(shape[-1]) % 2 == first, np.float32(np.nan), np.float32(-np.inf))
        return np.broadcast_to(x, shape).copy()

    run_evict(ctx, cv, cuda, oracle, "q8_0", "q4_0", 2, [80, 41], 40, make=alternate, kept=[0, 0], in_place=in_place)


@pytest.mark.parametrize("low", [np.nan, -np.inf])
def test_numbers_rank_above_both(ctx, cv, cuda, oracle, low):
    def make(rng, shape):
        x = np.full(shape, low, dtype=np.float32)
        x[..., 50:] = np.float32(-3.4e38)
        return x

    run_evict(ctx, cv, cuda, oracle, "q8_0", "q4_0", 2, [80], 40, make=make, kept=[0])


@pytest.mark.parametrize("L,budget", [(40960, 40000), (40961, 40001), (43000, 300), (43000, 42990)])
def test_evict_more_slots_than_a_cta_keeps_keys_of(ctx, cv, cuda, oracle, L, budget):
    """Slots from 40960 on have their keys formed again at every step; ties fall on both sides of that line."""
    def levels(rng, shape):
        return rng.integers(0, 40, shape) * 0.125

    run_evict(ctx, cv, cuda, oracle, "q8_0", "q4_0", 1, [L], budget, layers=1, sink=3, recent=17, make=levels)
