"""GPU: examples/speculative_decode.py, which runs draft verification, commit, scores and eviction together."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(cuda):
    path = Path(__file__).resolve().parent.parent / "examples" / "speculative_decode.py"
    spec = importlib.util.spec_from_file_location("speculative_decode", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_drafts_change_the_passes_and_not_the_tokens(example):
    one = example.generate(90, 128, 96, drafts=False)
    many = example.generate(90, 128, 96, drafts=True)
    assert one.tokens == many.tokens and len(many.tokens) == 90
    assert one.steps == 90 and many.steps <= 90
    assert one.evictions == many.evictions == 0


def test_a_full_cache_is_shrunk_and_decoding_goes_on(example):
    g = example.generate(300, 128, 64)
    assert g.evictions >= 300 // 128 and int(g.kv_len) <= 128 and int(g.total) >= 300
    kept = int(g.kept)
    assert kept == 64
    for layer in g.pos[:, 0, :, :kept].tolist():
        for head in layer:
            assert set(range(4)) <= set(head) and len(set(head)) == kept  # the first tokens stay, none is held twice
