"""CPU: what the Python launchers of tree attention, scores and eviction check and keep before they launch anything."""
from __future__ import annotations

import contextlib

import pytest
import torch

import cvattn as cv

D = 64


class Device(torch.Tensor):
    """A host tensor that says it is a CUDA tensor: launchers can be built on it, not called."""
    is_cuda = property(lambda self: True)


def on_device(t):
    return t.as_subclass(Device)


@pytest.fixture
def streams(monkeypatch):
    """The streams that are current, innermost last."""
    now = []

    @contextlib.contextmanager
    def enter(stream):
        now.append(stream)
        yield
        now.pop()

    monkeypatch.setattr(torch.cuda, "stream", enter)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: "current")
    return now


def test_one_shot_calls_allocate_on_the_stream_that_they_run_on(monkeypatch, streams):
    built, called, recorded = [], [], []

    class Plan:
        def __init__(self, *args, **kw):
            built.append(list(streams))

        def __call__(self, stream=None):
            called.append(stream)

    monkeypatch.setattr(cv, "TreeDecoder", Plan)
    monkeypatch.setattr(cv, "KVEvictor", Plan)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: recorded.append(s))
    q = torch.zeros(1, 2, 14, D)
    cv.tree_decode(None, q, None, None, None, None, None, 5, stream="side")
    cv.tree_decode(None, q, None, None, None, None, None, 5, out=torch.empty_like(q), stream="side")
    cv.kv_evict(None, None, None, None, None, None, None, None, 5, stream="side")
    assert built == [["side"]] * 3 and called == ["side"] * 3 and recorded == ["current"]
    cv.tree_decode(None, q, None, None, None, None, None, 5)
    cv.kv_evict(None, None, None, None, None, None, None, None, 5)
    assert built[3:] == [[], []] and called[3:] == [None, None] and recorded == ["current"]
