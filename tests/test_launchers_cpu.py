"""CPU: what the Python launchers of tree attention, scores and eviction check and keep before they launch anything."""
from __future__ import annotations

import contextlib
import gc
import weakref

import pytest
import torch

import cvattn as cv

D = 64


class Device(torch.Tensor):
    """A host tensor that says it is a CUDA tensor: launchers can be built on it, not called."""
    is_cuda = property(lambda self: True)


def on_device(t):
    return t.as_subclass(Device)


class Handle:
    cuda_stream = 77


@pytest.mark.parametrize("missing", [None, "_cuda_getCurrentRawStream", "_cuda_getDevice"])
def test_the_current_stream_without_private_functions(monkeypatch, missing):
    """The handle comes from functions of torch that are not public where there are such, else from the stream object."""
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Handle)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 3, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 55 + device, raising=False)
    if missing:
        monkeypatch.delattr(torch._C, missing)
    assert cv._stream(None) == (77 if missing else 58)
    assert cv._stream(5) == 5 and cv._stream(Handle) == 77


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


def tree_arguments(S=2, n=4, L=640):
    made = {name: cv.kv_tensor(on_device(torch.zeros(S * rows * 136, dtype=torch.uint8)), cv.Q8_0, 2, D, rows, S)
            for name, rows in (("k", L), ("v", L), ("k_draft", n), ("v_draft", n))}
    q = on_device(torch.zeros(S, n, 14, D))
    return {**made, "q": q, "out": on_device(torch.zeros(S, n, 14, D)), "kv_len": on_device(torch.zeros(S, dtype=torch.int32)), "max_kv_len": L,
            "workspace": on_device(torch.zeros(cv.tree_decode_workspace_size(cv.Q8_0, cv.Q8_0, S, L, n, 14, 2), dtype=torch.uint8))}


def scores_arguments(S=2, n=4, L=64):
    return {"k": cv.kv_tensor(on_device(torch.zeros(S * L * 136, dtype=torch.uint8)), cv.Q8_0, 2, D, L, S), "q": on_device(torch.zeros(S, n, 14, D)),
            "lse": on_device(torch.zeros(S, n, 14)), "kv_len": on_device(torch.zeros(S, dtype=torch.int32)),
            "scores": on_device(torch.zeros(S, 2, L)), "scores_out": on_device(torch.zeros(S, 2, L))}


def evict_arguments(S=2, L=64, budget=32):
    kv = [[cv.kv_tensor(on_device(torch.zeros(S * L * 136, dtype=torch.uint8)), cv.Q8_0, 2, D, L, S)] for _ in "kv"]
    f = lambda: on_device(torch.zeros(1, S, 2, L))  # noqa: E731
    i = lambda: on_device(torch.zeros(1, S, 2, L, dtype=torch.int32))  # noqa: E731
    n = lambda: on_device(torch.zeros(S, dtype=torch.int32))  # noqa: E731
    need = int(cv.lib.cvattn_kv_evict_workspace_size(1, S, 2, L, budget))
    return {"k": kv[0], "v": kv[1], "scores": f(), "pos": i(), "kv_len": n(), "kept_len": n(), "n_tokens": n(), "budget": budget,
            "scores_out": f(), "pos_out": i(), "kv_len_out": n(), "workspace": on_device(torch.zeros(need, dtype=torch.uint8))}


LAUNCHERS = [(cv.TreeDecoder, tree_arguments), (cv.KVScorer, scores_arguments), (cv.KVEvictor, evict_arguments)]


def optional(cls, S=2):
    table = {name: on_device(torch.zeros(S, dtype=torch.int64)) for name in ("k_seq_ptrs", "v_seq_ptrs")}
    if cls is cv.TreeDecoder:
        return {**table, "lse": on_device(torch.zeros(S, 4, 14)), "mask": on_device(torch.zeros(S, 4, 1, dtype=torch.int32)),
                "n_nodes": on_device(torch.zeros(S, dtype=torch.int32))}
    if cls is cv.KVScorer:
        return {"k_seq_ptrs": table["k_seq_ptrs"], "rows": on_device(torch.zeros(S, 3, dtype=torch.int32)),
                "n_rows": on_device(torch.zeros(S, dtype=torch.int32))}
    return {}


@pytest.mark.parametrize("cls,arguments", LAUNCHERS, ids=lambda x: getattr(x, "__name__", None))
def test_host_tensors_are_refused(cls, arguments):
    """Every tensor whose address a kernel gets."""
    given = {**arguments(), **optional(cls)}
    cls(None, **given)
    tensors = [name for name, x in given.items() if isinstance(x, torch.Tensor)]
    assert len(tensors) >= 7
    for name in tensors:
        with pytest.raises(ValueError):
            cls(None, **{**given, name: given[name].as_subclass(torch.Tensor)})


@pytest.mark.parametrize("cls,arguments,name", [(cv.TreeDecoder, tree_arguments, "k_seq_ptrs"), (cv.TreeDecoder, tree_arguments, "v_seq_ptrs"),
                                                (cv.KVScorer, scores_arguments, "k_seq_ptrs")])
def test_tables_of_addresses_have_an_address_for_each_sequence(cls, arguments, name):
    for table in (torch.zeros(1, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int64)[::2]):
        with pytest.raises(ValueError):
            cls(None, **arguments(), **{name: on_device(table)})


def test_a_workspace_counts_its_bytes():
    for cls, arguments in (LAUNCHERS[0], LAUNCHERS[2]):
        given = arguments()
        words = on_device(torch.zeros((given["workspace"].numel() + 3) // 4, dtype=torch.float32))
        assert cls(None, **{**given, "workspace": words}).params.workspace_size == 4 * words.numel()


def commit_arguments(S=2, n=4, L=64):
    of = lambda rows: [cv.kv_tensor(on_device(torch.zeros(S * rows * 136, dtype=torch.uint8)), cv.Q8_0, 2, D, rows, S) for _ in "kv"]  # noqa: E731
    ints = lambda *s: on_device(torch.zeros(s, dtype=torch.int32))  # noqa: E731
    return {"caches": of(L), "drafts": of(n), "accepted": ints(S, n), "n_accepted": ints(S), "kv_len": ints(S), "kv_len_out": ints(S)}


@pytest.mark.parametrize("cls,arguments", [*LAUNCHERS, (cv.TreeCommitter, commit_arguments)], ids=lambda x: getattr(x, "__name__", None))
def test_a_launcher_keeps_its_buffers(cls, arguments):
    """Tensors, and the buffers behind descriptors, live as long as the launcher that will use them again."""
    given = {**arguments(), **(optional(cls) if cls is not cv.TreeCommitter else {})}
    refs = []
    for x in given.values():
        for y in x if isinstance(x, list) else [x]:
            if isinstance(y, torch.Tensor):
                refs.append(weakref.ref(y))
            elif isinstance(y, cv.Tensor):
                refs.append(weakref.ref(y._buf))
    plan = cls(None, **given)
    assert len(refs) >= 8
    del given, x, y
    gc.collect()
    assert all(r() is not None for r in refs)
    del plan
    gc.collect()
    assert all(r() is None for r in refs)


@pytest.mark.parametrize("cls,arguments", LAUNCHERS[:2], ids=lambda x: getattr(x, "__name__", None))
@pytest.mark.parametrize("heads,head_dim", [(14, 128), (7, 128), (28, 32)])
def test_queries_have_the_head_size_of_the_cache(cls, arguments, heads, head_dim):
    """Wider heads would pass the checks of strides and be read as other heads."""
    given = arguments()
    q = on_device(torch.zeros(2, 4, heads, head_dim))
    given |= {"q": q, "out": q.clone()} if cls is cv.TreeDecoder else {"q": q, "lse": on_device(torch.zeros(2, 4, heads))}
    with pytest.raises(ValueError):
        cls(None, **given)


@pytest.mark.parametrize("cls,arguments", [*LAUNCHERS, (cv.TreeCommitter, commit_arguments)], ids=lambda x: getattr(x, "__name__", None))
def test_descriptors_of_host_memory_are_refused(cls, arguments):
    given = arguments()
    cls(None, **given)
    host = cv.kv_tensor(torch.zeros(2 * 640 * 136, dtype=torch.uint8), cv.Q8_0, 2, D, 64, 2)
    seen = 0
    for name, x in given.items():
        if isinstance(x, cv.Tensor) or (isinstance(x, list) and isinstance(x[0], cv.Tensor)):
            seen += 1
            with pytest.raises(ValueError):
                cls(None, **{**given, name: [host, *x[1:]] if isinstance(x, list) else host})
    assert seen >= 1
