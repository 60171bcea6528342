"""GPU: assignment and compaction of the pages of a cache, against books kept on the host."""
from __future__ import annotations

import numpy as np
import pytest

from paged_reference import assign

pytestmark = pytest.mark.gpu


def ints(torch, v):
    return torch.tensor(np.asarray(v, np.int32), device="cuda")


def pools(torch, cv, n, pages, size, heads=2, apart=False):
    made = []
    for _ in range(n):
        k, v = (torch.randint(0, 256, (pages, heads + apart, size * 64), dtype=torch.uint8, device="cuda")[:, :heads] for _ in "kv")
        ks, vs = (torch.rand(pages, heads + apart, size // 16, device="cuda")[:, :heads] for _ in "kv")
        made.append(cv.PagePool(k, v, ks, vs, 0))
    return made


def parts(pool):
    return [pool.k, pool.v, pool.k_scale, pool.v_scale]


def check(cv, ctx, torch, table, src, keep, need, size, pages, layers=2, in_place=False, src_given=True, heads=2, apart=False):
    S = len(table)
    made = pools(torch, cv, layers, pages, size, heads, apart)
    before = [[t.clone() for t in parts(x)] for x in made]
    t = ints(torch, table)
    out = t if in_place else torch.full_like(t, 99)
    refs, room = torch.full((pages,), 9, dtype=torch.int32, device="cuda"), torch.full((S,), 9, dtype=torch.int32, device="cuda")
    cv.PageAssigner(ctx, made, t, ints(torch, keep), ints(torch, need), src=ints(torch, src) if src_given else None,
                    table_out=None if in_place else out, refs=refs, room=room)()
    want, held, rooms, moves = assign(table, src, keep, need, size, pages)
    assert np.array_equal(out.cpu().numpy(), want)
    assert np.array_equal(refs.cpu().numpy(), held)
    assert np.array_equal(room.cpu().numpy(), rooms)
    if not in_place:
        assert np.array_equal(t.cpu().numpy(), table)
    for x, old in zip(made, before):
        for now, was in zip(parts(x), old):
            for a, b in moves:
                was[b] = was[a].clone()
            assert torch.equal(now, was)
    return want, moves


def random_state(rng, S, size, pages, width, shared):
    """A table, partly of shared pages, and lengths."""
    L = rng.integers(0, width * size // 2, S)
    t, at, order = np.full((S, width), -1, np.int32), 0, rng.permutation(pages)
    for s in range(S):
        if shared and s % 3 and L[s - 1]:
            L[s] = min(L[s], L[s - 1])
            t[s, :-(-L[s] // size)] = t[s - 1, :-(-L[s] // size)]
            continue
        m = -(-L[s] // size)
        t[s, :m] = order[at:at + m]
        at += m
    return t, L, at


@pytest.mark.parametrize("seed", range(12))
def test_assign(ctx, cv, cuda, seed):
    rng = np.random.default_rng(seed)
    S, size = int(rng.integers(1, 80)), int(rng.choice([16, 32, 64, 128]))
    width = int(rng.integers(2, 30))
    pages = S * width // 2 + int(rng.integers(1, 200))
    table, L, _ = random_state(rng, S, size, pages, width, seed % 2)
    src = np.arange(S) if seed % 3 == 0 else rng.integers(0, S, S)
    keep = np.array([int(rng.integers(0, L[x] + 1)) if rng.random() < 0.4 else int(L[x]) for x in src])
    need = np.minimum(keep + rng.integers(-5, 3 * size, S), width * size).clip(0)
    check(cv, ctx, cuda, table, src, keep, need, size, pages, in_place=seed % 4 == 1, src_given=seed % 3 != 0, apart=seed % 5 == 0,
          heads=1 + seed % 3)


def test_assign_of_many_sequences(ctx, cv, cuda):
    """More sequences and pages than one pass of the books takes, and pools for two copy launches."""
    rng = np.random.default_rng(1)
    S, size, width, pages = 2500, 16, 4, 9000
    table, L, _ = random_state(rng, S, size, pages, width, True)
    src = np.arange(S)
    src[1::7] = src[::7][:len(src[1::7])]
    keep = L[src]
    check(cv, ctx, cuda, table, src, keep, np.minimum(keep + 3, width * size), size, pages, layers=50, heads=1)


def test_fork_copies_the_tail_but_for_one(ctx, cv, cuda):
    """Four candidates of one utterance write into its last page: three get copies; where it stays on too, all four do."""
    table = np.array([[5, 3, -1]] + [[-1, -1, -1]] * 4, np.int32)
    _, moves = check(cv, ctx, cuda, table, [0, 0, 0, 0, 0], [20, 20, 20, 20, 0], [21, 21, 21, 21, 0], 16, 12)
    assert moves == [(3, 0), (3, 1), (3, 2)]
    _, moves = check(cv, ctx, cuda, table, [0, 0, 0, 0, 0], [20, 20, 20, 20, 20], [20, 21, 21, 21, 21], 16, 12)
    assert moves == [(3, 0), (3, 1), (3, 2), (3, 4)]
    # at a border of pages there is nothing to copy, and shorter keeps share what they keep
    _, moves = check(cv, ctx, cuda, table, [0, 0, 0, 0, 0], [16, 16, 20, 5, 0], [17, 17, 20, 6, 0], 16, 12)
    assert moves == [(5, 2)]


def test_free_roll_back_and_swap(ctx, cv, cuda):
    table = np.array([[0, 1, 2, -1], [3, 4, -1, -1], [5, -1, -1, -1]], np.int32)
    want, moves = check(cv, ctx, cuda, table, [1, 0, 2], [20, 33, 0], [20, 33, 0], 16, 6, in_place=True)
    assert want.tolist() == [[3, 4, -1, -1], [0, 1, 2, -1], [-1] * 4] and not moves
    want, _ = check(cv, ctx, cuda, table, [0, 1, 2], [17, 0, 16], [17, 5, 40], 16, 6)
    assert want.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1], [5, 3, 4, -1]]


def test_too_few_pages(ctx, cv, cuda):
    """Sequences in order as long as what they ask for is there; one behind that asks for nothing has its room."""
    table = np.array([[0, -1, -1], [1, -1, -1], [2, -1, -1], [3, -1, -1]], np.int32)
    want, _ = check(cv, ctx, cuda, table, range(4), [16, 16, 16, 9], [17, 48, 17, 10], 16, 6)
    assert want.tolist() == [[0, 4, -1], [1, -1, -1], [2, -1, -1], [3, -1, -1]]
    # no free page at all
    check(cv, ctx, cuda, table, range(4), [16] * 4, [17] * 4, 16, 4)
    # a tail that cannot be copied stays shared, without room
    table = np.array([[0, -1], [0, -1]], np.int32)
    want, moves = check(cv, ctx, cuda, table, range(2), [9, 9], [9, 10], 16, 1)
    assert want.tolist() == [[0, -1], [0, -1]] and not moves


def test_bad_wishes_are_recorded(ctx, cv, cuda):
    torch = cuda
    table = np.array([[0, 1], [2, 7], [3, -1], [-1, -1], [4, -1], [5, -1]], np.int32)
    made = pools(torch, cv, 1, 7, 16)
    t, refs = ints(torch, table), torch.empty(7, dtype=torch.int32, device="cuda")
    a = cv.PageAssigner(ctx, made, t, ints(torch, [20, 20, -1, 5, 8, 8]), ints(torch, [20, 20, 0, 5, 33, 9]), src=ints(torch, [0, 1, 2, 3, 4, 6]), refs=refs)
    a()
    assert ctx.sync_status()[0] == 6
    assert t.tolist() == [[0, 1], [2, -1], [-1, -1], [-1, -1], [-1, -1], [-1, -1]]
    assert refs.tolist() == [1, 1, 1, 0, 0, 0, 0] and a.room.tolist() == [20, 20, 0, 5, 0, 0]


@pytest.mark.parametrize("seed", range(6))
def test_compact(ctx, cv, cuda, seed):
    torch, rng = cuda, np.random.default_rng(seed)
    S, size = int(rng.integers(1, 60)), int(rng.choice([16, 64]))
    width = int(rng.integers(2, 30))
    pages = S * width + int(rng.integers(1, 3000))
    table, _, _ = random_state(rng, S, size, pages, width, seed % 2)
    if seed == 4:
        table[:] = -1
    if seed == 5:
        table[0, 0] = pages  # out of range: dropped
    made = pools(torch, cv, 3, pages, size)
    before = [[t.clone() for t in parts(x)] for x in made]
    t = ints(torch, table)
    out = t if seed % 2 else torch.empty_like(t)
    refs = torch.empty(pages, dtype=torch.int32, device="cuda")
    c = cv.PageCompactor(ctx, made, t, table_out=out, refs=refs)
    c()
    live = sorted({int(p) for p in table.ravel() if 0 <= p < pages})
    free = sorted(set(range(len(live))) - set(live))
    to = dict(zip([p for p in live if p >= len(live)], free))
    want = np.array([[to.get(int(p), int(p)) if 0 <= p < pages else -1 for p in row] for row in table])
    assert int(c.n_live) == len(live)
    assert np.array_equal(out.cpu().numpy(), want)
    assert np.array_equal(refs.cpu().numpy(), np.bincount(want[want >= 0], minlength=pages))
    for x, old in zip(made, before):
        for now, was in zip(parts(x), old):
            for a, b in to.items():
                was[b] = was[a]
            assert torch.equal(now, was)


def test_books_in_a_graph(ctx, cv, cuda):
    """A replayed assignment reads the table, the wishes and the pages of its time; two graphs have books of their own."""
    torch = cuda
    made = pools(torch, cv, 2, 40, 16)
    table = torch.full((4, 6), -1, dtype=torch.int32, device="cuda")
    keep, need, src = (torch.zeros(4, dtype=torch.int32, device="cuda") for _ in range(3))
    src.copy_(torch.arange(4))
    plan = cv.PageAssigner(ctx, made, table, keep, need, src=src)
    plan()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan()
    host = np.full((4, 6), -1, np.int32)
    for k, n, f in (([0] * 4, [20, 5, 0, 40], range(4)), ([20, 20, 0, 33], [21, 22, 1, 70], [0, 0, 2, 3]), ([21, 0, 1, 70], [21, 0, 1, 71], range(4))):
        keep.copy_(ints(torch, k))
        need.copy_(ints(torch, n))
        src.copy_(ints(torch, list(f)))
        graph.replay()
        host, _, room, _ = assign(host, list(f), k, n, 16, 40)
        assert np.array_equal(table.cpu().numpy(), host) and plan.room.tolist() == room.tolist()
