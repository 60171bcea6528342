"""GPU: the paged cache and the verification as a serving loop uses them, against books, pages and sums kept on the host; and the
example."""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import pytest

from paged_reference import D, Pool, assign, attention, verify

pytestmark = pytest.mark.gpu

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))


def ints(torch, v):
    return torch.tensor(np.asarray(v, np.int32), device="cuda")


@pytest.mark.parametrize("fmt,size", [(0, 16), (1, 64)])
def test_prompt_fork_draft_verify_roll_back_free_compact(ctx, cv, cuda, fmt, size):
    torch, rng = cuda, np.random.default_rng(size)
    S, n, Hq, heads, V, prompt, pages, width = 5, 4, 14, 2, 300, 37, 64, 8
    host = [Pool(fmt, pages, size, heads, rng) for _ in range(2)]
    pools = [h.device(torch, cv) for h in host]
    table = np.full((S, width), -1, np.int32)
    t, refs = ints(torch, table), ints(torch, [0] * pages)
    keep, need, src, before, after = (ints(torch, [0] * S) for _ in range(5))
    plan = cv.PageAssigner(ctx, pools, t, keep, need, src=src, refs=refs)

    def books(k, m, f=None):
        nonlocal table
        f = list(range(S)) if f is None else f
        keep.copy_(ints(torch, k)), need.copy_(ints(torch, m)), src.copy_(ints(torch, f))
        plan()
        table, held, room, moves = assign(table, f, list(k), list(m), size, pages)
        assert np.array_equal(t.cpu().numpy(), table) and np.array_equal(refs.cpu().numpy(), held) and plan.room.tolist() == list(room)
        for h in host:
            for a, b in moves:
                for x in "kv":
                    h.codes[x][b], h.scales[x][b] = h.codes[x][a], h.scales[x][a]

    def forward(L, rows):
        """rows new tokens of every sequence (0: none) through both layers' pages; returns the last layer's output."""
        m = max(rows)
        q, k, v = (rng.standard_normal((S, m, h * D)).astype(np.float32) for h in (Hq, heads, heads))
        qd, kd, vd = (torch.from_numpy(x).cuda() for x in (q, k, v))
        count, out = ints(torch, rows), torch.empty(S, m, Hq, D, device="cuda")
        before.copy_(ints(torch, L)), after.copy_(ints(torch, np.add(L, rows)))
        for pool, h in zip(pools, host):
            cv.PageAppender(ctx, pool, kd, vd, t, before, n_new=count, refs=refs)()
            cv.PagedAttention(ctx, pool, qd.view(S, m, Hq, D), out, t, after, n_q=count)()
            for s in range(S):
                for x, data in (("k", k), ("v", v)):
                    h.append(x, table[s], L[s], data[s, :rows[s]].reshape(rows[s], heads, D))
            h.same(pool)
            for s in range(S):
                want, _ = attention(q[s].reshape(m, Hq, D), h.rows("k", table[s], L[s] + rows[s]), h.rows("v", table[s], L[s] + rows[s]), rows[s], D ** -0.5)
                # (as in the tests of attention alone: 2^-19 (1 + 64 |q k| / 8) of the largest value, which is below 5)
                assert np.abs(out[s].cpu().numpy() - want).max() <= 2.0 ** -19 * 40 * 5
        return out

    books([0] * S, [prompt] + [0] * (S - 1))
    forward([0] * S, [prompt] + [0] * (S - 1))
    L = [prompt] * S
    books(L, L, [0] * S)  # everyone holds the prompt's pages
    assert refs.max() == S
    for step in range(6):
        books(L, [x + n for x in L])
        assert refs.cpu().numpy()[[table[s, L[s] // size] for s in range(S)]].max() == 1  # nobody writes into a shared page
        out = forward(L, [n] * S)
        logits = (out.flatten(2) @ torch.from_numpy(rng.standard_normal((Hq * D, V)).astype(np.float32)).cuda()) * 0.2
        probs = torch.softmax(logits + 0.3 * torch.from_numpy(rng.standard_normal((S, n, V)).astype(np.float32)).cuda(), -1)
        tokens = np.array([[rng.choice(V, p=probs[s, max(i - 1, 0)].double().cpu().numpy() / float(probs[s, max(i - 1, 0)].double().sum()))
                            for i in range(n)] for s in range(S)], np.int32)
        u, last = rng.random((S, n)).astype(np.float32), rng.random(S).astype(np.float32)
        path, count, token = (torch.empty(x, dtype=torch.int32, device="cuda") for x in ((S, n), (S,), (S,)))
        cv.DraftVerifier(ctx, logits, ints(torch, tokens), torch.from_numpy(u).cuda(), torch.from_numpy(last).cuda(), path, count, token,
                         draft_probs=probs)()
        for s in range(S):
            want, end, _ = verify(logits[s].cpu().numpy(), tokens[s], np.arange(-1, n - 1), n, u[s].astype(np.float64), np.float64(last[s]), 1.0,
                                  probs[s].cpu().numpy())
            assert path[s, :len(want)].tolist() == want and int(count[s]) == len(want) and int(token[s]) == end
        L = [a + int(c) for a, c in zip(L, count)]
        if step == 2:  # one has ended, another takes its place as a fork of a third
            books([L[0], L[4], L[2], L[3], L[4]], [L[0], L[4], L[2], L[3], L[4]], [0, 4, 2, 3, 4])
            L[1] = L[4]
        if step == 4:  # one ends, and the pool is compacted
            L[3] = 0
            books(L, L)
            c = cv.PageCompactor(ctx, pools, t, refs=refs)
            c()
            live = sorted({int(p) for p in table.ravel() if p >= 0})
            to = dict(zip([p for p in live if p >= len(live)], sorted(set(range(len(live))) - set(live))))
            for h in host:
                for a, b in to.items():
                    for x in "kv":
                        h.codes[x][b], h.scales[x][b] = h.codes[x][a], h.scales[x][a]
            table = np.array([[to.get(int(p), int(p)) for p in row] for row in table], np.int32)
            assert np.array_equal(t.cpu().numpy(), table) and int(c.n_live) == len(live) == int((refs > 0).sum())


def test_calls_on_two_streams_at_once(ctx, cv, cuda):
    """Attention and verification of two batches with launchers of their own, under way together."""
    torch, rng = cuda, np.random.default_rng(0)
    batches, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in range(2):
        host = Pool(seed, 40, 32, 2, rng)
        table = rng.permutation(40)[:36].reshape(3, 12).astype(np.int32)
        for s in range(3):
            for x in "kv":
                host.append(x, table[s], 0, rng.standard_normal((384, 2, D)).astype(np.float32))
        pool = host.device(torch, cv)
        made = []
        for rows in (1, 40):
            q = torch.randn(3, rows, 14, D, device="cuda")
            made.append(cv.PagedAttention(ctx, pool, q, torch.empty_like(q), ints(torch, table), ints(torch, [384, 100, 200])))
        logits = torch.randn(3, 4, 20000, device="cuda") * 3
        ids = torch.randint(20000, (3, 4), dtype=torch.int32, device="cuda")
        outs = [torch.empty(s, dtype=torch.int32, device="cuda") for s in ((3, 4), (3,), (3,))]
        made.append(cv.DraftVerifier(ctx, logits, ids, torch.zeros(3, 4, device="cuda"), torch.rand(3, device="cuda"), *outs))
        results = [made[0]._keep[2], made[1]._keep[2], *outs]
        for m in made:
            m()
        batches.append((made, results, [r.clone() for r in results]))
    torch.cuda.synchronize()
    for _ in range(20):
        for (made, _, _), stream in zip(batches, streams):
            for m in made:
                m(stream)
    torch.cuda.synchronize()
    for _, results, want in batches:
        assert all(torch.equal(a, b) for a, b in zip(results, want))


def test_example(cuda):
    import paged_serving as ex
    for temperature in (0.0, 0.5):
        s = ex.serve(4, 40, prompt=45, temperature=temperature)
        assert all(len(t) > 45 + 30 for t in s.tokens) and all(0 <= x < ex.VOCAB for t in s.tokens for x in t)
        assert bool((s.refs[s.refs > 0] >= 1).all()) and int(s.refs.max()) == 4  # the prompt's whole page is shared
        held = int((s.refs > 0).sum())
        assert s.finish([0, 2]) < held
        assert int(s.refs.max()) == 2
        s.ctx.close()
