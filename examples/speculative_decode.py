"""Speculative decoding in a bounded cache: drafts are verified as a tree, the accepted path is committed, its attention weight
added up, and the cache shrunk to a budget when it is full.

A random model (embedding, attention layers of 14 query and 2 KV heads, output projection) stands in for the LLM; drafts come from a
lookup of what followed the last token before (two candidates of three tokens).  Greedy decoding accepts a draft when it is the
token that the model would have chosen, so until the first eviction `--no-drafts` prints the same tokens, in more passes.

    python examples/speculative_decode.py --tokens 400 --budget 256
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "cosyvoice.cpp_b200"))
import cvattn as cv  # noqa: E402

HQ, HKV, D, HIDDEN, LAYERS, VOCAB = 14, 2, 64, 896, 2, 96
PARENTS = [-1, 0, 1, 2, 0, 4, 5]  # the pending token, then two chains of three drafts
DEPTH = [0, 1, 2, 3, 1, 2, 3]


def norm(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


class Generator:
    def __init__(self, capacity: int, budget: int, drafts: bool, seed: int = 0):
        g = torch.Generator().manual_seed(seed)
        mk = lambda *s: (torch.randn(s, generator=g) / s[0] ** 0.5).cuda()  # noqa: E731
        self.embed, self.head = torch.randn((VOCAB, HIDDEN), generator=g).cuda(), mk(HIDDEN, VOCAB)
        self.layers = [[mk(HIDDEN, HQ * D) * 2, mk(HIDDEN, HKV * D) * 2, mk(HIDDEN, HKV * D), mk(HQ * D, HIDDEN)] for _ in range(LAYERS)]
        self.n = n = len(PARENTS) if drafts else 1
        self.capacity, self.budget = capacity, budget
        self.ctx = cv.Context(0)
        ints = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.cache = [[cv.alloc_kv(cv.Q8_0, HKV, D, capacity)[1] for _ in "kv"] for _ in range(LAYERS)]
        self.draft = [[cv.alloc_kv(cv.Q8_0, HKV, D, n)[1] for _ in "kv"] for _ in range(LAYERS)]
        self.kv_len, self.kept, self.total, self.count = ints(1), ints(1), ints(1), ints(1)
        self.path, self.node = ints(1, 4), torch.arange(n, dtype=torch.int32, device="cuda")
        self.depth = torch.tensor(DEPTH[:n], dtype=torch.int32, device="cuda")
        self.scores = torch.zeros((LAYERS, 1, HKV, capacity), device="cuda")
        self.pos = ints(LAYERS, 1, HKV, capacity)
        self.q = torch.empty((LAYERS, 1, n, HQ, D), device="cuda")
        self.out, self.lse = torch.empty_like(self.q[0]), torch.empty((LAYERS, 1, n, HQ), device="cuda")
        self.rope = cv.rope_params(cv.ROPE_NEOX, D, D, 1e6)
        mask = cv.pack_tree_mask(torch.tensor([PARENTS[:n]])).cuda()
        self.verify = [cv.TreeDecoder(self.ctx, *self.cache[i], *self.draft[i], self.q[i], self.out, self.kv_len, capacity,
                                      lse=self.lse[i], mask=mask) for i in range(LAYERS)]
        self.commit = cv.TreeCommitter(self.ctx, [t for kv in self.cache for t in kv], [t for kv in self.draft for t in kv],
                                       self.path, self.count, self.kv_len, self.kv_len)
        self.weigh = [cv.KVScorer(self.ctx, self.cache[i][0], self.q[i], self.lse[i], self.kv_len, self.scores[i], rows=self.path,
                                  n_rows=self.count, decay=0.99) for i in range(LAYERS)]
        self.shrink = cv.KVEvictor(self.ctx, [kv[0] for kv in self.cache], [kv[1] for kv in self.cache], self.scores, self.pos,
                                   self.kv_len, self.kept, self.total, budget, kv_len_out=self.kv_len, n_sink=4, n_recent=budget // 4)
        self.tokens, self.steps, self.evictions, self.used = [1], 0, 0, 0

    def proposals(self) -> list[int]:
        """The pending token and two continuations that followed it earlier (else whatever: they will be rejected)."""
        t = self.tokens
        found = [i for i in range(len(t) - 2, -1, -1) if t[i] == t[-1]]
        chains = []
        for k in range(2):
            at = found[k] if k < len(found) else len(t)
            chains.append((t[at + 1:at + 4] + [0, 0, 0])[:3])
        return ([t[-1]] + chains[0] + chains[1])[:self.n]

    def step(self) -> int:
        """One pass of the model over the tree; returns how many tokens it gave."""
        if self.used + 4 > self.capacity:
            self.shrink()
            self.kept.copy_(self.kv_len)
            self.used = self.budget
            self.evictions += 1
        ids = self.proposals()
        x = self.embed[torch.tensor(ids, device="cuda")]
        at = self.total + self.depth
        for i, (wq, wk, wv, wo) in enumerate(self.layers):
            h = norm(x)
            cv.rope((h @ wq).view(self.n, HQ * D), at, self.rope, out=self.q[i].view(self.n, HQ * D))
            cv.kv_append(self.ctx, self.draft[i][0], cv.rope(h @ wk, at, self.rope)[None], self.node)
            cv.kv_append(self.ctx, self.draft[i][1], (h @ wv)[None], self.node)
            self.verify[i]()
            x = x + self.out.view(self.n, HQ * D) @ wo
        best = (norm(x) @ self.head).argmax(-1).tolist()
        path = [0]
        while True:
            child = [j for j in range(self.n) if PARENTS[j] == path[-1] and ids[j] == best[path[-1]]]
            if not child:
                break
            path.append(child[0])
        self.path.copy_(torch.tensor([(path + [0, 0, 0])[:4]], dtype=torch.int32))
        self.count.fill_(len(path))
        self.commit()
        self.total += self.count
        for w in self.weigh:
            w()
        self.tokens += [best[j] for j in path]
        self.used += len(path)
        self.steps += 1
        return len(path)


def generate(tokens: int, capacity: int, budget: int, drafts: bool = True, seed: int = 0) -> Generator:
    g = Generator(capacity, budget, drafts, seed)
    while len(g.tokens) <= tokens:
        g.step()
    g.tokens = g.tokens[1:tokens + 1]
    status, detail = g.ctx.sync_status()
    if status:
        raise RuntimeError(f"device status {status} ({detail})")
    return g


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    p.add_argument("--tokens", type=int, default=400)
    p.add_argument("--capacity", type=int, default=320)
    p.add_argument("--budget", type=int, default=256)
    p.add_argument("--no-drafts", action="store_true")
    p.add_argument("--seed", type=int, default=0)
    a = p.parse_args()
    g = generate(a.tokens, a.capacity, a.budget, not a.no_drafts, a.seed)
    print(" ".join(map(str, g.tokens)))
    print(f"{len(g.tokens)} tokens in {g.steps} passes, {g.evictions} evictions, {int(g.kv_len)} of {int(g.total)} positions kept")


if __name__ == "__main__":
    main()
