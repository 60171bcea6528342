"""Several utterances over one voice prompt in a paged 8-bit cache: the prompt's pages are shared, drafts are verified by
speculative sampling, rejected ones rolled back, finished utterances' pages given back and the pool compacted.

A random model (embedding, attention layers of 14 query and 2 KV heads, output projection) stands in for the LLM; drafts come
from a lookup of what followed the last two tokens before in the same utterance.

    python examples/paged_serving.py --utterances 6 --tokens 120
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "cosyvoice.cpp_b200"))
import cvattn as cv  # noqa: E402

HQ, HKV, D, HIDDEN, LAYERS, VOCAB, PAGE = 14, 2, 64, 896, 2, 96, 32
DRAFTS = 4  # the pending token and three drafted ones


def norm(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


class Server:
    def __init__(self, utterances: int, most: int, prompt: int, temperature: float, seed: int = 0):
        g = torch.Generator().manual_seed(seed)
        mk = lambda *s: (torch.randn(s, generator=g) / s[0] ** 0.5).cuda()  # noqa: E731
        self.embed, self.head = torch.randn((VOCAB, HIDDEN), generator=g).cuda(), mk(HIDDEN, VOCAB) * 3
        self.layers = [[mk(HIDDEN, HQ * D) * 2, mk(HIDDEN, HKV * D) * 2, mk(HIDDEN, HKV * D), mk(HQ * D, HIDDEN)] for _ in range(LAYERS)]
        self.random = torch.Generator("cuda").manual_seed(seed)
        self.ctx = cv.Context(0)
        S = self.S = utterances
        width = -(-(prompt + most + DRAFTS) // PAGE)
        pages = -(-prompt // PAGE) + S * -(-(most + DRAFTS + PAGE) // PAGE)
        self.pools = [cv.alloc_pages(cv.PAGE_I8, pages, PAGE, HKV) for _ in range(LAYERS)]
        ints = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        self.table, self.refs = torch.full((S, width), -1, dtype=torch.int32, device="cuda"), ints(pages)
        self.keep, self.need, self.src, self.len, self.seen = (ints(S) for _ in range(5))
        self.src.copy_(torch.arange(S))
        self.assign = cv.PageAssigner(self.ctx, self.pools, self.table, self.keep, self.need, src=self.src, refs=self.refs)
        self.compact = cv.PageCompactor(self.ctx, self.pools, self.table, refs=self.refs)
        self.rope = cv.rope_params(cv.ROPE_NEOX, D, D, 1e6)
        self.steps, self.accepted = {}, 0
        self.prompt, self.temperature = torch.randint(VOCAB, (prompt,), generator=g).tolist(), torch.full((S,), temperature, device="cuda")
        self.tokens = [list(self.prompt) for _ in range(S)]
        self.fill()

    def buffers(self, S: int, n: int) -> dict:
        """The tensors and launchers of a pass over n tokens of the first S sequences."""
        if (S, n) not in self.steps:
            f = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
            b = self.steps[S, n] = {"q": f(S, n, HQ, D), "out": f(S, n, HQ, D), "k": f(S, n, HKV * D), "v": f(S, n, HKV * D)}
            table, before, after = self.table[:S], self.len[:S], self.seen[:S]
            b["append"] = [cv.PageAppender(self.ctx, p, b["k"], b["v"], table, before, refs=self.refs) for p in self.pools]
            b["attend"] = [cv.PagedAttention(self.ctx, p, b["q"], b["out"], table, after) for p in self.pools]
        return self.steps[S, n]

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        """Logits [S, n, vocab] of ids [S, n], whose keys and values go to the end of the sequences' pages."""
        S, n = ids.shape
        b = self.buffers(S, n)
        torch.add(self.len[:S], n, out=self.seen[:S])
        at = (self.len[:S, None] + torch.arange(n, dtype=torch.int32, device="cuda")).flatten().int()
        x = self.embed[ids].view(S * n, HIDDEN)
        for i, (wq, wk, wv, wo) in enumerate(self.layers):
            h = norm(x)
            cv.rope((h @ wq), at, self.rope, out=b["q"].view(S * n, HQ * D))
            cv.rope((h @ wk), at, self.rope, out=b["k"].view(S * n, HKV * D))
            torch.matmul(h, wv, out=b["v"].view(S * n, HKV * D))
            b["append"][i]()
            b["attend"][i]()
            x = x + b["out"].view(S * n, HQ * D) @ wo
        return (norm(x) @ self.head).view(S, n, VOCAB)

    def fill(self) -> None:
        """The prompt, all but its last token, once; then every utterance forks it."""
        n = len(self.prompt) - 1
        self.need[0] = n
        self.assign()
        self.forward(torch.tensor([self.prompt[:n]], device="cuda"))
        self.len.fill_(n)
        self.src.zero_()
        self.keep.fill_(n)
        self.need.fill_(n)
        self.assign()
        self.src.copy_(torch.arange(self.S))

    def proposals(self, tokens: list[int]) -> list[int]:
        """The last token, and what followed the last two before (else whatever)."""
        for i in range(len(tokens) - 3, 0, -1):
            if tokens[i - 1:i + 1] == tokens[-2:]:
                return ([tokens[-1]] + tokens[i + 1:i + DRAFTS] + [0] * DRAFTS)[:DRAFTS]
        return [tokens[-1]] + [0] * (DRAFTS - 1)

    def step(self) -> None:
        """One pass for every utterance."""
        ids = torch.tensor([self.proposals(t) for t in self.tokens], dtype=torch.int32, device="cuda")
        self.keep.copy_(self.len)
        torch.add(self.len, DRAFTS, out=self.need)
        self.assign()
        logits = self.forward(ids)
        S, n = ids.shape
        u, last = (torch.rand(s, generator=self.random, device="cuda") for s in ((S, n), (S,)))
        path, count, token = (torch.empty(s, dtype=torch.int32, device="cuda") for s in ((S, n), (S,), (S,)))
        cv.DraftVerifier(self.ctx, logits, ids, u, last, path, count, token, temperature=self.temperature)()
        self.len += count  # (what lies behind is rolled back by the next assignment)
        for t, row, c, end in zip(self.tokens, ids.tolist(), count.tolist(), token.tolist()):
            t += row[1:c] + [end]
            self.accepted += c - 1

    def finish(self, which: list[int]) -> int:
        """Gives the pages of some utterances back and compacts the rest; returns how many pages are held."""
        for s in which:
            self.len[s] = 0
        self.keep.copy_(self.len)
        self.need.copy_(self.len)
        self.assign()
        self.compact()
        return int(self.compact.n_live)


def serve(utterances: int, tokens: int, prompt: int = 45, temperature: float = 0.3, seed: int = 0) -> Server:
    s = Server(utterances, tokens + DRAFTS, prompt, temperature, seed)
    while min(len(t) for t in s.tokens) < prompt + tokens and max(len(t) for t in s.tokens) < prompt + tokens + DRAFTS:
        s.step()
    status, detail = s.ctx.sync_status()
    if status:
        raise RuntimeError(f"device status {status} ({detail})")
    return s


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    p.add_argument("--utterances", type=int, default=6)
    p.add_argument("--tokens", type=int, default=120)
    p.add_argument("--prompt", type=int, default=45)
    p.add_argument("--temperature", type=float, default=0.3)
    p.add_argument("--seed", type=int, default=0)
    a = p.parse_args()
    s = serve(a.utterances, a.tokens, a.prompt, a.temperature, a.seed)
    for t in s.tokens:
        print(" ".join(map(str, t[a.prompt:a.prompt + 24])), "..")
    print(f"{sum(len(t) - a.prompt for t in s.tokens)} tokens, {s.accepted} of them drafted; {int((s.refs > 0).sum())} pages held,",
          f"{int((s.refs > 1).sum())} of them shared")
    print(f"{s.finish(list(range(0, a.utterances, 2)))} pages held after every second utterance has ended")


if __name__ == "__main__":
    main()
