"""Plain forms of the paged 8-bit cache and of draft verification, in 64 bits on the host, as include/cvattn.h defines them."""
from __future__ import annotations

import numpy as np

BLOCK, D = 16, 64
MOST = {0: 127.0, 1: 448.0}

E4M3 = np.array([(-1 if b & 128 else 1) * ((b & 7) * 2.0 ** -9 if (b >> 3 & 15) == 0 else (8 + (b & 7)) * 2.0 ** ((b >> 3 & 15) - 10))
                 for b in range(256)])
VALUES = {0: np.arange(256) - 128.0, 1: E4M3}
_T, _Dm = np.meshgrid(np.arange(BLOCK), np.arange(D), indexing="ij")
PLACE = {"k": _T * D + _Dm, "v": _Dm // 32 * 512 + (_Dm % 8 * 4 + _T // 4) * 16 + _Dm // 8 % 4 * 4 + _T % 4}


def nearest(fmt, x):
    """Codes of the values nearest to x (f64), ties to the even code, beyond the largest the largest."""
    if fmt == 0:
        return (np.clip(np.rint(x), -127, 127) + 128).astype(np.uint8)
    grid = E4M3[:127]  # 0 .. 448
    a = np.minimum(np.abs(x), 448.0)
    up = np.searchsorted(grid, a).clip(1, 126)
    lo, hi = grid[up - 1], grid[up]
    code = np.where(a - lo < hi - a, up - 1, np.where(a - lo > hi - a, up, np.where(up % 2 == 0, up, up - 1)))
    return (code + 128 * np.signbit(x)).astype(np.uint8)


class Pool:
    """Host copy of one layer's pages: codes uint8 [pages, heads, blocks, 1024], scales f32 [pages, heads, blocks]."""

    def __init__(self, fmt, pages, size, heads, rng=None):
        self.fmt, self.size, self.heads, self.pages = fmt, size, heads, pages
        shape = (pages, heads, size // BLOCK)
        self.codes = {x: np.zeros((*shape, BLOCK * D), np.uint8) for x in "kv"}
        self.scales = {x: np.zeros(shape, np.float32) for x in "kv"}
        if rng is not None:  # whatever: all codes, NaN as scales
            for x in "kv":
                self.codes[x] = rng.integers(0, 256, self.codes[x].shape, dtype=np.uint8)
                self.scales[x][:] = np.nan

    def append(self, x, table, L, rows):
        """rows f32 [n, heads, 64] of one sequence (table: its entries) to positions L .."""
        n = len(rows)
        for b in range(L // BLOCK, (L + n + BLOCK - 1) // BLOCK):
            t0, t1 = max(0, L - b * BLOCK), min(BLOCK, L + n - b * BLOCK)
            if t1 <= t0:
                continue
            page, part = table[b * BLOCK // self.size], b % (self.size // BLOCK)
            for h in range(self.heads):
                new = rows[b * BLOCK + t0 - L:b * BLOCK + t1 - L, h].astype(np.float32)
                fine = np.abs(new[np.isfinite(new)])
                with np.errstate(under="ignore"):
                    fresh = np.float32(fine.max() if fine.size else 0.0) / np.float32(MOST[self.fmt])
                if fresh < np.finfo(np.float32).tiny:
                    fresh = np.float32(0)
                was = self.scales[x][page, h, part] if t0 and self.scales[x][page, h, part] > 0 else np.float32(0)
                scale = max(was, fresh)
                block = self.codes[x][page, h, part][PLACE[x]]
                if t0 and scale > was:
                    block[:t0] = nearest(self.fmt, VALUES[self.fmt][block[:t0]] * np.float64(was) / np.float64(scale))
                v = new.astype(np.float64)
                with np.errstate(invalid="ignore", divide="ignore"):
                    v = np.where(np.isnan(v) | (scale == 0), 0.0, v / np.float64(scale))
                block[t0:t1] = nearest(self.fmt, v)
                self.codes[x][page, h, part][PLACE[x]] = block
                self.scales[x][page, h, part] = scale

    def rows(self, x, table, n):
        """f64 [n, heads, 64]: positions 0 .. n - 1 (positions of a page out of range: NaN)."""
        out = np.full((n, self.heads, D), np.nan)
        for b in range((n + BLOCK - 1) // BLOCK):
            page, part = table[b * BLOCK // self.size], b % (self.size // BLOCK)
            if not 0 <= page < self.pages:
                continue
            m = min(BLOCK, n - b * BLOCK)
            y = VALUES[self.fmt][self.codes[x][page, :, part][:, PLACE[x]]] * self.scales[x][page, :, part].astype(np.float64)[:, None, None]
            out[b * BLOCK:b * BLOCK + m] = y[:, :m].transpose(1, 0, 2)
        return out

    def device(self, torch, cv, apart=0):
        """A PagePool with this content; pages `apart` more elements apart than they are long."""
        made = []
        for data in (self.codes, self.scales):
            for x in "kv":
                a = torch.from_numpy(data[x].reshape(self.pages, self.heads, -1)).cuda()
                if apart:
                    wide = torch.full((self.pages, a[0].numel() + 16 * apart), 77, dtype=a.dtype, device="cuda")
                    view = wide[:, :a[0].numel()].view(a.shape)
                    view.copy_(a)
                    a = view
                made.append(a)
        return cv.PagePool(*made, self.fmt)

    def same(self, pool):
        """Codes and scales of a PagePool against this one's, bit for bit."""
        for x in "kv":
            assert np.array_equal(getattr(pool, x).cpu().numpy().reshape(self.codes[x].shape), self.codes[x]), x
            got = getattr(pool, x + "_scale").cpu().numpy().reshape(self.scales[x].shape)
            assert np.array_equal(got, self.scales[x], equal_nan=True), x


def attention(q, k, v, n, scale):
    """out, lse in f64 of rows q [n, Hq, 64], the last n positions of k, v [L, H, 64]; positions that are NaN are left out."""
    L, H = k.shape[:2]
    G = q.shape[1] // H
    out, lse = np.zeros((len(q), q.shape[1], D)), np.full((len(q), q.shape[1]), -np.inf)
    there = ~np.isnan(k).any((1, 2))
    for i in range(n):
        sees = there & (np.arange(L) <= L - n + i)
        if not sees.any():
            continue
        for h in range(q.shape[1]):
            x = scale * (k[sees, h // G] @ q[i, h].astype(np.float64))
            top = x.max()
            p = np.exp(x - top)
            lse[i, h] = top + np.log(p.sum())
            out[i, h] = p @ v[sees, h // G] / p.sum()
    return out, lse


def assign(table, src, keep, need, P, pages):
    """Next table, holders of each page, room and the (source, target) copies."""
    n, width = table.shape
    lists = [[p if 0 <= p < pages else -1 for p in table[src[s], :-(-keep[s] // P)]] for s in range(n)]
    refs = np.bincount([p for x in lists for p in x if p >= 0], minlength=pages)
    free, room, moves, asked, taken = [p for p in range(pages) if refs[p] == 0], list(keep), [], 0, 0
    by = {}
    for s in range(n):
        if need[s] > keep[s] and keep[s] % P and lists[s][-1] >= 0:
            by.setdefault(lists[s][-1], []).append(s)
    held = refs.copy()
    for s in range(n):
        tail = lists[s][-1] if need[s] > keep[s] and keep[s] % P else -1
        copy = tail >= 0 and held[tail] > 1 and not (len(by[tail]) == held[tail] and by[tail][0] == s)
        more = max(0, -(-need[s] // P) - len(lists[s]))
        asked += more + copy
        if asked > len(free):
            continue
        if copy:
            moves.append((tail, free[taken]))
            lists[s][-1] = free[taken]
        lists[s] += free[taken + copy:taken + copy + more]
        taken += copy + more
        room[s] = max(keep[s], need[s])
    out = np.full_like(table, -1)
    for s, x in enumerate(lists):
        out[s, :len(x)] = x
    return out, np.bincount(out[out >= 0], minlength=pages), np.array(room), moves


def verify(logits, tokens, parents, n, u, last, heat, probs=None):
    """(path, following token, log-probabilities) of one sequence: logits [nodes, vocab]."""
    if n == 0:
        return [], -1, []
    at, path, said = 0, [0], []
    while True:
        x = logits[at].astype(np.float64)
        x = np.where(np.isnan(x), -np.inf, x)
        top = x.max()
        if top == -np.inf:
            return path, -1, said
        if heat == 0:
            w = np.zeros(len(x))
            w[int(np.argmax(x))] = 1.0
        elif top == np.inf:
            w = (x == np.inf).astype(np.float64)
        else:
            w = np.exp((x - top) / np.float64(heat))
        first = p = w / w.sum()
        down = None
        for c in range(at + 1, n):
            if parents[c] != at:
                continue
            t = tokens[c]
            if probs is None:
                takes, left = u[c] < p[t], p.copy()
                left[t] = 0.0
            else:
                q = probs[at].astype(np.float64)
                q = np.where(q > 0, q, 0.0)
                takes, left = u[c] * q[t] < p[t], np.maximum(p - q, 0.0)
            if takes:
                down = c
                break
            if left.sum() > 0:
                p = left / left.sum()
        with np.errstate(divide="ignore"):
            logs = np.log(first)
        if down is None:
            sums = np.cumsum(w if p is first else p)  # (equal weights add up exactly)
            over = np.flatnonzero(sums > last * sums[-1])
            token = int(over[0]) if len(over) else int(np.flatnonzero(p > 0)[-1])
            return path, token, said + [logs[token]]
        said.append(logs[tokens[down]])
        path.append(down)
        at = down
