"""Launchers of the paged 8-bit cache and of the verification of drafts (include/cvattn.h).

As in the rest of the package a launcher checks its tensors and builds its parameters once; calling it launches on the given
or the current stream and reads the tensors' contents at that time.  Its scratch memory is its own (or the given workspace): what may
be under way at the same time, on two streams or in two graphs, wants launchers of its own."""
from __future__ import annotations

import ctypes
import math
from typing import Sequence

from . import Context, _dense, _device_bytes, _on, _rows4, _torch, _stream, check, lib
from ._lib import (PAGE_BLOCK, TREE_MAX_NODES, PagedAppendParams, PagedAttentionParams, PagedReadParams, PagePoolDesc,
                   PagesAssignParams, PagesCompactParams, VerifyParams)

PAGE_I8, PAGE_E4M3 = 0, 1
PAGE_SIZES = (16, 32, 64, 128)
_LOGITS = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 30}


class PagePool:
    """One layer's pages: k, v uint8 [n_pages, n_heads, page_size * 64], k_scale, v_scale f32 [n_pages, n_heads,
    page_size // 16], on the device; pages may lie apart, the rest is dense."""

    def __init__(self, k, v, k_scale, v_scale, format: int):
        torch = _torch()
        if k.dim() != 3 or k.shape[2] // 64 not in PAGE_SIZES or k.shape[2] % 64:
            raise ValueError("PagePool k: want [n_pages, n_heads, page_size * 64], page_size 16, 32, 64 or 128")
        pages, heads, size = k.shape[0], k.shape[1], k.shape[2] // 64
        for t, dtype, width, what in ((k, torch.uint8, size * 64, "k"), (v, torch.uint8, size * 64, "v"),
                                      (k_scale, torch.float32, size // PAGE_BLOCK, "k_scale"),
                                      (v_scale, torch.float32, size // PAGE_BLOCK, "v_scale")):
            if (t.dtype != dtype or not t.is_cuda or tuple(t.shape) != (pages, heads, width)
                    or (width > 1 and t.stride(2) != 1) or (heads > 1 and t.stride(1) != width)):
                raise ValueError(f"PagePool {what}: want a CUDA tensor of {dtype} and shape {(pages, heads, width)} with dense pages")
        apart = lambda t: t.shape[1] * t.shape[2] if pages == 1 else t.stride(0)  # noqa: E731
        if pages > 1 and (k.stride(0) != v.stride(0) or k_scale.stride(0) != v_scale.stride(0)):
            raise ValueError("PagePool: k and v, and their scales, want the same stride between pages")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.format, self.n_pages, self.n_heads, self.page_size = format, pages, heads, size
        self.desc = PagePoolDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), apart(k),
                                 apart(k_scale), format, heads, 64, size, pages, 0)


def alloc_pages(format: int, n_pages: int, page_size: int, n_heads: int, device="cuda") -> PagePool:
    """A pool with memory of its own."""
    torch = _torch()
    codes = torch.zeros((2, n_pages, n_heads, page_size * 64), dtype=torch.uint8, device=device)
    scales = torch.zeros((2, n_pages, n_heads, page_size // PAGE_BLOCK), dtype=torch.float32, device=device)
    return PagePool(codes[0], codes[1], scales[0], scales[1], format)


def _table(t, what, n_seq):
    """int32 [n_seq, entries] on the device, rows dense; its stride between sequences."""
    torch = _torch()
    if t.dtype != torch.int32 or not t.is_cuda or t.dim() != 2 or t.shape[0] != n_seq or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{what}: want a CUDA int32 tensor [n_seq, entries] with dense rows")
    return t.shape[1] if n_seq == 1 else t.stride(0)


def _counts(t, what, n_seq):
    torch = _torch()
    return None if t is None else _dense(t, (torch.int32,), what, (n_seq,)).data_ptr()


def _kv_rows(k, v, what, width):
    """k, v f32 [n_seq, rows, width] on the device in one layout with dense rows."""
    torch = _torch()
    for t, name in ((k, "k"), (v, "v")):
        if t.dtype != torch.float32 or not t.is_cuda or t.dim() != 3 or t.shape[2] != width or t.stride(2) != 1 or t.shape != k.shape:
            raise ValueError(f"{what} {name}: want a CUDA f32 tensor [n_seq, rows, {width}] with dense rows")
    if k.stride() != v.stride():
        raise ValueError(f"{what}: k and v in different layouts")
    return k.shape[0], k.shape[1], width if k.shape[1] == 1 else k.stride(1), k.stride(0)


class _Launcher:
    """Parameters built once, and what they point to."""
    _fn = _what = None

    def _ready(self, ctx: Context, params, *keep):
        self.ctx, self.params, self._ref, self._keep = ctx, params, ctypes.byref(params), keep

    def _scratch(self, workspace, need, device, what):
        torch = _torch()
        if workspace is None and need:
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
        self.workspace = workspace
        if workspace is None:
            return None, 0
        return workspace.data_ptr(), _device_bytes(workspace, f"{what} workspace")

    def __call__(self, stream=None) -> None:
        check(self._fn(self.ctx.handle, _stream(stream), self._ref), self._what)


class PageAppender(_Launcher):
    """Rounds rows k, v f32 [n_seq, max_new, n_heads * 64] into the pages of `pool` at positions kv_len[s] + i, i < n_new[s]
    (None: max_new).  table int32 [n_seq, entries]; kv_len, n_new int32 [n_seq]; refs int32 [n_pages] (PageAssigner's): pages
    that several entries hold are refused."""
    _fn, _what = lib.cvattn_paged_append, "paged_append"

    def __init__(self, ctx: Context, pool: PagePool, k, v, table, kv_len, n_new=None, refs=None):
        torch = _torch()
        n_seq, rows, nb_row, nb_seq = _kv_rows(k, v, "PageAppender", pool.n_heads * 64)
        p = PagedAppendParams()
        p.pool, p.k, p.v, p.nb_row, p.nb_seq = pool.desc, k.data_ptr(), v.data_ptr(), nb_row, nb_seq
        p.table_nb_seq, p.table, p.table_width = _table(table, "PageAppender table", n_seq), table.data_ptr(), table.shape[1]
        p.n_seq, p.max_new = n_seq, rows
        p.kv_len = _counts(kv_len, "PageAppender kv_len", n_seq)
        p.n_new = _counts(n_new, "PageAppender n_new", n_seq)
        if refs is not None:
            p.refs = _dense(refs, (torch.int32,), "PageAppender refs", (pool.n_pages,)).data_ptr()
        self._ready(ctx, p, pool, k, v, table, kv_len, n_new, refs)


class PageReader(_Launcher):
    """Reads positions first[s] + i (None: i), i < n_rows[s] (None: max_rows), back to rows of k, v f32 [n_seq, max_rows,
    n_heads * 64]; the other rows become zeros."""
    _fn, _what = lib.cvattn_paged_read, "paged_read"

    def __init__(self, ctx: Context, pool: PagePool, k, v, table, first=None, n_rows=None):
        n_seq, rows, nb_row, nb_seq = _kv_rows(k, v, "PageReader", pool.n_heads * 64)
        p = PagedReadParams()
        p.pool, p.k, p.v, p.nb_row, p.nb_seq = pool.desc, k.data_ptr(), v.data_ptr(), nb_row, nb_seq
        p.table_nb_seq, p.table, p.table_width = _table(table, "PageReader table", n_seq), table.data_ptr(), table.shape[1]
        p.n_seq, p.max_rows = n_seq, rows
        p.first = _counts(first, "PageReader first", n_seq)
        p.n_rows = _counts(n_rows, "PageReader n_rows", n_seq)
        self._ready(ctx, p, pool, k, v, table, first, n_rows)


def paged_attention_workspace_size(n_seq, max_q, max_kv_len, n_q_heads, n_kv_heads) -> int:
    return int(lib.cvattn_paged_attention_workspace_size(n_seq, max_q, max_kv_len, n_q_heads, n_kv_heads))


class PagedAttention(_Launcher):
    """Attention of the last n_q[s] (None: max_q) of kv_len[s] positions over the pages that table lists: q, out f32
    [n_seq, max_q, Hq, 64], lse f32 [n_seq, max_q, Hq] (optional); row i sees the positions before and at its own."""
    _fn, _what = lib.cvattn_paged_attention, "paged_attention"

    def __init__(self, ctx: Context, pool: PagePool, q, out, table, kv_len, max_kv_len: int | None = None, lse=None, n_q=None,
                 scale: float | None = None, workspace=None):
        torch = _torch()
        n_seq, rows, Hq, D = _rows4(q, "PagedAttention q", 64).shape
        if _rows4(out, "PagedAttention out", 64).shape != q.shape:
            raise ValueError("PagedAttention out: another shape than q")
        p = PagedAttentionParams()
        p.pool, p.q, p.out, p.q_nb_seq, p.out_nb_seq = pool.desc, q.data_ptr(), out.data_ptr(), q.stride(0), out.stride(0)
        p.q_nb_tok, p.out_nb_tok = (Hq * D, Hq * D) if rows == 1 else (q.stride(1), out.stride(1))
        if lse is not None:
            p.lse = _dense(lse, (torch.float32,), "PagedAttention lse", (n_seq, rows, Hq)).data_ptr()
        p.table_nb_seq, p.table, p.table_width = _table(table, "PagedAttention table", n_seq), table.data_ptr(), table.shape[1]
        p.kv_len = _counts(kv_len, "PagedAttention kv_len", n_seq)
        p.n_q = _counts(n_q, "PagedAttention n_q", n_seq)
        p.n_seq, p.max_q, p.n_q_heads = n_seq, rows, Hq
        p.max_kv_len = table.shape[1] * pool.page_size if max_kv_len is None else max_kv_len
        p.scale = 1.0 / math.sqrt(D) if scale is None else scale
        need = paged_attention_workspace_size(n_seq, rows, p.max_kv_len, Hq, pool.n_heads)
        p.workspace, p.workspace_size = self._scratch(workspace, need, q.device, "PagedAttention")
        self._ready(ctx, p, pool, q, out, lse, table, kv_len, n_q)


def paged_attention(ctx: Context, pool: PagePool, q, table, kv_len, max_kv_len: int | None = None, out=None, lse=None, stream=None, **kw):
    """One attention call; returns out f32 [n_seq, max_q, Hq, 64].  (Builds a PagedAttention each time: a program that keeps
    its buffers keeps one.)"""
    torch = _torch()
    with _on(stream):
        mine = out is None
        if mine:
            out = torch.empty(q.shape, dtype=torch.float32, device=q.device)
        plan = PagedAttention(ctx, pool, q, out, table, kv_len, max_kv_len, lse=lse, **kw)
    if mine and stream is not None:
        out.record_stream(torch.cuda.current_stream())  # (the caller may drop it there)
    plan(stream)
    return out


class _Books(_Launcher):
    """What assignment and compaction have in common."""

    def _tables(self, p, pools: Sequence[PagePool], table, table_out, refs, workspace, what):
        torch = _torch()
        if not pools:
            raise ValueError(f"{what}: one pool at least")
        table_out = table if table_out is None else table_out
        n_seq = table.shape[0]
        p.table_nb_seq, p.table, p.table_width, p.n_seq = _table(table, f"{what} table", n_seq), table.data_ptr(), table.shape[1], n_seq
        if _table(table_out, f"{what} table_out", n_seq) != p.table_nb_seq or table_out.shape != table.shape:
            raise ValueError(f"{what} table_out: want the layout of table")
        p.table_out = table_out.data_ptr()
        self._pools = (PagePoolDesc * len(pools))(*(x.desc for x in pools))
        p.pools, p.n_pools = self._pools, len(pools)
        if refs is not None:
            p.refs = _dense(refs, (torch.int32,), f"{what} refs", (pools[0].n_pages,)).data_ptr()
        need = int(lib.cvattn_pages_workspace_size(n_seq, table.shape[1], pools[0].n_pages))
        p.workspace, p.workspace_size = self._scratch(workspace, need, table.device, what)
        return table_out, n_seq


class PageAssigner(_Books):
    """What the tables hold next: sequence s keeps keep[s] positions of src[s] (None: of itself) and gets pages for need[s],
    in every pool of `pools`.  table, table_out (None: in place) int32 [n_seq, entries]; keep, need, src, room int32 [n_seq];
    refs int32 [n_pages] receives how many entries hold each page."""
    _fn, _what = lib.cvattn_pages_assign, "pages_assign"

    def __init__(self, ctx: Context, pools: Sequence[PagePool], table, keep, need, src=None, table_out=None, refs=None, room=None,
                 workspace=None):
        torch = _torch()
        p = PagesAssignParams()
        table_out, n_seq = self._tables(p, pools, table, table_out, refs, workspace, "PageAssigner")
        room = torch.empty(n_seq, dtype=torch.int32, device=table.device) if room is None else room
        p.keep, p.need = _counts(keep, "PageAssigner keep", n_seq), _counts(need, "PageAssigner need", n_seq)
        p.src, p.room = _counts(src, "PageAssigner src", n_seq), _counts(room, "PageAssigner room", n_seq)
        self.table, self.room, self.refs = table_out, room, refs
        self._ready(ctx, p, list(pools), table, table_out, keep, need, src, refs, room)


class PageCompactor(_Books):
    """Moves the pages that the tables hold to the front of every pool; n_live int32 [1] receives their number."""
    _fn, _what = lib.cvattn_pages_compact, "pages_compact"

    def __init__(self, ctx: Context, pools: Sequence[PagePool], table, n_live=None, table_out=None, refs=None, workspace=None):
        torch = _torch()
        p = PagesCompactParams()
        table_out, _ = self._tables(p, pools, table, table_out, refs, workspace, "PageCompactor")
        n_live = torch.empty(1, dtype=torch.int32, device=table.device) if n_live is None else n_live
        p.n_live = _counts(n_live, "PageCompactor n_live", 1)
        self.table, self.n_live, self.refs = table_out, n_live, refs
        self._ready(ctx, p, list(pools), table, table_out, n_live, refs)


class DraftVerifier(_Launcher):
    """Which drafted tokens stand.  logits f32, f16 or bf16 [n_seq, max_nodes, vocab]; tokens int32, accept_u f32
    [n_seq, max_nodes]; sample_u f32 [n_seq]; accepted int32 [n_seq, max_nodes], n_accepted, next_token int32 [n_seq] are
    written, and log_probs f32 [n_seq, max_nodes] if given.  parents int32 [n_seq or 1, max_nodes] (None: chains), n_nodes
    int32 [n_seq] (None: max_nodes), draft_probs f32 like logits (None: drafts not drawn at random), temperature f32 [n_seq]
    (None: 1)."""
    _fn, _what = lib.cvattn_verify_drafts, "verify_drafts"

    def __init__(self, ctx: Context, logits, tokens, accept_u, sample_u, accepted, n_accepted, next_token, parents=None, n_nodes=None,
                 draft_probs=None, temperature=None, log_probs=None, workspace=None):
        torch = _torch()
        if str(logits.dtype) not in _LOGITS or not logits.is_cuda or logits.dim() != 3 or (logits.shape[2] > 1 and logits.stride(2) != 1):
            raise ValueError("DraftVerifier logits: want a CUDA f32, f16 or bf16 tensor [n_seq, max_nodes, vocab] with dense rows")
        n_seq, n, vocab = logits.shape
        if n > TREE_MAX_NODES:
            raise ValueError(f"DraftVerifier: at most {TREE_MAX_NODES} nodes")
        p = VerifyParams()
        p.logits, p.logits_type, p.n_seq, p.max_nodes, p.vocab = logits.data_ptr(), _LOGITS[str(logits.dtype)], n_seq, n, vocab
        p.logits_nb_node, p.logits_nb_seq = vocab if n == 1 else logits.stride(1), logits.stride(0)
        if draft_probs is not None:
            t = draft_probs
            if t.dtype != torch.float32 or not t.is_cuda or t.shape != logits.shape or (vocab > 1 and t.stride(2) != 1):
                raise ValueError("DraftVerifier draft_probs: want a CUDA f32 tensor in the shape of logits with dense rows")
            p.draft_probs, p.probs_nb_node, p.probs_nb_seq = t.data_ptr(), vocab if n == 1 else t.stride(1), t.stride(0)
        each, one = (n_seq, n), (n_seq,)
        p.tokens = _dense(tokens, (torch.int32,), "DraftVerifier tokens", each).data_ptr()
        p.accept_u = _dense(accept_u, (torch.float32,), "DraftVerifier accept_u", each).data_ptr()
        p.sample_u = _dense(sample_u, (torch.float32,), "DraftVerifier sample_u", one).data_ptr()
        p.accepted, p.accepted_stride = _dense(accepted, (torch.int32,), "DraftVerifier accepted", each).data_ptr(), n
        p.n_accepted = _dense(n_accepted, (torch.int32,), "DraftVerifier n_accepted", one).data_ptr()
        p.next_token = _dense(next_token, (torch.int32,), "DraftVerifier next_token", one).data_ptr()
        if log_probs is not None:
            p.log_probs = _dense(log_probs, (torch.float32,), "DraftVerifier log_probs", each).data_ptr()
        if parents is not None:
            _dense(parents, (torch.int32,), "DraftVerifier parents")
            if tuple(parents.shape) not in ((n_seq, n), (1, n)):
                raise ValueError("DraftVerifier parents: want [n_seq or 1, max_nodes]")
            p.parents, p.parents_nb_seq = parents.data_ptr(), 0 if parents.shape[0] == 1 else n
        p.n_nodes = _counts(n_nodes, "DraftVerifier n_nodes", n_seq)
        if temperature is not None:
            p.temperature = _dense(temperature, (torch.float32,), "DraftVerifier temperature", one).data_ptr()
        need = int(lib.cvattn_verify_workspace_size(n_seq, n, vocab))
        p.workspace, p.workspace_size = self._scratch(workspace, need, logits.device, "DraftVerifier")
        self._ready(ctx, p, logits, tokens, accept_u, sample_u, accepted, n_accepted, next_token, parents, n_nodes, draft_probs,
                    temperature, log_probs)
