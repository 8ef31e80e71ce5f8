"""Paged key/value cache, attention of a ragged batch over it, and the sampler that ends a decode step (include/ttq.h,
``ttq_paged_*`` and ``ttq_sample``).  The reference keeps one growing contiguous cache per sequence (attn.nim:97-104) and has no
sampler."""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Union

import torch

from . import _lib
from ._lib import KvPages, PagedBatchArgs, Sampling, TtqError, check
from .layers import Context, _dt, _stream_ptr


# The checks below are on the path of every call of a decode step: plain comparisons, no views and no temporary tensors.

def _elsewhere(name: str) -> TtqError:
    return TtqError(1, f"{name} must live on the context's CUDA device")


def _on(ctx: Context, t: torch.Tensor, name: str) -> torch.Tensor:
    if t.get_device() != (ctx.device.index or 0):
        raise _elsewhere(name)
    return t


class PagedBatch:
    """A ragged batch (``ttq_paged_batch``): rows ``q_start[b] .. q_start[b+1]-1`` are the newest of the ``kv_len[b]`` tokens of
    sequence b, whose pages are ``block_table[b]``.  int32 tensors on the device; their contents may change between calls (a
    captured graph follows them), ``max_q`` is the most new tokens of any sequence (it selects the kernel only; 0: unknown, slow for
    many short ones).
    With ``prefix_len`` all sequences begin with the tokens of ``prefix_table``'s pages; ``kv_len`` counts them, the
    block tables start behind them."""

    def __init__(self, q_start: torch.Tensor, kv_len: torch.Tensor, block_table: torch.Tensor, max_q: int = 0, prefix_len: int = 0,
                 prefix_table: Optional[torch.Tensor] = None):
        n = kv_len.numel()
        for name, t, dim in (("q_start", q_start, 1), ("kv_len", kv_len, 1), ("block_table", block_table, 2), ("prefix_table", prefix_table, 1)):
            if t is None:
                continue
            if t.dtype != torch.int32 or t.dim() != dim or not t.is_cuda:
                raise TtqError(1, f"{name} must be a {dim}-D int32 tensor on the device")
            if t.numel() and t.stride(-1) != 1:
                raise TtqError(2, f"{name} must be contiguous along its last dimension")
            if t.device != q_start.device:
                raise TtqError(1, f"{name} is on another device than q_start")
        if q_start.numel() != n + 1 or block_table.shape[0] != n:
            raise TtqError(2, f"q_start and block_table do not fit {n} sequences")
        self.q_start, self.kv_len, self.block_table, self.prefix_table = q_start, kv_len, block_table, prefix_table
        self.n_seqs, self.max_q, self.prefix_len, self.device = n, max_q, prefix_len, q_start.get_device()
        self._args = PagedBatchArgs(n, 0, max_q, q_start.data_ptr(), kv_len.data_ptr(), block_table.data_ptr(), block_table.shape[1],
                                    block_table.stride(0) if n > 1 else block_table.shape[1], prefix_len,
                                    None if prefix_table is None else prefix_table.data_ptr())
        self._page_entries = 0 if prefix_table is None else prefix_table.numel()

    def _for(self, plan: "PagedAttention", n_tokens: int) -> PagedBatchArgs:
        if self.device != plan.device:
            raise _elsewhere("the batch's tensors")
        page_size = plan.page_size
        if self.prefix_len > self._page_entries * page_size:
            raise TtqError(2, f"prefix_table has {self._page_entries} pages of {page_size}, prefix_len is {self.prefix_len}")
        args = self._args
        if args.n_tokens != n_tokens:  # (a copy: another thread's call may hold the present ones)
            args = PagedBatchArgs.from_buffer_copy(args)
            args.n_tokens = n_tokens
            self._args = args
        return args


class PagedAttention:
    """Head geometry and workspace of paged attention (``ttq_paged_create``); one object serves all layers of a model, its calls
    follow each other on one stream.  ``max_prefix_tokens`` (default: ``max_tokens``) makes room for calls with a
    shared prefix, (head_dim + 1) * 4 bytes per token and query head; 0 where no batch has one.  A layer's cache is a pair of tensors ``[n_pages, n_kv_heads, page_size, head_dim]`` (any
    strides with a contiguous head dimension, so a permuted view of another layout will do)."""

    def __init__(self, ctx: Context, n_q_heads: int, n_kv_heads: int, head_dim: int, page_size: int, max_seqs: int, max_tokens: int,
                 dtype: torch.dtype = torch.bfloat16, max_prefix_tokens: Optional[int] = None):
        self.ctx, self.hq, self.hkv, self.d, self.page_size, self.dtype = ctx, n_q_heads, n_kv_heads, head_dim, page_size, dtype
        self.device, self.scale = ctx.device.index or 0, 1.0 / math.sqrt(head_dim)
        h = ctypes.c_void_p()
        check(ctx.handle, ctx._lib.ttq_paged_create(ctx.handle, _dt(dtype), n_q_heads, n_kv_heads, head_dim, page_size, max_seqs, max_tokens,
                                                    max_tokens if max_prefix_tokens is None else max_prefix_tokens, ctypes.byref(h)))
        self.handle = h

    def _pages(self, k_pages: torch.Tensor, v_pages: torch.Tensor) -> KvPages:
        shape, st = k_pages.shape, k_pages.stride()
        if len(shape) != 4 or shape[1] != self.hkv or shape[2] != self.page_size or shape[3] != self.d or v_pages.shape != shape:
            raise TtqError(2, f"pages must be [n_pages, {self.hkv}, {self.page_size}, {self.d}], k and v alike")
        if k_pages.dtype != self.dtype or v_pages.dtype != self.dtype:
            raise TtqError(1, f"pages must be {self.dtype}")
        if k_pages.get_device() != self.device or v_pages.get_device() != self.device:
            raise _elsewhere("k_pages and v_pages")
        if st != v_pages.stride() or st[3] != 1:
            raise TtqError(2, "k and v pages must have the same strides and a contiguous head dimension")
        return KvPages(k_pages.data_ptr(), v_pages.data_ptr(), shape[0], st[0], st[1], st[2])

    def _rows(self, t: torch.Tensor, heads: int, name: str):
        """``t`` as rows of ``heads`` x head_dim values: a tensor that owns them, their number and pitch."""
        shape, width = t.shape, heads * self.d
        if len(shape) == 3:
            if shape[1] != heads or shape[2] != self.d:
                raise TtqError(2, f"{name} is {tuple(shape)}, expected [rows, {heads}, {self.d}]")
        elif len(shape) != 2 or shape[1] != width:
            raise TtqError(2, f"{name} is {tuple(shape)}, expected [rows, {width}]")
        if t.dtype != self.dtype:
            raise TtqError(1, f"{name} must be {self.dtype}")
        if t.get_device() != self.device:
            raise _elsewhere(name)
        st = t.stride()
        if st[-1] != 1 or (len(shape) == 3 and st[1] != self.d and heads > 1):
            t = t.contiguous()
            st = t.stride()
        return t, shape[0], st[0] if shape[0] > 1 else width

    def _out(self, out: Optional[torch.Tensor], n: int, like: torch.Tensor, name: str):
        """The result tensor and its row pitch."""
        width = self.hq * self.d
        if out is None:
            return torch.empty((n, self.hq, self.d), dtype=self.dtype, device=like.device), width
        _on(self.ctx, out, name)
        if out.dtype != self.dtype or out.numel() != n * width or out.shape[0] != n:
            raise TtqError(2, f"{name} must be [{n}, {self.hq}, {self.d}] {self.dtype}")
        inner = out.stride()[1:]
        if inner != ((self.d, 1) if out.dim() == 3 else (1,)):
            raise TtqError(2, f"the rows of {name} must be contiguous")
        return out, out.stride(0) if n > 1 else width

    def append(self, qkv: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, batch: PagedBatch, cos: torch.Tensor, sin: torch.Tensor,
               q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
               q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Normalises (where weights ``[head_dim]`` are given) and rotates the q and k heads of fused qkv rows, writes k and v into the
        sequences' pages, returns q ``[n_tokens, n_q_heads, head_dim]``.  ``cos`` / ``sin``: ``[positions, head_dim]``, f32 or the
        plan's dtype."""
        rows, n, ld = self._rows(qkv, self.hq + 2 * self.hkv, "qkv")
        if cos.shape != sin.shape or cos.dim() != 2 or cos.shape[1] != self.d or cos.dtype != sin.dtype:
            raise TtqError(2, f"cos and sin must be [positions, {self.d}], alike")
        cos, sin = _on(self.ctx, cos, "cos").contiguous(), _on(self.ctx, sin, "sin").contiguous()
        norms = []
        for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
            if w is not None and (w.dtype != self.dtype or w.numel() != self.d or not w.is_contiguous()):
                raise TtqError(2, f"{name} must be {self.d} contiguous values of {self.dtype}")
            norms.append(None if w is None else _on(self.ctx, w, name).data_ptr())
        q_out, ld_q = self._out(q_out, n, rows, "q_out")
        ctx = self.ctx
        st = ctx._lib.ttq_paged_append(ctx.handle, self.handle, self._pages(k_pages, v_pages), batch._for(self, n), rows.data_ptr(), ld,
                                       norms[0], norms[1], eps, cos.data_ptr(), sin.data_ptr(),
                                       _dt(cos.dtype), cos.shape[0], q_out.data_ptr(), ld_q, _stream_ptr(rows.device))
        if st != 0:
            check(ctx.handle, st)
        return q_out

    def forward(self, q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, batch: PagedBatch, window: int = 0, sinks: int = 0,
                scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of the batch's rows ``q`` ``[n_tokens, n_q_heads, head_dim]`` over their sequences' pages.  With ``window``
        a token sees the ``window`` latest positions (its own among them) and the first ``sinks`` of the sequence."""
        rows, n, ld = self._rows(q, self.hq, "q")
        out, ld_out = self._out(out, n, rows, "out")
        ctx = self.ctx
        st = ctx._lib.ttq_paged_attention(ctx.handle, self.handle, self._pages(k_pages, v_pages), batch._for(self, n), rows.data_ptr(),
                                          ld, self.scale if scale is None else scale, window, sinks, out.data_ptr(), ld_out, _stream_ptr(rows.device))
        if st != 0:
            check(ctx.handle, st)
        return out

    __call__ = forward

    def close(self) -> None:
        if getattr(self, "handle", None):
            self.ctx._lib.ttq_paged_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def sample(ctx: Context, logits: torch.Tensor, u: torch.Tensor, temperature: Union[float, torch.Tensor] = 1.0, top_k: Union[int, torch.Tensor] = 0,
           top_p: Union[float, torch.Tensor] = 1.0, min_p: Union[float, torch.Tensor] = 0.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The next token (int64) of every row of ``logits`` ``[rows, vocabulary]``, drawn with the random numbers ``u`` ``[rows]`` (f32 in
    [0, 1); others count as the nearest, NaN as 0).  ``logits`` may be one row expanded to many.  Settings are one value for all rows or a tensor of one per row; top-k, then top-p, then min-p, as ``ttq_sample`` defines
    them.  A temperature of 0 takes the largest logit, the lowest index among equals; a row with nothing but -inf (or NaN) gives -1."""
    if logits.dim() != 2:
        raise TtqError(2, "logits must be [rows, vocabulary]")
    _on(ctx, logits, "logits")
    m, v = logits.shape
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    s = Sampling()
    keep = []
    for name, value, dtype in (("temperature", temperature, torch.float32), ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32),
                               ("top_k", top_k, torch.int32)):
        if isinstance(value, torch.Tensor):
            if value.numel() != m or value.dtype != dtype or not value.is_contiguous():
                raise TtqError(2, f"{name} must be one value or {m} contiguous values of {dtype}")
            keep.append(_on(ctx, value, name))
            setattr(s, name + "_dev", value.data_ptr())
        else:
            setattr(s, name, max(0, min(value, 2 ** 31 - 1)) if name == "top_k" else value)  # (ctypes would wrap it)
    if u.numel() != m or u.dtype != torch.float32 or not u.is_contiguous():
        raise TtqError(2, f"u must be {m} contiguous values of float32")
    _on(ctx, u, "u")
    if out is None:
        out = torch.empty((m,), dtype=torch.int64, device=logits.device)
    elif _on(ctx, out, "out").dtype != torch.int64 or out.numel() != m or not out.is_contiguous():
        raise TtqError(2, f"out must be {m} contiguous int64 values")
    st = ctx._lib.ttq_sample(ctx.handle, logits.data_ptr(), _dt(logits.dtype), m, v, logits.stride(0) if m > 1 else v, ctypes.byref(s), u.data_ptr(),
                             out.data_ptr(), _stream_ptr(logits.device))
    if st != 0:
        check(ctx.handle, st)
    return out
