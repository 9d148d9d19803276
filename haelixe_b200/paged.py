"""Attention one token at a time over a paged key/value cache.

The reference attends over whole sequences only (`MultiHeadAttention::forward`,
src/nn/attention.rs:46-98) and keeps no keys between calls. A model that answers
token by token appends each new token's keys and values to a cache
(`paged_append`, which rotates k and q by their positions on the way, the pairs of
src/kernels/rope.rs:5-44) and attends from the new queries to the cached
positions (`paged_attention`, the formula of `Tensor::flash_attention`,
src/tensor.rs:644-666, for one query a sequence).

Both are for inference: they have no backward and refuse tensors that would
need one. Calls of several host threads may overlap: each runs on its thread's
current stream.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _native as N
from .attention import _DTYPES, context


def _no_grad_needed(who: str, *ts: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise RuntimeError(f"{who} has no backward: call it under torch.no_grad()")


class PagedKVCache:
    """Keys and values of many sequences in pages, and the table that maps them.

    k, v: [pages, slots, heads, head_dim] on one device, f32 or bf16, with equal
    strides and a contiguous head_dim (a multiple of 8, at most 256); a transposed
    view of [pages, heads, slots, head_dim] storage is as good. block_table:
    int32 [sequences, columns]; entry (s, c) is the page of positions
    [c * slots, (c + 1) * slots) of sequence s. The tensors stay the caller's:
    their values, the table's among them, may change between calls.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor):
        for t in (k, v, block_table):
            if not t.is_cuda:
                raise RuntimeError("the paged cache requires CUDA tensors")
        if k.dtype not in _DTYPES:
            raise TypeError(f"unsupported dtype {k.dtype}; f32 and bf16 are supported")
        if block_table.dtype != torch.int32:
            raise TypeError("block_table must be int32")
        if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
            raise ValueError("k and v must be [pages, slots, heads, head_dim] of one dtype and device")
        if block_table.dim() != 2 or block_table.device != k.device:
            raise ValueError("block_table must be [sequences, columns] on the cache's device")
        if k.stride(3) != 1 or any(n > 1 and a != b for n, a, b in zip(k.shape, k.stride(), v.stride())):
            raise ValueError("k and v must share strides, with a contiguous head dimension")
        if block_table.shape[1] > 1 and block_table.stride(1) != 1:
            raise ValueError("rows of block_table must be contiguous")
        pages, slots, heads, dim = k.shape
        # The stride of a dimension of size 1 never moves an address: give it one that is in order.
        sh = k.stride(2) if heads > 1 else dim
        ss = k.stride(1) if slots > 1 else max(dim, heads * sh)
        sp = k.stride(0) if pages > 1 else slots * ss
        seqs, columns = block_table.shape
        self._k, self._v, self._table = k, v, block_table
        self._c = N.PagedCache(k.data_ptr(), v.data_ptr(), block_table.data_ptr(), sp, ss, sh,
                               block_table.stride(0) if seqs > 1 else columns, pages, slots, heads, dim, seqs, columns)
        self._ref = ctypes.byref(self._c)
        self._dt = _DTYPES[k.dtype]
        self._workspace: dict[int, int] = {}  # bytes by query heads
        self.dtype, self.device = k.dtype, k.device
        self.num_seqs, self.heads, self.head_dim = seqs, heads, dim
        self.workspace_bytes(heads)  # refuses a cache that the kernels cannot address

    @classmethod
    def allocate(cls, pages: int, slots: int, heads: int, head_dim: int, block_table: torch.Tensor,
                 dtype=torch.bfloat16) -> "PagedKVCache":
        """A cache of zeros on the table's device."""
        k, v = (torch.zeros(pages, slots, heads, head_dim, dtype=dtype, device=block_table.device) for _ in range(2))
        return cls(k, v, block_table)

    @property
    def k(self) -> torch.Tensor:
        return self._k

    @property
    def v(self) -> torch.Tensor:
        return self._v

    @property
    def block_table(self) -> torch.Tensor:
        return self._table

    def workspace_bytes(self, query_heads: int) -> int:
        n = self._workspace.get(query_heads)
        if n is None:
            out = ctypes.c_uint64()
            st = N.lib().hx_paged_attention_workspace_size(self._dt, self._ref, query_heads, ctypes.byref(out))
            if st != N.HX_OK:
                raise N.HxError(st, f"no paged attention for {query_heads} query heads over a cache of shape "
                                    f"{tuple(self._k.shape)} (head_dim a multiple of 8 up to 256, 16-byte aligned "
                                    "strides, query heads a multiple of the cache's)")
            n = self._workspace[query_heads] = out.value
        return n


def _rows(cache: PagedKVCache, who: str, name: str, t: torch.Tensor, rows: int, heads: Optional[int]) -> N.Rows:
    if t.dim() != 3 or t.shape[0] != rows or t.shape[2] != cache.head_dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{who}: {name} must be [{rows}, {heads or 'heads'}, {cache.head_dim}], got {tuple(t.shape)}")
    if t.dtype != cache.dtype or t.device != cache.device:
        raise ValueError(f"{who}: {name} must have the cache's dtype and device")
    s0, s1, s2 = t.stride()
    if s2 != 1:
        raise ValueError(f"{who}: the head dimension of {name} must be contiguous")
    # The stride of a dimension of size 1 never moves an address.
    if t.shape[1] == 1:
        s1 = cache.head_dim
    if rows == 1:
        s0 = t.shape[1] * s1
    return N.Rows(t.data_ptr(), s0, s1)


def _indices(cache: PagedKVCache, who: str, name: str, t: torch.Tensor, n: int):
    if t.dtype != torch.int32:
        raise TypeError(f"{who}: {name} must be int32")
    if t.dim() != 1 or t.shape[0] != n or t.device != cache.device or not t.is_contiguous():
        raise ValueError(f"{who}: {name} must be a contiguous vector of {n} on the cache's device")
    return t.data_ptr()


def paged_append(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor, seq_ids: torch.Tensor,
                 positions: torch.Tensor, rope_base: Optional[float] = None, q: Optional[torch.Tensor] = None,
                 out_q: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes k and v [tokens, heads, head_dim] of new tokens to their places in the cache.

    Token t is position positions[t] of sequence seq_ids[t] (int32 on the device).
    With rope_base, k is rotated by its position, and so is q [tokens, query
    heads, head_dim], in the same launch; the result is out_q (a new tensor by
    default; q itself for in place). A negative seq_id marks padding: nothing of
    that token is written, its row of out_q included. A token whose sequence or
    position the table does not hold, or whose entry there is no page, writes
    nothing to the cache and NaN to its row of out_q.
    """
    who = "paged_append"
    _no_grad_needed(who, k, v, q)
    n = k.shape[0]
    kr, vr = _rows(cache, who, "k", k, n, cache.heads), _rows(cache, who, "v", v, n, cache.heads)
    ids, pos = _indices(cache, who, "seq_ids", seq_ids, n), _indices(cache, who, "positions", positions, n)
    heads, qr, orr = 0, None, None
    if q is not None:
        qr = _rows(cache, who, "q", q, n, None)
        heads = q.shape[1]
        if out_q is None:
            out_q = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        orr = _rows(cache, who, "out_q", out_q, n, heads)
        qr, orr = ctypes.byref(qr), ctypes.byref(orr)
    elif out_q is not None:
        raise ValueError("paged_append: out_q without q")
    base = 0.0
    if rope_base is not None:
        base = float(rope_base)
        if not base > 0.0:
            raise ValueError("paged_append: rope_base must be positive")
    ctx = context(cache.device.index)
    with ctx.lock:
        ctx.use_stream()
        N.check(N.lib().hx_paged_append(ctx.handle, cache._dt, cache._ref, n, ctypes.byref(kr), ctypes.byref(vr), ids,
                                        pos, heads, qr, orr, base), ctx.handle)
    return out_q


def paged_attention(cache: PagedKVCache, q: torch.Tensor, seq_lens: torch.Tensor, scale: float,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None):
    """Attention of one query a sequence over its first seq_lens[s] cached positions.

    q: [sequences, query heads, head_dim], query heads a multiple of the cache's;
    seq_lens: int32 [sequences] on the device. Returns (o like q, lse f32
    [sequences, query heads]). A length of 0 gives zeros and an lse of -inf; a
    length past the table row, or a table entry that is no page, gives NaN. What
    the cache holds at or past seq_lens is not read.
    """
    who = "paged_attention"
    _no_grad_needed(who, q)
    qr = _rows(cache, who, "q", q, cache.num_seqs, None)
    heads = q.shape[1]
    lens = _indices(cache, who, "seq_lens", seq_lens, cache.num_seqs)
    need = cache.workspace_bytes(heads)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    orr = _rows(cache, who, "out", out, cache.num_seqs, heads)
    if lse is None:
        lse = torch.empty(q.shape[0], heads, dtype=torch.float32, device=q.device)
    elif lse.shape != q.shape[:2] or lse.dtype != torch.float32 or lse.device != q.device or not lse.is_contiguous():
        raise ValueError("paged_attention: lse must be a contiguous f32 [sequences, query heads]")
    # A tensor of the current stream, so that calls on other streams and captured graphs have their own.
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    ctx = context(cache.device.index)
    with ctx.lock:
        ctx.use_stream()
        N.check(N.lib().hx_paged_attention(ctx.handle, cache._dt, cache._ref, heads, ctypes.byref(qr),
                                           ctypes.byref(orr), lse.data_ptr(), lens, float(scale), ws.data_ptr(), need),
                ctx.handle)
    return out, lse
