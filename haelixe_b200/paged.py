"""Attention one token at a time over a paged key/value cache.

The reference attends over whole sequences only (`MultiHeadAttention::forward`,
src/nn/attention.rs:46-98) and keeps no keys between calls. A model that answers
token by token appends each new token's keys and values to a cache
(`paged_append`, which rotates k and q by their positions on the way, the pairs of
src/kernels/rope.rs:5-44) and attends from the new queries to the cached
positions (`paged_attention`, the formula of `Tensor::flash_attention`,
src/tensor.rs:644-666, for one query a sequence).

Both are for inference: they have no backward and refuse tensors that would
need one. They may be called from several host threads at once: each call runs
on its thread's current stream.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _native as N
from .attention import _DTYPES, context, has_tangent


class PagedKVCache:
    """Keys and values of many sequences in pages, and the table that maps them.

    k, v: [pages, slots, heads, head_dim] on one device, f32 or bf16, with equal
    strides and a contiguous head_dim (a multiple of 8, at most 256); a transposed
    view of [pages, heads, slots, head_dim] storage is as good. block_table:
    int32 [sequences, columns]; entry (s, c) is the page of positions
    [c * slots, (c + 1) * slots) of sequence s. The tensors stay the caller's:
    their values, the table's among them, may change between calls, their memory may not.
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
        N.check_sizes("the paged cache", *k.shape, *block_table.shape)
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
        self._dev = k.get_device()
        self._ctx = context(self._dev)
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


# The calls are made once a layer and token, so their checks are kept to a few
# attribute reads. Operands go to the library as hx_rows: address, stride of a row, stride of a
# head, packed into bytes, which cost a fraction of a ctypes structure.
_pack_rows = struct.Struct("Pqq").pack


def _rows(cache: PagedKVCache, who: str, name: str, t: torch.Tensor, rows: int, heads: int) -> bytes:
    if t.shape != (rows, heads, cache.head_dim):
        raise ValueError(f"{who}: {name} must be [{rows}, {heads}, {cache.head_dim}], got {tuple(t.shape)}")
    if t.dtype is not cache.dtype or t.get_device() != cache._dev:
        raise ValueError(f"{who}: {name} must have the cache's dtype and device")
    s0, s1, s2 = t.stride()
    if s2 != 1:
        raise ValueError(f"{who}: the head dimension of {name} must be contiguous")
    # The stride of a dimension of size 1 never moves an address.
    if heads == 1:
        s1 = cache.head_dim
    if rows == 1:
        s0 = heads * s1
    return _pack_rows(t.data_ptr(), s0, s1)


def _indices(cache: PagedKVCache, who: str, name: str, t: torch.Tensor, n: int) -> int:
    if t.dtype is not torch.int32:
        raise TypeError(f"{who}: {name} must be int32")
    if t.dim() != 1 or t.shape[0] != n or t.get_device() != cache._dev or not t.is_contiguous():
        raise ValueError(f"{who}: {name} must be a contiguous vector of {n} on the cache's device")
    return t.data_ptr()


def _refuse_derivative(who: str, grad: bool) -> None:
    raise RuntimeError(f"{who} has no backward: call it under torch.no_grad()" if grad else
                       f"{who} has no forward-mode derivative")


def paged_append(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor, seq_ids: torch.Tensor,
                 positions: torch.Tensor, rope_base: Optional[float] = None, q: Optional[torch.Tensor] = None,
                 out_q: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes k and v [tokens, heads, head_dim] of new tokens to their places in the cache.

    Token t is position positions[t] of sequence seq_ids[t] (int32 on the device).
    With rope_base, k is rotated by its position, and so is q [tokens, query
    heads, head_dim], in the same launch; the result is out_q (a new tensor by
    default; q itself for in place; memory of its own otherwise). A negative seq_id marks padding: nothing of
    that token is written, its row of out_q included. No two tokens may have the same
    place. A token whose sequence or
    position the table does not hold, or whose entry there is no page, writes
    nothing to the cache and NaN to its row of out_q.
    """
    who = "paged_append"
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or cache._k.requires_grad or cache._v.requires_grad
                                    or q is not None and q.requires_grad or out_q is not None and out_q.requires_grad):
        _refuse_derivative(who, True)
    if forward_ad._current_level >= 0 and has_tangent(cache._k, cache._v, k, v, q, out_q):
        _refuse_derivative(who, False)
    n = k.shape[0]
    if n > 0x7fffffff:
        N.check_sizes(who, n)
    kr, vr = _rows(cache, who, "k", k, n, cache.heads), _rows(cache, who, "v", v, n, cache.heads)
    ids, pos = _indices(cache, who, "seq_ids", seq_ids, n), _indices(cache, who, "positions", positions, n)
    base = 0.0
    if rope_base is not None:
        base = float(rope_base)
        if not base >= 1e-30:  # 0 stands for no rotation below
            raise ValueError("paged_append: rope_base must be positive")
    if q is not None:
        heads = q.shape[1] if q.dim() == 3 else 0
        qr = _rows(cache, who, "q", q, n, heads)
        if out_q is None:
            out_q = torch.empty_like(q)
        outr = qr if out_q is q else _rows(cache, who, "out_q", out_q, n, heads)
    else:
        if out_q is not None:
            raise ValueError("paged_append: out_q without q")
        heads, qr, outr = 0, None, None
    cache._ctx.call(N.lib().hx_paged_append, cache._dt, cache._ref, n, kr, vr, ids, pos, heads, qr, outr, base)
    return out_q


def paged_attention(cache: PagedKVCache, q: torch.Tensor, seq_lens: torch.Tensor, scale: float,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None):
    """Attention of one query a sequence over its first seq_lens[s] cached positions.

    q: [sequences, query heads, head_dim], every row on a 16-byte boundary, query
    heads a multiple of the cache's; seq_lens: int32 [sequences] on the device.
    Returns (o like q, or out, which may be q itself or else memory of its own; lse f32 [sequences, query
    heads]). A length of 0 gives zeros and an lse of -inf; a length past the table
    row, or a table entry that is no page, gives NaN. What
    the cache holds at or past seq_lens is not read.
    """
    who = "paged_attention"
    if torch.is_grad_enabled() and (q.requires_grad or cache._k.requires_grad or cache._v.requires_grad or
                                    out is not None and out.requires_grad or lse is not None and lse.requires_grad):
        _refuse_derivative(who, True)
    if forward_ad._current_level >= 0 and has_tangent(cache._k, cache._v, q, out, lse):
        _refuse_derivative(who, False)
    n, heads = cache.num_seqs, q.shape[1] if q.dim() == 3 else 0
    qr = _rows(cache, who, "q", q, n, heads)
    lens = _indices(cache, who, "seq_lens", seq_lens, n)
    need = cache.workspace_bytes(heads)
    if out is None:
        out = torch.empty_like(q)
    outr = qr if out is q else _rows(cache, who, "out", out, n, heads)
    if lse is None:
        lse = q.new_empty((n, heads), dtype=torch.float32)
    elif lse.shape != (n, heads) or lse.dtype is not torch.float32 or lse.get_device() != cache._dev or not lse.is_contiguous():
        raise ValueError("paged_attention: lse must be a contiguous f32 [sequences, query heads]")
    # A tensor of the current stream, so that calls on other streams and captured graphs have their own.
    ws = q.new_empty(need, dtype=torch.uint8)
    cache._ctx.call(N.lib().hx_paged_attention, cache._dt, cache._ref, heads, qr, outr, lse.data_ptr(), lens, float(scale),
                    ws.data_ptr(), need)
    return out, lse
