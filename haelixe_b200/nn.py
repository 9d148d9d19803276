"""Device-resident layers around the fused kernel.

Mirrors haelixe's `nn` modules: `RMSNorm` (src/nn/rms_norm.rs,
kernels/rms_norm.rs), `Linear` (src/nn/linear.rs), `MultiHeadAttention`
(src/nn/attention.rs:46-98), `FeedForward` (src/nn/mlp.rs) and
`TransformerBlock` (src/nn/transformer.rs), plus the pieces a language-model
training step over a block stack needs: a token `Embedding` (the reference
has none), `cross_entropy` (src/tensor.rs:754-801) and `BlockStack`, and those
that it answers with: `prefill` and `decode` over paged key/value caches,
`token_logprobs`, and Linear weights in 4 bits (`LinearW4`). Every op
runs on the GPU through the library's C ABI: RMSNorm and GELU kernels, Linear
as cuBLAS GEMMs (weights stored [in, out] as in linear.rs:41) with the bias
and the block's residual add folded into the GEMM's C operand, and the fused
attention with RoPE. The reference's head split/merge copies
(`view -> transpose -> view`, attention.rs:62-73, 91-94) become strided
[B, H, S, D] views of the projection outputs: no data moves. Gradients flow
through torch.autograd, one Function per op, like the reference's `Op` nodes.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _native as N
from .attention import _DTYPES, context, flash_attention, has_tangent
from .paged import PagedKVCache, paged_append, paged_attention


def _p(t: Optional[torch.Tensor]) -> Optional[int]:
    """t's address; the caller keeps t until the call is made."""
    return None if t is None else t.data_ptr()


def _context_of(t: torch.Tensor):
    """The context of t's device."""
    if not t.is_cuda:
        raise RuntimeError("the attention block runs on CUDA tensors")
    if t.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {t.dtype}; f32 and bf16 are supported")
    return context(t.get_device())


class _RMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(fctx, x, w, eps):
        c = _context_of(x)
        x = x.contiguous()
        hidden = x.shape[-1]
        y = torch.empty_like(x)
        wc = w.contiguous()
        c.call(N.lib().hx_rmsnorm_fwd, _DTYPES[x.dtype], x.data_ptr(), wc.data_ptr(), y.data_ptr(), x.numel() // hidden,
               hidden, float(eps))
        fctx.save_for_backward(x, w)
        fctx.eps = eps
        return y

    @staticmethod
    def backward(fctx, dy):
        x, w = fctx.saved_tensors
        c = _context_of(x)
        dy = dy.contiguous()
        hidden = x.shape[-1]
        dx = torch.empty_like(x)
        dw = torch.empty(hidden, dtype=torch.float32, device=x.device)
        wc = w.contiguous()
        c.call(N.lib().hx_rmsnorm_bwd, _DTYPES[x.dtype], dy.data_ptr(), x.data_ptr(), wc.data_ptr(), dx.data_ptr(),
               dw.data_ptr(), x.numel() // hidden, hidden, float(fctx.eps))
        return dx, dw.to(w.dtype), None


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(fctx, x, w, b, r=None):
        c = _context_of(x)
        in_f, out_f = w.shape
        x2 = x.reshape(-1, in_f).contiguous()
        y = torch.empty(x2.shape[0], out_f, dtype=x.dtype, device=x.device)
        wc, bc = w.contiguous(), None if b is None else b.contiguous()
        if r is None:
            c.call(N.lib().hx_linear_fwd, _DTYPES[x.dtype], x2.data_ptr(), wc.data_ptr(), _p(bc), y.data_ptr(),
                   x2.shape[0], in_f, out_f)
        else:
            r2 = r.reshape(x2.shape[0], out_f).contiguous()
            c.call(N.lib().hx_linear_residual_fwd, _DTYPES[x.dtype], x2.data_ptr(), wc.data_ptr(), _p(bc),
                   r2.data_ptr(), y.data_ptr(), x2.shape[0], in_f, out_f)
        fctx.save_for_backward(x2, w)
        fctx.in_shape, fctx.has_bias, fctx.has_res = x.shape, b is not None, r is not None
        return y.view(*x.shape[:-1], out_f)

    @staticmethod
    def backward(fctx, dy):
        x2, w = fctx.saved_tensors
        c = _context_of(x2)
        in_f, out_f = w.shape
        dy2 = dy.reshape(-1, out_f).contiguous()
        need_x, need_w, need_b = fctx.needs_input_grad[:3]
        dx = torch.empty_like(x2) if need_x else None
        dw = torch.empty_like(w) if need_w else None
        db = torch.empty(out_f, dtype=w.dtype, device=w.device) if (need_b and fctx.has_bias) else None
        wc = w.contiguous()
        c.call(N.lib().hx_linear_bwd, _DTYPES[x2.dtype], x2.data_ptr(), wc.data_ptr(), dy2.data_ptr(), _p(dx), _p(dw),
               _p(db), x2.shape[0], in_f, out_f)
        dr = dy if fctx.has_res else None  # y = r + ...: the residual's gradient is dy itself
        return (None if dx is None else dx.view(fctx.in_shape)), dw, db, dr


class _GeluFn(torch.autograd.Function):
    @staticmethod
    def forward(fctx, x):
        c = _context_of(x)
        x = x.contiguous()
        y = torch.empty_like(x)
        c.call(N.lib().hx_gelu_fwd, _DTYPES[x.dtype], x.data_ptr(), y.data_ptr(), x.numel())
        fctx.save_for_backward(x)
        return y

    @staticmethod
    def backward(fctx, dy):
        (x,) = fctx.saved_tensors
        c = _context_of(x)
        dy = dy.contiguous()
        dx = torch.empty_like(x)
        c.call(N.lib().hx_gelu_bwd, _DTYPES[x.dtype], dy.data_ptr(), x.data_ptr(), dx.data_ptr(), x.numel())
        return dx


def _ids(ids: torch.Tensor) -> torch.Tensor:
    if ids.dtype not in (torch.int32, torch.int64, torch.uint32):
        raise TypeError("token ids / targets must be an integer tensor")
    return ids.reshape(-1).to(torch.int32).contiguous()  # read as uint32 by the kernels


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(fctx, ids, table):
        c = _context_of(table)
        vocab, dim = table.shape
        flat = _ids(ids)
        out = torch.empty(flat.numel(), dim, dtype=table.dtype, device=table.device)
        rows = table.contiguous()
        c.call(N.lib().hx_embedding_fwd, _DTYPES[table.dtype], rows.data_ptr(), flat.data_ptr(), out.data_ptr(),
               flat.numel(), vocab, dim)
        fctx.save_for_backward(flat)
        fctx.vocab, fctx.table_dtype = vocab, table.dtype
        return out.view(*ids.shape, dim)

    @staticmethod
    def backward(fctx, dout):
        (flat,) = fctx.saved_tensors
        c = _context_of(dout)
        dim = dout.shape[-1]
        dout = dout.contiguous()
        dtable = torch.zeros(fctx.vocab, dim, dtype=torch.float32, device=dout.device)
        c.call(N.lib().hx_embedding_bwd, _DTYPES[dout.dtype], dout.data_ptr(), flat.data_ptr(), dtable.data_ptr(),
               flat.numel(), fctx.vocab, dim)
        return None, dtable.to(fctx.table_dtype)


class _CrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(fctx, logits, targets):
        c = _context_of(logits)
        rows, classes = logits.shape
        logits = logits.contiguous()
        flat = _ids(targets)
        if flat.numel() != rows:
            raise ValueError("targets length must match the number of logit rows")
        loss = torch.empty((), dtype=torch.float32, device=logits.device)
        dlogits = torch.empty_like(logits) if fctx.needs_input_grad[0] else None
        c.call(N.lib().hx_cross_entropy, _DTYPES[logits.dtype], logits.data_ptr(), flat.data_ptr(), loss.data_ptr(),
               _p(dlogits), rows, classes)
        fctx.dlogits = dlogits
        return loss

    @staticmethod
    def backward(fctx, _dloss):
        # Like ops/cross_entropy.rs:18-50 the loss is the graph's root: the
        # stored (softmax - onehot) / rows is the gradient, the upstream one is 1.
        d, fctx.dlogits = fctx.dlogits, None
        return d, None


class TokenLogprobs(NamedTuple):
    """What token_logprobs returns; the top_ fields are None without alternatives."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_ids: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]


def _token_logprobs(logits, flat, top_k, with_stats):
    rows, classes = logits.shape
    stride = logits.stride(0) if rows > 1 else classes
    c = _context_of(logits)
    logprob = logits.new_empty(rows, dtype=torch.float32)
    entropy = torch.empty_like(logprob)
    stats = logits.new_empty((rows, 3), dtype=torch.float32) if with_stats else None
    ids = top = None
    if top_k:
        ids = logits.new_empty((rows, top_k), dtype=torch.int32)
        top = logits.new_empty((rows, top_k), dtype=torch.float32)
    c.call(N.lib().hx_token_logprobs_fwd, _DTYPES[logits.dtype], logits.data_ptr(), stride, flat.data_ptr(),
           logprob.data_ptr(), entropy.data_ptr(), stats.data_ptr() if with_stats else None, top_k,
           ids.data_ptr() if top_k else None, top.data_ptr() if top_k else None, rows, classes)
    return logprob, entropy, ids, top, stats


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(fctx, logits, flat, top_k):
        logprob, entropy, ids, top, stats = _token_logprobs(logits, flat, top_k, True)
        fctx.save_for_backward(logits, flat, stats)
        fctx.set_materialize_grads(False)
        if top_k:
            fctx.mark_non_differentiable(ids, top)
        return logprob, entropy, ids, top

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(fctx, g_logprob, g_entropy, _ids, _top):
        logits, flat, stats = fctx.saved_tensors
        rows, classes = logits.shape
        if g_logprob is None and g_entropy is None:
            return None, None, None
        stride = logits.stride(0) if rows > 1 else classes
        # Rows at the logits' stride, so that 16-byte pieces line up in both (unless that wastes memory).
        dstride = stride if stride <= 2 * classes else classes
        d = torch.empty_strided((rows, classes), (dstride, 1), dtype=logits.dtype, device=logits.device)
        gl = None if g_logprob is None else g_logprob.contiguous()
        gh = None if g_entropy is None else g_entropy.contiguous()
        _context_of(logits).call(N.lib().hx_token_logprobs_bwd, _DTYPES[logits.dtype], logits.data_ptr(), stride,
                                 flat.data_ptr(), stats.data_ptr(), _p(gl), _p(gh), d.data_ptr(), dstride, rows, classes)
        return d, None, None


def gelu(x: torch.Tensor) -> torch.Tensor:
    """Tensor::gelu (kernels/activations.rs:192-237, tanh form) with its backward."""
    return _GeluFn.apply(x)


def embedding(ids: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """table[ids]: [..., dim] rows of a [vocab, dim] table; its gradient is a scatter-add."""
    return _EmbeddingFn.apply(ids, table)


def cross_entropy(logits: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    """Tensor::cross_entropy (src/tensor.rs:754-801): mean over rows of
    logsumexp(row) - row[target], a device scalar; logits [rows, classes]."""
    return _CrossEntropyFn.apply(logits, targets)


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """log softmax(logits)[r, targets[r]] and the entropy of each row, f32 [rows];
    logits [rows, classes] with contiguous rows, targets an integer vector.
    With top_k (at most 32) also the likeliest classes of each row, int32 and f32
    [rows, top_k], the lower index first among equals. The row terms of
    `cross_entropy`, differentiable in the log probability and the entropy; the
    alternatives carry no gradient. A target (read as 32 bits) outside
    [0, classes) gives NaN; so does a row with NaN, +inf or no finite logit."""
    if logits.dim() != 2 or logits.stride(1) != 1 and logits.shape[1] > 1:
        raise ValueError("logits must be [rows, classes] with contiguous rows")
    if max(logits.shape) > 0x7fffffff:
        N.check_sizes("token_logprobs", *logits.shape)
    if logits.shape[0] > 1 and logits.stride(0) < logits.shape[1]:
        logits = logits.contiguous()
    flat = targets
    if targets.dtype is not torch.int32 or targets.dim() != 1 or not targets.is_contiguous():
        flat = _ids(targets)
    if flat.numel() != logits.shape[0]:
        raise ValueError("targets length must match the number of logit rows")
    if flat.get_device() != logits.get_device():
        raise ValueError("targets must be on the logits' device")
    top_k = int(top_k)
    if not 0 <= top_k <= min(32, logits.shape[1]):
        raise ValueError("top_k must be 0 to 32 and at most the number of classes")
    # A dual tensor goes there too: autograd refuses it, for there is no forward-mode derivative.
    if logits.requires_grad and torch.is_grad_enabled() or forward_ad._current_level >= 0 and has_tangent(logits):
        return TokenLogprobs(*_TokenLogprobsFn.apply(logits, flat, top_k))
    return TokenLogprobs(*_token_logprobs(logits, flat, top_k, False)[:4])


def quantize_w4(weight: torch.Tensor, group: int = 128):
    """(packed, scales) of a finite weight [in, out] for linear_w4: int32
    [ceil(in / 8), out] with 8 consecutive inputs' q in a word, the first in the
    lowest 4 bits, and [ceil(in / group), out] scales in the weight's dtype;
    weight is about (q - 8) * scale."""
    if weight.dim() != 2:
        raise ValueError("weight must be [in, out]")
    N.check_sizes("quantize_w4", *weight.shape, group)
    c = _context_of(weight)
    w = weight.detach().contiguous()
    in_f, out_f = w.shape
    if group <= 0 or group % 32:
        raise ValueError("group must be a multiple of 32")
    packed = torch.empty(-(-in_f // 8), out_f, dtype=torch.int32, device=w.device)
    scales = torch.empty(-(-in_f // group), out_f, dtype=w.dtype, device=w.device)
    c.call(N.lib().hx_quantize_w4, _DTYPES[w.dtype], w.data_ptr(), packed.data_ptr(), scales.data_ptr(), in_f, out_f,
           group)
    return packed, scales


def linear_w4(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group: int,
              bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`linear` with 4-bit weights (quantize_w4's layout), for the few rows of a decode
    step: x [..., in] -> [..., out], x, scales, bias and residual of one dtype.
    For inference: it has no backward and refuses tensors that would need one."""
    if torch.is_grad_enabled() and (x.requires_grad or scales.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        raise RuntimeError("linear_w4 has no backward: call it under torch.no_grad()")
    if forward_ad._current_level >= 0 and has_tangent(x, scales, bias, residual):
        raise RuntimeError("linear_w4 has no forward-mode derivative")
    c = _context_of(x)
    lead, in_f, out_f = x.shape[:-1], x.shape[-1], packed.shape[-1]
    if group <= 0 or group % 32:
        raise ValueError("group must be a multiple of 32")
    if packed.dtype is not torch.int32 or packed.shape != (-(-in_f // 8), out_f) or not packed.is_contiguous():
        raise ValueError(f"packed must be contiguous int32 [{-(-in_f // 8)}, out] for {in_f} inputs")
    if scales.shape != (-(-in_f // group), out_f) or not scales.is_contiguous():
        raise ValueError(f"scales must be contiguous [{-(-in_f // group)}, {out_f}]")
    dt, dev = x.dtype, x.get_device()
    shape = (*lead, out_f)
    if bias is not None:
        if bias.shape != (out_f,) or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous vector of {out_f}")
        if bias.dtype is not dt or bias.get_device() != dev:
            raise ValueError("bias must have x's dtype and device")
    if residual is not None:
        if residual.shape != shape:
            raise ValueError(f"residual must be {shape}")
        if residual.dtype is not dt or residual.get_device() != dev:
            raise ValueError("residual must have x's dtype and device")
        residual = residual.contiguous()
    if scales.dtype is not dt or scales.get_device() != dev or packed.get_device() != dev:
        raise ValueError("packed and scales must be on x's device, scales in its dtype")
    rows = 1
    for n in lead:
        rows *= n
    if max(rows, in_f, out_f, group) > 0x7fffffff:
        N.check_sizes("linear_w4", rows, in_f, out_f, group)
    x = x.contiguous()
    y = x.new_empty(shape)
    if rows == 0 or out_f == 0:
        return y
    c.call(N.lib().hx_linear_w4_fwd, _DTYPES[dt], x.data_ptr(), packed.data_ptr(), scales.data_ptr(),
           None if bias is None else bias.data_ptr(), None if residual is None else residual.data_ptr(), y.data_ptr(),
           rows, in_f, out_f, group)
    return y


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """kernels/rms_norm.rs:20-55 over the last dimension, with its backward."""
    return _RMSNormFn.apply(x, weight, float(eps))


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x @ weight + bias with weight stored [in, out] (nn/linear.rs:54-56);
    `residual` (same shape as the output) is added in the same GEMM, the
    residual add of nn/transformer.rs:32, 37."""
    return _LinearFn.apply(x, weight, bias, residual)


class RMSNorm:
    """src/nn/rms_norm.rs: weight initialised to ones, eps 1e-5."""

    def __init__(self, hidden_dim: int, device=None, dtype=torch.float32):
        self.weight = torch.ones(hidden_dim, device=device, dtype=dtype, requires_grad=True)
        self.eps = 1e-5

    def forward(self, x):
        return rms_norm(x, self.weight, self.eps)

    __call__ = forward

    def parameters(self):
        return [self.weight]


class Linear:
    """src/nn/linear.rs: weight [in, out] uniform in +-sqrt(6 / in), bias zeros."""

    def __init__(self, in_features: int, out_features: int, device=None, dtype=torch.float32,
                 generator: Optional[torch.Generator] = None):
        bound = math.sqrt(6.0 / in_features)
        w = torch.rand(in_features, out_features, generator=generator, dtype=torch.float32) * 2 * bound - bound
        self.weight = w.to(device=device, dtype=dtype).requires_grad_()
        self.bias = torch.zeros(out_features, device=device, dtype=dtype, requires_grad=True)

    def forward(self, x, residual=None):
        return linear(x, self.weight, self.bias, residual)

    __call__ = forward

    def parameters(self):
        return [self.weight, self.bias]


class LinearW4:
    """A Linear for inference with its weight in 4 bits (quantize_w4); bias as it was."""

    def __init__(self, linear: Linear, group: int = 128):
        self.group = int(group)
        self.packed, self.scales = quantize_w4(linear.weight, self.group)
        self.bias = linear.bias.detach()

    def forward(self, x, residual=None):
        return linear_w4(x, self.packed, self.scales, self.group, self.bias, residual)

    __call__ = forward

    def parameters(self):
        return []


class MultiHeadAttention:
    """src/nn/attention.rs:5-98: pre-RMSNorm, Q/K/V projections, heads as strided
    views, RoPE (base 10000, attention.rs:76) on Q and K, the fused attention
    with scale 1/sqrt(head_dim), heads merged by a view, output projection.
    `causal` adds the mask the reference's layer lacks (False reproduces it)."""

    def __init__(self, hidden_dim: int, num_heads: int, device=None, dtype=torch.float32,
                 rope_base: float = 10000.0, causal: bool = False, seed: Optional[int] = None):
        if hidden_dim % num_heads:
            raise ValueError("hidden_dim must be divisible by num_heads")
        g = torch.Generator().manual_seed(seed) if seed is not None else None
        self.num_heads, self.head_dim = num_heads, hidden_dim // num_heads
        self.rope_base, self.causal = float(rope_base), bool(causal)
        self.norm = RMSNorm(hidden_dim, device, dtype)
        self.q_proj, self.k_proj, self.v_proj, self.out_proj = (
            Linear(hidden_dim, hidden_dim, device, dtype, g) for _ in range(4))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        B, S, Hd = x.shape
        H, D = self.num_heads, self.head_dim
        n = self.norm(x)

        def heads(t):  # [B, S, H*D] -> [B, H, S, D] view (attention.rs:62-73 without the copies)
            return t.view(B, S, H, D).transpose(1, 2)

        q, k, v = heads(self.q_proj(n)), heads(self.k_proj(n)), heads(self.v_proj(n))
        o = flash_attention(q, k, v, 1.0 / math.sqrt(D), self.causal, rope_base=self.rope_base)
        # [B, H, S, D] with [B, S, H, D] memory: the head merge is a view (attention.rs:91-94)
        return self.out_proj(o.transpose(1, 2).reshape(B, S, Hd), residual)

    __call__ = forward

    def _answers(self) -> None:
        if not self.causal:
            raise ValueError("answering from a cache needs a causal layer")

    def prefill(self, x: torch.Tensor, cache: PagedKVCache, seq_ids: torch.Tensor, positions: torch.Tensor,
                residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        """forward of prompts [B, S, hidden] from position 0 whose rotated keys and values also enter
        the cache: token (b, s) at positions[b * S + s] of seq_ids[b * S + s], padding negative. The layer is causal."""
        self._answers()
        B, S, Hd = x.shape
        H, D = self.num_heads, self.head_dim
        n = self.norm(x)
        q, k, v = (p(n).view(B, S, H, D) for p in (self.q_proj, self.k_proj, self.v_proj))
        paged_append(cache, k.view(-1, H, D), v.view(-1, H, D), seq_ids, positions, rope_base=self.rope_base)
        o = flash_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), 1.0 / math.sqrt(D), True,
                            rope_base=self.rope_base)
        return self.out_proj(o.transpose(1, 2).reshape(B, S, Hd), residual)

    def decode(self, x: torch.Tensor, cache: PagedKVCache, seq_ids: torch.Tensor, positions: torch.Tensor,
               seq_lens: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        """forward of one new token a sequence [sequences, hidden]: its keys and values enter the cache
        and it attends to the seq_lens positions that are there then. The layer is causal."""
        self._answers()
        T, H, D = x.shape[0], self.num_heads, self.head_dim
        n = self.norm(x)
        q, k, v = (p(n).view(T, H, D) for p in (self.q_proj, self.k_proj, self.v_proj))
        paged_append(cache, k, v, seq_ids, positions, rope_base=self.rope_base, q=q, out_q=q)
        o, _ = paged_attention(cache, q, seq_lens, 1.0 / math.sqrt(D))
        return self.out_proj(o.view(T, H * D), residual)

    def parameters(self):
        return (self.norm.parameters() + self.q_proj.parameters() + self.k_proj.parameters()
                + self.v_proj.parameters() + self.out_proj.parameters())


class FeedForward:
    """src/nn/mlp.rs: linear1 (hidden -> 4 hidden), GELU, linear2 (4 hidden -> hidden)."""

    def __init__(self, hidden_dim: int, device=None, dtype=torch.float32, seed: Optional[int] = None):
        g = torch.Generator().manual_seed(seed) if seed is not None else None
        self.linear1 = Linear(hidden_dim, 4 * hidden_dim, device, dtype, g)
        self.linear2 = Linear(4 * hidden_dim, hidden_dim, device, dtype, g)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return self.linear2(gelu(self.linear1(x)), residual)

    __call__ = forward

    def parameters(self):
        return self.linear1.parameters() + self.linear2.parameters()


class TransformerBlock:
    """src/nn/transformer.rs:17-40, pre-norm with residuals:
    x = x + mha(norm1(x)); x = x + mlp(norm2(x)). The MultiHeadAttention
    keeps its own pre-RMSNorm (nn/attention.rs:53), so the attention input is
    normalised twice, as in the reference. Each residual add is folded into
    the GEMM of the branch's last projection."""

    def __init__(self, hidden_dim: int, num_heads: int, device=None, dtype=torch.float32,
                 rope_base: float = 10000.0, causal: bool = False, seed: Optional[int] = None):
        self.norm1 = RMSNorm(hidden_dim, device, dtype)
        self.mha = MultiHeadAttention(hidden_dim, num_heads, device, dtype, rope_base, causal, seed)
        self.norm2 = RMSNorm(hidden_dim, device, dtype)
        self.mlp = FeedForward(hidden_dim, device, dtype, None if seed is None else seed + 1)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x = self.mha(self.norm1(x), residual=x)
        return self.mlp(self.norm2(x), residual=x)

    __call__ = forward

    def prefill(self, x, cache, seq_ids, positions):
        x = self.mha.prefill(self.norm1(x), cache, seq_ids, positions, residual=x)
        return self.mlp(self.norm2(x), residual=x)

    def decode(self, x, cache, seq_ids, positions, seq_lens):
        x = self.mha.decode(self.norm1(x), cache, seq_ids, positions, seq_lens, residual=x)
        return self.mlp(self.norm2(x), residual=x)

    def parameters(self):
        return (self.norm1.parameters() + self.mha.parameters() + self.norm2.parameters()
                + self.mlp.parameters())


class Embedding:
    """A [vocab, dim] token table (the reference has no embedding layer)."""

    def __init__(self, vocab: int, dim: int, device=None, dtype=torch.float32,
                 generator: Optional[torch.Generator] = None):
        w = torch.randn(vocab, dim, generator=generator, dtype=torch.float32) * 0.02
        self.weight = w.to(device=device, dtype=dtype).requires_grad_()

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return embedding(ids, self.weight)

    __call__ = forward

    def parameters(self):
        return [self.weight]


class BlockStack:
    """A language model over TransformerBlocks: token embedding, `layers`
    blocks, a final RMSNorm and an output Linear to `vocab` logits.
    forward(ids [B, S]) -> logits [B*S, vocab]; loss(ids, targets) adds the
    cross-entropy. `init_std` (e.g. 0.02) re-draws every Linear weight from
    N(0, init_std^2) instead of linear.rs's uniform init."""

    def __init__(self, vocab: int, hidden_dim: int, num_heads: int, layers: int, device=None,
                 dtype=torch.float32, rope_base: float = 10000.0, causal: bool = True,
                 init_std: Optional[float] = None, seed: int = 0):
        g = torch.Generator().manual_seed(seed)
        self.embed = Embedding(vocab, hidden_dim, device, dtype, g)
        self.blocks = [TransformerBlock(hidden_dim, num_heads, device, dtype, rope_base, causal, seed + 2 * i + 1)
                       for i in range(layers)]
        self.norm = RMSNorm(hidden_dim, device, dtype)
        self.head = Linear(hidden_dim, vocab, device, dtype, g)
        if init_std is not None:
            with torch.no_grad():
                for p in self.parameters():
                    if p.dim() == 2 and p is not self.embed.weight:
                        w = torch.randn(p.shape, generator=g, dtype=torch.float32) * init_std
                        p.copy_(w.to(p.device, p.dtype))

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        x = self.embed(ids)
        for blk in self.blocks:
            x = blk(x)
        y = self.head(self.norm(x))
        return y.reshape(-1, y.shape[-1])

    __call__ = forward

    def loss(self, ids: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        return cross_entropy(self(ids), targets)

    def caches(self, pages: int, slots: int, block_table: torch.Tensor) -> list:
        """One PagedKVCache a block, all on one table."""
        mha = self.blocks[0].mha
        return [PagedKVCache.allocate(pages, slots, mha.num_heads, mha.head_dim, block_table, self.embed.weight.dtype)
                for _ in self.blocks]

    def _answers(self, caches) -> None:
        for b in self.blocks:
            b.mha._answers()
        if len(caches) != len(self.blocks):
            raise ValueError("one cache a block")
        if any(c.num_seqs != caches[0].num_seqs for c in caches):
            raise ValueError("the caches must hold the same sequences")

    @torch.no_grad()
    def prefill(self, ids: torch.Tensor, caches: list, lens: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Prompts [B, S] (row b is sequence b of the caches; its first lens[b] ids count, all without
        lens; the table must hold them) into the caches. Returns the logits [B, vocab] after each prompt's
        last token: NaN for a length outside 1 to S."""
        self._answers(caches)
        B, S = ids.shape
        if B > caches[0].num_seqs:
            raise ValueError(f"{B} prompts for caches of {caches[0].num_seqs} sequences")
        if lens is None and any(S > c.block_table.shape[1] * c.k.shape[1] for c in caches):
            raise ValueError(f"the caches' tables do not hold {S} positions")
        positions = torch.arange(S, dtype=torch.int32, device=ids.device).repeat(B)
        seq_ids = torch.arange(B, dtype=torch.int32, device=ids.device).repeat_interleave(S)
        last, bad = torch.full((B,), S - 1, device=ids.device), None
        if lens is not None:
            bad = (lens < 1) | (lens > S)
            last = (lens.to(torch.int64) - 1).clamp(0, S - 1)
            seq_ids = torch.where(positions < lens.repeat_interleave(S), seq_ids, -1)
        x = self.embed(ids)
        for blk, cache in zip(self.blocks, caches):
            x = blk.prefill(x, cache, seq_ids, positions)
        x = x[torch.arange(B, device=ids.device), last]
        logits = self.head(self.norm(x))
        return logits if bad is None else logits.masked_fill_(bad[:, None], float("nan"))

    @torch.no_grad()
    def decode(self, ids: torch.Tensor, caches: list, positions: torch.Tensor) -> torch.Tensor:
        """One new token a sequence: ids [B], at positions [B] (int32; what the caches hold before them
        is what each attends to, itself included). A negative position leaves its sequence out.
        Returns the logits [B, vocab]: of no use for a sequence that is left out, NaN for a position
        outside the table."""
        self._answers(caches)
        if ids.shape[0] != caches[0].num_seqs:
            raise ValueError(f"{ids.shape[0]} ids for caches of {caches[0].num_seqs} sequences")
        every = torch.arange(ids.shape[0], dtype=torch.int32, device=ids.device)
        seq_ids = torch.where(positions < 0, -1, every)
        seq_lens = positions.clamp(-1, 2**31 - 2) + 1  # the last int32 stays outside the table
        x = self.embed(ids)
        for blk, cache in zip(self.blocks, caches):
            x = blk.decode(x, cache, seq_ids, positions, seq_lens)
        return self.head(self.norm(x))

    def quantize_w4(self, group: int = 128) -> "BlockStack":
        """Puts every Linear's weight in 4 bits, for inference; the stack can then no longer be trained."""
        for blk in self.blocks:
            for part, names in ((blk.mha, ("q_proj", "k_proj", "v_proj", "out_proj")), (blk.mlp, ("linear1", "linear2"))):
                for name in names:
                    setattr(part, name, LinearW4(getattr(part, name), group))
        self.head = LinearW4(self.head, group)
        return self

    def parameters(self):
        ps = self.embed.parameters()
        for blk in self.blocks:
            ps += blk.parameters()
        return ps + self.norm.parameters() + self.head.parameters()
