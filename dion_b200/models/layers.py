"""Building blocks of the Llama model: RMSNorm, rotary embedding, causal
grouped-query attention (full, or with a sliding window and visible first
tokens), SwiGLU, a memory-lean linear + cross-entropy, and distillation from a
teacher's top logits (their selection and the loss, both behind the LM head).

Each op uses the package's fused sm_100a kernel for CUDA bf16 inputs when
the extension provides it, and plain PyTorch otherwise (CPU runs and
autograd reference)."""
from __future__ import annotations

import math
from contextlib import contextmanager
from typing import Optional, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from .. import ops
from ..ops import fused as _fused
from ..ops.fused import TopLogits

__all__ = [
    "RMSNorm",
    "rope_table",
    "apply_rope",
    "causal_attention",
    "window_attention",
    "swiglu",
    "linear_cross_entropy",
    "TopLogits",
    "top_logits",
    "linear_top_logits",
    "linear_distillation",
]


class RMSNorm(nn.Module):
    def __init__(self, dim: int, eps: float = 1e-5):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if _fused.enabled(x):
            return _fused.rms_norm(x, self.weight, self.eps)
        return F.rms_norm(x.float(), (x.shape[-1],), self.weight.float(), self.eps).to(x.dtype)

    def add_forward(self, x: torch.Tensor, a: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """(x + a, norm(x + a)): the residual add fused into the norm where the kernel applies."""
        if _fused.add_rms_enabled(x) and a.dtype == x.dtype and a.shape == x.shape:
            return _fused.add_rms_norm(x, a, self.weight, self.eps)
        h = x + a
        return h, self(h)

    def reset_parameters(self):
        nn.init.ones_(self.weight)


def rope_table(head_dim: int, max_seq_len: int, theta: float) -> torch.Tensor:
    """[max_seq_len, head_dim/2, 2] table of (cos, sin), fp32."""
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim))
    t = torch.arange(max_seq_len, dtype=torch.float64)
    ang = torch.outer(t, inv)
    return torch.stack([ang.cos(), ang.sin()], dim=-1).float()


def apply_rope(q: torch.Tensor, k: torch.Tensor, rope: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rotate interleaved (even, odd) pairs of the head dim; q,k: [b, s, h, d]."""
    if _fused.enabled(q):
        return _fused.rope(q, k, rope)
    return _rope_ref(q, rope), _rope_ref(k, rope)


def _rope_ref(x: torch.Tensor, rope: torch.Tensor) -> torch.Tensor:
    xf = x.float().reshape(*x.shape[:-1], -1, 2)
    c = rope[: x.shape[1], None, :, 0]
    s = rope[: x.shape[1], None, :, 1]
    x0, x1 = xf[..., 0], xf[..., 1]
    out = torch.stack([x0 * c - x1 * s, x0 * s + x1 * c], dim=-1)
    return out.flatten(-2).to(x.dtype)


def causal_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """q: [b, s, hq, d], k/v: [b, s, hkv, d] -> [b, s, hq, d]."""
    qt, kt, vt = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
    gqa = qt.shape[1] != kt.shape[1]
    o = F.scaled_dot_product_attention(qt, kt, vt, is_causal=True, enable_gqa=gqa)
    return o.transpose(1, 2)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0) -> torch.Tensor:
    """Causal attention over the last ``window`` positions and the first
    ``sinks`` ones: i sees j <= i where i - j < window or j < sinks.
    q: [b, s, hq, d], k/v: [b, s, hkv, d] -> [b, s, hq, d]."""
    if _fused.window_enabled(q):
        return _fused.window_attention(q, k, v, window, sinks)
    _fused._check_window(q, k, v, window, sinks)
    return _window_ref(q, k, v, window, sinks)


def _window_ref(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int) -> torch.Tensor:
    pos = torch.arange(q.shape[1], device=q.device)
    i, j = pos[:, None], pos[None, :]
    seen = (j <= i) & ((i - j < window) | (j < sinks))
    qt, kt, vt = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
    o = F.scaled_dot_product_attention(qt, kt, vt, attn_mask=seen, enable_gqa=qt.shape[1] != kt.shape[1])
    return o.transpose(1, 2)


def swiglu(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    if _fused.enabled(a):
        return _fused.swiglu(a, b)
    return F.silu(a) * b


class _LinearCE(torch.autograd.Function):
    """loss = mean CE(h @ W^T, labels) with the gradient computed chunk by
    chunk during forward, so the [tokens, vocab] logits never exist in fp32
    all at once."""

    @staticmethod
    def forward(ctx, h, W, labels, chunk: int):
        T = h.shape[0]
        grad_h = torch.empty_like(h)
        grad_W = torch.zeros_like(W, dtype=torch.float32)
        total = torch.zeros((), device=h.device, dtype=torch.float32)
        for s in range(0, T, chunk):
            e = min(T, s + chunk)
            hc = h[s:e]
            logits = hc @ W.t()
            lab = labels[s:e]
            loss_c, g = _fused.cross_entropy_fwd_bwd(logits, lab, 1.0 / T)
            total += loss_c
            grad_h[s:e] = g @ W
            # grad_W (fp32) += g^T @ hc on the tensor cores, accumulating in place
            ops.matmul(g.t(), hc, out=grad_W, C=grad_W, beta=1.0)
        ctx.save_for_backward(grad_h, grad_W.to(W.dtype))
        return total / T

    @staticmethod
    def backward(ctx, go):
        grad_h, grad_W = ctx.saved_tensors
        return grad_h * go, grad_W * go, None, None


def linear_cross_entropy(h: torch.Tensor, W: torch.Tensor, labels: torch.Tensor, chunk: int = 8192) -> torch.Tensor:
    h2 = h.reshape(-1, h.shape[-1])
    lab = labels.reshape(-1)
    if not h.is_cuda:
        return F.cross_entropy((h2 @ W.t()).float(), lab)
    if not (torch.is_grad_enabled() and (h.requires_grad or W.requires_grad)):
        # evaluation: the same chunked loss without the gradient products
        T = h2.shape[0]
        total = torch.zeros((), device=h.device, dtype=torch.float32)
        for s in range(0, T, chunk):
            e = min(T, s + chunk)
            loss_c, _ = _fused.cross_entropy_fwd_bwd(h2[s:e] @ W.t(), lab[s:e], 1.0 / T)
            total += loss_c
        return total / T
    return _LinearCE.apply(h2, W, lab, chunk)


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """The k largest logits of every row of [T, V] with their columns, and the
    row's log-sum-exp at ``temperature`` (see :func:`dion_b200.ops.fused.top_logits`)."""
    return _fused.top_logits(logits, k, temperature)


def _mm_fp32(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """a @ b with the sum and the result in fp32. (A bf16 logit of 8 is off by
    up to 2^-6, and a softmax turns that into as large a relative error of its
    probability; a bf16 result also lets the library add parts of a long sum
    in bf16.)"""
    if a.dtype == torch.float32:
        return a @ b
    if a.is_cuda:
        return torch.mm(a, b, out_dtype=torch.float32)
    return a.float() @ b.float()


@contextmanager
def _head(h: torch.Tensor, W: torch.Tensor):
    """h and W in the type that F.linear would take them in, and autocast off for what is done with
    them: it would round the products' fp32 results to its type."""
    dev = h.device.type
    if not torch.is_autocast_enabled(dev):
        yield h, W
        return
    dtype = torch.get_autocast_dtype(dev)
    h, W = h.to(dtype), W.to(dtype)
    with torch.autocast(dev, enabled=False):
        yield h, W


@torch.no_grad()
def linear_top_logits(h: torch.Tensor, W: torch.Tensor, k: int, temperature: float = 1.0,
                      chunk: int = 4096) -> TopLogits:
    """``top_logits`` of the LM head's h @ W^T, ``chunk`` tokens at a time, so
    that the [tokens, vocab] logits never exist at once. h: [..., dim]; the
    results are [..., k] and [...]."""
    with _head(h.reshape(-1, h.shape[-1]), W) as (h2, W):
        parts = [_fused.top_logits(_mm_fp32(c, W.t()), k, temperature) for c in h2.split(max(1, chunk))]
    values, indices, lse = (torch.cat(p) if len(p) > 1 else p[0] for p in zip(*parts))
    lead = h.shape[:-1]
    return TopLogits(values.view(*lead, k), indices.view(*lead, k), lse.view(lead))


class _LinearDistillation(torch.autograd.Function):
    """Mean distillation loss behind the LM head, its gradient computed chunk by
    chunk during forward as in :class:`_LinearCE`. The chunk's gradient of the
    logits is that of the sum over the rows, in h's dtype, times a factor of
    :meth:`_scale`. The number of rows in the loss, known on the device only, and
    that factor are applied with the incoming gradient in backward, before the
    one rounding of each result."""

    @staticmethod
    def _scale(dtype, labels, temperature, alpha):
        """Factor of the logits' gradient between the loss and the head's products.
        1 / (1 - alpha) with labels: the entry of a label is then close to -1, which
        rounds to itself, where -(1 - alpha) would be off by the same part in every
        row. In fp16 a power of two on top: an entry of a 128k vocabulary is 8e-6 on
        average, among the subnormals (spacing 6e-8), while no entry exceeds
        (1 - alpha) + alpha * temperature times the teacher's mass; with a mass of 1 that
        bound is brought to 2^13 ... 2^14, so that one of 3 (columns that come twice under
        a log-sum-exp of the row) stays finite as well."""
        hard = 1.0 - alpha if labels is not None and alpha < 1 else 0.0
        scale = 1.0 / hard if hard else 1.0
        if dtype == torch.float16:
            scale *= 2.0 ** (14 - math.ceil(math.log2((hard + alpha * temperature) * scale)))
        return scale

    @staticmethod
    def forward(ctx, h, W, labels, top_values, top_indices, top_lse, temperature, alpha, chunk, need_grad):
        T, V = h.shape[0], W.shape[0]
        scale = _LinearDistillation._scale(h.dtype, labels, temperature, alpha)
        total = torch.zeros((), device=h.device, dtype=torch.float32)
        grad_h = torch.empty(h.shape, device=h.device, dtype=torch.float32) if need_grad else None
        make = torch.empty if T else torch.zeros
        grad_W = make(W.shape, device=W.device, dtype=torch.float32) if need_grad else None
        for s in range(0, T, chunk):
            e = min(T, s + chunk)
            hc = h[s:e]
            loss_c, g = _fused.distillation_fwd_bwd(
                _mm_fp32(hc, W.t()), None if labels is None else labels[s:e], top_values[s:e], top_indices[s:e],
                None if top_lse is None else top_lse[s:e], temperature, alpha, scale, h.dtype, need_grad)
            total += loss_c
            if need_grad:
                grad_h[s:e] = _mm_fp32(g, W)
                # grad_W (fp32) = or += g^T @ hc
                if h.is_cuda and h.dtype == torch.bfloat16:
                    ops.matmul(g.t(), hc, out=grad_W, C=grad_W if s else None, beta=1.0 if s else 0.0)
                elif s:
                    grad_W += g.t().float() @ hc.float()
                else:
                    grad_W = g.t().float() @ hc.float()
        n = max(T, 1) if labels is None else ((labels >= 0) & (labels < V)).sum().clamp_min(1).float()
        ctx.n = n * scale
        ctx.save_for_backward(grad_h, grad_W)
        ctx.dtypes = h.dtype, W.dtype
        return total / n

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        grad_h, grad_W = ctx.saved_tensors
        f = go / ctx.n
        return (_fused.scale_cast(grad_h, f, ctx.dtypes[0]), _fused.scale_cast(grad_W, f, ctx.dtypes[1])) + (None,) * 8


def linear_distillation(h: torch.Tensor, W: torch.Tensor, labels: Optional[torch.Tensor], top_values: torch.Tensor,
                        top_indices: torch.Tensor, top_lse: Optional[torch.Tensor] = None, temperature: float = 1.0,
                        alpha: float = 1.0, chunk: int = 4096) -> torch.Tensor:
    """Mean distillation loss of the student logits h @ W^T against a teacher's
    top logits (see :func:`dion_b200.ops.fused.distillation_fwd_bwd` for the
    loss). h: [..., dim], labels: [...] or None, top_values / top_indices:
    [..., k], top_lse: [...]. Rows whose label is outside [0, V) are left out
    of the sum and of the mean; the loss is 0 if that leaves none.

    The mean is over this call's rows. Where data parallelism averages gradients
    over ranks that leave out unequally many, that is not the mean over all rows:
    multiply each rank's loss by ranks * (its rows in the loss) / (those of all
    ranks), which one all-reduce of the counts gives."""
    h2 = h.reshape(-1, h.shape[-1])
    flat = lambda t: None if t is None else t.reshape(-1)  # noqa: E731
    rows = lambda t: t.reshape(math.prod(t.shape[:-1]), t.shape[-1])  # noqa: E731
    teacher = flat(labels), rows(top_values), rows(top_indices), flat(top_lse), temperature, alpha
    # of all rows at once: the chunks are slices, which would pass over a row too many
    _fused._check_distillation((h2.shape[0], W.shape[0]), *teacher)
    need = torch.is_grad_enabled() and (h.requires_grad or W.requires_grad)
    with _head(h2, W) as (h2, W):
        return _LinearDistillation.apply(h2, W, *teacher, max(1, chunk), need)
