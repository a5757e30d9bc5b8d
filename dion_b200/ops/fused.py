"""Fused model-side ops (RMSNorm, rotary embedding, sliding-window attention,
SwiGLU, cross-entropy, distillation from a teacher's top logits).

The CUDA versions are sm_100a kernels of the ``dion_b200._C`` extension,
wrapped in autograd Functions; ``enabled(x)`` says whether a tensor takes the
fused path (CUDA, bf16, extension present, not disabled through
``DION_B200_FUSED=0``)."""
from __future__ import annotations

import os
from typing import NamedTuple, Optional, Tuple

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from ._ext import ext, has_ext

_DISABLED = os.environ.get("DION_B200_FUSED", "1") == "0"
_ADDNORM_DISABLED = os.environ.get("DION_B200_FUSED_ADDNORM", "1") == "0"


def enabled(x: torch.Tensor) -> bool:
    return (not _DISABLED) and x.is_cuda and x.dtype == torch.bfloat16 and has_ext() and hasattr(ext(), "rms_norm_fwd")


# ---------------------------------------------------------------- RMSNorm
class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, eps):
        x2 = x.reshape(-1, x.shape[-1]).contiguous()
        y = torch.empty_like(x2)
        rstd = torch.empty(x2.shape[0], device=x.device, dtype=torch.float32)
        ext().rms_norm_fwd(x2, w, y, rstd, float(eps))
        ctx.save_for_backward(x2, w, rstd)
        ctx.shape = x.shape
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, gy):
        x2, w, rstd = ctx.saved_tensors
        gy2 = gy.reshape(-1, gy.shape[-1]).contiguous()
        gx = torch.empty_like(x2)
        gw = torch.empty(w.shape, device=w.device, dtype=torch.float32)
        ext().rms_norm_bwd(gy2, x2, w, rstd, gx, gw)
        return gx.view(ctx.shape), gw.to(w.dtype), None


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    return _RMSNorm.apply(x, w, eps)


class _AddRMSNorm(torch.autograd.Function):
    """h = x + a and y = rms_norm(h) * w in one pass (the residual add of a
    transformer block fused into the next norm); the backward adds the
    residual gradient into the norm's input gradient in the same pass."""

    @staticmethod
    def forward(ctx, x, a, w, eps):
        x2 = x.reshape(-1, x.shape[-1]).contiguous()
        a2 = a.reshape(-1, a.shape[-1]).contiguous()
        h = torch.empty_like(x2)
        y = torch.empty_like(x2)
        rstd = torch.empty(x2.shape[0], device=x.device, dtype=torch.float32)
        ext().add_rms_norm_fwd(x2, a2, w, h, y, rstd, float(eps))
        ctx.save_for_backward(h, w, rstd)
        ctx.shape = x.shape
        return h.view(x.shape), y.view(x.shape)

    @staticmethod
    def backward(ctx, gh, gy):
        h, w, rstd = ctx.saved_tensors
        gy2 = gy.reshape(-1, gy.shape[-1]).contiguous()
        gh2 = gh.reshape(-1, gh.shape[-1]).contiguous()
        gx = torch.empty_like(h)
        gw = torch.empty(w.shape, device=w.device, dtype=torch.float32)
        ext().rms_norm_bwd_res(gy2, h, w, rstd, gh2, gx, gw)
        g = gx.view(ctx.shape)
        return g, g, gw.to(w.dtype), None


def add_rms_enabled(x: torch.Tensor) -> bool:
    """Fused add + RMSNorm: bf16 rows of 1024-8192 (multiple of 256) features."""
    d = x.shape[-1]
    return (not _ADDNORM_DISABLED and enabled(x) and hasattr(ext(), "add_rms_norm_fwd") and d % 256 == 0
            and 1024 <= d <= 8192)


def add_rms_norm(x: torch.Tensor, a: torch.Tensor, w: torch.Tensor, eps: float):
    """Returns (x + a, rms_norm(x + a) * w)."""
    return _AddRMSNorm.apply(x, a, w, eps)


# ---------------------------------------------------------------- RoPE
class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, rope):
        qo = torch.empty_like(q, memory_format=torch.contiguous_format)
        ko = torch.empty_like(k, memory_format=torch.contiguous_format)
        ext().rope_fwd(q.contiguous(), k.contiguous(), rope, qo, ko, False)
        ctx.save_for_backward(rope)
        return qo, ko

    @staticmethod
    def backward(ctx, gq, gk):
        (rope,) = ctx.saved_tensors
        gqo = torch.empty_like(gq, memory_format=torch.contiguous_format)
        gko = torch.empty_like(gk, memory_format=torch.contiguous_format)
        ext().rope_fwd(gq.contiguous(), gk.contiguous(), rope, gqo, gko, True)
        return gqo, gko, None


def rope(q: torch.Tensor, k: torch.Tensor, table: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    return _Rope.apply(q, k, table)


# ---------------------------------------------------------------- sliding-window attention
def _check_window(q, k, v, window, sinks) -> None:
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"window_attention: q [b, s, hq, d] and k, v [b, s, hkv, d], got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    if q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"window_attention: q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch, positions or "
                         "head dimension")
    if k.shape[2] < 1 or q.shape[2] % k.shape[2]:
        raise ValueError(f"window_attention: {q.shape[2]} query heads do not divide over {k.shape[2]} key heads")
    if not (q.dtype == k.dtype == v.dtype) or not (q.device == k.device == v.device):
        raise ValueError("window_attention: q, k and v of one type on one device")
    if int(window) < 1 or int(sinks) < 0:
        raise ValueError(f"window_attention: window >= 1 and sinks >= 0, got {window} and {sinks}")


def window_enabled(q: torch.Tensor) -> bool:
    """Window attention kernels: bf16 or fp16, head dimension a multiple of 8 up to 128."""
    return ((not _DISABLED) and q.is_cuda and q.dtype in (torch.bfloat16, torch.float16) and q.shape[-1] % 8 == 0
            and 8 <= q.shape[-1] <= 128 and has_ext() and hasattr(ext(), "window_attention_fwd"))


def _tile_rows(x: torch.Tensor) -> torch.Tensor:
    """x itself where the kernels' tiled copies can read it in place (head dim
    contiguous, every other stride a positive multiple of 16 bytes, aligned
    base), a packed copy otherwise."""
    st = x.stride()
    ok = x.data_ptr() % 16 == 0 and st[3] == 1 and all(n == 1 or (t > 0 and t % 8 == 0) for n, t in zip(x.shape[:3], st))
    return x if ok else x.clone(memory_format=torch.contiguous_format)


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks):
        q, k, v = _tile_rows(q), _tile_rows(k), _tile_rows(v)
        o, o_low, lse = torch.ops.dion_b200.window_attention_fwd(q, k, v, window, sinks, True)
        ctx.save_for_backward(q, k, v, o, o_low, lse)
        ctx.window, ctx.sinks = window, sinks
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        q, k, v, o, o_low, lse = ctx.saved_tensors
        dq, dk, dv = ext().window_attention_bwd(_tile_rows(go), q, k, v, o, o_low, lse, ctx.window, ctx.sinks)
        return dq, dk, dv, None, None


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0) -> torch.Tensor:
    """Causal attention in which position i sees position j <= i where
    ``i - j < window`` or ``j < sinks``. q: [b, s, hq, d], k/v: [b, s, hkv, d]
    (query head h reads key head h // (hq / hkv)) -> [b, s, hq, d]; scores are
    scaled by 1 / sqrt(d). A row that sees one key (the first one; every one with
    window 1 and no first tokens) adds exactly 0 to the gradients of q and k.
    Inputs are finite. A NaN is not lost (one in a key reaches o in every row that
    sees the key), but a non-finite value, and in the backward pass a non-finite
    query, key or output's gradient as well, also reaches rows up to a tile of 128
    beyond those that see it. The backward pass holds P (dP - delta) in the inputs'
    type, so in fp16 that is bounded by 65504."""
    _check_window(q, k, v, window, sinks)
    if not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)):
        return torch.ops.dion_b200.window_attention_fwd(_tile_rows(q), _tile_rows(k), _tile_rows(v), int(window),
                                                        int(sinks), False)[0]
    return _WindowAttention.apply(q, k, v, int(window), int(sinks))


# ---------------------------------------------------------------- SwiGLU
class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b):
        a, b = a.contiguous(), b.contiguous()
        out = torch.empty_like(a)
        ext().swiglu_fwd(a, b, out)
        ctx.save_for_backward(a, b)
        return out

    @staticmethod
    def backward(ctx, go):
        a, b = ctx.saved_tensors
        ga = torch.empty_like(a)
        gb = torch.empty_like(b)
        ext().swiglu_bwd(go.contiguous(), a, b, ga, gb)
        return ga, gb


def swiglu(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    return _SwiGLU.apply(a, b)


# ---------------------------------------------------------------- cross-entropy
def cross_entropy_fwd_bwd(logits: torch.Tensor, labels: torch.Tensor, grad_scale: float):
    """Return (sum of per-row losses (fp32 scalar), grad_scale * (softmax - onehot) in logits' dtype)."""
    if enabled(logits) and hasattr(ext(), "cross_entropy_fwd_bwd"):
        loss = torch.empty((), device=logits.device, dtype=torch.float32)
        grad = torch.empty_like(logits)
        ext().cross_entropy_fwd_bwd(logits.contiguous(), labels.contiguous(), grad, loss, float(grad_scale))
        return loss, grad
    lf = logits.float()
    lse = torch.logsumexp(lf, dim=-1)
    picked = lf.gather(1, labels.view(-1, 1)).squeeze(1)
    loss = (lse - picked).sum()
    p = torch.exp(lf - lse.unsqueeze(1))
    p.scatter_add_(1, labels.view(-1, 1), torch.full_like(picked.view(-1, 1), -1.0))
    return loss, (p * grad_scale).to(logits.dtype)


# ---------------------------------------------------------------- distillation
class TopLogits(NamedTuple):
    """A teacher's largest logits per row: values (fp32) and indices [T, k] in
    falling order, and log sum exp(logits / temperature) of the whole row [T]."""

    values: torch.Tensor
    indices: torch.Tensor
    lse: Optional[torch.Tensor]


MAX_TOP = 1024


def _check_temperature(op: str, temperature: float) -> None:
    # its square and its inverse are fp32 factors
    if not 1e-18 <= temperature <= 1e18:
        raise ValueError(f"{op}: temperature > 0 (1e-18 to 1e18), got {temperature}")


def _check_distillation(shape, labels, top_values, top_indices, top_lse, temperature, alpha) -> None:
    """Refuses what does not go with logits of ``shape``, or a shape that is not [T, V]."""
    if len(shape) != 2 or top_values.dim() != 2 or top_values.shape != top_indices.shape:
        raise ValueError(f"distillation: logits [T, V], top_values and top_indices [T, k], got {tuple(shape)}, "
                         f"{tuple(top_values.shape)}, {tuple(top_indices.shape)}")
    T, k = shape[0], top_values.shape[1]
    if top_values.shape[0] != T or not 1 <= k <= MAX_TOP:
        raise ValueError(f"distillation: {T} rows of 1 to {MAX_TOP} teacher entries, got {tuple(top_values.shape)}")
    if top_indices.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"distillation: int32 or int64 top_indices, got {top_indices.dtype}")
    for name, t in (("labels", labels), ("top_lse", top_lse)):
        if t is not None and t.shape != (T,):
            raise ValueError(f"distillation: {name} [{T}], got {tuple(t.shape)}")
    _check_temperature("distillation", temperature)
    if not 0 <= alpha <= 1:
        raise ValueError(f"distillation: 0 <= alpha <= 1, got {alpha}")
    if labels is None and alpha != 1:
        raise ValueError("distillation: alpha < 1 needs labels")
    if labels is not None and labels.dtype != torch.int64:
        raise ValueError(f"distillation: int64 labels, got {labels.dtype}")


def _rows_enabled(x: torch.Tensor) -> bool:
    return ((not _DISABLED) and x.is_cuda and x.dtype in (torch.bfloat16, torch.float16, torch.float32) and has_ext()
            and hasattr(ext(), "top_logits"))


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """The k largest logits of every row of [T, V] in falling order (equal ones
    by the lower index, a NaN above all), with the row's log-sum-exp at
    ``temperature`` (1e-18 to 1e18). 1 <= k <= min(V, 1024); V up to 2^20 on CUDA."""
    if logits.dim() != 2:
        raise ValueError(f"top_logits: logits [T, V], got {tuple(logits.shape)}")
    T, V = logits.shape
    if not 1 <= k <= min(V, MAX_TOP):
        raise ValueError(f"top_logits: 1 <= k <= min(V, {MAX_TOP}), got k = {k} with V = {V}")
    _check_temperature("top_logits", temperature)
    if _rows_enabled(logits):
        x = logits if logits.stride(1) == 1 or V == 1 else logits.contiguous()
        values = torch.empty(T, k, device=x.device, dtype=torch.float32)
        indices = torch.empty(T, k, device=x.device, dtype=torch.int64)
        lse = torch.empty(T, device=x.device, dtype=torch.float32)
        ext().top_logits(x, values, indices, lse, float(temperature))
        return TopLogits(values, indices, lse)
    x = logits.float()
    indices = (x + 0.0).sort(dim=1, descending=True, stable=True).indices[:, :k].contiguous()
    return TopLogits(x.gather(1, indices), indices, torch.logsumexp(x / temperature, dim=1))


def distillation_fwd_bwd(logits: torch.Tensor, labels: Optional[torch.Tensor], top_values: torch.Tensor,
                         top_indices: torch.Tensor, top_lse: Optional[torch.Tensor] = None, temperature: float = 1.0,
                         alpha: float = 1.0, grad_scale: float = 1.0, grad_dtype: Optional[torch.dtype] = None,
                         need_grad: bool = True):
    """Sum over the rows of
    ``(1 - alpha) CE(logits, label) + alpha temperature^2 KL(teacher || softmax(logits / temperature))``
    (fp32 scalar), and grad_scale times its gradient with respect to the logits
    (in their dtype, or ``grad_dtype`` for fp32 logits; None without ``need_grad``).

    logits: [T, V] (V up to 2^20 on CUDA); top_values / top_indices: [T, k], k <= 1024,
    the teacher's logits (constants: no gradient flows to them) and their columns (int32 or int64; a column outside [0, V) marks an
    unused entry, a column may come twice). ``top_lse`` [T] is the teacher's
    log-sum-exp at the temperature: the teacher's probability outside its
    entries then counts as one outcome more, held against the student's
    probability outside them. Without it the entries are normalised among
    themselves. labels: int64 [T] (a row whose label is outside [0, V) is left
    out: loss and gradient 0), or None with alpha = 1. Temperatures from 1e-18 to 1e18."""
    _check_distillation(logits.shape, labels, top_values, top_indices, top_lse, temperature, alpha)
    T, V = logits.shape
    gdt = grad_dtype or logits.dtype
    if gdt != logits.dtype and (logits.dtype != torch.float32 or gdt not in (torch.bfloat16, torch.float16)):
        raise ValueError(f"distillation: a {gdt} gradient of {logits.dtype} logits")
    if _rows_enabled(logits):
        x = logits if logits.stride(1) == 1 or V == 1 else logits.contiguous()
        loss = torch.empty((), device=x.device, dtype=torch.float32)
        grad = torch.empty((T, V), device=x.device, dtype=gdt) if need_grad else None
        ext().distill_fwd_bwd(x, None if labels is None else labels.contiguous(), top_values.float().contiguous(),
                              top_indices.contiguous(), None if top_lse is None else top_lse.float().contiguous(), grad,
                              loss, float(temperature), float(alpha), float(grad_scale))
        return loss, grad
    loss, grad = _distillation_ref(logits.float(), labels, top_values.float(), top_indices.long(),
                                   None if top_lse is None else top_lse.float(), temperature, alpha, need_grad)
    return loss, (grad * grad_scale).to(gdt) if need_grad else None


def scale_cast(x: torch.Tensor, f: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """fp32 x times the scalar tensor f, rounded once to ``dtype``."""
    if _rows_enabled(x) and x.dtype == torch.float32 and x.is_contiguous() and x.data_ptr() % 32 == 0:
        out = torch.empty(x.shape, device=x.device, dtype=dtype)
        ext().scale_cast(x, f.to(x.device, torch.float32), out)
        return out
    return (x * f).to(dtype)


def _distillation_ref(z, labels, top_values, top_indices, top_lse, tau, alpha, need_grad=True):
    V = z.shape[1]
    ninf = float("-inf")
    valid = (top_indices >= 0) & (top_indices < V)
    at = top_indices.clamp(0, V - 1)
    t = torch.where(valid, top_values, ninf)
    # to the row's maximum, before anything is rounded: an offset that all of a row have means nothing
    relative = lambda x: x - x.amax(1, keepdim=True).clamp_min(torch.finfo(x.dtype).min)  # noqa: E731
    if top_lse is None:
        t = relative(t) / tau
        logp = t - torch.logsumexp(t, 1, keepdim=True)
    else:
        t = t / tau
        logp = t - top_lse[:, None]
    p = torch.where(t == ninf, 0.0, logp.exp())
    logq = torch.log_softmax(relative(z) / tau, 1)
    kl = torch.where(p == 0, 0.0, p * (logp - logq.gather(1, at))).sum(1)
    q = logq.exp() if need_grad else None
    # not 1 where columns come twice, or where the whole vocabulary is in the set and mass elsewhere
    mass = p.sum(1, keepdim=True)
    soft = torch.where(mass == 0, 0.0, mass * q) if need_grad else None
    if top_lse is not None:
        inside = torch.zeros_like(z).scatter_add(1, at, valid.to(z.dtype)) > 0
        p_rest = torch.where(inside.all(1, keepdim=True), 0.0, (1 - mass).clamp_min(0))
        q_set = torch.where(inside, logq.exp(), 0.0).sum(1, keepdim=True)
        rest = torch.logsumexp(logq.masked_fill(inside, ninf), 1, keepdim=True)
        # where the set holds little, from its sums: their roundings are far smaller than those of two numbers near 1
        ratio = torch.where((mass < 0.5) & (q_set < 0.5), (-mass).log1p() - (-q_set).log1p(), p_rest.log() - rest)
        kl = kl + torch.where(p_rest > 0, p_rest * ratio, 0.0)[:, 0]
        if need_grad:
            outside = (mass - q_set) * (logq - rest).exp()
            soft = torch.where(p_rest > 0, torch.where(inside | (rest == ninf), q, outside), soft)
    loss = alpha * tau * tau * kl if alpha > 0 else torch.zeros_like(kl)
    grad = None
    if need_grad:
        grad = soft.scatter_add(1, at, -p) * (alpha * tau)
    if labels is not None:
        live = (labels >= 0) & (labels < V)
        y = labels.clamp(0, V - 1)[:, None]
        if alpha != 1:
            logs = torch.log_softmax(z, 1)
            loss = loss - (1 - alpha) * logs.gather(1, y)[:, 0]
            if need_grad:
                grad = grad + (1 - alpha) * logs.exp().scatter_add(1, y, -torch.ones_like(y, dtype=z.dtype))
        loss = torch.where(live, loss, 0.0)
        grad = torch.where(live[:, None], grad, 0.0) if need_grad else None
    return loss.sum(), grad
