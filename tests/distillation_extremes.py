"""Rows of logits that the distillation loss does not tell from ordinary ones: a common offset, the type's lowest value
throughout. Shared by the CPU and the GPU tests."""
import torch

from dion_b200.ops import fused

from operator_oracles import assert_within, distill_oracle, halves
from test_distillation_cpu import distill_case

OFFSET = 2.0 ** 14


def check_offset(tau, rest, alpha, device, dtype=torch.float32):
    """The softmax does not know a common offset of its logits. Values are multiples of 2^-8 (the log-sum-exp of 2^-9),
    so that adding the offset is exact in fp32: what changes is the kernel's rounding alone. The oracle, and its
    tolerance, are those of the rows without it."""
    z, labels, val, idx, lse = distill_case(9, 700, 12, rest, tau=tau, device=device)
    z, val = ((t * 256).round() / 256 for t in (z, val))
    if rest:
        lse = (lse * 512).round() / 512
    labels = labels if alpha < 1 else None
    want, wg, tl, tg = distill_oracle(z, labels, val, idx, lse, tau, alpha)
    for off_z, off_t in ((0.0, 0.0), (OFFSET, 0.0), (-OFFSET, 0.0), (0.0, OFFSET), (0.0, -OFFSET)):
        if off_t and rest:
            continue  # their log-sum-exp is an input, rounded by whoever gave it
        loss, grad = fused.distillation_fwd_bwd(z + off_z, labels, val + off_t, idx, lse, tau, alpha)
        assert abs(loss.item() - want.item()) <= tl.item(), (off_z, off_t, loss.item(), want.item(), tl.item())
        assert_within(grad, wg, halves(grad.dtype)[0] * wg.abs() + tg + 1e-30, f"grad {off_z} {off_t}")


def check_lowest(rest, alpha, device, dtype):
    """Every logit of a row at its type's lowest value: as a row of zeros. So are the teacher's entries where they are
    normalised among themselves."""
    z, labels, val, idx, lse = distill_case(6, 500, 8, rest, device=device)
    labels[:] = idx[:, 0]
    labels[1] = 499
    z, zeros = z.to(dtype), torch.zeros(6, 500, device=device)
    zeros[3:] = z[3:].float()
    z[:3] = torch.finfo(dtype).min
    tv = val.clone()
    if not rest:
        val[2], tv[2] = 0.0, torch.finfo(torch.float32).min
    want, wg, tl, tg = distill_oracle(zeros, labels, val, idx, lse, 1.0, alpha)
    loss, grad = fused.distillation_fwd_bwd(z, labels, tv, idx, lse, 1.0, alpha)
    assert abs(loss.item() - want.item()) <= tl.item(), (loss.item(), want.item(), tl.item())
    half, small = halves(grad.dtype)
    assert_within(grad, wg, half * wg.abs() + tg + small + 1e-30, "grad")


def check_masked_vocabulary(rest, device, dtype):
    """A student whose vocabulary is masked by the type's lowest value outside a few columns, the teacher's among them."""
    z, labels, val, idx, lse = distill_case(4, 500, 8, rest, device=device)
    keep = torch.zeros(4, 500, dtype=torch.bool, device=device).scatter_(1, idx, True)
    keep[:, :3] = True
    labels[:] = 1
    z = z.to(dtype).masked_fill(~keep, torch.finfo(dtype).min)
    out = z.float().masked_fill(~keep, float("-inf"))
    want, wg, tl, tg = distill_oracle(out, labels, val, idx, lse, 2.0, 0.5)
    loss, grad = fused.distillation_fwd_bwd(z, labels, val, idx, lse, 2.0, 0.5)
    assert abs(loss.item() - want.item()) <= tl.item(), (loss.item(), want.item(), tl.item())
    half, small = halves(grad.dtype)
    assert_within(grad, wg, half * wg.abs() + tg + small + 1e-30, "grad")


def check_high_temperature(tau, V, k, device, gdt=None):
    """The teacher's entries hold little, and little more than the student gives them. Tolerances, with e = 2^-24: a
    log-probability is off by 2^-20 of itself (its fp32 sum, 2^x to 2 e, its argument's rounding), so a probability by
    2^-19 of itself for logarithms to 12, and p and q, their sums over the set and their difference by 2^-18 (p + q).
    Outside the set the gradient is alpha tau q (sum p - sum q) / q_rest; the loss sum p (log p - log q) + p_rest (log(1 - sum p) -
    log(1 - sum q)). Twice each."""
    z, _, val, idx, lse = distill_case(7, V, k, True, tau=tau, seed=3, device=device)
    want, wg, _, _ = distill_oracle(z, None, val, idx, lse, tau, 1.0)
    loss, grad = fused.distillation_fwd_bwd(z, None, val, idx, lse, tau, 1.0, 1.0, gdt)
    logq = torch.log_softmax(z.double() / tau, 1)
    lp, lq = val.double() / tau - lse.double()[:, None], logq.gather(1, idx)
    both = lp.exp().sum(1) + lq.exp().sum(1)
    tl = tau * tau * ((lp.exp() * (lp.abs() + lq.abs())).sum(1) * 2.0 ** -19 + both * 2.0 ** -17).sum()
    assert abs(loss.item() - want.item()) <= tl.item() + 2.0 ** -20 * want.abs().item(), (loss.item(), want.item(), tl.item())
    out = torch.ones_like(z, dtype=torch.bool).scatter_(1, idx, False)
    tol = tau * logq.exp() * (both * 2.0 ** -17)[:, None]
    half, small = halves(grad.dtype)
    tol = tol + (half + 2.0 ** -18) * wg.abs() + small
    tol = torch.where(out, tol, tol + tau * (logq.exp() * 2.0 ** -17).scatter_add(1, idx, lp.exp() * 2.0 ** -17))
    assert_within(grad, wg, tol, "grad")


def check_other_masses(tau, alpha, device, dtype=torch.float32):
    """A teacher's probabilities whose sum with the rest's is not 1: columns that come twice under a log-sum-exp of the whole
    row (more than 1, nothing left for the rest), a log-sum-exp that is too small, entries over the student's whole
    vocabulary with mass elsewhere. The gradient is that of the loss as it stands."""
    z, labels, val, idx, lse = distill_case(9, 40, 40, True, dtype, tau=tau, seed=4, device=device)
    order = torch.stack([torch.randperm(40, generator=torch.Generator().manual_seed(r)) for r in range(9)]).to(device)
    val, idx = val.gather(1, order), idx.gather(1, order)
    top = idx.clone()
    top[0:3, 20:] = idx[0:3, :20]     # twenty columns, twice each
    val[0:3, 20:] = val[0:3, :20]
    lse[1] -= 1.0
    lse[3] -= 0.5                     # all columns, a sum above 1
    lse[4:7] += 0.7                   # all columns, a sum of 1/2
    top[7, 5:] = -1                   # few columns, a sum above 1 for five of them
    lse[7] = torch.logsumexp(val[7, :5] / tau, 0) - 0.3
    labels = labels.clamp_min(0) if alpha < 1 else None
    want, wg, tl, tg = distill_oracle(z, labels, val, top, lse, tau, alpha)
    loss, grad = fused.distillation_fwd_bwd(z, labels, val, top, lse, tau, alpha)
    assert abs(loss.item() - want.item()) <= tl.item(), (loss.item(), want.item(), tl.item())
    half, small = halves(grad.dtype)
    assert_within(grad, wg, half * wg.abs() + tg + small + 1e-30, "grad")
