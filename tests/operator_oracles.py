"""64-bit oracles of the window-attention and distillation operators, with the
elementwise error that their kernels' roundings allow.

``half`` below is the largest relative error of one rounding to the output
type (finfo.eps / 2); ``small`` half the spacing of its subnormals; ``SLOP``
covers the fp32 arithmetic (scores of up to 128 products, 2^x to 2^-18, sums)."""
import math

import torch

SLOP = 2.0 ** -14


def halves(dtype):
    f = torch.finfo(dtype)
    return f.eps / 2, (f.smallest_normal * f.eps / 2 if dtype == torch.float16 else 0.0)


def window_oracle(q, k, v, window, sinks, do=None):
    """{name: (value, tolerance)} for o and, with ``do``, dq, dk, dv.

    o: P is rounded (half of P), o is rounded. dv likewise. dq / dk: dS is
    rounded; its delta = do . o takes the rounded o, so it is off by up to
    |do| . tolerance(o), times P."""
    half, small = halves(q.dtype)
    s, hq, d = q.shape[1:]
    g = hq // k.shape[2]
    x = [t.detach().double().transpose(1, 2) for t in (q, k, v)]
    Q, K, V = x[0], x[1].repeat_interleave(g, 1), x[2].repeat_interleave(g, 1)
    pos = torch.arange(s, device=q.device)
    i, j = pos[:, None], pos[None, :]
    seen = (j <= i) & ((i - j < window) | (j < sinks))
    sc = 1 / math.sqrt(d)
    P = torch.softmax((Q @ K.mT * sc).masked_fill(~seen, float("-inf")), -1)
    O = P @ V
    seen_n = seen.double().expand_as(P)
    tol_p = (half + SLOP) * P + small * seen_n
    tol_o = tol_p @ V.abs() + half * O.abs() + small
    out = {"o": (O, tol_o)}
    if do is not None:
        G = do.detach().double().transpose(1, 2)
        dP = G @ V.mT
        delta = (G * O).sum(-1, keepdim=True)
        dS = P * (dP - delta)
        err = (half + SLOP) * dS.abs() + P * (G.abs() * tol_o).sum(-1, keepdim=True) + small * seen_n \
            + SLOP * P * (G.abs() @ V.abs().mT + (G * O).abs().sum(-1, keepdim=True))
        fold = lambda t: t.unflatten(1, (-1, g)).sum(2)  # noqa: E731
        dq, dk, dv = dS @ K * sc, fold(dS.mT @ Q) * sc, fold(P.mT @ G)
        out["dq"] = (dq, err @ K.abs() * sc + half * dq.abs() + small)
        out["dk"] = (dk, fold(err.mT @ Q.abs()) * sc + half * dk.abs() + small)
        out["dv"] = (dv, fold(tol_p.mT @ G.abs()) + half * dv.abs() + small)
    return {n: (a.transpose(1, 2), b.transpose(1, 2)) for n, (a, b) in out.items()}


def assert_within(got, want, tol, what=""):
    diff = (got.detach().double() - want).abs()
    bad = ~(diff <= tol)
    if bad.any():
        at = tuple(int(c) for c in bad.nonzero()[0])
        worst = (diff / tol.clamp_min(1e-300)).nan_to_num(1e9).max().item()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {worst:.3g} x the tolerance, "
                             f"first at {at}: {got[at].item()} for {want[at].item()}")


def distill_oracle(z, labels, top_values, top_indices, top_lse, tau, alpha):
    """Loss and gradient by autograd on the definition in 64 bits, row by row
    over the distinct columns; the gradient's tolerance is relative to the
    terms that cancel in it."""
    T, V = z.shape
    z = z.detach().double().requires_grad_()
    loss, mag = torch.zeros(2, dtype=torch.float64, device=z.device)
    tol = torch.zeros_like(z)
    for r in range(T):
        if labels is not None and not 0 <= int(labels[r]) < V:
            continue
        soft = torch.log_softmax(z[r] / tau, 0)
        sel = (top_indices[r] >= 0) & (top_indices[r] < V)
        idx, t = top_indices[r][sel].long(), top_values[r][sel].double() / tau
        kl = torch.zeros((), dtype=torch.float64, device=z.device)
        terms = torch.zeros(V, dtype=torch.float64, device=z.device)
        if idx.numel():
            logp = t - (top_lse[r].double() if top_lse is not None else torch.logsumexp(t, 0))
            p = torch.where(t == -math.inf, 0.0, logp.exp())
            kl = kl + torch.where(p > 0, p * (logp - soft[idx]), 0.0).sum()
            mag = mag + alpha * tau * tau * torch.where(p > 0, p * (logp.abs() + soft[idx].detach().abs()), 0.0).sum()
            terms.index_add_(0, idx, p)
        else:
            p = torch.zeros(1, dtype=torch.float64, device=z.device)
        soft_terms = soft.detach().exp() if p.sum() > 0 or top_lse is not None else 0 * terms
        if top_lse is not None:
            inside = torch.zeros(V, dtype=torch.bool, device=z.device)
            inside[idx] = True
            p_rest = (1 - p.sum()).clamp_min(0)
            if p_rest > 0 and not inside.all():
                rest = torch.logsumexp(soft[~inside], 0)
                kl = kl + p_rest * (p_rest.log() - rest)
                mag += alpha * tau * tau * p_rest * (p_rest.log().abs() + rest.detach().abs() + 1)
                terms += torch.where(inside, 0.0, p_rest * (soft.detach() - rest.detach()).exp())
        if alpha > 0:
            loss = loss + alpha * tau * tau * kl
        tol[r] = alpha * tau * (soft_terms + terms)
        if labels is not None and alpha < 1:
            hard = torch.log_softmax(z[r], 0)
            loss = loss - (1 - alpha) * hard[labels[r]]
            mag += (1 - alpha) * (torch.logsumexp(z[r].detach(), 0).abs() + z[r, labels[r]].detach().abs())
            tol[r] += (1 - alpha) * hard.detach().exp()
            tol[r, labels[r]] += 1 - alpha
    grad = torch.autograd.grad(loss, z)[0] if loss.requires_grad else torch.zeros_like(z)
    return loss.detach(), grad.nan_to_num(0.0), mag * 2.0 ** -16 + 1e-6, tol * 2.0 ** -15
