"""Factor of the logits' gradient behind the LM head: the bound it rests on, and its ranges (CPU)."""
import pytest
import torch

from dion_b200.models.layers import _LinearDistillation
from dion_b200.ops import fused

from test_distillation_cpu import distill_case


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("labelled,alpha", [(True, 0.0), (True, 0.5), (True, 0.95), (True, 1 - 1e-9), (True, 1.0), (False, 1.0)])
@pytest.mark.parametrize("tau", [0.25, 1.0, 3.0, 1000.0])
def test_scaled_entries_stay_in_fp16(labelled, alpha, tau, rest):
    """Sure students and sure teachers, right and wrong ones: no entry leaves fp16, the bound is used to half, and the
    factor is a power of two but for 1 / (1 - alpha)."""
    z, labels, val, idx, lse = distill_case(40, 50, 4, rest, tau=tau)
    z[::2] *= 100
    val[::3, 0] += 200 * tau
    labels = labels.clamp_min(0) if labelled else None
    if rest:
        lse = torch.logsumexp(val / tau, 1) + 0.1
    scale = _LinearDistillation._scale(torch.float16, labels, tau, alpha)
    grad = fused.distillation_fwd_bwd(z, labels, val, idx, lse, tau, alpha, scale, torch.float16)[1]
    assert grad.isfinite().all()
    bound = ((1 - alpha if labelled else 0) + alpha * tau) * scale
    assert 2.0 ** 13 < bound <= 2.0 ** 14 * (1 + 1e-12) and grad.abs().max() <= 2.0 ** 14 * (1 + 2.0 ** -10)
    wide = _LinearDistillation._scale(torch.bfloat16, labels, tau, alpha)
    assert wide == (1 / (1 - alpha) if labelled and alpha < 1 else 1.0)
    mantissa = torch.frexp(torch.tensor(scale / wide, dtype=torch.float64)).mantissa.item()
    assert mantissa == 0.5


@pytest.mark.parametrize("tau", [1.0, 4.0])
def test_a_mass_of_three_stays_finite(tau):
    """Every column three times, all of the mass in one that the student holds for impossible, and the other way round."""
    z, _, _, _, _ = distill_case(2, 8, 2, True)
    idx = torch.arange(8).repeat(2, 3)
    val = torch.zeros(2, 24)
    val[:, 1::8] = 60.0 * tau
    z[0, 1], z[1, 1] = -100.0 * tau, 100.0 * tau
    lse = torch.logsumexp(val[:, :8] / tau, 1)
    scale = _LinearDistillation._scale(torch.float16, None, tau, 1.0)
    grad = fused.distillation_fwd_bwd(z, None, val, idx, lse, tau, 1.0, scale, torch.float16)[1]
    assert grad.isfinite().all() and abs(grad[0, 1].item() + 3 * tau * scale) <= 2.0 ** -10 * 3 * tau * scale
