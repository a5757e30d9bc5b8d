"""Distillation kernels on rows with extreme logits, and the head's gradient over a large vocabulary."""
import pytest
import torch

from dion_b200.models import layers as L

from distillation_extremes import check_lowest, check_masked_vocabulary, check_offset
from operator_oracles import distill_oracle, halves
from test_distillation_cpu import distill_case
from test_distillation_gpu import TYPES

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (1.0, 0.5), (2.0, 0.5), (1.5, 1.0)])
def test_common_offset(tau, alpha, rest):
    check_offset(tau, rest, alpha, DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("alpha", [1.0, 0.5])
def test_rows_of_the_lowest_value(alpha, rest, dtype):
    check_lowest(rest, alpha, DEV, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rest", [False, True])
def test_vocabulary_masked_by_the_lowest_value(rest, dtype):
    check_masked_vocabulary(rest, DEV, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("labelled,alpha,tau", [(True, 0.5, 1.0), (True, 0.0, 1.0), (True, 0.95, 2.0), (True, 0.999999, 1.0), (False, 1.0, 1.0)])
def test_head_gradient_over_a_large_vocabulary(labelled, alpha, tau, dtype):
    """The head's rows that are neither labels nor teacher entries sum gradients of 1e-5 and less, the labels' rows one
    of nearly 1 - alpha. In the mean square over such rows, two roundings (the logits' gradient, the result), each
    half / sqrt(3) of its value, and a quarter more for all that is fp32. (The loss is scaled as fp16 wants, so that
    the result itself is not among the subnormals.)"""
    T, V, D = 96, 128256, 64
    _, labels, val, idx, lse = distill_case(T, V, 16, True, tau=tau, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    h = torch.randn(T, D, device=DEV, generator=g).to(dtype).requires_grad_()
    W = (torch.randn(V, D, device=DEV, generator=g) * 0.1).to(dtype).requires_grad_()
    labels = labels if labelled else None
    up = 2.0 ** 13
    (L.linear_distillation(h, W, labels, val, idx, lse, tau, alpha, chunk=64) * up).backward()
    hd, Wd = h.detach().double(), W.detach().double()
    wg = distill_oracle(hd @ Wd.t(), labels, val, idx, lse, tau, alpha)[1]
    n = (labels >= 0).sum() if labelled else T
    want = up * wg.t() @ hd / n
    kind = torch.zeros(V, dtype=torch.long, device=DEV)
    kind[idx.flatten()] = 1
    if labelled:
        kind[labels[labels >= 0]] = 2
    bound = 1.25 * (2 / 3) ** 0.5 * halves(dtype)[0]
    off = {}
    for name, m in (("rest", kind == 0), ("entries", kind == 1), ("labels", kind == 2)):
        if m.any() and not (name == "entries" and alpha == 0):
            off["W " + name] = ((W.grad.double() - want)[m].norm() / want[m].norm()).item()
    wh = up * wg @ Wd / n
    off["h"] = ((h.grad.double() - wh).norm() / wh.norm()).item()
    assert all(v <= bound for v in off.values()), (off, bound)
