"""Distillation kernels on rows with extreme logits, and the head's gradient over a large vocabulary."""
import pytest
import torch

from dion_b200.models import layers as L

from distillation_extremes import (check_high_temperature, check_lowest, check_masked_vocabulary, check_offset,
                                    check_other_masses)
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
@pytest.mark.parametrize("labelled,alpha,tau", [(True, 0.5, 1.0), (True, 0.0, 1.0), (True, 0.95, 2.0), (True, 0.999999, 1.0), (False, 1.0, 1.0),
                                                (False, 1.0, 30.0)])
def test_head_gradient_over_a_large_vocabulary(labelled, alpha, tau, dtype):
    """The head's rows that are neither labels nor teacher entries sum gradients of 1e-5 and less, the labels' rows one
    of nearly 1 - alpha. In the mean square over such rows, two roundings (the logits' gradient, the result), each
    half / sqrt(3) of its value, and a quarter more for all that is fp32. (The loss is scaled as fp16 wants, so that
    the result itself is not among the subnormals.) In fp16 an entry of the logits' gradient that is a subnormal under
    its factor, 2^13 / temperature at least, is off by up to 2^-25 whatever its size, 2^-25 / sqrt(3) in the mean
    square, so each of the head's entries by that / factor * sqrt(sum h^2): what is 2^-38 of the largest possible
    entry (at temperature 30 without labels, the rows in question are) keeps fewer bits."""
    T, V, D = 96, 128256, 64
    _, labels, val, idx, lse = distill_case(T, V, 16, True, tau=tau, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    h = torch.randn(T, D, device=DEV, generator=g).to(dtype).requires_grad_()
    W = (torch.randn(V, D, device=DEV, generator=g) * 0.1).to(dtype).requires_grad_()
    labels = labels if labelled else None
    up = 2.0 ** (13 if labelled else 21)  # 7e-9 * 96^-1/2 at temperature 30 would be 7e-6 under 2^13, a subnormal
    (L.linear_distillation(h, W, labels, val, idx, lse, tau, alpha, chunk=64) * up).backward()
    hd, Wd = h.detach().double(), W.detach().double()
    wg = distill_oracle(hd @ Wd.t(), labels, val, idx, lse, tau, alpha)[1]
    n = (labels >= 0).sum() if labelled else T
    want = up * wg.t() @ hd / n
    kind = torch.zeros(V, dtype=torch.long, device=DEV)
    kind[idx.flatten()] = 1
    if labelled:
        kind[labels[labels >= 0]] = 2
    half, small = halves(dtype)
    sub = small / 3 ** 0.5 / L._LinearDistillation._scale(dtype, labels, tau, alpha) * up / n
    off = {}
    for name, m in (("rest", kind == 0), ("entries", kind == 1), ("labels", kind == 2)):
        if m.any() and not (name == "entries" and alpha == 0):
            flat = (sub * hd.norm(dim=0)).norm() * m.sum() ** 0.5 / want[m].norm()
            off["W " + name] = ((W.grad.double() - want)[m].norm() / want[m].norm()).item(), \
                1.25 * (2 / 3 * half ** 2 + flat.item() ** 2) ** 0.5
    wh = up * wg @ Wd / n
    flat = (sub * Wd.norm(dim=0)).norm() * T ** 0.5 / wh.norm()
    off["h"] = ((h.grad.double() - wh).norm() / wh.norm()).item(), 1.25 * (2 / 3 * half ** 2 + flat.item() ** 2) ** 0.5
    assert all(v <= bound for v, bound in off.values()), off


@pytest.mark.parametrize("gdt", [None, torch.bfloat16])
@pytest.mark.parametrize("tau,V,k", [(10.0, 5003, 4), (30.0, 20000, 16), (100.0, 20000, 64), (30.0, 128256, 16), (30.0, 128256, 256)])
def test_high_temperature(tau, V, k, gdt):
    check_high_temperature(tau, V, k, DEV, gdt)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast(dtype):
    """As the call with its inputs in autocast's type, on an fp32 model's hidden states and head."""
    T, V, D = 70, 2051, 64
    _, labels, val, idx, lse = distill_case(T, V, 8, True, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    h = torch.randn(T, D, device=DEV, generator=g).requires_grad_()
    W = (torch.randn(V, D, device=DEV, generator=g) * 0.1).requires_grad_()
    with torch.autocast("cuda", dtype):
        loss = L.linear_distillation(h, W, labels, val, idx, lse, 1.0, 0.5, chunk=32)
        top = L.linear_top_logits(h, W, 6)
    got = torch.autograd.grad(loss, (h, W))
    hl, Wl = h.detach().to(dtype).requires_grad_(), W.detach().to(dtype).requires_grad_()
    want = L.linear_distillation(hl, Wl, labels, val, idx, lse, 1.0, 0.5, chunk=32)
    assert torch.equal(loss, want)
    for a, b in zip(got, torch.autograd.grad(want, (hl, Wl))):
        assert a.dtype == torch.float32 and a.isfinite().all() and torch.equal(a, b.float())
    assert all(torch.equal(a, b) for a, b in zip(top, L.linear_top_logits(hl, Wl, 6)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("wanted", ["h", "W"])
def test_one_gradient_wanted(wanted, dtype):
    T, V, D = 70, 2056, 64
    _, labels, val, idx, lse = distill_case(T, V, 8, True, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    x = {"h": torch.randn(T, D, device=DEV, generator=g).to(dtype), "W": (torch.randn(V, D, device=DEV, generator=g) * 0.1).to(dtype)}
    both = {n: t.clone().requires_grad_() for n, t in x.items()}
    one = {n: t.clone().requires_grad_(n == wanted) for n, t in x.items()}
    want, got = (torch.autograd.grad(L.linear_distillation(**a, labels=labels, top_values=val, top_indices=idx, top_lse=lse, alpha=0.5,
                                                           chunk=32), a[wanted])[0] for a in (both, one))
    assert torch.equal(want, got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (2.0, 0.5), (1.5, 0.5), (1.0, 0.5)])
def test_masses_that_do_not_sum_to_one(tau, alpha, dtype):
    check_other_masses(tau, alpha, DEV, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_without_rows(dtype):
    _, labels, val, idx, lse = (t[:0] for t in distill_case(3, 24, 4, True, device=DEV))
    h = torch.randn(0, 8, device=DEV).to(dtype).requires_grad_()
    W = torch.randn(24, 8, device=DEV).to(dtype).requires_grad_()
    loss = L.linear_distillation(h, W, labels, val, idx, lse, 1.0, 0.5)
    gh, gW = torch.autograd.grad(loss, (h, W))
    assert loss.item() == 0 and gh.shape == (0, 8) and not gW.any()
    top = L.linear_top_logits(h.detach().view(2, 0, 8), W, 4)
    assert top.values.shape == (2, 0, 4) and top.indices.shape == (2, 0, 4) and top.lse.shape == (2, 0)
