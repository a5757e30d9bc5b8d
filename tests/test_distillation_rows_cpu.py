"""Distillation: refusals behind the LM head, and its ranges (CPU)."""
import pytest
import torch

from dion_b200.models import layers as L
from dion_b200.ops import fused

from distillation_extremes import (check_high_temperature, check_lowest, check_masked_vocabulary, check_offset,
                                    check_other_masses)
from test_distillation_cpu import distill_case


# ------------------------------------------------------------------ refusals
def linear_case(T=6):
    z, labels, val, idx, lse = distill_case(T, 24, 3, True)
    h, W = torch.randn(T, 8), torch.randn(24, 8)
    return dict(h=h, W=W, labels=labels, top_values=val, top_indices=idx, top_lse=lse, alpha=0.5)


@pytest.mark.parametrize("name", ["labels", "top_values", "top_indices", "top_lse", "top_values,top_indices", "h"])
@pytest.mark.parametrize("chunk", [2, 4096])
def test_linear_refuses_other_numbers_of_rows(name, chunk):
    """More rows than tokens are not cut, fewer are not an empty chunk."""
    for rows in (slice(0, 4), [0, 1, 2, 3, 4, 5, 0, 1]):
        kw = linear_case()
        for n in name.split(","):
            kw[n] = kw[n][rows]
        with pytest.raises(ValueError, match="distillation"):
            L.linear_distillation(**kw, chunk=chunk)


@pytest.mark.parametrize("change,message", [
    (dict(top_indices=torch.zeros(3, 6).long()), "top_indices"),   # as many entries in other rows
    (dict(alpha=1.5), "alpha"), (dict(alpha=float("nan")), "alpha"), (dict(labels=None), "needs labels"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(top_values=torch.zeros(6, 0), top_indices=torch.zeros(6, 0).long()), "1 to 1024"),
    (dict(labels=torch.zeros(6)), "int64 labels"),
])
def test_linear_refusals(change, message):
    kw = linear_case()
    kw.update(change)
    with pytest.raises(ValueError, match=message):
        L.linear_distillation(**kw)
    empty = {n: t[:0] if torch.is_tensor(t) and n != "W" else t for n, t in kw.items()}
    with pytest.raises(ValueError, match=message):
        L.linear_distillation(**empty)


@pytest.mark.parametrize("temperature", [float("inf"), float("nan"), 1e-30, 1e30])
def test_temperatures_out_of_range(temperature):
    z, labels, val, idx, lse = distill_case(3, 16, 2, True)
    with pytest.raises(ValueError, match="temperature"):
        fused.distillation_fwd_bwd(z, labels, val, idx, lse, temperature, 0.5)
    with pytest.raises(ValueError, match="temperature"):
        L.top_logits(z, 2, temperature)


def test_linear_without_rows():
    kw = {n: t[:0] if torch.is_tensor(t) and n != "W" else t for n, t in linear_case().items()}
    kw["h"], kw["W"] = kw["h"].requires_grad_(), kw["W"].requires_grad_()
    loss = L.linear_distillation(**kw)
    loss.backward()
    assert loss.item() == 0 and kw["h"].grad.shape == (0, 8) and not kw["W"].grad.any()


# ------------------------------------------------------------------ extreme logits
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (1.0, 0.5), (2.0, 0.5), (1.5, 1.0)])
def test_common_offset(tau, alpha, rest):
    check_offset(tau, rest, alpha, "cpu")


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("alpha", [1.0, 0.5])
def test_rows_of_the_lowest_value(alpha, rest):
    check_lowest(rest, alpha, "cpu", torch.float32)


@pytest.mark.parametrize("rest", [False, True])
def test_vocabulary_masked_by_the_lowest_value(rest):
    check_masked_vocabulary(rest, "cpu", torch.float32)


@pytest.mark.parametrize("tau,V,k", [(10.0, 5003, 4), (30.0, 20000, 16), (100.0, 20000, 64)])
def test_high_temperature(tau, V, k):
    check_high_temperature(tau, V, k, "cpu")


# ------------------------------------------------------------------ autocast
def test_autocast():
    """As the call with its inputs in autocast's type: the fp32 products stay fp32, the gradients come back in the inputs' type."""
    kw = linear_case()
    kw["h"], kw["W"] = kw["h"].requires_grad_(), kw["W"].requires_grad_()
    with torch.autocast("cpu", torch.bfloat16):
        loss = L.linear_distillation(**kw)
        top = L.linear_top_logits(kw["h"], kw["W"], 4)
    got = torch.autograd.grad(loss, (kw["h"], kw["W"]))
    low = dict(kw, h=kw["h"].detach().bfloat16().requires_grad_(), W=kw["W"].detach().bfloat16().requires_grad_())
    want = L.linear_distillation(**low)
    assert torch.equal(loss, want) and loss.dtype == torch.float32
    for a, b in zip(got, torch.autograd.grad(want, (low["h"], low["W"]))):
        assert a.dtype == torch.float32 and torch.equal(a, b.float())
    for a, b in zip(top, L.linear_top_logits(low["h"], low["W"], 4)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("wanted", ["h", "W"])
def test_one_gradient_wanted(wanted):
    """A frozen head, or hidden states without a gradient: the other's is as with both."""
    both = linear_case()
    both["h"], both["W"] = both["h"].requires_grad_(), both["W"].requires_grad_()
    want = torch.autograd.grad(L.linear_distillation(**both), both[wanted])[0]
    one = dict(both, h=both["h"].detach(), W=both["W"].detach())
    one[wanted] = one[wanted].requires_grad_()
    loss = L.linear_distillation(**one)
    loss.backward()
    assert torch.equal(one[wanted].grad, want) and one["hW".replace(wanted, "")].grad is None


def test_unequal_rows_over_ranks():
    """Two ranks' losses, each times ranks * (its rows) / (all rows) and averaged as data parallelism does, have the gradient
    of the mean over all rows; the plain average has not."""
    T = 12
    kw = linear_case(T)
    kw["labels"][:5] = -100
    kw["labels"][5:] = torch.arange(T - 5)

    def grad(rows, factor=1.0):
        part = {n: t[rows] if torch.is_tensor(t) and n != "W" else t for n, t in kw.items()}
        part["W"] = kw["W"].clone().requires_grad_()
        return torch.autograd.grad(L.linear_distillation(**part) * factor, part["W"])[0]

    halves = slice(0, 6), slice(6, T)
    live = [int((kw["labels"][r] >= 0).sum()) for r in halves]
    assert live == [1, 6]
    whole = grad(slice(0, T))
    scaled = sum(grad(r, 2 * n / sum(live)) for r, n in zip(halves, live)) / 2
    torch.testing.assert_close(scaled, whole, rtol=1e-5, atol=1e-7)
    assert not torch.allclose(sum(grad(r) for r in halves) / 2, whole, rtol=1e-2, atol=1e-4)


@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (2.0, 0.5), (1.5, 0.5)])
def test_masses_that_do_not_sum_to_one(tau, alpha):
    check_other_masses(tau, alpha, "cpu")
