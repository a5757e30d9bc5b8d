"""Products with one row, one column or an inner dimension of one: the stride of the single row is any number."""
import pytest
import torch

from dion_b200 import ops
from dion_b200.models import layers as L

from operator_oracles import distill_oracle
from test_distillation_cpu import distill_case

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("M,N", [(2051, 64), (50257, 64), (129, 8), (7, 24)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_outer_product(M, N, accumulate):
    """a^T b of one row each, a of odd length: one product per entry, exact in fp32, and one addition."""
    g = torch.Generator(device=DEV).manual_seed(M)
    a, b = torch.randn(1, M, device=DEV, generator=g).bfloat16(), torch.randn(1, N, device=DEV, generator=g).bfloat16()
    out = torch.randn(M, N, device=DEV, generator=g)
    want = a.t().float() * b.float() + (out if accumulate else 0.0)
    ops.matmul(a.t(), b, out=out, C=out if accumulate else None, beta=1.0 if accumulate else 0.0)
    ops.check_status()
    torch.testing.assert_close(out, want, rtol=2.0 ** -22, atol=2.0 ** -22)


@pytest.mark.parametrize("T,chunk", [(1, 4096), (65, 64), (3, 1)])
def test_linear_distillation_with_a_chunk_of_one_row(T, chunk):
    V, D = 2051, 64
    _, labels, val, idx, lse = distill_case(T, V, 8, True, device=DEV)
    labels = labels.clamp_min(0)
    g = torch.Generator(device=DEV).manual_seed(0)
    h = torch.randn(T, D, device=DEV, generator=g).bfloat16().requires_grad_()
    W = (torch.randn(V, D, device=DEV, generator=g) * 0.1).bfloat16().requires_grad_()
    loss = L.linear_distillation(h, W, labels, val, idx, lse, 1.0, 0.5, chunk=chunk)
    gh, gW = torch.autograd.grad(loss, (h, W))
    hd, Wd = h.detach().double(), W.detach().double()
    want, wg, _, _ = distill_oracle(hd @ Wd.t(), labels, val, idx, lse, 1.0, 0.5)
    assert abs(loss.item() - want.item() / T) <= 1e-5 * want.abs().item()
    for got, exact in ((gh, wg @ Wd / T), (gW, wg.t() @ hd / T)):
        # two roundings to bf16, in the mean square half / sqrt(3) each, and a quarter more for all that is fp32
        off = ((got.double() - exact).norm() / exact.norm()).item()
        assert off <= 1.25 * (2 / 3) ** 0.5 * 2.0 ** -8, off
