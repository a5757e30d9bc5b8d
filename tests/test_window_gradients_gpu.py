"""Sliding-window attention: the gradients' accuracy where dP - delta cancels, over head dimensions, odd lengths and layouts.

delta = do . o is taken from o and from what o's rounding left out. In rows of two or three keys of which one has nearly
all of the mass, delta from the rounded o alone would be off by more than dP - delta itself, which a bound on single
elements (with the rounding of o among its terms) does not show; the norm over all rows does."""
import pytest
import torch

from dion_b200.models import layers as L
from dion_b200.ops import check_status

from operator_oracles import window_oracle
from test_window_attention_gpu import make

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check_norms(q, k, v, do, window, sinks):
    """Roundings between the inputs and each gradient, each at most half / sqrt(3) of its value in the mean square: of P or
    dS, of the result, and for dq and dk of P within o. The last leaves the key with nearly all (whose exponential is 1)
    as it is; the other's, P2, puts P1 P2 half dP2 on dS_1 = P1 P2 (dP1 - dP2), where dP1 and dP2 are independent: half of a
    rounding's square. A quarter more for all that is fp32 and for the remainder's own rounding."""
    grads = torch.autograd.grad(L.window_attention(q, k, v, window, sinks), (q, k, v), do)
    check_status()
    want = window_oracle(q, k, v, window, sinks, do)
    for got, name in zip(grads, ("dq", "dk", "dv")):
        exact = want[name][0]
        off = ((got.double() - exact).norm() / exact.norm()).item()
        assert off <= 1.25 * (2.5 / 3) ** 0.5 * torch.finfo(q.dtype).eps / 2, (name, off)


@pytest.mark.parametrize("d", [8, 16, 40, 64, 72, 80, 96, 128])
@pytest.mark.parametrize("s", [333, 513])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_dims_and_odd_lengths(d, s, dtype):
    """Scores of some standard deviations, whatever the head dimension: one key of two has nearly all in most rows."""
    q, k, v, do = make(2, s, 6, 2, d, dtype, scale=2.0)
    check_norms(q, k, v, do, 2, 0)
    check_norms(q, k, v, do, 1, 1)


@pytest.mark.parametrize("layout", ["packed", "heads_first", "odd_offset"])
@pytest.mark.parametrize("d", [64, 80])
def test_layouts(layout, d):
    q, k, v, do = make(2, 257, 4, 2, d, packed=layout == "packed", scale=2.0)
    if layout == "heads_first":
        q, k, v, do = (t.detach().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_() for t in (q, k, v, do))
    if layout == "odd_offset":
        def shifted(t):
            buf = torch.empty(t.numel() + 1, device=DEV, dtype=t.dtype)
            buf[1:] = t.detach().reshape(-1)
            return buf[1:].view(t.shape).requires_grad_()
        q, k, v, do = (shifted(t) for t in (q, k, v, do))
    check_norms(q, k, v, do, 2, 1)
