"""Top logits: the ways that a row can take through the kernel, at the sizes where they change."""
import pytest
import torch

from dion_b200.ops import fused

from test_distillation_gpu import TYPES, check_top

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("k,V", [(8, 2048), (17, 40000), (64, 128256), (100, 50009)])
def test_second_bound_over_the_candidates(k, V):
    """Some 128 to 512 candidates a row, thinned out by one warp's search while the others wait: thousands of rows at
    once, beside another stream's work on the same SMs, and the same rows again."""
    T = min(4096, 60_000_000 // V)
    x = torch.randn(T, V, device=DEV, generator=torch.Generator(device=DEV).manual_seed(k))
    val, idx, lse = check_top(x, k)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        with torch.cuda.stream(other):
            fused.top_logits(x, k)
        again = fused.top_logits(x, k)
        assert torch.equal(val, again.values) and torch.equal(idx, again.indices) and torch.equal(lse, again.lse)
    torch.cuda.current_stream().wait_stream(other)


# rows of every lead (the odd widths and strides), widths whose last group of 8 columns a lead takes, so that the row
# has a round of groups less than the width says, and more entries than one set of columns per thread gives a bound for
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rounds,k", [(1, 257), (1, 512), (1, 1024), (2, 300), (2, 700), (3, 300), (3, 500), (5, 300), (8, 257)])
def test_widths_with_a_round_less_in_some_rows(rounds, k, dtype):
    for extra in (8, 9, 11, 14, 15):
        V = 4096 * rounds + extra
        x = torch.randn(9, V, device=DEV, generator=torch.Generator(device=DEV).manual_seed(V + k)).to(dtype)
        check_top(x, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,stride", [(4104, 4105), (4104, 4111), (8200, 8203), (4109, 4200), (32776, 32777)])
@pytest.mark.parametrize("k", [257, 512, 1000])
def test_padded_rows(V, stride, k, dtype):
    x = torch.randn(9, stride, device=DEV, generator=torch.Generator(device=DEV).manual_seed(V)).to(dtype)
    check_top(x[:, :V], k)
    check_top(x[:, stride - V:], k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [100, 700, 5003])
def test_rows_of_the_lowest_value(dtype, V):
    """A row that is masked throughout by the type's lowest value (its log-sum-exp is that value, to rounding), one that is
    masked but for a few columns, and one of the largest values."""
    x = torch.randn(4, V, device=DEV, generator=torch.Generator(device=DEV).manual_seed(V)).to(dtype)
    x[0] = torch.finfo(dtype).min
    x[1, 5:] = torch.finfo(dtype).min
    x[2, ::2] = torch.finfo(dtype).max
    for tau in (1.0, 2.0, 1.5):
        lse = check_top(x, 7, tau)[2]
        assert lse.isfinite().all()
