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
