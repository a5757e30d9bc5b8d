"""The dispatcher op beneath the sliding-window attention (CPU)."""
import pytest
import torch

from dion_b200.ops import has_ext


@pytest.mark.skipif(not has_ext(), reason="extension not built")
def test_a_direct_call_does_not_drop_a_gradient():
    """The op has no CPU kernel: with gradients off it is that which is missing, with them on the call is refused first."""
    q = torch.zeros(1, 3, 2, 8, dtype=torch.bfloat16)
    for grads in ((True, False, False), (False, True, False), (False, False, True)):
        args = [q.clone().requires_grad_(g) for g in grads]
        with pytest.raises(RuntimeError, match="records no gradient"):
            torch.ops.dion_b200.window_attention_fwd(*args, 2, 0, False)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="CPU"):
            torch.ops.dion_b200.window_attention_fwd(*args, 2, 0, False)
