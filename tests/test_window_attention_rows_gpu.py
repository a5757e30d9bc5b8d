"""Sliding-window attention: rows whose gradients are known exactly, and non-finite inputs."""
import math

import pytest
import torch

from dion_b200.models import layers as L
from dion_b200.ops import check_status

from operator_oracles import assert_within, window_oracle
from test_window_attention_gpu import make

pytestmark = pytest.mark.gpu
DEV = "cuda"


def run(q, k, v, do, window, sinks):
    o = L.window_attention(q, k, v, window, sinks)
    grads = torch.autograd.grad(o, (q, k, v), do)
    check_status()
    return (o.detach(),) + grads


# ------------------------------------------------------------------ rows that see one key
@pytest.mark.parametrize("d", [16, 64, 80, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("s,window,sinks", [(1, 1, 0), (1, 7, 3), (128, 1, 0), (333, 1, 0)])
def test_one_visible_key_in_every_row(s, window, sinks, d, dtype):
    """The softmax of one score is 1 whatever the score: o is the value, dq and dk are zeros."""
    q, k, v, do = make(2, s, 6, 2, d, dtype)
    o, dq, dk, dv = run(q, k, v, do, window, sinks)
    assert torch.equal(o, v.detach().repeat_interleave(3, 2))
    assert not dq.any() and not dk.any()
    assert_within(dv, *window_oracle(q, k, v, window, sinks, do)["dv"], "dv")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,s,window,sinks", [(2, 300, 40, 0), (2, 300, 40, 2), (1, 2100, 1, 1), (1, 2100, 700, 130)])
def test_first_row_sees_one_key(b, s, window, sinks, d):
    """Row 0 sees key 0 alone. With a gradient in row 0 only, dq and dk are zeros everywhere and dv is that gradient."""
    q, k, v, do = make(b, s, 4, 2, d)
    assert not run(q, k, v, do, window, sinks)[1][:, 0].any()
    do[:, 1:] = 0
    _, dq, dk, dv = run(q, k, v, do, window, sinks)
    assert not dq.any() and not dk.any() and not dv[:, 1:].any()
    assert_within(dv, *window_oracle(q, k, v, window, sinks, do)["dv"], "dv")
