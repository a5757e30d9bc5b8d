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


# ------------------------------------------------------------------ non-finite inputs
def sees(s, window, sinks, j):
    i = torch.arange(s, device=DEV)
    return (j <= i) & ((i - j < window) | (j < sinks))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_non_finite_keys_reach_every_row_that_sees_them(d, bad):
    """At every place of a step's 64 keys: NaN in o and dq of each row that sees the key, in dv of each key that such a
    row sees; o of the other rows is finite."""
    s, window, sinks = 200, 30, 1
    for j in list(range(64, 128)) + [0, 199]:
        q, k, v, do = make(1, s, 2, 1, d, seed=j)
        with torch.no_grad():
            q.abs_()
            k[:, j, :, 3] = bad
        o, dq, _, dv = run(q, k, v, do, window, sinks)
        rows = sees(s, window, sinks, j)
        assert o[:, rows].isnan().all() and o[:, ~rows].isfinite().all(), j
        # a row whose only key has a NaN score has no other value either
        assert dq[:, rows].isnan().all(), j
        keys = torch.stack([sees(s, window, sinks, t)[rows].any() for t in range(s)])
        assert dv[:, keys].isnan().all(), j


def test_non_finite_queries_and_gradients():
    """NaN in a query: in its row of o and dq. NaN in the output's gradient: in its row of dq and in dv of the keys that it sees."""
    s, window, sinks = 200, 30, 1
    for i in (0, 5, 6, 7, 130, 199):
        q, k, v, do = make(1, s, 2, 1, 64, seed=i)
        with torch.no_grad():
            q[:, i, :, 3] = math.nan
        o, dq, _, _ = run(q, k, v, do, window, sinks)
        others = torch.arange(s, device=DEV) != i
        assert o[:, i].isnan().all() and dq[:, i].isnan().all() and o[:, others].isfinite().all()
        q, k, v, do = make(1, s, 2, 1, 64, seed=i)
        do[:, i] = math.nan
        _, dq, _, dv = run(q, k, v, do, window, sinks)
        keys = torch.tensor([bool(sees(s, window, sinks, t)[i]) for t in range(s)], device=DEV)
        assert dq[:, i].isnan().all() and dv[:, keys].isnan().all()


def test_a_direct_call_of_the_op_does_not_drop_a_gradient():
    q, k, v, _ = make(1, 40, 4, 2, 64)
    with pytest.raises(RuntimeError, match="records no gradient"):
        torch.ops.dion_b200.window_attention_fwd(q, k, v, 8, 1, False)
    with torch.no_grad():
        o = torch.ops.dion_b200.window_attention_fwd(q, k, v, 8, 1, False)[0]
    assert torch.equal(o, L.window_attention(q, k, v, 8, 1).detach())
