"""Sliding-window attention kernels against the 64-bit oracle (tolerances derived there)."""
import pytest
import torch

from dion_b200.models import layers as L
from dion_b200.models.llama3 import Transformer, llama3_config
from dion_b200.ops import check_status, fused

from operator_oracles import assert_within, window_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(b, s, hq, hkv, d, dtype=torch.bfloat16, packed=False, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda h: (torch.randn(b, s, h, d, device=DEV, generator=g) * scale).to(dtype)  # noqa: E731
    if packed:
        q, k, v = r(hq + 2 * hkv).split([hq, hkv, hkv], dim=2)
    else:
        q, k, v = r(hq), r(hkv), r(hkv)
    return [t.detach().requires_grad_() for t in (q, k, v)] + [r(hq)]


def check(q, k, v, do, window, sinks):
    o = L.window_attention(q, k, v, window, sinks)
    grads = torch.autograd.grad(o, (q, k, v), do)
    check_status()
    want = window_oracle(q, k, v, window, sinks, do)
    for got, name in zip((o,) + grads, ("o", "dq", "dk", "dv")):
        assert_within(got, *want[name], name)
    return (o.detach(),) + grads


# lengths around the tile of 128; windows of one, within a tile, of whole tiles, beyond the sequence; first tokens none,
# one, some, more than a tile, more than the sequence
@pytest.mark.parametrize("s,window,sinks", [
    (1, 1, 0), (2, 1, 1), (31, 7, 0), (64, 64, 0), (127, 1, 0), (128, 128, 4), (129, 128, 0), (130, 3, 129), (200, 17, 3),
    (256, 256, 0), (257, 129, 1), (300, 1000, 0), (384, 127, 200), (513, 128, 4), (640, 255, 130), (700, 300, 5),
    (1000, 64, 128), (1025, 511, 1), (90, 40, 500),
])
def test_lengths_windows_sinks(s, window, sinks):
    check(*make(2, s, 4, 2, 64), window, sinks)


@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_dims_types(d, dtype):
    check(*make(1, 333, 3, 1, d, dtype), 100, 2)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (5, 5), (12, 4), (8, 1), (32, 8)])
@pytest.mark.parametrize("d", [64, 128])
def test_heads(hq, hkv, d):
    check(*make(2, 270, hq, hkv, d), 70, 4)


@pytest.mark.parametrize("d", [16, 64, 128])
def test_large_scores(d):
    """Scores of tens, rising along the sequence: the running maximum moves many times."""
    q, k, v, do = make(1, 600, 2, 1, d, scale=3.0)
    with torch.no_grad():
        k *= torch.linspace(0.1, 2.0, 600, device=DEV)[None, :, None, None].to(k.dtype)
    check(q, k, v, do, 400, 3)


@pytest.mark.parametrize("d", [64, 128])
def test_unseen_keys_with_far_larger_scores(d):
    """Keys that a row does not see, in the tiles that it reads, score hundreds more than those that it sees."""
    q, k, v, do = make(1, 400, 2, 1, d)
    with torch.no_grad():
        q[..., 0] = 4.0
        k[..., 0] = 0.0
        k[:, 60::97, :, 0] = 512.0
    check(q, k, v, do, 40, 1)


@pytest.mark.parametrize("window,sinks", [(1, 1), (2, 0), (2, 1), (5, 2)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_few_keys_with_one_that_has_nearly_all(window, sinks, d, dtype):
    """dP - delta cancels there. Two roundings lie between the inputs and each gradient (of P or dS, and of the
    result), each at most half / sqrt(3) of the value in the mean square; a quarter more for all that is fp32."""
    q, k, v, do = make(2, 500, 4, 2, d, dtype, scale=1.3)
    with torch.no_grad():
        k[:, :sinks] *= 2
    o = L.window_attention(q, k, v, window, sinks)
    want = window_oracle(q, k, v, window, sinks, do)
    for got, name in zip(torch.autograd.grad(o, (q, k, v), do), ("dq", "dk", "dv")):
        exact = want[name][0]
        off = ((got.double() - exact).norm() / exact.norm()).item()
        assert off <= 1.25 * (2 / 3) ** 0.5 * torch.finfo(dtype).eps / 2, (name, off)


def test_equal_and_zero_inputs():
    q, k, v, do = make(1, 300, 2, 2, 64)
    with torch.no_grad():
        q.zero_()
    check(q, k, v, do, 129, 1)
    with torch.no_grad():
        v.fill_(1.0)
    o = L.window_attention(q, k, v, 50, 2)
    assert (o - 1).abs().max() <= 2.0 ** -8  # one rounding of P each way cancels but for the sum's


@pytest.mark.parametrize("layout", ["packed", "batch_last", "heads_first", "odd_offset", "expanded_grad", "odd_head_stride"])
def test_strides(layout):
    q, k, v, do = make(2, 200, 4, 2, 64, packed=layout == "packed")
    if layout == "batch_last":
        q, k, v = (t.detach().permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3).requires_grad_() for t in (q, k, v))
    if layout == "heads_first":
        q, k, v, do = (t.detach().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_() for t in (q, k, v, do))
    if layout == "odd_offset":
        def shifted(t):
            buf = torch.empty(t.numel() + 1, device=DEV, dtype=t.dtype)
            buf[1:] = t.detach().reshape(-1)
            return buf[1:].view(t.shape).requires_grad_()
        q, k, v, do = (shifted(t) for t in (q, k, v, do))
    if layout == "odd_head_stride":
        q, k, v = (torch.cat([t.detach(), t.detach()[..., :3]], -1)[..., :64].requires_grad_() for t in (q, k, v))
    if layout == "expanded_grad":
        do = torch.ones((), device=DEV, dtype=q.dtype).expand(q.shape)
    check(q, k, v, do, 60, 3)


def test_repeatable_and_independent_of_the_batch():
    q, k, v, do = make(3, 500, 8, 2, 64)
    a, b = check(q, k, v, do, 150, 4), check(q, k, v, do, 150, 4)
    one = check(*(t.detach()[1:2].requires_grad_() for t in (q, k, v)), do[1:2], 150, 4)
    for x, y, z in zip(a, b, one):
        assert torch.equal(x, y) and torch.equal(x[1:2], z)


def test_empty():
    for b, s in ((0, 5), (2, 0)):
        q, k, v, do = make(b, s, 4, 2, 64)
        o = L.window_attention(q, k, v, 4, 1)
        assert o.shape == q.shape and all(g.shape == t.shape for g, t in zip(torch.autograd.grad(o, (q, k, v), do), (q, k, v)))


def test_against_full_attention_and_fp32_fallback():
    q, k, v, _ = make(2, 190, 4, 2, 64)
    with torch.no_grad():
        full = L.causal_attention(q, k, v)
        torch.testing.assert_close(L.window_attention(q, k, v, 190).float(), full.float(), rtol=2 ** -6, atol=2 ** -6)
        x = [t.float() for t in (q, k, v)]
        assert_within(L.window_attention(*x, 33, 2), *window_oracle(*x, 33, 2)["o"], "fp32")


def test_side_stream():
    q, k, v, do = make(2, 400, 4, 2, 64)
    want = check(q, k, v, do, 100, 4)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = check(q, k, v, do, 100, 4)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_two_streams_at_once():
    sets = [make(1, 700, 4, 2, 64, seed=i) for i in range(2)]
    want = [check(*x, 200, 4) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for n, (x, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                o = L.window_attention(*x[:3], 200, 4)
                got[n] = (o.detach(),) + torch.autograd.grad(o, x[:3], x[3])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_and_replayed():
    q, k, v, do = make(1, 300, 4, 2, 64)

    def step():
        o = L.window_attention(q, k, v, 90, 2)
        return (o.detach(),) + torch.autograd.grad(o, (q, k, v), do)

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    other = make(1, 300, 4, 2, 64, seed=9)
    with torch.no_grad():
        for t, x in zip((q, k, v, do), other):
            t.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, check(*other, 90, 2)):
        assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    """More than 2^31 elements per tensor: the last rows equal those of a short call on the same window."""
    b, s, h, d = 3, 90000, 64, 128
    g = torch.Generator(device=DEV).manual_seed(0)
    k = torch.randn(b, s, h, d, device=DEV, dtype=torch.bfloat16, generator=g)
    assert k.numel() > 2 ** 31
    q = k.roll(1, 1)
    with torch.no_grad():
        o = L.window_attention(q, k, q, 64)
        tail = slice(s - 256, s)
        want = window_oracle(q[-1:, tail], k[-1:, tail], q[-1:, tail], 64, 0)["o"]
    assert_within(o[-1:, s - 128:], want[0][:, 128:], want[1][:, 128:], "tail")


def test_refusals():
    q, k, v, _ = make(1, 16, 4, 2, 64)
    ext = fused.ext()
    with pytest.raises(RuntimeError, match="multiple of 8"):
        fused.window_attention(q[..., :20], k[..., :20], v[..., :20], 4)
    with pytest.raises(RuntimeError, match="bf16 or fp16"):
        ext.window_attention_fwd(q.float(), k.float(), v.float(), 4, 0, False)
    with pytest.raises(RuntimeError, match="window >= 1"):
        ext.window_attention_fwd(q.detach(), k.detach(), v.detach(), 0, 0, False)
    with pytest.raises(ValueError, match="one device"):
        fused.window_attention(q, k.cpu(), v.cpu(), 4)


@pytest.mark.parametrize("mode", [("full", "1"), ("selective", "op")])
def test_model_and_activation_checkpointing(mode):
    """A model with a window trains with the same gradients under activation checkpointing, and selective op
    checkpointing keeps the attention's output instead of computing it again."""
    cfg = llama3_config("debug", attn_window=50, attn_sinks=2, n_layers=2)
    tokens = torch.randint(0, cfg.vocab_size, (2, 130), device=DEV)
    grads, launches = [], []
    for m in (("none", "1"), mode):
        with torch.device(DEV):
            model = Transformer(cfg)
        model.init_weights(generator=torch.Generator(device=DEV).manual_seed(1))
        model = model.bfloat16()
        model.set_activation_checkpointing(*m)
        calls = 0

        class Count(torch.utils._python_dispatch.TorchDispatchMode):
            def __torch_dispatch__(self, func, types, args=(), kwargs=None):
                nonlocal calls
                calls += func is torch.ops.dion_b200.window_attention_fwd.default
                return func(*args, **(kwargs or {}))

        with Count():
            model.loss(tokens[:, :-1], tokens[:, 1:]).backward()
        grads.append([p.grad for p in model.parameters()])
        launches.append(calls)
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    assert launches == [2, 4 if mode[0] == "full" else 2]
