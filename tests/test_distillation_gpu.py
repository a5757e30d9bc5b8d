"""Top-logits and distillation kernels against the 64-bit oracle (tolerances derived there)."""
import math

import pytest
import torch

from dion_b200.models import layers as L
from dion_b200.models.llama3 import Transformer, llama3_config
from dion_b200.ops import fused

from operator_oracles import assert_within, distill_oracle, halves
from test_distillation_cpu import distill_case

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


# ------------------------------------------------------------------ top logits
def check_top(x, k, tau=1.0):
    val, idx, lse = fused.top_logits(x, k, tau)
    xf = x.float()
    order = (xf + 0.0).sort(dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(idx, order)
    assert torch.equal(val.nan_to_num(1e30), xf.gather(1, order).nan_to_num(1e30))
    want = torch.logsumexp(x.double() / tau, 1)
    fine = want.isfinite()
    assert ((lse.double() - want)[fine].abs() <= 2.0 ** -18 * (1 + want[fine].abs())).all()
    return val, idx, lse


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,k", [(1, 1, 1), (3, 7, 7), (5, 100, 3), (4, 2048, 8), (2, 2049, 1024), (3, 4096, 1024), (7, 5003, 64),
                                   (2, 50009, 200), (9, 32768, 256), (2, 32771, 257), (3, 128256, 64), (2, 131073, 1000)])
def test_top_logits(dtype, T, V, k):
    g = torch.Generator(device=DEV).manual_seed(V)
    check_top((3 * torch.randn(T, V, device=DEV, generator=g)).to(dtype), k, 1.0 if V % 2 else 2.0)


@pytest.mark.parametrize("V,k", [(600, 600), (5000, 100), (40000, 17), (40000, 1024)])
def test_top_logits_many_equal(V, k):
    """Equal values throughout, two values, few large ones among equal ones, sorted rows, -inf, NaN, both zeros."""
    x = torch.zeros(8, V, device=DEV)
    x[1, ::3] = 1
    x[2, V - 5:] = torch.arange(5.0, device=DEV)
    x[3] = torch.arange(V, device=DEV)
    x[4] = -torch.arange(V, device=DEV).float()
    x[5] = -math.inf
    x[5, V // 2] = 0
    x[6, V // 3] = math.nan
    x[7, ::2] = -0.0
    check_top(x, k)
    check_top(x.bfloat16(), k)


def test_top_logits_layouts():
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(6, 3001, device=DEV, generator=g).bfloat16()
    check_top(x[:, :3000], 20)            # row stride beyond the row, odd
    check_top(x[:, 5:], 20)               # rows that start unaligned
    check_top(x.t()[:, :5], 3)            # columns contiguous instead
    check_top(x[::2], 20)
    assert all(t.shape[0] == 0 for t in fused.top_logits(x[:0], 4))


def test_top_logits_captured_and_streams():
    x = torch.randn(40, 5000, device=DEV)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        fused.top_logits(x, 9)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fused.top_logits(x, 9)
    x.normal_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, check_top(x, 9)))


def test_top_logits_offsets_beyond_32_bits():
    x = torch.zeros(17000, 128256, device=DEV, dtype=torch.bfloat16)
    assert x.numel() > 2 ** 31
    x[-3:].normal_()
    val, idx, _ = fused.top_logits(x, 5)
    a, b, _ = check_top(x[-3:], 5)
    assert torch.equal(val[-3:], a) and torch.equal(idx[-3:], b)


# ------------------------------------------------------------------ distillation
def check_distill(z, labels, val, idx, lse, tau, alpha, scale=1.0, grad_dtype=None):
    loss, grad = fused.distillation_fwd_bwd(z, labels, val, idx, lse, tau, alpha, scale, grad_dtype)
    want, wg, tl, tg = distill_oracle(z, labels, val, idx, lse, tau, alpha)
    assert abs(loss.item() - want.item()) <= tl.item(), (loss.item(), want.item(), tl.item())
    half, small = halves(grad.dtype)
    assert grad.dtype == (grad_dtype or z.dtype)
    assert_within(grad, wg * scale, half * (wg * scale).abs() + abs(scale) * tg + small + 1e-30, "grad")
    only, none = fused.distillation_fwd_bwd(z, labels, val, idx, lse, tau, alpha, scale, grad_dtype, need_grad=False)
    assert none is None and torch.equal(only, loss)
    return loss, grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("T,V,k,tau,alpha", [(1, 1, 1, 1.0, 0.5), (3, 9, 9, 2.0, 0.5), (5, 100, 3, 1.0, 1.0), (6, 2048, 8, 1.0, 0.3),
                                             (4, 2051, 1024, 3.0, 0.9), (3, 32771, 64, 2.0, 0.6), (3, 128256, 64, 2.0, 0.0),
                                             (2, 128256, 200, 1.5, 0.5), (2, 131071, 33, 0.5, 0.5)])
def test_distillation(dtype, rest, T, V, k, tau, alpha):
    z, labels, val, idx, lse = distill_case(T, V, k, rest, dtype, seed=V + k, tau=tau, device=DEV)
    check_distill(z, labels, val, idx, lse, tau, alpha, scale=0.25)
    check_distill(z, None, val, idx.int(), lse, tau, 1.0)


@pytest.mark.parametrize("gdt", [torch.bfloat16, torch.float16])
def test_fp32_logits_with_a_half_gradient(gdt):
    z, labels, val, idx, lse = distill_case(5, 10007, 16, True, tau=2.0, device=DEV)
    check_distill(z, labels, val, idx, lse, 2.0, 0.5, grad_dtype=gdt)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_unused_repeated_and_masked_entries(rest, dtype):
    z, labels, val, idx, lse = distill_case(9, 2300, 40, rest, dtype, seed=2, device=DEV)
    labels[:] = 3
    idx[0, 1] = -1
    idx[1] = 2300
    idx[2, 1:9] = idx[2, 0]
    labels[2] = idx[2, 0]
    val[3, 2:] = -math.inf
    keep = torch.ones(2300, dtype=torch.bool, device=DEV)
    keep[idx[4]] = False
    keep[3] = False
    z[4, keep] = torch.where(torch.arange(int(keep.sum()), device=DEV) < 700, -math.inf, z[4, keep].float()).to(dtype)
    z[5] = 0.0
    idx[6] = -5
    val[7] = -math.inf
    labels[8] = 2300
    check_distill(z, labels, val, idx, lse, 1.5, 0.5)


def test_sure_students():
    """A student far surer than the teacher, and one that is sure of another column: nothing cancels to 0 or NaN."""
    z, labels, val, idx, lse = distill_case(4, 3001, 8, True, device=DEV)
    labels[:] = 11
    z *= 0.01
    z[0, idx[0, 0]] = 30.0
    z[1, idx[1, 1]] = 200.0
    z[2, 7] = 90.0
    z[3] = torch.linspace(-300, 300, 3001, device=DEV)
    check_distill(z, labels, val, idx, lse, 1.0, 0.5)


def test_layouts():
    z, labels, val, idx, lse = distill_case(6, 3001, 8, True, torch.bfloat16, device=DEV)
    val, idx = val.t().contiguous().t(), idx.repeat_interleave(2, 1)[:, ::2]
    idx = idx.clamp(max=2990)
    check_distill(z[:, :3000], labels.clamp(max=2990), val, idx, lse, 1.0, 0.5)
    check_distill(z[:, 5:], labels.clamp(max=2990), val, idx, lse, 1.0, 0.5)
    check_distill(z.t().contiguous().t(), labels, val, idx, lse, 1.0, 0.5)
    wide = torch.zeros(6, 3008, device=DEV, dtype=torch.bfloat16)
    wide[:, :3000] = z[:, :3000]
    check_distill(wide[:, :3000], labels.clamp(max=2990), val, idx, lse, 1.0, 0.5)
    loss, grad = fused.distillation_fwd_bwd(z[:0], labels[:0], val[:0], idx[:0], lse[:0])
    assert loss.item() == 0 and grad.shape == (0, 3001)


def test_rows_behind_keep_their_values_and_runs_repeat():
    """The gradient's rows only are written, and two runs give the same bits."""
    z, labels, val, idx, lse = distill_case(12, 5000, 20, True, torch.bfloat16, device=DEV)
    buf = torch.full((14, 5000), 7.0, device=DEV, dtype=torch.bfloat16)
    loss = torch.empty((), device=DEV)
    fused.ext().distill_fwd_bwd(z, labels, val, idx, lse, buf[1:13], loss, 2.0, 0.5, 1.0)
    assert (buf[0] == 7).all() and (buf[13] == 7).all()
    for _ in range(2):
        l2, g2 = fused.distillation_fwd_bwd(z, labels, val, idx, lse, 2.0, 0.5)
        assert torch.equal(l2, loss) and torch.equal(g2, buf[1:13])


def test_captured_and_replayed():
    z, labels, val, idx, lse = distill_case(16, 5003, 20, True, torch.bfloat16, device=DEV)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        fused.distillation_fwd_bwd(z, labels, val, idx, lse, 2.0, 0.5)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fused.distillation_fwd_bwd(z, labels, val, idx, lse, 2.0, 0.5)
    z2 = distill_case(16, 5003, 20, True, torch.bfloat16, seed=5, device=DEV)[0]
    z.copy_(z2)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, check_distill(z, labels, val, idx, lse, 2.0, 0.5)))


def test_offsets_beyond_32_bits():
    T, V = 17000, 128256
    z = torch.zeros(T, V, device=DEV, dtype=torch.bfloat16)
    tail, labels, val, idx, lse = distill_case(3, V, 8, True, torch.bfloat16, device=DEV)
    z[-3:] = tail
    pad = lambda t, fill: torch.cat([torch.full((T - 3,) + t.shape[1:], fill, device=DEV, dtype=t.dtype), t])  # noqa: E731
    loss, grad = fused.distillation_fwd_bwd(z, pad(labels, -100), pad(val, 0.0), pad(idx, 0), pad(lse, 0.0), 1.0, 0.5)
    a, b = check_distill(tail, labels, val, idx, lse, 1.0, 0.5)
    assert torch.equal(grad[-3:], b) and not grad[:-3].any() and abs(loss.item() - a.item()) <= 1e-5 * abs(a.item())


def test_refusals():
    z, labels, val, idx, lse = distill_case(2, 64, 4, True, device=DEV)
    ext, loss = fused.ext(), torch.empty((), device=DEV)
    with pytest.raises(RuntimeError, match="logits"):
        ext.distill_fwd_bwd(z.double(), labels, val, idx, lse, None, loss, 1.0, 0.5, 1.0)
    with pytest.raises(RuntimeError, match="labels"):
        ext.distill_fwd_bwd(z, labels.cpu(), val, idx, lse, None, loss, 1.0, 0.5, 1.0)
    with pytest.raises(RuntimeError, match="grad"):
        ext.distill_fwd_bwd(z, labels, val, idx, lse, torch.empty(2, 63, device=DEV), loss, 1.0, 0.5, 1.0)
    with pytest.raises(RuntimeError, match="k <= min"):
        ext.top_logits(z, torch.empty(2, 65, device=DEV), idx, lse, 1.0)


# ------------------------------------------------------------------ behind the LM head, and all together
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_distillation(dtype):
    """Three roundings lie on the way to the gradients: the logits' gradient, the product's result and the final
    division; sums of T or V products in fp32 are covered by the slop."""
    T, V, D = 300, 4096, 256
    z, labels, val, idx, lse = distill_case(T, V, 16, True, tau=1.5, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    h = torch.randn(T, D, device=DEV, generator=g).to(dtype).requires_grad_()
    W = (torch.randn(V, D, device=DEV, generator=g) * 0.1).to(dtype).requires_grad_()
    loss = L.linear_distillation(h, W, labels, val, idx, lse, 1.5, 0.6, chunk=128)
    loss.backward()
    hd, Wd = h.detach().double(), W.detach().double()
    want, wg, tl, tg = distill_oracle(hd @ Wd.t(), labels, val, idx, lse, 1.5, 0.6)
    n = (labels >= 0).sum()
    half, small = halves(dtype)
    logit = 2.0 ** -20 * (hd.abs() @ Wd.abs().t())          # fp32 sums of D products
    tg = tg + half * wg.abs() + small + logit.amax(1, keepdim=True) * tg * 2.0 ** 15 * 2
    assert abs(loss.item() - want.item() / n.item()) <= (tl.item() + 2 * logit.amax().item() * T) / n.item()
    for got, exact, err, m in ((h.grad, wg @ Wd / n, tg @ Wd.abs() / n, None), (W.grad, wg.t() @ hd / n, tg.t() @ hd.abs() / n, None)):
        assert_within(got, exact, err + 2 * half * exact.abs() + small * 3, "linear")


@pytest.mark.parametrize("n", [1, 7, 8, 9, 4099, 1 << 20])
@pytest.mark.parametrize("dtype", TYPES)
def test_scale_cast(n, dtype):
    x = torch.randn(n, device=DEV)
    f = torch.tensor(0.37, device=DEV)
    assert torch.equal(fused.scale_cast(x, f, dtype), (x * f).to(dtype))
    assert torch.equal(fused.scale_cast(x[1:], f, dtype), (x[1:] * f).to(dtype))


def test_linear_top_logits():
    g = torch.Generator(device=DEV).manual_seed(0)
    h = torch.randn(2, 150, 256, device=DEV, generator=g).bfloat16()
    W = torch.randn(4096, 256, device=DEV, generator=g).bfloat16()
    val, idx, lse = L.linear_top_logits(h, W, 12, 2.0, chunk=64)
    z = h.reshape(300, 256).double() @ W.double().t()
    slack = 2.0 ** -20 * (h.reshape(300, 256).double().abs() @ W.double().abs().t()).amax()
    assert ((z.gather(1, idx.view(300, 12)) - val.view(300, 12)).abs() <= slack).all()
    assert (val.view(300, 12)[:, -1:] >= z.topk(12).values[:, -1:] - slack).all()
    assert ((torch.logsumexp(z / 2, 1) - lse.view(300)).abs() <= slack + 1e-5).all()


def test_window_student_from_a_teacher():
    """Teacher's top logits -> window student's loss -> gradients, as they are used: against the oracle's loss gradient
    sent back through the same student, and captured into a graph."""
    t_cfg, s_cfg = llama3_config("debug", n_layers=2), llama3_config("debug", n_layers=2, attn_window=40, attn_sinks=2)
    models = []
    for cfg, seed in ((t_cfg, 1), (s_cfg, 2)):
        with torch.device(DEV):
            m = Transformer(cfg)
        m.init_weights(std=0.05, generator=torch.Generator(device=DEV).manual_seed(seed))
        models.append(m.bfloat16())
    teacher, student = models
    tokens = torch.randint(0, 2048, (2, 151), device=DEV)
    x, y = tokens[:, :-1], tokens[:, 1:].clone()
    y[0, -20:] = -100

    def step():
        top = teacher.top_logits(x, 16, temperature=2.0)
        loss = student.distillation_loss(x, y, top, temperature=2.0, alpha=0.5)
        return top, loss.detach(), torch.autograd.grad(loss, list(student.parameters()))

    top, loss, grads = step()
    h = student(x, return_hidden=True)
    flat = (y.reshape(-1), top.values.view(-1, 16), top.indices.view(-1, 16), top.lse.view(-1))
    hd = h.detach().reshape(-1, 256).double()
    W = student.output.weight.detach().double()
    want, wg, *_ = distill_oracle(hd @ W.t(), *flat, 2.0, 0.5)
    n = (y >= 0).sum().item()
    assert abs(loss.item() - want.item() / n) <= 1e-4 * abs(loss.item())
    rest = [p for p in student.parameters() if p is not student.output.weight]
    plain = torch.autograd.grad(h, rest, (wg @ W / n).view(h.shape).bfloat16())
    got = [g for p, g in zip(student.parameters(), grads) if p is not student.output.weight]
    for a, b in zip(got, plain):
        # the two gradients of the hidden states differ by a few roundings; norms over whole matrices average them
        assert (a.double() - b.double()).norm() <= 2.0 ** -6 * b.double().norm() + 1e-12
    del h, plain
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, loss2, grads2 = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss, loss2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))
