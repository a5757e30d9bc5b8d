"""Distillation from a teacher's top logits: the plain path against the oracle, refusals, the model's use of it (CPU)."""
import math

import pytest
import torch

from dion_b200.models import layers as L
from dion_b200.models.llama3 import Transformer, llama3_config
from dion_b200.ops import fused

from operator_oracles import assert_within, distill_oracle


def distill_case(T, V, k, rest, dtype=torch.float32, seed=0, tau=1.0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    teacher = 2 * torch.randn(T, V, generator=g)
    z = (teacher * 0.7 + torch.randn(T, V, generator=g)).to(dtype)
    val, idx = teacher.topk(k, 1)
    lse = torch.logsumexp(teacher / tau, 1) if rest else None
    labels = torch.randint(0, V, (T,), generator=g)
    labels[::4] = -100
    labels[1::5] = idx[1::5, 0]  # labels inside the teacher's set as well as outside
    return [t if t is None else t.to(device) for t in (z, labels, val, idx, lse)]


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (1.0, 0.4), (2.5, 0.7), (2.0, 0.0)])
def test_loss_and_gradient(rest, tau, alpha):
    z, labels, val, idx, lse = distill_case(9, 37, 5, rest, tau=tau)
    loss, grad = fused.distillation_fwd_bwd(z, labels, val, idx, lse, tau, alpha, 0.5)
    want, wg, tl, tg = distill_oracle(z, labels, val, idx, lse, tau, alpha)
    assert abs(loss.item() - want.item()) <= tl.item()
    assert_within(grad, wg * 0.5, tg * 0.5 + 1e-9, "grad")
    assert fused.distillation_fwd_bwd(z, labels, val, idx, lse, tau, alpha, need_grad=False)[1] is None


def test_gradient_by_differences():
    z, labels, val, idx, lse = distill_case(3, 11, 4, True, tau=2.0)
    labels[:] = torch.tensor([2, 5, 7])
    z = z.double()
    grad = distill_oracle(z, labels, val, idx, lse, 2.0, 0.6)[1]
    for at in [(0, 2), (1, 0), (2, int(idx[2, 0]))]:
        e = torch.zeros_like(z)
        e[at] = 1e-5
        d = distill_oracle(z + e, labels, val, idx, lse, 2.0, 0.6)[0] - distill_oracle(z - e, labels, val, idx, lse, 2.0, 0.6)[0]
        assert abs(d.item() / 2e-5 - grad[at].item()) < 1e-6


@pytest.mark.parametrize("rest", [False, True])
def test_unused_repeated_and_masked_entries(rest):
    """Unused entries, rows without any, a column that comes twice, entries at -inf, vocabulary at -inf."""
    z, labels, val, idx, lse = distill_case(8, 23, 4, rest, seed=2)
    labels[:] = 3
    idx[0, 1] = -1
    idx[1] = 99
    idx[2, 1] = idx[2, 0]
    val[3, 2:] = -math.inf
    z[4, [t for t in range(23) if t not in idx[4].tolist() + [3]][:6]] = -math.inf
    z[5] = 0.0
    idx[6] = -5
    val[7] = -math.inf
    loss, grad = fused.distillation_fwd_bwd(z, labels, val, idx, lse, 1.5, 0.5)
    want, wg, tl, tg = distill_oracle(z, labels, val, idx, lse, 1.5, 0.5)
    assert abs(loss.item() - want.item()) <= tl.item()
    assert_within(grad, wg, tg + 1e-9, "grad")


def test_every_row_left_out():
    z, labels, val, idx, lse = distill_case(4, 16, 2, True)
    loss, grad = fused.distillation_fwd_bwd(z, torch.full((4,), -100), val, idx, lse, 1.0, 0.5)
    assert loss.item() == 0 and not grad.any()
    h, W = torch.randn(4, 8, requires_grad=True), torch.randn(16, 8, requires_grad=True)
    loss = L.linear_distillation(h, W, torch.full((4,), 16), val, idx, lse, alpha=0.5)
    loss.backward()
    assert loss.item() == 0 and not h.grad.any() and not W.grad.any()


@pytest.mark.parametrize("chunk", [3, 100])
def test_linear_distillation(chunk):
    torch.manual_seed(0)
    z, labels, val, idx, lse = distill_case(10, 24, 3, True, tau=1.5)
    h, W = torch.randn(2, 5, 8, requires_grad=True), torch.randn(24, 8, requires_grad=True)
    shape = (2, 5)
    args = (labels.view(shape), val.view(2, 5, 3), idx.view(2, 5, 3), lse.view(shape))
    loss = L.linear_distillation(h, W, *args, temperature=1.5, alpha=0.6, chunk=chunk)
    loss.backward()
    hd, Wd = h.detach().double().requires_grad_(), W.detach().double().requires_grad_()
    zd = hd.view(10, 8) @ Wd.t()
    want, wg, *_ = distill_oracle(zd, labels, val, idx, lse, 1.5, 0.6)
    n = (labels >= 0).sum().item()
    assert abs(loss.item() - want.item() / n) < 1e-4
    torch.testing.assert_close(h.grad.double().view(10, 8), wg @ Wd.detach() / n, rtol=1e-4, atol=1e-5)
    torch.testing.assert_close(W.grad.double(), wg.t() @ hd.detach().view(10, 8) / n, rtol=1e-4, atol=1e-5)
    with torch.no_grad():
        assert abs(L.linear_distillation(h, W, *args, temperature=1.5, alpha=0.6, chunk=chunk).item() - loss.item()) < 1e-6


def test_top_logits():
    x = torch.tensor([[1.0, 3.0, 3.0, -0.0, 0.0], [float("-inf"), 2.0, float("nan"), 2.0, 2.0]])
    val, idx, lse = L.top_logits(x, 4)
    assert idx.tolist() == [[1, 2, 0, 3], [2, 1, 3, 4]] and val[0].tolist() == [3, 3, 1, 0]
    assert abs(lse[0].item() - torch.logsumexp(x[0].double(), 0).item()) < 1e-6 and math.isnan(lse[1])
    h, W = torch.randn(2, 3, 8), torch.randn(32, 8)
    got = L.linear_top_logits(h, W, 5, temperature=2.0, chunk=4)
    want = L.top_logits((h.view(6, 8) @ W.t()), 5, 2.0)
    assert torch.equal(got.indices.view(6, 5), want.indices) and got.values.shape == (2, 3, 5) and got.lse.shape == (2, 3)
    torch.testing.assert_close(got.lse.view(6), want.lse)


@pytest.mark.parametrize("change,message", [
    (dict(logits=torch.zeros(4)), "logits \\[T, V\\]"),
    (dict(top_values=torch.zeros(4, 3)), "top_indices"),
    (dict(top_values=torch.zeros(3, 2), top_indices=torch.zeros(3, 2).long()), "4 rows"),
    (dict(top_values=torch.zeros(4, 0), top_indices=torch.zeros(4, 0).long()), "1 to 1024"),
    (dict(top_values=torch.zeros(4, 1025), top_indices=torch.zeros(4, 1025).long()), "1 to 1024"),
    (dict(top_indices=torch.zeros(4, 2)), "int32 or int64"),
    (dict(labels=torch.zeros(3).long()), "labels \\[4\\]"),
    (dict(labels=torch.zeros(4)), "int64 labels"),
    (dict(labels=None, alpha=0.5), "needs labels"),
    (dict(top_lse=torch.zeros(4, 1)), "top_lse \\[4\\]"),
    (dict(temperature=0.0), "temperature"),
    (dict(alpha=1.5), "alpha"),
    (dict(grad_dtype=torch.float64), "gradient"),
    (dict(logits=torch.zeros(4, 8).bfloat16(), grad_dtype=torch.float16), "gradient"),
])
def test_refusals(change, message):
    kw = dict(logits=torch.zeros(4, 8), labels=torch.zeros(4).long(), top_values=torch.zeros(4, 2),
              top_indices=torch.zeros(4, 2).long())
    kw.update(change)
    with pytest.raises(ValueError, match=message):
        fused.distillation_fwd_bwd(**kw)


@pytest.mark.parametrize("x,k,tau,message", [
    (torch.zeros(8), 1, 1.0, "logits"), (torch.zeros(2, 8), 0, 1.0, "k"), (torch.zeros(2, 8), 9, 1.0, "k"),
    (torch.zeros(2, 2000), 1025, 1.0, "k"), (torch.zeros(2, 8), 2, -1.0, "temperature"),
])
def test_top_logits_refusals(x, k, tau, message):
    with pytest.raises(ValueError, match=message):
        L.top_logits(x, k, tau)


def test_window_student_from_a_teacher():
    """A full-attention teacher's top logits train a sliding-window student: gradients against plain autograd, and a few steps run."""
    kw = dict(dim=64, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=512, ffn_dim=128, max_seq_len=64)
    teacher, student = Transformer(llama3_config("tiny", **kw)), Transformer(llama3_config("tiny", attn_window=5, attn_sinks=1, **kw))
    teacher.init_weights(std=0.1, generator=torch.Generator().manual_seed(1))
    student.init_weights(std=0.1, generator=torch.Generator().manual_seed(2))
    tokens = torch.randint(0, 512, (2, 20), generator=torch.Generator().manual_seed(0))
    x, y = tokens[:, :-1], tokens[:, 1:].clone()
    y[0, -3:] = -100
    top = teacher.top_logits(x, 8, temperature=2.0)
    assert top.indices.shape == (2, 19, 8) and not top.values.requires_grad
    student.distillation_loss(x, y, top, temperature=2.0, alpha=0.5).backward()
    got = {n: p.grad.clone() for n, p in student.named_parameters()}
    student.zero_grad()
    z = student(x).reshape(38, 512)
    flat = (y.reshape(-1), top.values.reshape(38, 8), top.indices.reshape(38, 8), top.lse.reshape(38))
    g = distill_oracle(z, *flat, 2.0, 0.5)[1] / (y >= 0).sum()
    z.backward(g.float())
    for n, p in student.named_parameters():
        torch.testing.assert_close(got[n], p.grad, rtol=1e-3, atol=1e-6)
    opt = torch.optim.SGD(student.parameters(), lr=0.1)
    for _ in range(3):
        opt.zero_grad()
        loss = student.distillation_loss(x, y, teacher.top_logits(x, 8, temperature=2.0), temperature=2.0, alpha=0.5)
        loss.backward()
        opt.step()
        assert torch.isfinite(loss)


def test_refused_under_sequence_parallelism():
    m = Transformer(llama3_config("tiny", dim=64, n_layers=1, vocab_size=64, ffn_dim=64))
    m.sp = object()
    x = torch.zeros(1, 4, dtype=torch.long)
    with pytest.raises(ValueError, match="sequence-parallel"):
        m.top_logits(x, 4)
