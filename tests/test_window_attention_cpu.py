"""Sliding-window attention: the plain path against the oracle, refusals, and the model's use of it (CPU)."""
import pytest
import torch

from dion_b200.models import layers as L
from dion_b200.models.llama3 import Transformer, llama3_config
from dion_b200.ops import fused

from operator_oracles import assert_within, window_oracle


@pytest.mark.parametrize("s,window,sinks", [(1, 1, 0), (7, 1, 0), (7, 3, 2), (33, 8, 1), (33, 100, 0), (20, 4, 50)])
def test_plain_form(s, window, sinks):
    torch.manual_seed(0)
    q, k, v = torch.randn(2, s, 4, 8), torch.randn(2, s, 2, 8), torch.randn(2, s, 2, 8)
    for t in (q, k, v):
        t.requires_grad_()
    o = L.window_attention(q, k, v, window, sinks)
    do = torch.randn_like(o)
    grads = torch.autograd.grad(o, (q, k, v), do)
    want = window_oracle(q, k, v, window, sinks, do)
    for got, name in zip((o,) + grads, ("o", "dq", "dk", "dv")):
        assert_within(got, *want[name], name)


def test_oracle_gradients_by_differences():
    """The oracle's closed-form gradients against central differences of its own output."""
    torch.manual_seed(1)
    q, k, v = (torch.randn(1, 6, h, 8, dtype=torch.float64) for h in (2, 1, 1))
    do = torch.randn(1, 6, 2, 8, dtype=torch.float64)
    want = window_oracle(q, k, v, 3, 1, do)
    f = lambda: (window_oracle(q, k, v, 3, 1)["o"][0] * do).sum()  # noqa: E731
    for t, name in ((q, "dq"), (k, "dk"), (v, "dv")):
        for at in [(0, 0, 0, 0), (0, 3, 0, 5), (0, 5, 0, 7)]:
            keep = t[at].item()
            t[at] = keep + 1e-5
            up = f()
            t[at] = keep - 1e-5
            down = f()
            t[at] = keep
            assert abs((up - down).item() / 2e-5 - want[name][0][at].item()) < 1e-7


@pytest.mark.parametrize("change,message", [
    (dict(window=0), "window >= 1"),
    (dict(sinks=-1), "sinks >= 0"),
    (dict(k=(2, 5, 3, 8), v=(2, 5, 3, 8)), "do not divide"),
    (dict(v=(2, 5, 1, 8)), "q \\[b, s, hq, d\\]"),
    (dict(k=(2, 4, 2, 8), v=(2, 4, 2, 8)), "differ"),
    (dict(k=(2, 5, 2, 16), v=(2, 5, 2, 16)), "differ"),
    (dict(dtype=torch.float64), "one type"),
])
def test_refusals(change, message):
    shape = {"q": (2, 5, 4, 8), "k": (2, 5, 2, 8), "v": (2, 5, 2, 8)}
    shape.update({n: c for n, c in change.items() if n in shape})
    q, k, v = (torch.randn(shape[n]) for n in "qkv")
    k = k.to(change.get("dtype", k.dtype))
    for f in (L.window_attention, fused.window_attention):
        with pytest.raises(ValueError, match=message):
            f(q, k, v, change.get("window", 3), change.get("sinks", 0))


def test_model_with_a_window():
    """A window that covers the sequence gives the full-attention model; a short one does not, and counts fewer FLOPs."""
    torch.manual_seed(0)
    tokens = torch.randint(0, 512, (2, 24))
    kw = dict(dim=64, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=512, ffn_dim=128, max_seq_len=64)
    losses = []
    for extra in ({}, {"attn_window": 24}, {"attn_window": 5, "attn_sinks": 2}):
        cfg = llama3_config("tiny", **kw, **extra)
        m = Transformer(cfg)
        m.init_weights(std=0.2, generator=torch.Generator().manual_seed(3))
        loss = m.loss(tokens[:, :-1], tokens[:, 1:])
        loss.backward()
        assert all(torch.isfinite(p.grad).all() for p in m.parameters())
        losses.append(loss.item())
    assert abs(losses[0] - losses[1]) < 1e-5 and abs(losses[0] - losses[2]) > 1e-4
    full, short = llama3_config("1B"), llama3_config("1B", attn_window=1024, attn_sinks=4)
    assert full.flops_per_token(8192) - short.flops_per_token(8192) == 12 * 16 * 2048 * (8192 - 1028)
    assert short.flops_per_token(512) == full.flops_per_token(512)


def test_activation_checkpointing_gives_the_same_gradients():
    tokens = torch.randint(0, 512, (2, 17), generator=torch.Generator().manual_seed(0))
    grads = []
    for mode in (("none", "1"), ("full", "1"), ("selective", "op")):
        m = Transformer(llama3_config("tiny", dim=64, n_layers=2, vocab_size=512, ffn_dim=128, attn_window=6, attn_sinks=1))
        m.init_weights(generator=torch.Generator().manual_seed(3))
        m.set_activation_checkpointing(*mode)
        m.loss(tokens[:, :-1], tokens[:, 1:]).backward()
        grads.append([p.grad for p in m.parameters()])
    for g in grads[1:]:
        for a, b in zip(grads[0], g):
            torch.testing.assert_close(a, b)


def test_command_line_window():
    """--model.attn_window and --model.attn_sinks reach the model's configuration."""
    from dion_b200.integration.config import apply_overrides
    from dion_b200.integration.config_registry import get_config
    from dion_b200.train import trainer_config_from_job

    job = get_config("llama3_160m_dion")
    assert trainer_config_from_job(job).model_overrides == job.model.overrides
    apply_overrides(job, ["--model.attn_window", "9", "--model.attn_sinks", "2"])
    cfg = trainer_config_from_job(job)
    assert cfg.model_overrides["attn_window"] == 9 and cfg.model_overrides["attn_sinks"] == 2
    job.model.attn_window = None
    with pytest.raises(ValueError, match="attn_window"):
        trainer_config_from_job(job)
