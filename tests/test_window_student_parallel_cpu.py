"""A sliding-window student under tensor, sequence, pipeline and fully sharded data parallelism on CPU (gloo), against
one process: training on labels through the trainer, and the distillation loss with its gradients."""
import functools

import pytest
import torch

from test_distributed_cpu import spawn

WINDOW = dict(n_layers=2, vocab_size=512, max_seq_len=64, attn_window=6, attn_sinks=2)


def _trainer(**kw):
    from dion_b200.integration.hybrid_optimizer import HybridOptimizersContainer
    from dion_b200.integration.trainer import Trainer, TrainerConfig

    opt = HybridOptimizersContainer.Config(name="Muon", lr=0.02, scalar_lr=3e-3)
    torch.manual_seed(0)
    return Trainer(TrainerConfig(**{**dict(model="tiny", model_overrides=dict(WINDOW), seq_len=32, local_batch_size=4, steps=3,
                                           warmup_steps=0, optimizer=opt, seed=5), **kw}), device=torch.device("cpu"))


def _train_body(kw, rank, world):
    tr = _trainer(**kw)
    return [float(tr.train_step(*tr.data.next())) for _ in range(3)]


@functools.lru_cache(None)
def _alone(body):
    (status, res), = spawn(functools.partial(body, {}), world=1).values()
    assert status == "ok", res
    return res


@pytest.mark.parametrize("kw", [dict(tp=2, sequence_parallel=False), dict(tp=2, sequence_parallel=True),
                                dict(pp=2, pp_microbatches=2, use_fsdp=False)])
def test_training_matches_one_process(kw):
    out = spawn(functools.partial(_train_body, kw), world=2)
    for status, res in out.values():
        assert status == "ok", res
    want = torch.tensor(_alone(_train_body))
    assert torch.allclose(want, torch.tensor(out[0][1]), rtol=2e-3, atol=2e-3), (want, out[0][1])


def _distill_body(kw, rank, world):
    from dion_b200.models.llama3 import Transformer, llama3_config

    tr = _trainer(param_dtype="float32", **kw)  # so that the order of sums is all that differs
    teacher = Transformer(llama3_config("tiny", n_layers=2, vocab_size=512, max_seq_len=64))
    teacher.init_weights(std=0.1, generator=torch.Generator().manual_seed(1))
    tokens = torch.randint(0, 512, (4, 21), generator=torch.Generator().manual_seed(2))
    x, y = tokens[:, :-1], tokens[:, 1:].clone()
    y[:, -4:] = -100  # as many on every rank: each takes the mean over its own rows
    if kw.get("dp_shard", 1) > 1:
        x, y = x[2 * rank:2 * rank + 2], y[2 * rank:2 * rank + 2]
    top = teacher.top_logits(x, 8, temperature=2.0)
    own = tr.model.top_logits(x, 4)
    loss = tr.model.distillation_loss(x, y, top, temperature=2.0, alpha=0.5)
    loss.backward()
    full = lambda g: g.full_tensor() if hasattr(g, "full_tensor") else g  # noqa: E731
    return (loss.item(), {n: full(p.grad).clone().numpy() for n, p in tr.model.named_parameters()},
            own.indices.numpy(), own.lse.detach().numpy())


@pytest.mark.parametrize("kw", [dict(dp_shard=2, local_batch_size=2), dict(tp=2, sequence_parallel=False)])
def test_distillation_matches_one_process(kw):
    out = spawn(functools.partial(_distill_body, kw), world=2)
    for status, res in out.values():
        assert status == "ok", res
    (loss, grads, idx, lse), ranks = _alone(_distill_body), [out[r][1] for r in range(2)]
    cut = "dp_shard" in kw
    assert abs(sum(r[0] for r in ranks) / 2 - loss) < 1e-5 * loss
    for r, (_, g, i, z) in enumerate(ranks):
        rows = slice(2 * r, 2 * r + 2) if cut else slice(None)
        assert (i == idx[rows]).all() and abs(z - lse[rows]).max() < 1e-4
        for n, want in grads.items():
            torch.testing.assert_close(torch.as_tensor(g[n]), torch.as_tensor(want), rtol=1e-3, atol=1e-6, msg=lambda m: f"{n}: {m}")
