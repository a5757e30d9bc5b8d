"""Cases of the operators that train a sliding-window student from a teacher's top logits.

Three operators are measured, each in its plain form (``own = False``: elementary
torch operations in 32 bits, rounded once at the end) and through the package's
entry points (``own = True``):

* ``attention``: causal attention with a sliding window and a few first tokens
  that stay visible (``dion_b200.models.layers.window_attention``), forward
  alone or forward and backward;
* ``top``: a teacher's k largest logits of each row with their indices and the
  row's log-sum-exp (``layers.top_logits``);
* ``distill``: the distillation loss against those and its gradient with respect
  to the student's logits in one call (``ops.fused.distillation_fwd_bwd``);
  ``linear``: the same through the LM head, chunk by chunk
  (``layers.linear_distillation``), with the gradients of the hidden states and
  of the head's weight.
"""
import math

import torch

own = False

IGNORED = -100  # label of a position that takes no part in the loss


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one evaluation pass over one sequence of the smallest model (4 heads of 64): latency
        attention("window eval, smallest", b=1, s=256, hq=4, hkv=4, d=64, window=64, sinks=4, train=False),
        # a training step's attention of the debug model (16 heads of 16) on a ragged batch of odd length
        attention("window train, heads of 16", b=3, s=777, hq=16, hkv=16, d=16, window=100, sinks=1),
        # the 160M model's attention at the trainer's default batch (8 x 2048, 12 query and 4 key heads)
        attention("window train, 160M", b=8, s=2048, hq=12, hkv=4, d=64, window=512, sinks=4),
        # the 1B model's attention at a 4096-token context
        attention("window train, 1B", b=2, s=4096, hq=32, hkv=8, d=64, window=1024, sinks=4),
        # the 8B model's attention at its full context, q / k / v as slices of one fused projection
        attention("window train, 8B", b=1, s=8192, hq=32, hkv=8, d=128, window=2048, sinks=16, packed=True),
        # a long evaluation sequence of odd length in fp16, one key head for all query heads
        attention("window eval, long fp16", b=1, s=32763, hq=8, hkv=1, d=128, window=4096, sinks=64, train=False,
                  dtype="float16"),
        # the debug model as a teacher of one short sequence: latency
        top("top 8, smallest", t=64, v=2048, k=8),
        # a Llama-vocabulary teacher on half a micro-batch of 8192 tokens
        top("top 64, Llama vocabulary", t=4096, v=128256, k=64),
        # fp32 logits over an odd vocabulary, many entries kept
        top("top 200, odd fp32", t=1500, v=50009, k=200, dtype="float32"),
        # a short sequence of the debug model distilled without labels: latency
        distill("distill 8, smallest", t=64, v=2048, k=8, dtype="float32", labels=False, alpha=1.0, rest=False),
        # half a micro-batch over the Llama vocabulary: soft and hard targets, the rest of the teacher's mass kept
        distill("distill 64, Llama vocabulary", t=4096, v=128256, k=64, alpha=0.5, temperature=2.0, rest=True),
        # the 160M student's LM head with the loss behind it: the head's three products dominate
        distill("linear distill, 160M", t=4096, v=128256, k=32, dim=768, alpha=0.7, temperature=1.5, rest=True),
    ]


def attention(name=None, **kw):
    c = {"op": "attention", "train": True, "packed": False, "dtype": "bfloat16", **kw}
    return {"name": name, **c} if name else c


def top(name=None, **kw):
    c = {"op": "top", "dtype": "bfloat16", "temperature": 1.0, **kw}
    return {"name": name, **c} if name else c


def distill(name=None, **kw):
    c = {"op": "distill", "dtype": "bfloat16", "labels": True, "alpha": 0.5, "temperature": 1.0, "rest": True, "dim": 0, **kw}
    return {"name": name, **c} if name else c


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attention", "attention", "attention", "top", "distill", "distill"])
    if op == "attention":
        s = spread(1, 8192)
        b = min(spread(1, 8), max(1, 8192 // s))
        d = rng.choice([16, 32, 64, 80, 96, 128])
        hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4])
        window, sinks = spread(1, 1800), rng.choice([0, 0, 1, 4, 16, rng.randrange(1, 200)])
        train = rng.random() < 0.7
        return attention(b=b, s=s, hq=hkv * group, hkv=hkv, d=d, window=window, sinks=sinks, train=train,
                         packed=rng.random() < 0.4, dtype=rng.choice(["bfloat16", "bfloat16", "float16"]))
    v = spread(512, 128256)
    t = spread(1, min(4096, 260_000_000 // v))
    k = min(spread(1, 256), v)
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "top":
        return top(t=t, v=v, k=k, dtype=dtype, temperature=rng.choice([1.0, 1.0, 2.0]))
    labels = rng.random() < 0.7
    kw = dict(t=t, v=v, k=k, labels=labels, alpha=round(rng.uniform(0.1, 0.9), 2) if labels else 1.0,
              temperature=rng.choice([1.0, 1.0, 2.0, 3.0]), rest=rng.random() < 0.5)
    if rng.random() < 0.25:
        return distill(dim=rng.choice([256, 512, 768]), **kw)
    return distill(dtype=dtype, **kw)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    dt = getattr(torch, case["dtype"])
    if case["op"] == "attention":
        b, s, hq, hkv, d = (case[n] for n in ("b", "s", "hq", "hkv", "d"))
        if case["packed"]:
            qkv = randn(b, s, hq + 2 * hkv, d).to(dt)
            q, k, v = qkv.split([hq, hkv, hkv], dim=2)
        else:
            q, k, v = (randn(b, s, h, d).to(dt) for h in (hq, hkv, hkv))
        k[:, : case["sinks"]] *= 2  # first tokens draw much attention
        st = {"case": case, "q": q.detach(), "k": k.detach(), "v": v.detach()}
        if case["train"]:
            st = {n: x.requires_grad_() if n in "qkv" else x for n, x in st.items()}
            st["do"] = randn(b, s, hq, d).to(dt)
        return st
    t, v, k = case["t"], case["v"], case["k"]
    if case["op"] == "top":
        return {"case": case, "logits": (2.5 * randn(t, v)).to(dt)}
    # the teacher's logits and a student that has learnt some of them
    teacher = 2.5 * randn(t, v)
    if case["dim"]:
        st = {"h": randn(t, case["dim"]).to(dt).requires_grad_(),
              "W": (randn(v, case["dim"]) * (1.5 / math.sqrt(case["dim"]))).to(dt).requires_grad_()}
    else:
        st = {"logits": (0.8 * teacher).add_(randn(t, v)).to(dt)}
    tau = case["temperature"]
    val, idx = teacher.topk(k, dim=1)
    st["top_values"], st["top_indices"] = val, idx
    st["top_lse"] = torch.logsumexp(teacher / tau, dim=1) if case["rest"] else None
    labels = None
    if case["labels"]:
        labels = torch.randint(0, v, (t,), device="cuda", generator=g)
        labels = torch.where(torch.rand(t, device="cuda", generator=g) < 0.1, IGNORED, labels)  # padded positions
    return {"case": case, "labels": labels, **st}


# ------------------------------------------------------------------ one pass
def run(st):
    case = st["case"]
    if case["op"] == "attention":
        q, k, v = st["q"], st["k"], st["v"]
        if own:
            from dion_b200.models import layers

            if not case["train"]:
                with torch.no_grad():
                    return layers.window_attention(q, k, v, case["window"], case["sinks"])
            o = layers.window_attention(q, k, v, case["window"], case["sinks"])
            return (o.detach(), *torch.autograd.grad(o, (q, k, v), st["do"]))
        with torch.no_grad():
            return window_plain(q, k, v, case["window"], case["sinks"], st.get("do"))
    if case["op"] == "top":
        if own:
            from dion_b200.models import layers

            return layers.top_logits(st["logits"], case["k"], temperature=case["temperature"])
        return top_plain(st["logits"], case["k"], case["temperature"])
    teacher = (st["labels"], st["top_values"], st["top_indices"], st["top_lse"], case["temperature"], case["alpha"])
    if case["dim"]:
        h, W = st["h"], st["W"]
        if own:
            from dion_b200.models import layers

            loss = layers.linear_distillation(h, W, *teacher)
            return (loss.detach(), *torch.autograd.grad(loss, (h, W)))
        with torch.no_grad():
            return linear_plain(h, W, *teacher)
    if own:
        from dion_b200.ops import fused

        return fused.distillation_fwd_bwd(st["logits"], *teacher, 1.0)
    loss, grad = distill_plain(st["logits"].float(), *teacher)
    return loss, grad.to(st["logits"].dtype)


# ------------------------------------------------------------------ plain forms
def window_plain(q, k, v, window, sinks, do=None):
    """Blocks of queries against the band of keys that their windows cover, and
    the first keys beside it. Returns o, or (o, dq, dk, dv)."""
    b, s, hq, d = q.shape
    hkv, g, dt = k.shape[2], hq // k.shape[2], q.dtype
    window, sinks = min(window, s), min(sinks, s)
    blk = max(64, window // 4)
    nb = -(-s // blk)
    L, front, scale = blk + window - 1, window - 1, d ** -0.5
    n = torch.arange(nb, device=q.device)
    qpos = n[:, None] * blk + torch.arange(blk, device=q.device)          # [nb, blk]
    kpos = n[:, None] * blk - front + torch.arange(L, device=q.device)    # [nb, L]
    dist = qpos[:, :, None] - kpos[:, None, :]
    seen = (dist >= 0) & (dist < window) & (kpos[:, None, :] >= 0) & (kpos[:, None, :] < s)
    first = torch.arange(sinks, device=q.device)
    seen = torch.cat([(qpos[:, :, None] - first) >= window, seen], dim=2)   # keys: first ones, then the band
    seen = seen[None, :, None, None]                                        # [1, nb, 1, 1, blk, sinks + L]

    def queries(x):  # [b, s, hq, d] -> [b, nb, hkv, g * blk, d]
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, nb * blk - s))
        return x.view(b, nb, blk, hkv, g, d).permute(0, 1, 3, 4, 2, 5).reshape(b, nb, hkv, g * blk, d)

    def from_queries(x):
        return x.view(b, nb, hkv, g, blk, d).permute(0, 1, 4, 2, 3, 5).reshape(b, nb * blk, hq, d)[:, :s].to(dt)

    def keys(x):  # [b, s, hkv, d] -> [b, nb, hkv, sinks + L, d]
        x = x.float()
        band = torch.nn.functional.pad(x, (0, 0, 0, 0, front, nb * blk - s)).unfold(1, L, blk).transpose(3, 4)
        head = x[:, :sinks].transpose(1, 2)[:, None].expand(b, nb, hkv, sinks, d)
        return torch.cat([head, band], dim=3)

    def from_keys(x):  # the sum over every block that used a key
        out = x.new_zeros(b, nb * blk + front, hkv, d)
        at = (kpos + front).reshape(-1)
        out.index_add_(1, at, x[:, :, :, sinks:].transpose(2, 3).reshape(b, nb * L, hkv, d))
        out = out[:, front:front + s]
        out[:, :sinks] += x[:, :, :, :sinks].sum(1).transpose(1, 2)
        return out.to(dt)

    Q, K, V = queries(q), keys(k), keys(v)
    S = (Q @ K.transpose(-1, -2)).mul_(scale).view(b, nb, hkv, g, blk, sinks + L)
    S.masked_fill_(~seen, float("-inf"))
    # queries behind the last position see nothing: their maximum is set to 0
    m = S.amax(-1, keepdim=True)
    P = S.sub_(torch.where(m == float("-inf"), 0.0, m)).exp_()
    P = P.div_(P.sum(-1, keepdim=True).clamp_min(1e-30)).view(b, nb, hkv, g * blk, sinks + L)
    O = P @ V
    if do is None:
        return from_queries(O)
    dO = queries(do)
    dV = P.transpose(-1, -2) @ dO
    dS = (dO @ V.transpose(-1, -2)).sub_((dO * O).sum(-1, keepdim=True)).mul_(P).mul_(scale)
    return from_queries(O), from_queries(dS @ K), from_keys(dS.transpose(-1, -2) @ Q), from_keys(dV)


def top_plain(logits, k, temperature):
    x = logits.float() + 0.0  # -0 becomes 0
    v = x.shape[1]
    # one whole number per logit: its order, then the lower index first
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * (1 << 32) + (v - 1 - torch.arange(v, device=x.device))
    index = v - 1 - (key.topk(k, dim=1).values & 0xFFFFFFFF)
    x = x / temperature
    m = x.amax(1, keepdim=True)
    lse = m[:, 0] + (x - m).exp().sum(1).log()
    return logits.float().gather(1, index), index, lse


def distill_plain(z, labels, top_values, top_indices, top_lse, temperature, alpha):
    """Sum over the rows of (1 - alpha) CE + alpha t^2 KL, and its gradient, from fp32 logits."""
    tau = temperature
    live = torch.ones(z.shape[0], 1, device=z.device, dtype=torch.bool) if labels is None else labels[:, None] >= 0

    def softmax_log(x):
        x = x - x.amax(1, keepdim=True)
        e = x.exp()
        s = e.sum(1, keepdim=True)
        return x - s.log(), e / s

    logq, q = softmax_log(z / tau)
    t = top_values / tau
    p = (t - top_lse[:, None]).exp() if top_lse is not None else softmax_log(t)[1]
    lq = logq.gather(1, top_indices)
    kl = torch.where(p > 0, p * (p.log() - lq), 0.0).double().sum(1)
    grad = q
    if top_lse is not None:
        # the teacher's mass outside its top entries against the student's there
        p_rest = (1 - p.double().sum(1, keepdim=True)).clamp_min(0)
        q_rest = q.scatter(1, top_indices, 0.0).double().sum(1, keepdim=True)
        kl += torch.where(p_rest > 0, p_rest * (p_rest / q_rest).log(), 0.0)[:, 0]
        keep = grad.gather(1, top_indices)
        grad = grad * (1 - p_rest / q_rest).float()
        grad.scatter_(1, top_indices, keep)
    grad = grad.scatter_add(1, top_indices, -p) * (alpha * tau)
    loss = alpha * tau * tau * kl
    if labels is not None:
        logq, q = softmax_log(z)
        y = labels.clamp_min(0)[:, None]
        loss = loss - (1 - alpha) * logq.gather(1, y)[:, 0].double()
        grad = grad + (1 - alpha) * q.scatter_add(1, y, -torch.ones_like(y, dtype=q.dtype))
    return torch.where(live[:, 0], loss, 0.0).sum().float(), torch.where(live, grad, 0.0)


def linear_plain(h, W, labels, *teacher):
    hf, Wf = h.float(), W.float()
    loss, grad = distill_plain(hf @ Wf.t(), labels, *teacher)
    n = h.shape[0] if labels is None else (labels >= 0).sum().clamp_min(1)
    return loss / n, ((grad @ Wf) / n).to(h.dtype), ((grad.t() @ hf) / n).to(W.dtype)


# ------------------------------------------------------------------ work and exact values
def work(case):
    size = torch.empty(0, dtype=getattr(torch, case["dtype"])).element_size()
    if case["op"] == "attention":
        b, s, hq, hkv, d = (case[n] for n in ("b", "s", "hq", "hkv", "d"))
        pairs = seen_pairs(s, case["window"], case["sinks"])
        rows = 4 * hq + 4 * hkv if case["train"] else 2 * hq + 2 * hkv  # q o do dq, k v dk dv
        return {"bytes": rows * b * s * d * size, "flops": (14 if case["train"] else 4) * b * hq * d * pairs}
    t, v, k = case["t"], case["v"], case["k"]
    if case["op"] == "top":
        return {"bytes": t * v * size + t * (12 * k + 4), "flops": 3 * t * v}
    teacher = t * (12 * k + (4 if case["rest"] else 0) + (8 if case["labels"] else 0))
    if case["dim"]:
        return {"bytes": 2 * (t + v) * case["dim"] * size + teacher, "flops": 6 * t * v * case["dim"]}
    return {"bytes": 2 * t * v * size + teacher, "flops": 8 * t * v}


def seen_pairs(s, window, sinks):
    """Pairs (i, j) with j <= i and (i - j < window or j < sinks)."""
    i = torch.arange(s, dtype=torch.int64)
    band = torch.clamp(i + 1, max=window)
    return int((band + torch.minimum(torch.clamp(i + 1 - window, min=0), torch.tensor(sinks))).sum())


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attention":
        return exact_attention(st, case)
    if case["op"] == "top":
        z = st["logits"].double()
        order = torch.sort(z, dim=1, descending=True, stable=True)
        return order.values[:, : case["k"]], order.indices[:, : case["k"]], torch.logsumexp(z / case["temperature"], 1)
    if case["dim"]:
        h, W = st["h"].detach().double().requires_grad_(), st["W"].detach().double().requires_grad_()
        loss = exact_loss(h @ W.t(), st, case)
        loss = loss / (case["t"] if st["labels"] is None else max(1, int((st["labels"] >= 0).sum())))
        return (loss.detach(), *torch.autograd.grad(loss, (h, W)))
    z = st["logits"].double().requires_grad_()
    loss = exact_loss(z, st, case)
    return (loss.detach(), *torch.autograd.grad(loss, z))


def exact_attention(st, case):
    """The definition, one head of one sequence at a time, its gradients by autograd."""
    s, group = case["s"], case["hq"] // case["hkv"]
    i, j = torch.arange(s, device="cuda")[:, None], torch.arange(s, device="cuda")[None, :]
    hidden = (j > i) | ((i - j >= case["window"]) & (j >= case["sinks"]))
    q, k, v = (st[n].detach().double() for n in "qkv")
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(case["b"]):
        for h in range(case["hq"]):
            x = [t.detach().requires_grad_(case["train"]) for t in (q[b, :, h], k[b, :, h // group], v[b, :, h // group])]
            a = (x[0] @ x[1].t() / math.sqrt(case["d"])).masked_fill(hidden, float("-inf"))
            y = torch.softmax(a, dim=1) @ x[2]
            del a
            o[b, :, h] = y.detach()
            if case["train"]:
                grads = torch.autograd.grad(y, x, st["do"][b, :, h].double())
                dq[b, :, h] = grads[0]
                dk[b, :, h // group] += grads[1]
                dv[b, :, h // group] += grads[2]
    return (o, dq, dk, dv) if case["train"] else o


def exact_loss(z, st, case):
    tau, t = case["temperature"], st["top_values"].double() / case["temperature"]
    logq = torch.log_softmax(z / tau, dim=1)
    if case["rest"]:
        logp = t - st["top_lse"].double()[:, None]
        p_rest = 1 - logp.exp().sum(1)
        rest = torch.logsumexp(logq.scatter(1, st["top_indices"], float("-inf")), dim=1)
        kl = torch.where(p_rest > 0, torch.xlogy(p_rest, p_rest) - p_rest * rest, torch.zeros_like(rest))
    else:
        logp, kl = torch.log_softmax(t, dim=1), 0.0
    kl = kl + (logp.exp() * (logp - logq.gather(1, st["top_indices"]))).sum(1)
    loss = case["alpha"] * tau * tau * kl
    if st["labels"] is not None:
        ce = -torch.log_softmax(z, dim=1).gather(1, st["labels"].clamp_min(0)[:, None])[:, 0]
        loss = torch.where(st["labels"] >= 0, loss + (1 - case["alpha"]) * ce, torch.zeros_like(ce))
    return loss.sum()
