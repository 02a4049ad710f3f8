"""Performance cases of the operators at the two ends of a model whose embedding
is also its output layer: the loss over the vocabulary and its gradients from
hidden rows and the embedding, distillation from a teacher's top logits, and the
lookup of tokens with its gradient.

Kinds of case (the "kind" of a case):

  loss     softmax cross entropy of x w^T against one target a token
           (head.cross_entropy).  "train": the gradients of x and w too
           (head.cross_entropy_grad), times a number for each token or for all.
  distill  the divergence of softmax(x w^T / temperature) from a teacher's
           distribution over its top logits (head.distill_grad), with gradients.
  embed    rows of a table by token, scaled (embed.lookup).  "train": the
           table's gradient in fp32 too (embed.lookup_grad).

A token whose target is -100 (a prompt's, a padded one) has no loss and gives no
gradient; a teacher's entry of index -1 is left out.
"""
import math

import torch

own = False

DEV = "cuda"
NONE = -100
LOSS_SCALE = 65536.0  # shared by 256 tokens at least: dw has to fit fp16
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}

MOST_BYTES = 5.0e8    # what the largest listed cases cost
MOST_FLOPS = 6.45e12


def listed():
    return [
        # scoring: the next token of 8 sequences, the 237M model
        {"name": "loss_score_few", "kind": "loss", "tokens": 8, "columns": 768, "vocab": 32000,
         "type": "f16", "train": False, "masked": 0.0, "weights": False},
        # evaluation: an odd number of tokens, the 1.3B model
        {"name": "loss_eval_1p3b", "kind": "loss", "tokens": 4099, "columns": 2048,
         "vocab": 32000, "type": "bf16", "train": False, "masked": 0.0, "weights": False},
        # a short micro-batch of a small model, nothing a multiple of anything
        {"name": "loss_train_odd", "kind": "loss", "tokens": 333, "columns": 901, "vocab": 5003,
         "type": "f16", "train": True, "masked": 0.1, "weights": True},
        # training, 2 sequences of 2048 tokens, the 237M model
        {"name": "loss_train_237m_batch", "kind": "loss", "tokens": 4096, "columns": 768,
         "vocab": 32000, "type": "f16", "train": True, "masked": 0.0, "weights": False},
        # training on answers, 8 sequences of 2048 tokens, prompts masked
        {"name": "loss_train_237m", "kind": "loss", "tokens": 16384, "columns": 768,
         "vocab": 32000, "type": "f16", "train": True, "masked": 0.25, "weights": False},
        # training, 8 sequences of 2048 tokens, the 1.3B model
        {"name": "loss_train_1p3b", "kind": "loss", "tokens": 16384, "columns": 2048,
         "vocab": 32000, "type": "bf16", "train": True, "masked": 0.0, "weights": False},
        # a short micro-batch against a teacher's few best
        {"name": "distill_few", "kind": "distill", "tokens": 517, "columns": 768, "vocab": 32308,
         "type": "bf16", "top": 8, "temperature": 1.0, "masked": 0.1},
        # distillation of the 237M model, 64 logits a token
        {"name": "distill_237m", "kind": "distill", "tokens": 4096, "columns": 768,
         "vocab": 32000, "type": "f16", "top": 64, "temperature": 2.0, "masked": 0.0},
        # serving: one token of each of 8 sequences
        {"name": "embed_decode", "kind": "embed", "tokens": 8, "columns": 768, "vocab": 32000,
         "type": "f16", "train": False, "scale": 1.0},
        # a long prompt of the 1.3B model, rows scaled
        {"name": "embed_prompt", "kind": "embed", "tokens": 16384, "columns": 2048,
         "vocab": 32000, "type": "bf16", "train": False, "scale": 45.25},
        # training, 8 sequences of 2048 tokens, the 237M model
        {"name": "embed_train_237m", "kind": "embed", "tokens": 16384, "columns": 768,
         "vocab": 32000, "type": "f16", "train": True, "scale": 1.0},
        # odd rows in fp32
        {"name": "embed_train_odd", "kind": "embed", "tokens": 5003, "columns": 901,
         "vocab": 5003, "type": "f32", "train": True, "scale": 30.0},
    ]


def _log(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    kind = rng.choice(["loss", "loss", "loss", "distill", "distill", "embed", "embed"])
    while True:
        columns = _log(rng, 64, 4096) if rng.random() < 0.3 else 64 * _log(rng, 1, 64)
        vocab = rng.choice([32000, 32308, _log(rng, 300, 131072), _log(rng, 300, 131072)])
        c = {"kind": kind, "tokens": _log(rng, 1, 16384), "columns": columns, "vocab": vocab}
        if kind == "loss":
            c.update({"type": rng.choice(["f16", "bf16"]), "train": rng.random() < 0.7,
                      "masked": rng.choice([0.0, 0.0, 0.1, 0.5]),
                      "weights": rng.random() < 0.4})
        elif kind == "distill":
            c.update({"type": rng.choice(["f16", "bf16"]), "top": _log(rng, 1, 128),
                      "temperature": rng.choice([1.0, 2.0, 4.0]),
                      "masked": rng.choice([0.0, 0.2])})
        else:
            c.update({"type": rng.choice(["f16", "bf16", "f32"]), "train": rng.random() < 0.6,
                      "scale": rng.choice([1.0, 30.0])})
        w = work(c)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return c


def work(case):
    t, d, v, es = case["tokens"], case["columns"], case["vocab"], SIZE[case["type"]]
    if case["kind"] == "embed":
        n = t * d
        reads = min(t, v) * d * es + 8 * t
        if not case["train"]:
            return {"bytes": reads + es * n, "flops": n}
        return {"bytes": reads + 2 * es * n + 4 * v * d, "flops": 2 * n}
    train = case.get("train", True)
    live = t * (1.0 - case["masked"])
    b = es * (t + v) * d * (2 if train else 1) + 12 * t
    if case["kind"] == "distill":
        b += t * case["top"] * 8
    return {"bytes": b, "flops": (6 if train else 2) * live * v * d}


# ---- inputs -----------------------------------------------------------------

def _rare(gen, n, vocab):
    """Tokens as text has them: the k-th most frequent about 1 / k as often."""
    u = torch.rand((n,), generator=gen, device=DEV, dtype=torch.float64)
    rank = torch.exp(u * math.log(vocab + 1.0)).long().clamp(1, vocab) - 1
    return torch.randperm(vocab, generator=gen, device=DEV)[rank]


def _mask(gen, case):
    """The tokens without a loss: runs of them, as prompts are."""
    t = case["tokens"]
    out = torch.zeros((t,), dtype=torch.bool, device=DEV)
    n = int(t * case["masked"])
    if n:
        at = torch.arange(t, device=DEV)
        runs = max(1, t // 2048)
        out = (at % -(-t // runs)) < n // runs
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype, t, d, v = TYPES[case["type"]], case["tokens"], case["columns"], case["vocab"]
    s = {"case": case}
    if case["kind"] == "embed":
        s["table"] = torch.randn((v, d), generator=gen, device=DEV).mul_(0.02).to(dtype)
        s["tokens"] = _rare(gen, t, v)
        if case["train"]:
            s["dy"] = (0.05 * torch.randn((t, d), generator=gen, device=DEV)).to(dtype)
        return s
    # logits a few units wide, and above that a target's, by nothing to a lot
    w = torch.randn((v, d), generator=gen, device=DEV) * (2.0 / math.sqrt(d))
    target = _rare(gen, t, v)
    x = torch.randn((t, d), generator=gen, device=DEV)
    x += 4.0 * torch.rand((t, 1), generator=gen, device=DEV) * w[target]
    s["x"], s["w"] = x.to(dtype), w.to(dtype)
    masked = _mask(gen, case)
    if case["kind"] == "loss":
        s["targets"] = torch.where(masked, NONE, target)
        s["grad"] = LOSS_SCALE / max(t, 256)
        if case["weights"]:
            s["grad"] = s["grad"] * torch.rand((t,), generator=gen, device=DEV)
        return s
    # a teacher's best: the target among them, the others anywhere, falling logits;
    # in some rows fewer of them
    k = min(case["top"], v)
    first = torch.randint(0, v, (t, 1), generator=gen, device=DEV)
    step = torch.randint(1, max(2, v // k), (t, 1), generator=gen, device=DEV)
    index = (first + step * torch.arange(k, device=DEV)) % v
    index[:, 0] = torch.where((index == target[:, None]).any(1), index[:, 0], target)
    falls = torch.empty((t, k), device=DEV).exponential_(2.0, generator=gen).cumsum(1)
    few = 1 + torch.randint(0, 2 * k, (t, 1), generator=gen, device=DEV)
    out = (torch.arange(k, device=DEV) >= few) | masked[:, None]
    s["index"] = torch.where(out, -1, index).int()
    s["logits"] = 15.0 - falls
    s["grad"] = (LOSS_SCALE / max(t, 256) * case["temperature"] ** 2
                 * torch.rand((t,), generator=gen, device=DEV))
    return s


# ---- the plain forms --------------------------------------------------------

def run(state):
    return _own(state) if own else _plain(state)


def _plain(state):
    case, kind = state["case"], state["case"]["kind"]
    dtype = TYPES[case["type"]]
    if kind == "embed":
        out = {"y": (state["table"][state["tokens"]].float() * case["scale"]).to(dtype)}
        if case["train"]:
            dw = torch.zeros(state["table"].shape, device=DEV)
            out["dw"] = dw.index_add_(0, state["tokens"], state["dy"].float() * case["scale"])
        return out
    x, w = state["x"].float(), state["w"].float()
    if kind == "loss":
        z = x @ w.t()
        live = state["targets"] >= 0
        target = state["targets"].clamp_min(0)[:, None]
        most = z.amax(1, keepdim=True)
        lse = most + (z - most).exp().sum(1, keepdim=True).log()
        nll = ((lse - z.gather(1, target))[:, 0] * live).contiguous()
        if not case["train"]:
            return nll
        dz = (z - lse).exp()
        dz.scatter_add_(1, target, torch.full_like(lse, -1.0))
        dz *= (live * state["grad"])[:, None]
        return {"loss": nll, "dx": (dz @ w).to(dtype), "dw": (dz.t() @ x).to(dtype)}
    tau = case["temperature"]
    z = (x @ w.t()) / tau
    most = z.amax(1, keepdim=True)
    lse = most + (z - most).exp().sum(1, keepdim=True).log()
    there = state["index"] >= 0
    live = there.any(1, keepdim=True)
    index = state["index"].clamp_min(0).long()
    a = torch.where(there, state["logits"] / tau, -1e30)
    a = a - a.amax(1, keepdim=True)
    e = a.exp() * there
    total = e.sum(1, keepdim=True)
    p = e / total.clamp_min(1e-30)
    log_p = a - total.clamp_min(1e-30).log()
    loss = torch.where(there, p * (log_p - (z.gather(1, index) - lse)), 0.0).sum(1)
    dz = (z - lse).exp() * live
    dz.scatter_add_(1, index, -p)
    dz *= state["grad"][:, None] / tau
    return {"loss": loss, "dx": (dz @ w).to(dtype), "dw": (dz.t() @ x).to(dtype)}


# ---- the framework's kernels --------------------------------------------------

def _own(state):
    from ark_amd import embed, head
    case, kind = state["case"], state["case"]["kind"]
    if kind == "embed":
        out = {"y": embed.lookup(state["table"], state["tokens"], scale=case["scale"])}
        if case["train"]:
            out["dw"] = embed.lookup_grad(state["dy"], state["tokens"], case["vocab"],
                                          scale=case["scale"])
        return out
    if kind == "loss":
        if not case["train"]:
            return head.cross_entropy(state["x"], state["w"], state["targets"])
        loss, dx, dw = head.cross_entropy_grad(state["x"], state["w"], state["targets"],
                                               grad=state["grad"])
    else:
        loss, dx, dw = head.distill_grad(state["x"], state["w"], state["index"], state["logits"],
                                         grad=state["grad"], temperature=case["temperature"])
    return {"loss": loss, "dx": dx, "dw": dw}


# ---- the definitions in 64 bits -----------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    f64 = torch.float64
    if case["kind"] == "embed":
        table = state["table"].to(f64)
        out = {"y": torch.index_select(table, 0, state["tokens"]) * case["scale"]}
        if case["train"]:
            order = torch.argsort(state["tokens"], stable=True)
            rows = torch.cumsum(state["dy"].to(f64)[order] * case["scale"], 0)
            ends = torch.searchsorted(state["tokens"][order],
                                      torch.arange(case["vocab"], device=DEV), right=True)
            upto = torch.cat([torch.zeros_like(rows[:1]), rows])[ends]
            out["dw"] = torch.diff(upto, dim=0, prepend=torch.zeros_like(rows[:1]))
        return out
    tau = case.get("temperature", 1.0)
    x, w = state["x"].to(f64), state["w"].to(f64)
    t, v = len(x), len(w)
    loss, dx, dw = x.new_zeros((t,)), torch.zeros_like(x), torch.zeros_like(w)
    grad = torch.as_tensor(state["grad"], dtype=f64, device=DEV).expand(t)
    train = case.get("train", True)
    for lo in range(0, t, 2048):
        at = slice(lo, lo + 2048)
        log_q = torch.log_softmax(torch.matmul(x[at], w.t()) / tau, 1)
        # the distribution wanted, written out over the whole vocabulary
        want = torch.zeros_like(log_q)
        row = torch.arange(len(log_q), device=DEV)
        if case["kind"] == "loss":
            ok = state["targets"][at] != NONE
            want[row[ok], state["targets"][at][ok]] = 1.0
            loss[at] = -(want * log_q).sum(1)
        else:
            index, logits = state["index"][at].long(), state["logits"][at].to(f64) / tau
            ok = (index >= 0).any(1)
            logits = logits.masked_fill(index < 0, -math.inf)
            p = torch.softmax(torch.where(ok[:, None], logits, torch.zeros_like(logits)), 1)
            p = p.masked_fill(index < 0, 0.0)
            want.scatter_add_(1, index.clamp_min(0), p)
            loss[at] = torch.special.xlogy(p, p).sum(1) - (want * log_q).sum(1)
        if train:
            dz = (log_q.exp() * ok[:, None] - want) * grad[at, None] / tau
            dx[at] = torch.matmul(dz, w)
            dw += torch.matmul(dz.t(), x[at])
    return {"loss": loss, "dx": dx, "dw": dw} if train else loss
