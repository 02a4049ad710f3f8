"""Performance cases of the operators on either side of a layer's matrix
products: rotary positions, the norms of queries and keys with the rotation in
the same pass, and activations kept in 8 bits for the backward pass, with the
weight gradient that reads them.

Kinds of case (the "kind" of a case):

  rope   queries and keys rotated by their positions (Rope.apply), or rotated
         back, as their gradients are.
  norm   a pass of Rope.norm: RMS norm of every head of q and k, its gain, the
         rotation.  "train": also the backward pass, which gives the gradients
         of q, k and both gains; "keep8": q and k are kept in 8 bits by the
         forward pass, and the backward pass reads them from there.
  keep   an activation packed into 8 bits and unpacked again (act.pack,
         act.unpack).
  grad   a linear layer's weight gradient from its input, kept in 8 bits since
         the forward pass: act.pack, then act.weight_grad into fp32.

The 8-bit form: 32 consecutive tokens of one column share a power of two 2^e,
the smallest with max |x| <= 127 * 2^e, and keep q = round(x / 2^e).
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5
BASE = 10000.0
GROUP = 32          # tokens that share an exponent
LONG = 131072       # positions a scaled model reaches
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
SCALING = {
    "none": None,
    "linear": {"kind": "linear", "factor": 8.0},
    "ntk": {"kind": "ntk", "factor": 8.0},
    "yarn": {"kind": "yarn", "factor": 32.0, "original": 4096},
    "bands": {"kind": "bands", "factor": 8.0, "original": 8192, "low": 1.0, "high": 4.0},
}

MOST_BYTES = 1.35e9   # what the largest listed cases cost
MOST_FLOPS = 3.69e11


def listed():
    return [
        # serving: one new token of each of 8 sequences, the 237M model's heads
        {"name": "rope_decode", "kind": "rope", "tokens": 8, "heads": 12, "kv_heads": 12,
         "head": 64, "rotary": 64, "layout": "half", "scaling": "none", "type": "f16",
         "inverse": False},
        # a long prompt, half of each head rotated, pairs interleaved, far positions
        {"name": "rope_prompt_long", "kind": "rope", "tokens": 16384, "heads": 16, "kv_heads": 16,
         "head": 128, "rotary": 64, "layout": "interleaved", "scaling": "yarn", "type": "bf16",
         "inverse": False},
        # gradients of q and k rotated back, an odd number of tokens, fp32
        {"name": "rope_back_odd", "kind": "rope", "tokens": 5003, "heads": 12, "kv_heads": 12,
         "head": 64, "rotary": 64, "layout": "half", "scaling": "linear", "type": "f32",
         "inverse": True},
        # serving: 32 sequences, the 1.3B model's heads over shared keys
        {"name": "norm_decode", "kind": "norm", "tokens": 32, "heads": 16, "kv_heads": 4,
         "head": 128, "rotary": 128, "layout": "half", "scaling": "bands", "type": "bf16",
         "train": False, "keep8": False},
        # a prompt of an odd length through the 237M model's heads
        {"name": "norm_prompt_odd", "kind": "norm", "tokens": 4099, "heads": 12, "kv_heads": 12,
         "head": 64, "rotary": 64, "layout": "half", "scaling": "none", "type": "f16",
         "train": False, "keep8": False},
        # a training pass, 8 sequences of 2048 tokens, the 237M model
        {"name": "norm_train_237m", "kind": "norm", "tokens": 16384, "heads": 12, "kv_heads": 12,
         "head": 64, "rotary": 64, "layout": "half", "scaling": "none", "type": "f16",
         "train": True, "keep8": True},
        # a training pass of the 1.3B model, 16 sequences of 2048 tokens
        {"name": "norm_train_1p3b", "kind": "norm", "tokens": 32768, "heads": 16, "kv_heads": 16,
         "head": 128, "rotary": 128, "layout": "half", "scaling": "none", "type": "bf16",
         "train": True, "keep8": True},
        # a hidden activation kept and read back, 8 sequences of 2048 tokens
        {"name": "keep_hidden", "kind": "keep", "tokens": 16384, "columns": 2048, "type": "f16"},
        # a small model's odd sizes, fp32
        {"name": "keep_odd_f32", "kind": "keep", "tokens": 1001, "columns": 901, "type": "f32"},
        # a short micro-batch of a small model, odd sizes
        {"name": "grad_small_odd", "kind": "grad", "tokens": 333, "columns": 333, "outputs": 901,
         "type": "f16", "layout": "in_out"},
        # the 237M model's w1, 8 sequences of 2048 tokens
        {"name": "grad_237m", "kind": "grad", "tokens": 16384, "columns": 768, "outputs": 2048,
         "type": "f16", "layout": "in_out"},
        # the 1.3B model's w1, weights stored output-major
        {"name": "grad_1p3b", "kind": "grad", "tokens": 16384, "columns": 2048, "outputs": 5504,
         "type": "bf16", "layout": "out_in"},
    ]


def _log(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def _heads(rng):
    heads = _log(rng, 1, 32)
    kv = rng.choice([h for h in range(1, heads + 1) if heads % h == 0])
    head = rng.choice([64, 64, 128, 128, 256, 2 * _log(rng, 16, 120)])
    rotary = head if rng.random() < 0.6 else max(2, head // rng.choice([2, 4]) // 2 * 2)
    return {"heads": heads, "kv_heads": kv, "head": head, "rotary": rotary,
            "layout": rng.choice(["half", "half", "interleaved"]),
            "scaling": rng.choice(["none", "none", "linear", "ntk", "yarn", "bands"])}


def draw(rng):
    kind = rng.choice(["rope", "rope", "norm", "norm", "norm", "keep", "grad", "grad"])
    kinds = rng.choice(["f16", "bf16", "f32"])
    while True:
        if kind == "rope":
            c = {"kind": kind, "tokens": _log(rng, 1, 32768), **_heads(rng), "type": kinds,
                 "inverse": rng.random() < 0.4}
        elif kind == "norm":
            train = rng.random() < 0.6
            c = {"kind": kind, "tokens": _log(rng, 1, 32768), **_heads(rng), "type": kinds,
                 "train": train, "keep8": train and rng.random() < 0.7}
        elif kind == "keep":
            c = {"kind": kind, "tokens": _log(rng, 1, 32768), "columns": _log(rng, 32, 8192),
                 "type": kinds}
        else:
            odd = rng.random() < 0.4
            side = (lambda hi: _log(rng, 32, hi)) if odd else (lambda hi: 64 * _log(rng, 1, hi / 64))
            c = {"kind": kind, "tokens": _log(rng, 32, 32768), "columns": side(4096),
                 "outputs": side(8192), "type": rng.choice(["f16", "bf16"]),
                 "layout": rng.choice(["in_out", "out_in"])}
        w = work(c)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and 3072 not in _widths(c):
            return c


def _widths(c):
    """Row lengths of a case (3072 is left to programs that have it)."""
    d = c.get("head", 0)
    return (c.get("columns", 0), c.get("outputs", 0), d * c.get("heads", 0),
            d * c.get("kv_heads", 0))


def work(case):
    es, t = SIZE[case["type"]], case["tokens"]
    if case["kind"] in ("rope", "norm"):
        d = case["head"]
        n = t * d * (case["heads"] + case["kv_heads"])
        kept = n + n / GROUP                       # 8-bit values and their exponents
        if case["kind"] == "rope":
            return {"bytes": 2 * es * n + 8 * t, "flops": 3 * n}
        if not case["train"]:
            return {"bytes": 2 * es * n + 8 * t + 4 * d, "flops": 7 * n}
        saved = 2 * kept if case["keep8"] else es * n
        return {"bytes": 4 * es * n + saved + 16 * t + 16 * d, "flops": 24 * n}
    n = t * case["columns"]
    kept = n + -(-t // GROUP) * case["columns"]
    if case["kind"] == "keep":
        return {"bytes": 2 * es * n + 2 * kept, "flops": 4 * n}
    m = case["outputs"]
    return {"bytes": es * n + 2 * kept + es * t * m + 4 * case["columns"] * m,
            "flops": 2 * n * m}


# ---- inputs -----------------------------------------------------------------

def _activation(gen, shape, dtype):
    """Activations: normal, a few channels twenty times as large as the rest."""
    x = torch.randn(shape, generator=gen, device=DEV)
    loud = torch.rand(shape[1:], generator=gen, device=DEV) < 0.02
    return (x * (1.0 + 19.0 * loud)).to(dtype)


def _positions(gen, case):
    """One token of each of many sequences, each anywhere; a prompt's tokens
    follow one another, several sequences end to end."""
    t = case["tokens"]
    reach = 4096 if case["scaling"] == "none" else LONG
    if t <= 64:
        return torch.randint(0, reach, (t,), generator=gen, device=DEV)
    at = torch.arange(t, device=DEV)
    starts = torch.randint(0, t, (t // 2048,), generator=gen, device=DEV).sort().values
    first = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), starts])
    p = at - first[torch.searchsorted(starts, at, right=True)]
    return p + (torch.randint(0, max(1, LONG - t), (1,), generator=gen, device=DEV)
                if reach == LONG else 0)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype, t = TYPES[case["type"]], case["tokens"]
    s = {"case": case}
    if case["kind"] in ("keep", "grad"):
        s["x"] = _activation(gen, (t, case["columns"]), dtype)
        if case["kind"] == "grad":
            # gradients carry a loss scale; their rows differ in size
            dy = torch.randn((t, case["outputs"]), generator=gen, device=DEV)
            size = torch.exp(torch.randn((t, 1), generator=gen, device=DEV))
            s["dy"] = (0.05 * dy * size).to(dtype)
        return s
    d = case["head"]
    s["q"] = _activation(gen, (t, case["heads"], d), dtype)
    s["k"] = _activation(gen, (t, case["kv_heads"], d), dtype)
    s["positions"] = _positions(gen, case)
    if case["kind"] == "norm":
        for g in ("gain_q", "gain_k"):
            s[g] = (1.0 + 0.2 * torch.randn((d,), generator=gen, device=DEV)).to(dtype)
        if case["train"]:
            s["dq"] = (0.05 * torch.randn(s["q"].shape, generator=gen, device=DEV)).to(dtype)
            s["dk"] = (0.05 * torch.randn(s["k"].shape, generator=gen, device=DEV)).to(dtype)
    # what a program makes once for a model: the plain form's table of every
    # position's cosines and sines, or the framework's handle
    if own:
        from ark_amd.rope import Rope
        s["rope"] = Rope(d, rotary_dim=case["rotary"], base=BASE, layout=case["layout"],
                         scaling=SCALING[case["scaling"]])
    else:
        freq, size = _frequencies(case)
        reach = 4096 if case["scaling"] == "none" else LONG
        reach = max(reach, t)
        a = torch.arange(reach, device=DEV, dtype=torch.float64)[:, None] * freq
        s["cos"], s["sin"] = (size * a.cos()).float(), (size * a.sin()).float()
    return s


def _frequencies(case):
    """The inverse frequency of every rotary pair, and the magnitude."""
    r, sc = case["rotary"], SCALING[case["scaling"]] or {"kind": "none"}
    i = torch.arange(r // 2, device=DEV, dtype=torch.float64)
    base = BASE
    if sc["kind"] == "ntk" and r > 2:
        base *= sc["factor"] ** (r / (r - 2))
    f = torch.exp(i * (-2.0 * math.log(base) / r))
    if sc["kind"] == "linear":
        f = f / sc["factor"]
    if sc["kind"] == "yarn":
        # pairs that turn more than 32 times over the original length keep
        # their frequency, pairs below one turn are stretched by the factor
        at = [r * math.log(sc["original"] / (2 * math.pi * turns)) / (2 * math.log(BASE))
              for turns in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), r - 1)
        slow = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f * (1 - slow) + f / sc["factor"] * slow, 0.1 * math.log(sc["factor"]) + 1.0
    if sc["kind"] == "bands":
        turns = sc["original"] * f / (2 * math.pi)
        keep = ((turns - sc["low"]) / (sc["high"] - sc["low"])).clamp(0, 1)
        f = f / sc["factor"] * (1 - keep) + f * keep
    return f, 1.0


# ---- the plain forms --------------------------------------------------------

def _rotate(x, cos, sin, case, back=False):
    """x (tokens, heads, head) in 32 bits, by the cosines and sines of its rows."""
    r = case["rotary"]
    cos, sin = cos[:, None], (-sin if back else sin)[:, None]
    if case["layout"] == "half":
        u, v = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([u * cos - v * sin, u * sin + v * cos, x[..., r:]], -1)
    u, v = x[..., 0:r:2], x[..., 1:r:2]
    y = torch.stack([u * cos - v * sin, u * sin + v * cos], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _norm(x, gain, cos, sin, case):
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return _rotate(x * r * gain, cos, sin, case)


def _norm_back(dy, x, gain, cos, sin, case):
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    dn = _rotate(dy, cos, sin, case, back=True)
    h = x * r
    dgain = (dn * h).sum((0, 1))
    dh = dn * gain
    return r * (dh - h * (dh * h).mean(-1, keepdim=True)), dgain


def _eight(x, kind):
    """x (tokens, columns) in 32 bits: the values its 8-bit form stands for."""
    t, c = x.shape
    g = torch.nn.functional.pad(x, (0, 0, 0, -t % GROUP)).view(-1, GROUP, c)
    m, e = torch.frexp(g.abs().amax(1, keepdim=True))
    e = torch.where(m > 127 / 128, e - 6, e - 7).clamp(-24 if kind == "f16" else -126, 121)
    up = ((e + 127) << 23).to(torch.int32).view(torch.float32)      # 2 ** e
    down = ((127 - e) << 23).to(torch.int32).view(torch.float32)    # 2 ** -e
    q = torch.round(g * down)
    most = torch.where(e >= 10, 63.0, 127.0) if kind == "f16" else torch.full_like(up, 127.0)
    return (torch.minimum(torch.maximum(q, -most), most) * up).view(-1, c)[:t]


def run(state):
    return _own(state) if own else _plain(state)


def _plain(state):
    case = state["case"]
    dtype = TYPES[case["type"]]
    if case["kind"] == "keep":
        return _eight(state["x"].float(), case["type"]).to(dtype)
    if case["kind"] == "grad":
        dw = _eight(state["x"].float(), case["type"]).t() @ state["dy"].float()
        return dw if case["layout"] == "in_out" else dw.t().contiguous()
    cos, sin = state["cos"][state["positions"]], state["sin"][state["positions"]]
    q, k = state["q"].float(), state["k"].float()
    if case["kind"] == "rope":
        return [_rotate(x, cos, sin, case, case["inverse"]).to(dtype) for x in (q, k)]
    gq, gk = state["gain_q"].float(), state["gain_k"].float()
    out = {"q": _norm(q, gq, cos, sin, case).to(dtype), "k": _norm(k, gk, cos, sin, case).to(dtype)}
    if case["train"]:
        if case["keep8"]:
            q, k = (_eight(x.flatten(1), case["type"]).view(x.shape) for x in (q, k))
        dq, out["dgain_q"] = _norm_back(state["dq"].float(), q, gq, cos, sin, case)
        dk, out["dgain_k"] = _norm_back(state["dk"].float(), k, gk, cos, sin, case)
        out["dq"], out["dk"] = dq.to(dtype), dk.to(dtype)
    return out


# ---- the framework's kernels --------------------------------------------------

def _own(state):
    from ark_amd import act
    case = state["case"]
    if case["kind"] == "keep":
        return act.unpack(act.pack(state["x"]))
    if case["kind"] == "grad":
        return act.weight_grad(act.pack(state["x"]), state["dy"], layout=case["layout"])
    rope, q, k, p = state["rope"], state["q"], state["k"], state["positions"]
    if case["kind"] == "rope":
        return list(rope.apply(q, k, positions=p, inverse=case["inverse"]))
    gains = state["gain_q"], state["gain_k"]
    if not case["train"]:
        yq, yk = rope.norm(q, k, *gains, positions=p, eps=EPS)
        return {"q": yq, "k": yk}
    if case["keep8"]:
        yq, yk, kept_q, kept_k = rope.norm(q, k, *gains, positions=p, eps=EPS, keep8=True)
    else:
        yq, yk = rope.norm(q, k, *gains, positions=p, eps=EPS)
        kept_q, kept_k = q, k
    dq, dk, dgq, dgk = rope.norm_backward(state["dq"], state["dk"], kept_q, kept_k, *gains,
                                          positions=p, eps=EPS)
    return {"q": yq, "k": yk, "dq": dq, "dk": dk, "dgain_q": dgq, "dgain_k": dgk}


# ---- the definitions in 64 bits -----------------------------------------------

def _exact_turn(case):
    """(pairs' inverse frequencies, magnitude) from the definition, on the host."""
    r, sc = case["rotary"], SCALING[case["scaling"]]
    kind = sc["kind"] if sc else "none"
    base = BASE * (sc["factor"] ** (r / (r - 2.0)) if kind == "ntk" and r > 2 else 1.0)
    out = []
    for i in range(r // 2):
        f = base ** (-2.0 * i / r)
        if kind == "linear":
            f /= sc["factor"]
        elif kind == "yarn":
            pair = lambda turns: (r * math.log(sc["original"] / (2.0 * math.pi * turns))
                                  / (2.0 * math.log(BASE)))
            lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), r - 1)
            w = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = (1.0 - w) * f + w * f / sc["factor"]
        elif kind == "bands":
            wave = 2.0 * math.pi / f
            if wave > sc["original"] / sc["low"]:
                f /= sc["factor"]
            elif wave >= sc["original"] / sc["high"]:
                w = (sc["original"] / wave - sc["low"]) / (sc["high"] - sc["low"])
                f = (1.0 - w) * f / sc["factor"] + w * f
        out.append(f)
    return out, 0.1 * math.log(sc["factor"]) + 1.0 if kind == "yarn" else 1.0


def _exact_matrix(case, positions):
    """The rotation of every token as cosines and sines of whole heads and the
    place of each value's partner: y = x * c + x[partner] * s."""
    r, d = case["rotary"], case["head"]
    f, size = _exact_turn(case)
    c = torch.ones((len(positions), d), dtype=torch.float64, device=DEV)
    s = torch.zeros_like(c)
    partner = torch.arange(d, device=DEV)
    at = torch.arange(r // 2, device=DEV)
    u, v = (at, at + r // 2) if case["layout"] == "half" else (2 * at, 2 * at + 1)
    a = positions.double()[:, None] * torch.tensor(f, dtype=torch.float64, device=DEV)
    c[:, u] = c[:, v] = size * torch.cos(a)
    s[:, u], s[:, v] = -size * torch.sin(a), size * torch.sin(a)
    partner[u], partner[v] = v, u
    return c[:, None], s[:, None], partner


def _exact_eight(x, kind):
    """x (tokens, columns) in 64 bits: the exponent from the logarithm's floor,
    put right by comparison."""
    out = torch.empty_like(x)
    for lo in range(0, len(x), GROUP * 4096):
        part = x[lo:lo + GROUP * 4096]
        n = len(part)
        part = torch.cat([part, part.new_zeros((-n % GROUP, x.shape[1]))])
        part = part.reshape(-1, GROUP, x.shape[1])
        most = part.abs().max(1, keepdim=True).values
        e = torch.floor(torch.log2((most / 127).clamp_min(2.0 ** -140)))
        power = lambda k: ((k.long() + 1023) << 52).view(torch.float64)
        e = torch.where(most > 127 * power(e), e + 1, e)
        e = torch.where(most <= 127 * power(e - 1), e - 1, e)
        e = e.clamp(-24.0 if kind == "f16" else -126.0, 121.0)
        q = torch.round(part / power(e))
        top = torch.where((e >= 10) & (kind == "f16"), 63.0, 127.0).double()
        out[lo:lo + n] = (q.clamp(-top, top) * power(e)).reshape(-1, x.shape[1])[:n]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "keep":
        return _exact_eight(state["x"].double(), case["type"])
    if case["kind"] == "grad":
        x = _exact_eight(state["x"].double(), case["type"])
        dw = torch.matmul(state["dy"].double().t(), x)
        return dw if case["layout"] == "out_in" else dw.t().contiguous()
    c, s, partner = _exact_matrix(case, state["positions"])
    if case["kind"] == "rope":
        s = -s if case["inverse"] else s
        return [x.double() * c + x.double()[..., partner] * s for x in (state["q"], state["k"])]
    out = {}
    for name in ("q", "k"):
        x, g = state[name].double(), state["gain_" + name].double()
        size = torch.sqrt((x * x).sum(-1, keepdim=True) / case["head"] + EPS)
        n = x / size * g
        out[name] = n * c + n[..., partner] * s
        if not case["train"]:
            continue
        if case["keep8"]:
            x = _exact_eight(x.flatten(1), case["type"]).view(x.shape)
            size = torch.sqrt((x * x).sum(-1, keepdim=True) / case["head"] + EPS)
        dy = state["d" + name].double()
        dn = dy * c - dy[..., partner] * s
        out["dgain_" + name] = (dn * x / size).sum(1).sum(0)
        w = dn * g
        along = (w * x).sum(-1, keepdim=True) / (case["head"] * size ** 2)
        out["d" + name] = (w - x * along) / size
    return out
