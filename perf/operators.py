"""The operators of language-model training that stand beside batch norm, the elementwise layers and cross
entropy -- layer normalisation, dropout and the preference loss -- as measured cases: their inputs, their plain
form in elementary PyTorch operations, the calls of this package, and their definition in binary64."""
import math

import numpy as np
import torch

own = False  # True: run() calls repdl_amd; False: the plain forms

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # ---- layer normalisation ----
        # one token of a serving loop: a single row, forward only -- the latency of one launch
        {"name": "layer norm 1x4096 bf16", "op": "layer_norm", "rows": 1, "cols": 4096, "type": "bf16", "wtype": "bf16", "train": False},
        # a training step of a narrow model in binary32, forward and backward
        {"name": "layer norm 8192x1024 f32", "op": "layer_norm", "rows": 8192, "cols": 1024, "type": "f32", "wtype": "f32", "train": True},
        # odd rows of odd length, half precision with binary32 parameters
        {"name": "layer norm 5003x1001 f16", "op": "layer_norm", "rows": 5003, "cols": 1001, "type": "f16", "wtype": "f32", "train": True},
        # a long batch of a wide model, forward and backward
        {"name": "layer norm 16384x8192 bf16", "op": "layer_norm", "rows": 16384, "cols": 8192, "type": "bf16", "wtype": "bf16", "train": True},
        # ---- dropout ----
        # the hidden layer of a small classifier (64 images, 1000 units): launch-bound
        {"name": "dropout 64000 f32", "op": "dropout", "count": 64000, "type": "f32", "p": 0.5, "residual": False, "train": True},
        # an odd number of elements, in the residual form
        {"name": "dropout 12345677+res f32", "op": "dropout", "count": 12345677, "type": "f32", "p": 0.1, "residual": True, "train": True},
        # the residual branch of a wide model's layer, forward and backward
        {"name": "dropout 2^27+res bf16", "op": "dropout", "count": 1 << 27, "type": "bf16", "p": 0.1, "residual": True, "train": True},
        # activations without a residual
        {"name": "dropout 2^26 f32", "op": "dropout", "count": 1 << 26, "type": "f32", "p": 0.25, "residual": False, "train": True},
        # ---- preference loss ----
        # a toy vocabulary, one pair of short answers: three launches
        {"name": "preference 1x12x1000 f32", "op": "preference", "pairs": 1, "steps": 12, "vocab": 1000, "type": "f32", "view": False, "ref": True,
         "smoothing": 0.0, "train": True},
        # a few pairs of short answers over an odd vocabulary, the logits a view without their last step
        {"name": "preference 4x161x50257 f32", "op": "preference", "pairs": 4, "steps": 161, "vocab": 50257, "type": "f32", "view": True, "ref": True,
         "smoothing": 0.1, "train": True},
        # the evaluation of such a batch in half precision: the loss and the sequences' log probabilities alone
        {"name": "preference 8x512x32000 bf16", "op": "preference", "pairs": 8, "steps": 512, "vocab": 32000, "type": "bf16", "view": False, "ref": True,
         "smoothing": 0.0, "train": False},
        # a training step with a large vocabulary
        {"name": "preference 4x1024x131072 bf16", "op": "preference", "pairs": 4, "steps": 1024, "vocab": 131072, "type": "bf16", "view": False, "ref": False,
         "smoothing": 0.0, "train": True},
    ]


def _between(rng, low, high):
    """A whole number, spread evenly over the logarithm; odd ones as often as not."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["layer_norm", "dropout", "preference"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "layer_norm":
        cols = _between(rng, 16, 16384)
        rows = _between(rng, 1, min(65536, (1 << 26) // cols))
        return {"op": op, "rows": rows, "cols": cols, "type": kind, "wtype": rng.choice([kind, "f32"]), "train": rng.random() < 0.7}
    if op == "dropout":
        return {"op": op, "count": _between(rng, 1000, 1 << 26), "type": kind, "p": rng.choice([0.05, 0.1, 0.2, 0.5]), "residual": rng.random() < 0.5,
                "train": rng.random() < 0.7}
    vocab = _between(rng, 100, 131072)
    pairs = _between(rng, 1, 16)
    steps = _between(rng, 1, max(2, min(2048, (1 << 28) // (2 * pairs * vocab))))
    return {"op": op, "pairs": pairs, "steps": steps, "vocab": vocab, "type": kind, "view": rng.random() < 0.3, "ref": rng.random() < 0.7,
            "smoothing": rng.choice([0.0, 0.0, 0.1]), "train": rng.random() < 0.7}


_EPS = 1e-5
_BETA = 0.1
_IGNORE = -100


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    kind = _TYPES[case["type"]]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    state = {"case": case}
    if case["op"] == "layer_norm":
        rows, cols = case["rows"], case["cols"]
        # activations whose rows have different means and spreads, as a residual stream has
        x = normal(rows, cols) * (0.5 + normal(rows, 1).abs()) + normal(rows, 1)
        state["x"] = x.to(kind)
        state["w"] = (1 + 0.1 * normal(cols)).to(_TYPES[case["wtype"]])
        state["b"] = (0.1 * normal(cols)).to(_TYPES[case["wtype"]])
        if case["train"]:
            state["gy"] = normal(rows, cols).to(kind)
            state.update({k: state[k].requires_grad_() for k in ("x", "w", "b")})
    elif case["op"] == "dropout":
        n = case["count"]
        state["x"] = normal(n, dtype=kind)
        state["residual"] = normal(n, dtype=kind) if case["residual"] else None
        # the generator's state as a layer holds it: (seed, number of the call)
        state["rng"] = torch.tensor([7777777777 * (seed + 1), seed + 5], dtype=torch.int64, device="cuda")
        if case["train"]:
            state["gy"] = normal(n, dtype=kind)
            state["x"].requires_grad_()
    else:
        seqs, steps, vocab = 2 * case["pairs"], case["steps"], case["vocab"]
        kept = steps + (1 if case["view"] else 0)
        logits = normal(seqs, kept, vocab, dtype=kind).mul_(2.5)[:, :steps]
        target = torch.randint(0, vocab, (seqs, steps), generator=gen, device="cuda")
        # the prompt at the front and the padding at the end of each sequence are not counted
        prompt = torch.randint(0, max(1, steps // 4), (seqs, 1), generator=gen, device="cuda")
        end = steps - torch.randint(0, max(1, steps // 4), (seqs, 1), generator=gen, device="cuda")
        at = torch.arange(steps, device="cuda")
        state["target"] = torch.where((at >= prompt) & (at < end), target, _IGNORE)
        # a trained model gives the tokens of its own data more than chance: raise the target's logit on most steps
        lift = (3.0 * normal(seqs, steps).abs()).to(kind)
        logits.scatter_add_(2, target.unsqueeze(2), lift.unsqueeze(2))
        state["logits"] = logits.detach()
        if case["train"]:
            state["logits"].requires_grad_()
        # the reference model's log probabilities: near what the policy has, a little apart
        state["ref"] = None
        if case["ref"]:
            counted = (state["target"] != _IGNORE).sum(1)
            state["ref"] = -counted * (math.log(vocab) + 1.0) + 3.0 * normal(seqs)
    return state


def run(state):
    case = state["case"]
    if case["op"] == "layer_norm":
        return _own_layer_norm(state) if own else _plain_layer_norm(state)
    if case["op"] == "dropout":
        return _own_dropout(state) if own else _plain_dropout(state)
    return _own_preference(state) if own else _plain_preference(state)


# ---- the calls of this package ----


def _own_layer_norm(state):
    from repdl_amd.nn import functional as F

    y = F.layer_norm(state["x"], (state["case"]["cols"],), state["w"], state["b"], _EPS)
    if not state["case"]["train"]:
        return {"y": y}
    gx, gw, gb = torch.autograd.grad(y, (state["x"], state["w"], state["b"]), state["gy"])
    return {"y": y.detach(), "gx": gx, "gw": gw, "gb": gb}


def _own_dropout(state):
    from repdl_amd.nn import functional as F

    y = F.dropout(state["x"], state["case"]["p"], state["rng"], residual=state["residual"])
    if not state["case"]["train"]:
        return {"y": y}
    (gx,) = torch.autograd.grad(y, state["x"], state["gy"])
    return {"y": y.detach(), "gx": gx}


def _own_preference(state):
    from repdl_amd.nn import functional as F

    loss, logps = F.preference_loss(state["logits"], state["target"], state["ref"], beta=_BETA, label_smoothing=state["case"]["smoothing"],
                                    ignore_index=_IGNORE)
    if not state["case"]["train"]:
        return {"loss": loss, "logps": logps}
    (g,) = torch.autograd.grad(loss, state["logits"])
    return {"loss": loss.detach(), "logps": logps, "grad": g}


# ---- the plain forms ----


@torch.no_grad()
def _plain_layer_norm(state):
    x, w, b = state["x"].float(), state["w"].float(), state["b"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + _EPS)
    xh = centred * rstd
    y = (xh * w + b).to(state["x"].dtype)
    if not state["case"]["train"]:
        return {"y": y}
    gy = state["gy"].float()
    g = gy * w
    gx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return {"y": y, "gx": gx.to(state["x"].dtype), "gw": (gy * xh).sum(0).to(state["w"].dtype), "gb": gy.sum(0).to(state["b"].dtype)}


# The generator is Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011):
# element j takes word j % 4 of the block whose counter is (j / 4, call) and whose key is the seed.
_M0, _M1, _W0, _W1, _LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _philox_round(c, key):
    """One round on int64 tensors that hold 32-bit words: the products wrap at 64 bits, and all their bits are there."""
    a, b = c[0] * _M0, c[2] * _M1
    return ((b >> 32 & _LOW) ^ c[1] ^ key[0], b & _LOW, (a >> 32 & _LOW) ^ c[3] ^ key[1], a & _LOW), ((key[0] + _W0) & _LOW, (key[1] + _W1) & _LOW)


def _plain_words(n, rng):
    block = torch.arange((n + 3) // 4, dtype=torch.int64, device="cuda")
    seed, call = rng[0], rng[1]
    c = (block & _LOW, block >> 32, (call & _LOW).expand_as(block), (call >> 32 & _LOW).expand_as(block))
    key = (seed & _LOW, seed >> 32 & _LOW)
    for _ in range(10):
        c, key = _philox_round(c, key)
    return torch.stack(c, 1).reshape(-1)[:n]


@torch.no_grad()
def _plain_dropout(state):
    p = state["case"]["p"]
    x = state["x"].float()
    keep = _plain_words(x.numel(), state["rng"]) >= round(p * 2 ** 32)
    scale = 1.0 / (1.0 - p)
    y = torch.where(keep, x * scale, 0.0)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    y = y.to(state["x"].dtype)
    if not state["case"]["train"]:
        return {"y": y}
    return {"y": y, "gx": torch.where(keep, state["gy"].float() * scale, 0.0).to(state["x"].dtype)}


@torch.no_grad()
def _plain_preference(state):
    target, case = state["target"], state["case"]
    pairs = case["pairs"]
    x = state["logits"].float()
    counted = target != _IGNORE
    label = target.clamp(min=0).unsqueeze(2)
    m = x.amax(2, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(2, keepdim=True)
    lp = (x.gather(2, label) - m - torch.log(total)).squeeze(2)
    logps = torch.where(counted, lp, 0.0).double().sum(1)
    ref = state["ref"].double() if state["ref"] is not None else torch.zeros_like(logps)
    margin = logps - ref
    z = _BETA * (margin[:pairs] - margin[pairs:])
    eps = case["smoothing"]
    soft = torch.log1p(torch.exp(-z.abs()))  # softplus(-|z|)
    loss = ((1 - eps) * (soft + (-z).clamp(min=0)) + eps * (soft + z.clamp(min=0))).mean()
    out = {"loss": loss.float(), "logps": logps.float()}
    if case["train"]:
        sigma = 1.0 / (1.0 + torch.exp(-z))
        c = _BETA / pairs * (eps * sigma - (1 - eps) * (1.0 / (1.0 + torch.exp(z))))
        coef = torch.cat([c, -c]).float()[:, None] * counted
        g = e.mul_(-(coef.unsqueeze(2) / total))
        g.scatter_add_(2, label, coef.unsqueeze(2))
        out["grad"] = g.to(state["logits"].dtype)
    return out


# ---- what a pass cannot do without ----


def work(case):
    size = _BYTES[case["type"]]
    train = case["train"]
    if case["op"] == "layer_norm":
        n = case["rows"] * case["cols"]
        # x and y (8 operations an element); with the backward pass gy and gx too (16 more), and the parameters' gradients
        return {"bytes": (4 if train else 2) * n * size + (4 if train else 2) * case["cols"] * _BYTES[case["wtype"]], "flops": (24 if train else 8) * n}
    if case["op"] == "dropout":
        n = case["count"]
        # the generator's ten rounds are 20 products and 40 additions or exclusive ors for four elements
        return {"bytes": (2 + (1 if case["residual"] else 0) + (2 if train else 0)) * n * size, "flops": (34 if train else 17) * n}
    rows = 2 * case["pairs"] * case["steps"]
    n = rows * case["vocab"]
    # about three quarters of the steps are counted: their logits are read, and the gradient of every step is written
    return {"bytes": int(0.76 * n * size) + (n * size if train else 0) + 8 * rows, "flops": int(0.76 * n * (24 if train else 14))}


# ---- the definitions in 64 bits ----


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "layer_norm":
            return _exact_layer_norm(state, case)
        if case["op"] == "dropout":
            return _exact_dropout(state, case)
        return _exact_preference(state, case)


def _exact_layer_norm(state, case):
    """The rows in pieces of at most 2^25 elements, so that the largest case stays small in binary64."""
    w, b = state["w"].double(), state["b"].double()
    y, gx = [], []
    gw, gb = torch.zeros_like(w), torch.zeros_like(b)
    step = max(1, (1 << 25) // case["cols"])
    for at in range(0, case["rows"], step):
        x = state["x"][at:at + step].double()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        std = (var + _EPS).sqrt()
        xh = (x - mean) / std
        y.append(xh * w + b)
        if case["train"]:
            gy = state["gy"][at:at + step].double()
            gw += (gy * xh).sum(0)
            gb += gy.sum(0)
            d = gy * w
            gx.append((d - d.mean(1, keepdim=True) - xh * (d * xh).mean(1, keepdim=True)) / std)
    if not case["train"]:
        return {"y": torch.cat(y)}
    return {"y": torch.cat(y), "gx": torch.cat(gx), "gw": gw, "gb": gb}


def _exact_words(n, seed, call):
    """The same words from numpy's unsigned 64-bit integers."""
    u = np.uint64
    low, shift = u(_LOW), u(32)
    block = np.arange((n + 3) // 4, dtype=u)
    x0, x1 = block & low, block >> shift
    x2, x3 = np.full_like(block, u(call & _LOW)), np.full_like(block, u(call >> 32 & _LOW))
    k0, k1 = seed & _LOW, seed >> 32 & _LOW
    for _ in range(10):
        even, odd = x0 * u(_M0), x2 * u(_M1)
        x0, x1, x2, x3 = (odd >> shift) ^ x1 ^ u(k0), odd & low, (even >> shift) ^ x3 ^ u(k1), even & low
        k0, k1 = (k0 + _W0) & _LOW, (k1 + _W1) & _LOW
    words = np.empty((len(block), 4), dtype=np.uint32)
    words[:, 0], words[:, 1], words[:, 2], words[:, 3] = x0, x1, x2, x3
    return words.reshape(-1)[:n]


def _exact_dropout(state, case):
    n, p = case["count"], case["p"]
    seed, call = (int(v) for v in state["rng"].cpu())
    kept = torch.from_numpy(_exact_words(n, seed, call) >= np.uint32(round(p * 2 ** 32))).to("cuda")
    factor = kept.double() / (1.0 - p)
    y = state["x"].double() * factor
    if case["residual"]:
        y += state["residual"]
    if not case["train"]:
        return {"y": y}
    return {"y": y, "gx": factor.mul_(state["gy"])}


def _exact_preference(state, case):
    """Sequence by sequence: log_softmax in binary64, its rows picked and summed; then the pairs; then the gradient, again by sequence."""
    pairs, eps = case["pairs"], case["smoothing"]
    seqs = 2 * pairs
    total = torch.zeros(seqs, dtype=torch.float64, device="cuda")
    rows = [torch.nonzero(state["target"][i] != _IGNORE).squeeze(1) for i in range(seqs)]
    for i in range(seqs):
        if len(rows[i]):
            lp = torch.log_softmax(state["logits"][i, rows[i]].double(), 1)
            total[i] = lp[torch.arange(len(rows[i])), state["target"][i, rows[i]]].sum()
    ref = state["ref"].double() if state["ref"] is not None else 0.0 * total
    log_ratio = total - ref
    z = _BETA * (log_ratio[:pairs] - log_ratio[pairs:])
    sigmoid = torch.nn.functional.logsigmoid
    out = {"loss": -((1 - eps) * sigmoid(z) + eps * sigmoid(-z)).mean(), "logps": total}
    if case["train"]:
        slope = _BETA * (eps * torch.sigmoid(z) - (1 - eps) * torch.sigmoid(-z)) / pairs
        slope = torch.cat([slope, -slope])
        grad = torch.zeros(state["logits"].shape, dtype=torch.float64, device="cuda")
        for i in range(seqs):
            if len(rows[i]):
                d = -torch.softmax(state["logits"][i, rows[i]].double(), 1)
                d[torch.arange(len(rows[i])), state["target"][i, rows[i]]] += 1.0
                grad[i, rows[i]] = slope[i] * d
        out["grad"] = grad
    return out
