"""The language-model operators round the DenseGPA core, as measured cases.

Two operators of the training step and of scoring / generation:

* ``linear_cross_entropy``: softmax cross entropy of ``hidden @ weight.T`` over the vocabulary,
  without keeping the logits, with the gradients of hidden and weight ("step" cases) or the
  per-token losses alone ("score" cases);
* ``residual_norm`` / ``rms_norm``: the norm after a block, its gate and residual scale, the
  residual addition and the norm before the next block, forward alone ("token") or with every
  gradient ("step").

``run`` computes the plain form in 32-bit torch operations, or, with ``own`` set, calls the
framework's operators.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6


def listed():
    return [
        # the loss of one training step of the all-GPA LM: 8 sequences of 8192 tokens, vocabulary
        # 151936, the last position of each sequence without a label
        _loss("loss_step_lm", 8, 8192, 1024, 151936, "bf16", "mean", 0.0),
        # fine-tuning or policy-gradient step: 40 % of the positions are prompt (masked), every
        # token has a weight of its own, sizes that fill no tile
        _loss("loss_step_weighted", 3, 1365, 1000, 32003, "bf16", "none", 0.4),
        # half-precision training with a mid-sized vocabulary
        _loss("loss_step_fp16", 2, 1024, 2048, 50000, "fp16", "mean", 0.1),
        # full-precision training
        _loss("loss_step_fp32", 2, 513, 512, 16001, "fp32", "sum", 0.0),
        # the small model of the tests: launch latency counts
        _loss("loss_step_small", 2, 130, 128, 500, "bf16", "mean", 0.0),
        # evaluation: log-probabilities of four prompts
        _loss("score_prompt", 4, 509, 1024, 151936, "bf16", "none", 0.0, train=False),
        # scoring one new token for each of eight streams
        _loss("score_token", 8, 1, 1024, 151936, "bf16", "none", 0.0, train=False),
        # between two blocks of the LM in training: fp32 stream, bf16 block output
        _norm("block_step_lm", 8, 8192, 1024, "fp32", "bf16", "bf16"),
        # a block with a norm after it, a gate of every channel and a learned scale
        _norm("block_step_gated", 4, 2047, 2560, "bf16", "bf16", "bf16", post=True, gate="full", scale=True),
        # full precision, odd width, one gate value for each token
        _norm("block_step_odd", 3, 701, 1001, "fp32", "fp32", "fp32", post=True, gate="row", scale=True),
        # generation: one token of eight streams
        _norm("block_token", 8, 1, 1024, "fp32", "bf16", "bf16", train=False),
        # the norm of the query heads, a slice of the joint q/k/v projection, in training
        _heads("heads_step", 4, 4096, 16, 128, 32, "bf16"),
    ]


def _loss(name, batch, length, width, vocab, dtype, reduction, masked, train=True):
    return {"name": name, "op": "loss", "batch": batch, "length": length, "width": width, "vocab": vocab,
            "dtype": dtype, "reduction": reduction, "masked": masked, "train": train}


def _norm(name, batch, length, width, stream, update, out, post=False, gate="none", scale=False, train=True):
    return {"name": name, "op": "norm", "batch": batch, "length": length, "width": width, "stream": stream,
            "update": update, "out": out, "post": post, "gate": gate, "scale": scale, "train": train}


def _heads(name, batch, length, heads, width, of, dtype, train=True):
    return {"name": name, "op": "heads", "batch": batch, "length": length, "heads": heads, "width": width,
            "of": of, "dtype": dtype, "train": train}


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["loss", "loss", "norm", "norm", "heads"])
    if op == "loss":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = 3e11 if dtype != "fp32" else 3e10
        while True:
            batch, length = _log(rng, 1, 8), _log(rng, 1, 8192)
            width, vocab = _log(rng, 64, 4096), _log(rng, 256, 151936)
            if rng.random() < 0.5:
                width = max(64, width // 64 * 64)
            if batch * length * width * vocab <= most and width * vocab <= 2 ** 29:
                break
        c = _loss("", batch, length, width, vocab, dtype, rng.choice(["mean", "sum", "none"]),
                  rng.choice([0.0, 0.1, 0.6]), rng.random() < 0.7)
    elif op == "norm":
        stream, update = rng.choice([("fp32", "bf16"), ("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "fp32"), ("fp32", "fp16")])
        batch, length, width = _log(rng, 1, 8), _log(rng, 1, 8192), _log(rng, 64, 8192)
        if rng.random() < 0.6:
            width = max(64, width // 64 * 64)
        length = max(1, min(length, 2 ** 25 // (batch * width)))
        c = _norm("", batch, length, width, stream, update, update, rng.random() < 0.5,
                  rng.choice(["none", "row", "full"]), rng.random() < 0.5, rng.random() < 0.7)
    else:
        heads = _log(rng, 1, 32)
        c = _heads("", _log(rng, 1, 8), _log(rng, 1, 2048), heads, rng.choice([32, 64, 96, 128, 256, rng.randrange(33, 200)]),
                   heads * rng.choice([1, 2]), rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.7)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, scale, dtype):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(_TYPES[dtype])


def prepare(case, seed):
    g = _generator(seed)
    b, t, d = case["batch"], case["length"], case["width"]
    train = case["train"]
    if case["op"] == "loss":
        v, dtype = case["vocab"], case["dtype"]
        # hidden states as a final norm leaves them, logits of standard deviation about 2.5
        hidden = _normal(g, (b, t, d), 1.0, dtype)
        weight = _normal(g, (v, d), 2.5 / math.sqrt(d), dtype)
        # token frequencies fall off as in text: the label's rank is log-uniform
        labels = (torch.rand(b, t, generator=g, device="cuda") * math.log(v)).exp().long().clamp_(1, v) - 1
        if t > 1:
            labels[:, -1] = -100
        if case["masked"]:
            labels[torch.rand(b, t, generator=g, device="cuda") < case["masked"]] = -100
        up = torch.randn(b, t, generator=g, device="cuda") if train and case["reduction"] == "none" else None
        return {"case": case, "hidden": hidden.requires_grad_(train), "weight": weight.requires_grad_(train),
                "labels": labels, "up": up}
    if case["op"] == "heads":
        dtype = case["dtype"]
        joint = _normal(g, (b, t, case["of"] * d), 2.0, dtype)
        x = joint[..., :case["heads"] * d].unflatten(-1, (case["heads"], d))
        weight = 1 + 0.1 * torch.randn(d, generator=g, device="cuda")
        up = _normal(g, x.shape, 0.1, dtype) if train else None
        return {"case": case, "x": x.detach().requires_grad_(train), "weight": weight.requires_grad_(train), "up": up}
    s = {"case": case, "residual": _normal(g, (b, t, d), 3.0, case["stream"]),
         "update": _normal(g, (b, t, d), 0.7, case["update"]),
         "weight": 1 + 0.1 * torch.randn(d, generator=g, device="cuda"),
         "post_weight": 1 + 0.1 * torch.randn(d, generator=g, device="cuda") if case["post"] else None,
         "gate": None if case["gate"] == "none" else
         _normal(g, (b, t, d if case["gate"] == "full" else 1), 1.5, case["update"]),
         "scale": 0.3 + 0.05 * torch.randn(d, generator=g, device="cuda") if case["scale"] else None}
    for x in s.values():
        if isinstance(x, torch.Tensor):
            x.requires_grad_(train)
    s["up_stream"] = _normal(g, (b, t, d), 0.05, case["stream"]) if train else None
    s["up_normed"] = _normal(g, (b, t, d), 0.05, case["out"]) if train else None
    return s


_NORM_INPUTS = ("residual", "update", "weight", "post_weight", "gate", "scale")


# --------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    return _run_own(state, case) if own else _run_plain(state, case)


def _run_own(s, case):
    import gpa_b200
    if case["op"] == "loss":
        loss = gpa_b200.linear_cross_entropy(s["hidden"], s["weight"], s["labels"], reduction=case["reduction"])
        if not case["train"]:
            return {"loss": loss}
        dx, dw = torch.autograd.grad(loss, (s["hidden"], s["weight"]), s["up"])
        return {"loss": loss.detach(), "dhidden": dx, "dweight": dw}
    if case["op"] == "heads":
        y = gpa_b200.rms_norm(s["x"], s["weight"], _EPS)
        if not case["train"]:
            return {"y": y}
        dx, dw = torch.autograd.grad(y, (s["x"], s["weight"]), s["up"])
        return {"y": y.detach(), "dx": dx, "dweight": dw}
    h, n = gpa_b200.residual_norm(s["residual"], s["update"], s["weight"], _EPS, post_weight=s["post_weight"],
                                  gate=s["gate"], scale=s["scale"], out_dtype=_TYPES[case["out"]])
    if not case["train"]:
        return {"stream": h, "normed": n}
    names = [k for k in _NORM_INPUTS if s[k] is not None]
    grads = torch.autograd.grad((h, n), [s[k] for k in names], (s["up_stream"], s["up_normed"]))
    return {"stream": h.detach(), "normed": n.detach(), **{"d" + k: x for k, x in zip(names, grads)}}


def _run_plain(s, case):
    with torch.no_grad():
        if case["op"] == "loss":
            return _plain_loss(s, case)
        if case["op"] == "heads":
            x, w = s["x"].float(), s["weight"]
            r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
            y = (x * r * w).to(s["x"].dtype)
            if not case["train"]:
                return {"y": y}
            dx, dw = _plain_norm_grad(x, r, w, s["up"].float())
            return {"y": y, "dx": dx.to(s["x"].dtype), "dweight": dw}
        return _plain_norm(s, case)


def _plain_loss(s, case):
    x, w = s["hidden"].float().flatten(0, 1), s["weight"].float()
    y = s["labels"].flatten()
    keep = y != -100
    at = y.clamp_min(0)[:, None]
    z = x @ w.T
    top = z.amax(-1, keepdim=True)
    picked = z.gather(-1, at) - top
    z.sub_(top).exp_()
    total = z.sum(-1, keepdim=True)
    each = torch.where(keep, (total.log() - picked)[:, 0], 0.0)
    if case["reduction"] == "mean":
        g = keep.float() / keep.sum().clamp_min(1)
        loss = (each.double().sum() / keep.sum().clamp_min(1)).float()
    elif case["reduction"] == "sum":
        g, loss = keep.float(), each.double().sum().float()
    else:
        g, loss = keep.float(), each.view(s["labels"].shape)
    if not case["train"]:
        return {"loss": loss}
    if s["up"] is not None:
        g = g * s["up"].flatten()
    z.div_(total)
    z.scatter_add_(-1, at, torch.full_like(picked, -1.0))
    z.mul_(g[:, None])
    return {"loss": loss, "dhidden": (z @ w).view(s["hidden"].shape).to(s["hidden"].dtype),
            "dweight": (z.T @ x).to(s["weight"].dtype)}


def _plain_norm_grad(x, r, w, up):
    """(dx, dw) of x * r * w for the gradient `up`, r = rsqrt(mean x^2 + eps)."""
    a = up * w
    dx = r * (a - x * r * r * (a * x).mean(-1, keepdim=True))
    return dx, (up * x * r).flatten(0, -2).sum(0)


def _plain_norm(s, case):
    h, y, w = s["residual"].float(), s["update"].float(), s["weight"]
    r_y = torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS)
    u = y * r_y * s["post_weight"] if case["post"] else y
    gate = 1 / (1 + torch.exp(-s["gate"].float())) if s["gate"] is not None else 1.0
    c = s["scale"] if case["scale"] else 1.0
    stream = (h + c * gate * u).to(s["residual"].dtype)
    x = stream.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    out = {"stream": stream, "normed": (x * r * w).to(_TYPES[case["out"]])}
    if not case["train"]:
        return out
    dx, dw = _plain_norm_grad(x, r, w, s["up_normed"].float())
    dx = dx + s["up_stream"].float()
    out["dresidual"], out["dweight"] = dx.to(s["residual"].dtype), dw
    du = dx * c * gate
    if case["scale"]:
        out["dscale"] = (dx * gate * u).flatten(0, -2).sum(0)
    if s["gate"] is not None:
        da = dx * c * u * gate * (1 - gate)
        out["dgate"] = (da if case["gate"] == "full" else da.sum(-1, keepdim=True)).to(s["gate"].dtype)
    if case["post"]:
        du, out["dpost_weight"] = _plain_norm_grad(y, r_y, s["post_weight"], du)
    out["dupdate"] = du.to(s["update"].dtype)
    return out


# -------------------------------------------------------------------------- work and exact
def work(case):
    n, d = case["batch"] * case["length"], case["width"]
    if case["op"] == "loss":
        v, e = case["vocab"], _BYTES[case["dtype"]]
        rows = n * (1 - case["masked"]) - (case["batch"] if case["length"] > 1 else 0) * (1 - case["masked"])
        moved = (n * d + v * d) * e * (2 if case["train"] else 1) + 8 * n
        moved += 4 * n if case["reduction"] == "none" else 4
        return {"bytes": moved, "flops": max(rows, 0) * v * d * (6 if case["train"] else 2)}
    if case["op"] == "heads":
        n *= case["heads"]
        # x in, y out; in training the gradient in and dx out too
        return {"bytes": n * d * _BYTES[case["dtype"]] * (4 if case["train"] else 2) + 4 * d, "flops": n * d * (12 if case["train"] else 4)}
    hs, us, os = _BYTES[case["stream"]], _BYTES[case["update"]], _BYTES[case["out"]]
    gate = {"none": 0, "row": us / d, "full": us}[case["gate"]]
    each = 2 * hs + us + gate + os
    if case["train"]:  # gradients of stream and normed in; of residual, update and gate out
        each += 2 * hs + os + us + gate
    return {"bytes": n * d * each, "flops": n * d * (30 if case["train"] else 10)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "loss":
        return _exact_loss(s, case)
    leaf = {k: x.detach().double().requires_grad_(case["train"]) for k, x in s.items()
            if isinstance(x, torch.Tensor) and not k.startswith("up_") and k != "up"}

    def norm(x, w):
        return w * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + _EPS).sqrt()

    if case["op"] == "heads":
        y = norm(leaf["x"], leaf["weight"])
        if not case["train"]:
            return {"y": y}
        y.backward(s["up"].double())
        return {"y": y.detach(), "dx": leaf["x"].grad, "dweight": leaf["weight"].grad}
    u = norm(leaf["update"], leaf["post_weight"]) if case["post"] else leaf["update"]
    if "gate" in leaf:
        u = u * torch.sigmoid(leaf["gate"])
    if "scale" in leaf:
        u = u * leaf["scale"]
    h = leaf["residual"] + u
    # the stream is kept in its own type, and the next norm reads the kept values
    h = h + (h.detach().to(_TYPES[case["stream"]]).double() - h.detach())
    n = norm(h, leaf["weight"])
    if not case["train"]:
        return {"stream": h, "normed": n}
    torch.autograd.backward((h, n), (s["up_stream"].double(), s["up_normed"].double()))
    return {"stream": h.detach(), "normed": n.detach(), **{"d" + k: x.grad for k, x in leaf.items()}}


def _exact_loss(s, case):
    n = s["labels"].numel()
    if n * case["vocab"] * case["width"] > 1.2e13:
        return None
    train = case["train"]
    x = s["hidden"].detach().double().flatten(0, 1)
    w = s["weight"].detach().double().requires_grad_(train)
    y = s["labels"].flatten()
    count = int((y >= 0).sum())
    up = torch.ones(n, device=y.device, dtype=torch.float64) if s["up"] is None else s["up"].flatten().double()
    if case["reduction"] == "mean":
        up = up / max(count, 1)
    each, dx = torch.zeros(n, device=y.device, dtype=torch.float64), torch.zeros_like(x)
    dw = torch.zeros_like(w)
    some = max(1, 2 ** 30 // case["vocab"])
    for i in range(0, n, some):
        part = x[i:i + some].requires_grad_(train)
        l = torch.nn.functional.cross_entropy(part @ w.T, y[i:i + some], ignore_index=-100, reduction="none")
        each[i:i + some] = l.detach()
        if train:
            a, b = torch.autograd.grad(l, (part, w), up[i:i + some])
            dx[i:i + some], dw = a, dw + b
    loss = each.view(s["labels"].shape) if case["reduction"] == "none" else each.sum() / (max(count, 1) if case["reduction"] == "mean" else 1)
    if not train:
        return {"loss": loss}
    return {"loss": loss, "dhidden": dx.view(s["hidden"].shape), "dweight": dw.detach()}
