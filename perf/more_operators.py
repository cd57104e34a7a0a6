"""What the operators beside and behind blocks over tokens are timed on: the layer norm, the gated projection of a
feed-forward block, the cross entropy over a large vocabulary and the loss from a teacher's top logits, each forward and
backward.

A case is one operator in one direction with its sizes and type.  `prepare` makes what a program has in hand before
the call, `run` is one call with `own` true and the same operator in elementary torch operations with `own` false, and
`exact` is its definition in 64 bits.
"""

import math

import torch

own = False
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_queues = {}


def listed():
    return [
        # the norm behind the last block, over a batch of prompts, with the residual that the blocks hand on
        {"name": "norm_residual", "op": "norm", "type": "bfloat16", "rows": 16384, "channels": 2048, "bias": True,
         "residual": True},
        # a training step's backward pass through it
        {"name": "norm_grad", "op": "norm_grad", "type": "bfloat16", "rows": 8192, "channels": 2048, "bias": True,
         "residual": True},
        # a batch of prompts through the feed-forward block's first half
        {"name": "gated_prompts", "op": "gated", "type": "bfloat16", "rows": 8192, "channels": 2048, "features": 5504,
         "activation": "silu"},
        # serving: one token, where the weights are read for one row
        {"name": "gated_one", "op": "gated", "type": "bfloat16", "rows": 1, "channels": 2048, "features": 5504,
         "activation": "silu"},
        # serving: a token each of 48 requests
        {"name": "gated_48", "op": "gated", "type": "float16", "rows": 48, "channels": 2304, "features": 6144,
         "activation": "gelu"},
        # a training step's backward pass
        {"name": "gated_grad", "op": "gated_grad", "type": "bfloat16", "rows": 8192, "channels": 2048, "features": 5504,
         "activation": "silu"},
        # a training step: the loss of 8192 tokens over a large vocabulary
        {"name": "loss_training", "op": "loss", "type": "bfloat16", "rows": 8192, "channels": 2048, "words": 65536,
         "masked": 0.0},
        # its gradient, a fifth of the tokens (prompts, padding) not counted
        {"name": "loss_grad_training", "op": "loss_grad", "type": "bfloat16", "rows": 8192, "channels": 2048,
         "words": 65536, "masked": 0.2},
        # scoring a few tokens: the weights are read for few rows
        {"name": "loss_few", "op": "loss", "type": "bfloat16", "rows": 40, "channels": 2048, "words": 50021,
         "masked": 0.0},
        # a small model in 32 bits, sizes that nobody rounded, half of the tokens not counted
        {"name": "loss_grad_odd", "op": "loss_grad", "type": "float32", "rows": 1501, "channels": 300, "words": 10007,
         "masked": 0.5},
        # a student learns from a teacher's 64 largest logits
        {"name": "teacher_training", "op": "teacher", "type": "bfloat16", "rows": 4096, "channels": 1024, "words": 32000,
         "top": 64, "temperature": 2.0, "masked": 0.1},
        {"name": "teacher_grad", "op": "teacher_grad", "type": "bfloat16", "rows": 4096, "channels": 1024, "words": 32000,
         "top": 64, "temperature": 2.0, "masked": 0.1},
    ]


def _spread(rng, low, high):
    """A whole number between the two, evenly over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "gated", "gated", "gated_grad", "loss", "loss_grad", "loss_grad",
                     "teacher", "teacher_grad"])
    c = {"op": op, "type": rng.choice(["bfloat16", "bfloat16", "float32", "float16"])}
    slow = c["type"] == "float32"
    if op.startswith("norm"):
        c.update(rows=_spread(rng, 1, 16384), channels=_spread(rng, 48, 2048), bias=rng.random() < 0.7,
                 residual=rng.random() < 0.5)
        return c
    c["rows"] = _spread(rng, 1, 1024 if slow else 8192)
    # channels: rounded ones in most models, any in the others
    c["channels"] = 64 * _spread(rng, 2, 32) if rng.random() < 0.6 else _spread(rng, 64, 2048)
    if op.startswith("gated"):
        c.update(features=_spread(rng, 100, 5504), activation=rng.choice(["silu", "silu", "gelu"]))
        return c
    c.update(words=_spread(rng, 500, 20000 if slow else 65536), masked=rng.choice([0.0, 0.0, 0.1, 0.4, 0.8]))
    if op.startswith("teacher"):
        c.update(top=_spread(rng, 1, 100), temperature=rng.choice([1.0, 2.0, 4.0]))
    return c


# ------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape, scale=1.0, dtype=kind):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    def uniform(low, high, *shape):
        return torch.rand(*shape, generator=gen, device="cuda") * (high - low) + low

    op, s = case["op"], {"case": case}
    n, d = case["rows"], case["channels"]
    if op.startswith("norm"):
        # a row's mean is not zero: that is what the norm takes away
        s["x"] = (torch.randn(n, d, generator=gen, device="cuda") + uniform(-1.0, 1.0, n, 1)).to(kind)
        s["weight"] = uniform(0.5, 1.5, d)
        s["bias"] = normal(d, scale=0.1, dtype=torch.float32) if case["bias"] else None
        s["residual"] = normal(n, d, scale=2.0) if case["residual"] else None
        if op == "norm_grad":
            s["dout"] = normal(n, d)
            s["dv"] = normal(n, d) if case["residual"] else None
        return s
    s["x"] = normal(n, d)
    if op.startswith("gated"):
        s["gate"], s["up"] = (normal(case["features"], d, scale=d ** -0.5) for _ in range(2))
        if op == "gated_grad":
            s["dy"] = normal(n, case["features"])
        return s
    # logits of about two units, as in a model that has learned something
    s["weight"] = normal(case["words"], d, scale=2.0 * d ** -0.5)
    left_out = torch.rand(n, generator=gen, device="cuda") < case["masked"]
    z = None
    if op.startswith("loss"):
        s["labels"] = torch.randint(case["words"], (n,), generator=gen, device="cuda").masked_fill(left_out, -100)
    else:
        # the teacher and the student agree in part
        z = s["x"].float() @ s["weight"].float().t()
        top = torch.topk(z + 2.0 * torch.randn(z.shape, generator=gen, device="cuda"), min(case["top"], case["words"]))
        s["logits"] = top.values
        s["indices"] = top.indices.to(torch.int32).masked_fill(left_out[:, None], -1)
    if op.endswith("_grad"):
        # what the forward pass returned, and the gradient of the mean over the tokens that count, as a step scales it
        if z is None:
            z = s["x"].float() @ s["weight"].float().t()
        z = z / case.get("temperature", 1.0)
        s["lse"] = torch.logsumexp(z, -1)
        s["dloss"] = uniform(0.5, 1.5, n)
    return s


def _counted(case):
    """Rows that count, about."""
    return max(1.0, case["rows"] * (1.0 - case.get("masked", 0.0)))


def work(case):
    size = 4 if case["type"] == "float32" else 2
    op, n, d = case["op"], case["rows"], case["channels"]
    grad = op.endswith("_grad")
    if op.startswith("norm"):
        # x (and the residual) read, out (and v) written; x, residual, dout, dv read, the one gradient written
        arrays = (3 + 2 * case["residual"]) if grad else (2 + 2 * case["residual"])
        return {"bytes": n * d * size * arrays + d * 8 * (2 if grad else 1), "flops": n * d * (18 if grad else 9)}
    if op.startswith("gated"):
        f = case["features"]
        return {"bytes": ((n * d + 2 * f * d) * (2 if grad else 1) + n * f) * size, "flops": n * d * f * (12 if grad else 4)}
    v, rows = case["words"], _counted(case)
    per_row = case["top"] * 8 if op.startswith("teacher") else 8
    return {"bytes": (rows * d + v * d) * size * (2 if grad else 1) + n * (per_row + 8),
            "flops": rows * d * v * (6 if grad else 2)}


# ---------------------------------------------------------------------------------------------- the plain forms
def _activation(name, g):
    """f(g) and its derivative."""
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    cdf = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5


def _plain_norm(s, eps=1e-5):
    kind = s["x"].dtype
    v = s["x"].float()
    if s["residual"] is not None:
        v = v + s["residual"].float()
    off = v - v.mean(-1, keepdim=True)
    inv = 1 / torch.sqrt((off * off).mean(-1, keepdim=True) + eps)
    unit = off * inv
    if s["case"]["op"] == "norm":
        out = unit * s["weight"] if s["bias"] is None else unit * s["weight"] + s["bias"]
        return {"out": out.to(kind), "v": v.to(kind) if s["residual"] is not None else None}
    dout = s["dout"].float()
    e = dout * s["weight"]
    dx = (e - e.mean(-1, keepdim=True) - unit * (e * unit).mean(-1, keepdim=True)) * inv
    if s["dv"] is not None:
        dx = dx + s["dv"].float()
    return {"x": dx.to(kind), "weight": (dout * unit).sum(0), "bias": dout.sum(0) if s["bias"] is not None else None}


def _plain_gated(s):
    kind, x = s["x"].dtype, s["x"].float()
    gate, up = s["gate"].float(), s["up"].float()
    g, u = x @ gate.t(), x @ up.t()
    f, slope = _activation(s["case"]["activation"], g)
    if s["case"]["op"] == "gated":
        return (f * u).to(kind)
    dy = s["dy"].float()
    dg, du = dy * u * slope, dy * f
    return {"x": (dg @ gate + du @ up).to(kind), "gate": (dg.t() @ x).to(kind), "up": (du.t() @ x).to(kind)}


def _plain_targets(s):
    """(words, their shares) of each row; a row without any has the shares zero."""
    if "labels" in s:
        counted = (s["labels"] >= 0)[:, None]
        return s["labels"].clamp(min=0)[:, None], counted.float()
    inside = s["indices"] >= 0
    t = (s["logits"].float() / s["case"]["temperature"]).masked_fill(~inside, -math.inf)
    top = t.amax(-1, keepdim=True).clamp(min=-3e38)
    share = torch.exp(t - top)
    return s["indices"].clamp(min=0).long(), share / share.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_loss(s):
    kind = s["x"].dtype
    x, weight = s["x"].float(), s["weight"].float()
    temperature = s["case"].get("temperature", 1.0)
    words, share = _plain_targets(s)
    z = x @ weight.t()
    if temperature != 1.0:
        z = z / temperature
    counted = (share > 0).any(-1)
    if not s["case"]["op"].endswith("_grad"):
        top = z.amax(-1, keepdim=True)
        lse = (top + torch.log(torch.exp(z - top).sum(-1, keepdim=True)))[:, 0]
        at = torch.gather(z, 1, words)
        log_share = torch.log(torch.where(share > 0, share, 1.0))
        loss = (share * (log_share - (at - lse[:, None]))).sum(-1)
        return {"loss": torch.where(counted, loss, 0.0), "lse": torch.where(counted, lse, 0.0)}
    scale = torch.where(counted, s["dloss"], 0.0)[:, None] / temperature
    G = torch.exp(z - s["lse"][:, None]) * scale
    G.scatter_add_(1, words, -share * scale)
    return {"x": (G @ weight).to(kind), "weight": (G.t() @ x).to(kind)}


def _run_plain(s):
    op = s["case"]["op"]
    if op.startswith("norm"):
        return _plain_norm(s)
    if op.startswith("gated"):
        return _plain_gated(s)
    return _plain_loss(s)


# ------------------------------------------------------------------------------------------ the framework's calls
def _queue():
    """The program's queue, on the stream that its torch operations use."""
    stream = torch.cuda.current_stream()
    key = (stream.device_index, stream.cuda_stream)
    if key not in _queues:
        from nengo_ocl_amd.hipraggedarray import Queue

        _queues[key] = Queue(stream.device_index, stream=stream)
    return _queues[key]


def _run_own(s):
    from nengo_ocl_amd import hipra_tokens as ops

    queue, op = _queue(), s["case"]["op"]
    if op == "norm":
        out, v = ops.layer_norm(queue, s["x"], s["weight"], s["bias"], s["residual"], eps=1e-5)
        return {"out": out, "v": v}
    if op == "norm_grad":
        got = ops.layer_norm_grad(queue, s["dout"], s["x"], s["weight"], s["bias"], s["residual"], eps=1e-5, dv=s["dv"])
        return {"x": got.x, "weight": got.weight, "bias": got.bias}
    if op == "gated":
        return ops.gated_projection(queue, s["x"], s["gate"], s["up"], s["case"]["activation"])
    if op == "gated_grad":
        got = ops.gated_projection_grad(queue, s["dy"], s["x"], s["gate"], s["up"], s["case"]["activation"])
        return {"x": got.x, "gate": got.gate, "up": got.up}
    if op == "loss":
        loss, lse = ops.vocabulary_loss(queue, s["x"], s["weight"], s["labels"])
        return {"loss": loss, "lse": lse}
    if op == "loss_grad":
        got = ops.vocabulary_loss_grad(queue, s["dloss"], s["x"], s["weight"], s["labels"], s["lse"])
        return {"x": got.x, "weight": got.weight}
    temperature = s["case"]["temperature"]
    if op == "teacher":
        loss, lse = ops.teacher_loss(queue, s["x"], s["weight"], s["indices"], s["logits"], temperature)
        return {"loss": loss, "lse": lse}
    got = ops.teacher_loss_grad(queue, s["dloss"], s["x"], s["weight"], s["indices"], s["logits"], s["lse"], temperature)
    return {"x": got.x, "weight": got.weight}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_norm(s):
    v = s["x"].double() + (s["residual"].double() if s["residual"] is not None else 0.0)
    d = v.shape[1]
    b = s["bias"].double() if s["bias"] is not None else torch.zeros(d, dtype=torch.float64, device=v.device)
    if s["case"]["op"] == "norm":
        var, mean = torch.var_mean(v, -1, correction=0, keepdim=True)
        return {"out": (v - mean) * (var + 1e-5).rsqrt() * s["weight"].double() + b,
                "v": v if s["residual"] is not None else None}
    v.requires_grad_()
    w = s["weight"].double().requires_grad_()
    b.requires_grad_()
    out = torch.nn.functional.layer_norm(v, (d,), w, b, 1e-5)
    dv, dw, db = torch.autograd.grad(out, (v, w, b), s["dout"].double())
    return {"x": dv if s["dv"] is None else dv + s["dv"].double(), "weight": dw,
            "bias": db if s["bias"] is not None else None}


def _exact_gated(s):
    leaves = [s[k].double().requires_grad_() for k in ("x", "gate", "up")]
    x, gate, up = leaves
    act = torch.nn.functional.silu if s["case"]["activation"] == "silu" else torch.nn.functional.gelu
    if s["case"]["op"] == "gated":
        with torch.no_grad():
            return act(x @ gate.t()) * (x @ up.t())
    y = act(x @ gate.t()) * (x @ up.t())
    return dict(zip(("x", "gate", "up"), torch.autograd.grad(y, leaves, s["dy"].double())))


def _exact_loss(s):
    """Rows that count alone, 1024 at a time."""
    case = s["case"]
    x, w = s["x"].double(), s["weight"].double()
    n, temperature = x.shape[0], float(case.get("temperature", 1.0))
    if "labels" in s:
        rows = torch.nonzero(s["labels"] >= 0)[:, 0]
    else:
        rows = torch.nonzero((s["indices"] >= 0).all(-1))[:, 0]
    loss, lse = (torch.zeros(n, dtype=torch.float64, device=x.device) for _ in range(2))
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for part in rows.split(1024):
        z = x[part] @ w.t() / temperature
        logp = torch.log_softmax(z, -1)
        q = torch.zeros_like(z)
        if "labels" in s:
            q[torch.arange(len(part), device=x.device), s["labels"][part].long()] = 1.0
            loss[part] = -(q * logp).sum(-1)
        else:
            share = torch.softmax(s["logits"][part].double() / temperature, -1)
            q.scatter_(1, s["indices"][part].long(), share)
            loss[part] = torch.special.xlogy(q, q).sum(-1) - (q * logp).sum(-1)
        lse[part] = torch.logsumexp(z, -1)
        if case["op"].endswith("_grad"):
            G = (torch.exp(logp) - q) * (s["dloss"][part].double() / temperature)[:, None]
            dx[part] = G @ w
            dw += G.t() @ x[part]
    return {"x": dx, "weight": dw} if case["op"].endswith("_grad") else {"loss": loss, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("norm"):
        return _exact_norm(s)
    if case["op"].startswith("gated"):
        return _exact_gated(s)
    return _exact_loss(s)
