"""What the operators of blocks that filter selectively are timed on: the short causal convolution, the selective scan
and the gated norm, each for prompts, in training and (where it has a state) for single tokens.

A case is one operator in one direction with its sizes and type.  `prepare` makes what a program has in hand before
the call, `run` is one call with `own` true and the same operator in elementary torch operations with `own` false, and
`exact` is its definition in 64 bits: recurrences token by token.

Ragged sequences lie back to back, [tokens, ...], and `starts` (S + 1 offsets) says where each begins; others are
batches, [S, L, ...].
"""

import math

import torch

own = False
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
CHUNK = 64  # tokens that the plain form of the scan takes together
_queues = {}


def listed():
    return [
        # training or a batch of prompts: the convolution in front of the scan of 32 heads of 64 with 128 states
        {"name": "conv_prompts", "op": "conv", "type": "bfloat16", "seqs": 8, "tokens": 16384, "ragged": False,
         "channels": 2304, "width": 4, "silu": True},
        # its gradient over prompts of unequal lengths, channels and tokens that nobody rounded
        {"name": "conv_grad_ragged", "op": "conv_grad", "type": "float32", "seqs": 7, "tokens": 5003, "ragged": True,
         "channels": 1100, "width": 4, "silu": True},
        # serving: a token each of 64 requests, whose caches lie anywhere in the pool
        {"name": "conv_step_64", "op": "conv_step", "type": "bfloat16", "requests": 64, "slots": 96,
         "channels": 2304, "width": 4, "silu": True},
        # a batch of prompts
        {"name": "scan_prompts", "op": "scan", "type": "bfloat16", "seqs": 8, "tokens": 16384, "ragged": False,
         "heads": 32, "dim": 64, "states": 128, "groups": 1, "initial": False},
        # one long document, answered by few rows of work
        {"name": "scan_long", "op": "scan", "type": "bfloat16", "seqs": 1, "tokens": 32768, "ragged": False,
         "heads": 32, "dim": 64, "states": 128, "groups": 1, "initial": False},
        # prompts of unequal lengths that continue earlier ones, an empty one and single tokens among them; odd sizes
        {"name": "scan_ragged", "op": "scan", "type": "float32", "seqs": 9, "tokens": 4001, "ragged": True,
         "heads": 12, "dim": 48, "states": 72, "groups": 3, "initial": True},
        # a training step's backward pass
        {"name": "scan_grad", "op": "scan_grad", "type": "bfloat16", "seqs": 4, "tokens": 8192, "ragged": False,
         "heads": 32, "dim": 64, "states": 128, "groups": 1, "initial": False},
        # the same in 32 bits over sequences of unequal lengths, with gradients into and out of the states
        {"name": "scan_grad_ragged", "op": "scan_grad", "type": "float32", "seqs": 5, "tokens": 1500, "ragged": True,
         "heads": 6, "dim": 40, "states": 64, "groups": 2, "initial": True},
        # serving: a token each of 128 requests, the states of 64 heads
        {"name": "scan_step_128", "op": "scan_step", "type": "bfloat16", "requests": 128, "slots": 160,
         "heads": 64, "dim": 64, "states": 128, "groups": 8},
        # one request, where latency is all
        {"name": "scan_step_one", "op": "scan_step", "type": "float32", "requests": 1, "slots": 4,
         "heads": 24, "dim": 64, "states": 64, "groups": 1},
        # the gated norm behind the scan
        {"name": "norm_gated", "op": "norm", "type": "bfloat16", "rows": 16384, "channels": 2048, "groups": 4,
         "gate": True, "residual": False, "after": False},
        # the norm in front of the next block, with the residual's scale, in the backward pass
        {"name": "norm_grad_residual", "op": "norm_grad", "type": "bfloat16", "rows": 8192, "channels": 2048,
         "groups": 1, "gate": False, "residual": True, "after": False},
    ]


def _spread(rng, low, high):
    """A whole number between the two, evenly over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["conv", "conv_grad", "conv_step", "scan", "scan", "scan_grad", "scan_grad", "scan_step",
                     "norm", "norm_grad"])
    c = {"op": op, "type": rng.choice(["bfloat16", "bfloat16", "float32", "float16"])}
    if op in ("conv", "conv_grad", "scan", "scan_grad"):
        c["seqs"] = _spread(rng, 1, 24)
        c["ragged"] = rng.random() < 0.5
        tokens = max(c["seqs"], _spread(rng, 16, 16384 if op == "conv" else 8192))
        c["tokens"] = tokens if c["ragged"] else tokens // c["seqs"] * c["seqs"]
    if op.startswith("conv"):
        c.update(channels=_spread(rng, 64, 2304), width=rng.randint(2, 6), silu=rng.random() < 0.7)
    if op.startswith("scan"):
        c["groups"] = rng.choice([1, 1, 2, 4])
        most = 16 if op == "scan_grad" or c["type"] != "bfloat16" else 32
        c["heads"] = c["groups"] * rng.randint(1, most // c["groups"])
        c["dim"] = rng.choice([64, 64, 32, 48, 80, 128 if op == "scan_step" else 61])
        c["states"] = rng.choice([128, 64, 16, 100, 96])
        if op != "scan_step":
            c["initial"] = rng.random() < 0.5
    if op.endswith("_step"):
        c["requests"] = _spread(rng, 1, 128)
        c["slots"] = c["requests"] + rng.randint(0, 32)
    if op.startswith("norm"):
        c["groups"] = rng.choice([1, 1, 2, 8])
        c["channels"] = c["groups"] * _spread(rng, 48, 2048 // c["groups"])
        c["rows"] = _spread(rng, 1, 16384 if op == "norm" else 8192)
        c["gate"] = rng.random() < 0.5
        c["residual"] = not c["gate"] or rng.random() < 0.5
        c["after"] = rng.random() < 0.5
    return c


# ------------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """How long the sequences are: equal, or unequal with an empty one and a single token among them."""
    s, t = case["seqs"], case["tokens"]
    if not case["ragged"]:
        return [t // s] * s
    share = [1.0 + 0.8 * math.sin(2.3 * k + 0.7) for k in range(s)]
    lengths = [int(t * x / sum(share)) for x in share]
    if s >= 4:
        lengths[1], lengths[2] = 0, 1
    lengths[0] += t - sum(lengths)
    return lengths


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape, scale=1.0, dtype=kind):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    def uniform(low, high, *shape):
        return torch.rand(*shape, generator=gen, device="cuda") * (high - low) + low

    f32, op, s = torch.float32, case["op"], {"case": case}
    if op in ("conv", "conv_grad", "scan", "scan_grad"):
        lengths = _lengths(case)
        s["longest"], s["n"] = max(lengths), len(lengths)
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + n)
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if case["ragged"] else None
        rows = (starts[-1],) if case["ragged"] else (s["n"], s["longest"])
    elif op.endswith("_step"):
        rows = (case["requests"],)
        s["slots"] = torch.randperm(case["slots"], generator=gen, device="cuda")[:rows[0]].to(torch.int32)
    if op.startswith("conv"):
        d, k = case["channels"], case["width"]
        s["activation"] = "silu" if case["silu"] else None
        s["x"], s["weight"], s["bias"] = normal(*rows, d), normal(d, k, scale=k ** -0.5, dtype=f32), normal(d, scale=0.1, dtype=f32)
        if op == "conv_step":
            s["state"] = normal(case["slots"], k - 1, d)
        else:
            s["initial"] = normal(s["n"], k - 1, d) if case["ragged"] else None
        if op == "conv_grad":
            s["dy"] = normal(*rows, d)
            s["dfinal"] = normal(s["n"], k - 1, d) if case["ragged"] else None
    elif op.startswith("scan"):
        h, p, n, g = case["heads"], case["dim"], case["states"], case["groups"]
        # steps between 0.001 and 0.1 on average, rates between 1 and 16
        step = torch.exp(uniform(math.log(1e-3), math.log(1e-1), h))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["A"], s["D"] = -uniform(1.0, 16.0, h), uniform(0.5, 1.5, h)
        s["x"], s["dt"] = normal(*rows, h, p), normal(*rows, h, scale=0.7)
        s["B"], s["C"] = normal(*rows, g, n), normal(*rows, g, n, scale=n ** -0.5)
        if op == "scan_step":
            s["state"] = normal(case["slots"], h, p, n, scale=0.3, dtype=f32)
        else:
            s["initial"] = normal(s["n"], h, p, n, scale=0.3, dtype=f32) if case["initial"] else None
        if op == "scan_grad":
            s["dy"] = normal(*rows, h, p)
            s["dfinal"] = normal(s["n"], h, p, n, scale=0.3, dtype=f32) if case["initial"] else None
    else:
        r, d = case["rows"], case["channels"]
        s["x"], s["weight"] = normal(r, d), uniform(0.5, 1.5, d)
        s["gate"] = normal(r, d) if case["gate"] else None
        s["residual"] = normal(r, d) if case["residual"] else None
        s["scale"] = uniform(0.2, 1.0, d) if case["residual"] else None
        if op == "norm_grad":
            s["dout"] = normal(r, d)
            s["dv"] = normal(r, d) if case["residual"] and not case["after"] else None
    return s


def work(case):
    size = 4 if case["type"] == "float32" else 2
    op = case["op"]
    grad = op.endswith("_grad")
    if op in ("conv", "conv_grad"):
        t, d, k = case["tokens"], case["channels"], case["width"]
        edge = case["seqs"] * (k - 1) * d * size * (2 if case["ragged"] else 1)
        small = d * (k + 1) * 4
        return {"bytes": t * d * size * (3 if grad else 2) + edge * (2 if grad else 1) + small * (2 if grad else 1),
                "flops": t * d * (2 * k + 6) * (3 if grad else 1)}
    if op == "conv_step":
        r, d, k = case["requests"], case["channels"], case["width"]
        return {"bytes": r * d * size * 2 * k + d * (k + 1) * 4, "flops": r * d * (2 * k + 6)}
    if op in ("scan", "scan_grad"):
        t, h, p, n, g = (case[k] for k in ("tokens", "heads", "dim", "states", "groups"))
        ends = case["seqs"] * h * p * n * 4 * (2 if case["initial"] else 1)
        row = (2 * h * p + 2 * g * n + h) * size
        if grad:
            row = (3 * h * p + 4 * g * n + 2 * h) * size
            ends = case["seqs"] * h * p * n * 4 * (3 if case["initial"] else 0)
        return {"bytes": t * row + ends, "flops": t * h * p * n * (14 if grad else 5)}
    if op == "scan_step":
        r, h, p, n, g = (case[k] for k in ("requests", "heads", "dim", "states", "groups"))
        return {"bytes": r * (h * p * n * 8 + (2 * h * p + 2 * g * n + h) * size), "flops": r * h * p * n * 5}
    r, d = case["rows"], case["channels"]
    arrays = 2 + case["gate"] + case["residual"] + (case["residual"] and not case["after"])
    if grad:  # x, gate, residual (before), dout, dv read; dx, dgate, dresidual (before) written
        before = case["residual"] and not case["after"]
        arrays = 3 + 2 * case["gate"] + 3 * before + (case["residual"] and case["after"])
    return {"bytes": r * d * size * arrays + d * 8, "flops": r * d * (16 if grad else 8)}


# ---------------------------------------------------------------------------------------------- the plain forms
def _padded(s, v, front=0):
    """[S, front + longest, ...]: ragged rows each in its place, zeros in front of and behind each sequence."""
    if s["starts"] is not None:
        starts = s["starts"].long()
        places = starts[:-1, None] + torch.arange(s["longest"], device=v.device)
        inside = places < starts[1:, None]
        rows = v.index_select(0, torch.where(inside, places, 0).reshape(-1)).reshape(inside.shape + v.shape[1:])
        v = rows * inside.reshape(inside.shape + (1,) * (rows.dim() - 2)).to(v.dtype)
    if front:
        v = torch.cat([torch.zeros((v.shape[0], front) + v.shape[2:], dtype=v.dtype, device=v.device), v], 1)
    return v


def _packed(s, v, tokens):
    """Ragged rows back to back again; batches as they are."""
    if s["starts"] is None:
        return v[:, :s["longest"]]
    starts = s["starts"].long()
    t = torch.arange(tokens, device=v.device)
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    return v.flatten(0, 1).index_select(0, seq * v.shape[1] + t - starts[seq])


def _silu(v):
    return v / (1 + torch.exp(-v))


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))


def _plain_conv(s, x, weight, bias, initial):
    k = weight.shape[1]
    rows = _padded(s, x, front=k - 1)
    if initial is not None:
        rows = torch.cat([initial, rows[:, k - 1:]], 1)
    u = (rows.unfold(1, k, 1) * weight).sum(-1) + bias
    y = _packed(s, _silu(u) if s["activation"] else u, x.shape[0])
    if s["starts"] is None:
        return y, rows[:, s["longest"]:]
    last = s["starts"].long().diff()[:, None] + torch.arange(k - 1, device=x.device)
    return y, torch.gather(rows, 1, last[..., None].expand(-1, -1, x.shape[1]))


def _segment_sums(a):
    """[..., Q, Q]: the sum of a over (j, i], and -inf above the diagonal."""
    q = a.shape[-1]
    below = torch.tril(torch.ones(q, q, dtype=torch.bool, device=a.device), -1)
    sums = torch.cumsum(a[..., :, None].expand(a.shape + (q,)).masked_fill(~below, 0), -2)
    return sums.masked_fill(~torch.tril(torch.ones_like(below)), -math.inf)


def _plain_scan(s, x, dt, A, B, C, D, dt_bias, initial):
    tokens, (h, p), (g, n) = x.shape[0], x.shape[-2:], B.shape[-2:]
    step = _softplus(dt + dt_bias)
    chunks = max(1, -(-s["longest"] // CHUNK))

    def cut(v):  # [S, chunks, CHUNK, ...]
        v = _padded(s, v)
        more = chunks * CHUNK - v.shape[1]
        v = torch.cat([v, torch.zeros(v.shape[:1] + (more,) + v.shape[2:], device=v.device)], 1)
        return v.reshape((v.shape[0], chunks, CHUNK) + v.shape[2:])

    xs = cut(x).permute(0, 1, 3, 2, 4).contiguous()          # S c h q p
    steps = cut(step).permute(0, 1, 3, 2).contiguous()       # S c h q
    Bs = cut(B).permute(0, 1, 3, 2, 4).contiguous()          # S c g q n
    Cs = cut(C).permute(0, 1, 3, 2, 4).contiguous()
    a = steps * A[:, None]
    products = torch.matmul(Cs, Bs.transpose(-1, -2).contiguous()).repeat_interleave(h // g, 2)
    Bs, Cs = Bs.repeat_interleave(h // g, 2), Cs.repeat_interleave(h // g, 2)
    sums = _segment_sums(a)
    weights = products * torch.exp(sums) * steps[..., None, :]
    y = torch.matmul(weights, xs)
    to_end = torch.exp(sums[..., -1, :]) * steps
    states = torch.matmul((xs * to_end[..., None]).transpose(-1, -2).contiguous(), Bs)      # S c h p n
    first = torch.zeros_like(states[:, :1]) if initial is None else initial[:, None]
    states = torch.cat([first, states], 1).permute(0, 2, 1, 3, 4).reshape(s["n"], h, chunks + 1, p * n)
    totals = torch.cat([torch.zeros_like(a[:, :1, :, 0]), a.sum(-1)], 1).permute(0, 2, 1)   # S h 1+c
    states = torch.matmul(torch.exp(_segment_sums(totals.contiguous())), states).reshape(s["n"], h, chunks + 1, p, n)
    before = states[:, :, :-1].permute(0, 2, 1, 4, 3).contiguous()                          # S c h n p
    y = y + torch.exp(torch.cumsum(a, -1))[..., None] * torch.matmul(Cs, before) + D[:, None, None] * xs
    y = y.permute(0, 1, 3, 2, 4).reshape(s["n"], chunks * CHUNK, h, p)
    return _packed(s, y, tokens), states[:, :, -1]


def _plain_norm(s, x, weight, gate, residual, scale, eps=1e-6):
    groups, after = s["case"]["groups"], s["case"]["after"]
    u = x if gate is None else x * _silu(gate)
    if residual is not None and not after:
        u = residual + scale * u
    parts = u.reshape(u.shape[0], groups, -1)
    out = (parts / torch.sqrt((parts * parts).mean(-1, keepdim=True) + eps)).reshape(u.shape) * weight
    if residual is not None and after:
        return residual + scale * out, None
    return out, u if residual is not None else None


def _plain_step(s, state, x, dt, A, B, C, D, dt_bias):
    share = x.shape[1] // B.shape[1]
    B, C = B.repeat_interleave(share, 1), C.repeat_interleave(share, 1)
    step = _softplus(dt + dt_bias)
    state = torch.exp(step * A)[..., None, None] * state + (step[..., None] * x)[..., None] * B[:, :, None]
    return (state * C[:, :, None]).sum(-1) + D[:, None] * x, state


def _gradients(function, inputs, outputs):
    """The outputs' gradients with respect to the inputs, each rounded once to its input's type."""
    leaves = {k: v.float().requires_grad_() for k, v in inputs.items() if v is not None}
    pairs = [(y, dy.float()) for y, dy in zip(function(**leaves, **{k: None for k in inputs if k not in leaves}), outputs)
             if dy is not None]
    got = torch.autograd.grad([y for y, _ in pairs], list(leaves.values()), [dy for _, dy in pairs])
    return {k: v.to(inputs[k].dtype) for k, v in zip(leaves, got)}


def _wide(v):
    return None if v is None else v.float()


CONV = ("x", "weight", "bias", "initial")
SCAN = ("x", "dt", "A", "B", "C", "D", "dt_bias", "initial")
NORM = ("x", "weight", "gate", "residual", "scale")


def _run_plain(s):
    op = s["case"]["op"]
    kind = s["x"].dtype
    if op == "conv":
        y, final = _plain_conv(s, *[_wide(s[k]) for k in CONV])
        return {"y": y.to(kind), "final": final.to(kind)}
    if op == "conv_grad":
        return _gradients(lambda **v: _plain_conv(s, **v), {k: s[k] for k in CONV}, (s["dy"], s["dfinal"]))
    if op == "conv_step":
        slots = s["slots"].long()
        rows = torch.cat([s["state"][slots], s["x"][:, None]], 1)
        u = (rows.float() * s["weight"].t()).sum(1) + s["bias"]
        s["state"][slots] = rows[:, 1:]
        return {"y": (_silu(u) if s["activation"] else u).to(kind), "state": s["state"]}
    if op == "scan":
        y, final = _plain_scan(s, *[_wide(s[k]) for k in SCAN])
        return {"y": y.to(kind), "final": final}
    if op == "scan_grad":
        return _gradients(lambda **v: _plain_scan(s, **v), {k: s[k] for k in SCAN}, (s["dy"], s["dfinal"]))
    if op == "scan_step":
        slots = s["slots"].long()
        y, state = _plain_step(s, s["state"][slots], *[_wide(s[k]) for k in SCAN[:-1]])
        s["state"][slots] = state
        return {"y": y.to(kind), "state": s["state"]}
    if op == "norm":
        out, v = _plain_norm(s, *[_wide(s[k]) for k in NORM])
        return {"out": out.to(kind), "v": None if v is None else v.to(kind)}
    return _gradients(lambda **v: _plain_norm(s, **v), {k: s[k] for k in NORM}, (s["dout"], s["dv"]))


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
    from nengo_ocl_amd import hipra_selective as ops

    queue, op = _queue(), s["case"]["op"]
    if op.startswith("conv"):
        given = {"weight": s["weight"], "bias": s["bias"], "activation": s["activation"]}
        if op == "conv_step":
            y = ops.causal_conv_step(queue, s["state"], s["x"], slots=s["slots"], **given)
            return {"y": y, "state": s["state"]}
        given.update(initial=s["initial"], starts=s["starts"])
        if op == "conv":
            y, final = ops.causal_conv(queue, s["x"], **given)
            return {"y": y, "final": final}
        got = ops.causal_conv_grad(queue, s["dy"], s["x"], dfinal=s["dfinal"], **given)
        return {k: getattr(got, k) for k in CONV if s[k] is not None}
    if op.startswith("scan"):
        given = {k: s[k] for k in SCAN[:-1]}
        if op == "scan_step":
            y = ops.selective_step(queue, s["state"], softplus=True, slots=s["slots"], **given)
            return {"y": y, "state": s["state"]}
        given.update(softplus=True, initial=s["initial"], starts=s["starts"])
        if op == "scan":
            y, final = ops.selective_scan(queue, **given)
            return {"y": y, "final": final}
        got = ops.selective_scan_grad(queue, s["dy"], dfinal=s["dfinal"], **given)
        return {k: getattr(got, k) for k in SCAN if s[k] is not None}
    given = {k: s[k] for k in NORM}
    given.update(groups=s["case"]["groups"], after=s["case"]["after"], eps=1e-6)
    if op == "norm":
        out, v = ops.block_norm(queue, **given)
        return {"out": out, "v": v}
    got = ops.block_norm_grad(queue, s["dout"], dv=s["dv"], **given)
    return {k: getattr(got, k) for k in NORM if s[k] is not None}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------ the definition in 64 bits
def _laid_flat(s):
    """The same inputs with all tokens back to back, and where each sequence begins and ends."""
    s = dict(s)
    if s["starts"] is None:
        for k in ("x", "dt", "B", "C", "dy"):
            if k in s:
                s[k] = s[k].flatten(0, 1)
        s["starts"] = torch.arange(s["n"] + 1, device=s["x"].device) * s["longest"]
    at = s["starts"].tolist()
    return s, list(zip(at[:-1], at[1:]))


def _exact_conv(s, sequences, want_grad):
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    k, d = w.shape[1], x.shape[1]
    given = s["initial"].double() if s["initial"] is not None else x.new_zeros(s["n"], k - 1, d)
    y, final = torch.empty_like(x), torch.empty_like(given)
    dx, dw, db, dinitial = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b), torch.zeros_like(given)
    for i, (t0, t1) in enumerate(sequences):
        line = torch.cat([given[i], x[t0:t1]])
        n = t1 - t0
        u = b + sum(w[:, j] * line[j:j + n] for j in range(k))
        sig = torch.sigmoid(u)
        y[t0:t1] = u * sig if s["activation"] else u
        final[i] = line[n:]
        if want_grad:
            du = s["dy"][t0:t1].double()
            if s["activation"]:
                du = du * (sig + u * sig * (1 - sig))
            dline = torch.zeros_like(line)
            for j in range(k):
                dline[j:j + n] += du * w[:, j]
                dw[:, j] += (du * line[j:j + n]).sum(0)
            db += du.sum(0)
            if s["dfinal"] is not None:
                dline[n:] += s["dfinal"][i].double()
            dinitial[i], dx[t0:t1] = dline[:k - 1], dline[k - 1:]
    if not want_grad:
        return {"y": y, "final": final}
    got = {"x": dx, "weight": dw, "bias": db}
    return got if s["initial"] is None else dict(got, initial=dinitial)


def _exact_scan(s, want_grad):
    """The recurrence token by token, all sequences side by side; the gradient by the adjoint recurrence."""
    x, dt, A, B, C, D, bias = (s[k].double() for k in SCAN[:-1])
    h, p = x.shape[1:]
    share, n = h // B.shape[1], B.shape[2]
    raw = dt + bias
    step = torch.nn.functional.softplus(raw, threshold=60)
    decay = torch.exp(step * A)
    rows, longest = x.shape[0], s["longest"]
    starts = s["starts"].long()
    lengths = starts.diff()
    state = s["initial"].double() if s["initial"] is not None else x.new_zeros(s["n"], h, p, n)
    y = torch.zeros_like(x)
    kept = [None] * longest
    # sequences in order of length, so that those that go on at token t are the first of them
    order = torch.argsort(lengths, descending=True)
    begins, state, sizes = starts[order], state[order].clone(), sorted(lengths.tolist(), reverse=True)
    going = [sum(1 for v in sizes if v > t) for t in range(longest)]
    for t in range(longest):
        m = going[t]
        r = begins[:m] + t
        if want_grad:
            kept[t] = state[:m].clone()
        b = B[r].repeat_interleave(share, 1)
        state[:m] = decay[r][..., None, None] * state[:m] + (step[r][..., None] * x[r])[..., None] * b[:, :, None]
        y[r] = (state[:m] @ C[r].repeat_interleave(share, 1)[..., None])[..., 0] + D[:, None] * x[r]
    if not want_grad:
        final = torch.empty_like(state)
        final[order] = state
        return {"y": y, "final": final}
    dy = s["dy"].double()
    back = s["dfinal"].double()[order].clone() if s["dfinal"] is not None else torch.zeros_like(state)
    dx, dstep, dB, dC = D[:, None] * dy, torch.zeros_like(step), torch.zeros_like(B), torch.zeros_like(C)
    dA = torch.zeros_like(A)
    for t in range(longest - 1, -1, -1):
        m = going[t]
        r = begins[:m] + t
        c, b = C[r].repeat_interleave(share, 1), B[r].repeat_interleave(share, 1)
        old = kept[t]
        fresh = decay[r][..., None, None] * old + (step[r][..., None] * x[r])[..., None] * b[:, :, None]
        dC[r] = (dy[r][:, :, None] @ fresh)[:, :, 0].reshape(m, -1, share, n).sum(2)
        back[:m] += dy[r][..., None] * c[:, :, None]
        g = back[:m]
        gb = (g @ b[..., None])[..., 0]
        dx[r] += step[r][..., None] * gb
        dB[r] = ((step[r][..., None] * x[r])[:, :, None] @ g)[:, :, 0].reshape(m, -1, share, n).sum(2)
        da = (g * old).sum((-1, -2)) * decay[r]
        dstep[r] = (gb * x[r]).sum(-1) + da * A
        dA += (da * step[r]).sum(0)
        back[:m] = decay[r][..., None, None] * g
        kept[t] = None
    draw_ = dstep * torch.sigmoid(raw)
    dinitial = torch.empty_like(back)
    dinitial[order] = back
    got = {"x": dx, "dt": draw_, "A": dA, "B": dB, "C": dC, "D": (dy * x).sum((0, 2)), "dt_bias": draw_.sum(0)}
    return got if s["initial"] is None else dict(got, initial=dinitial)


def _exact_norm(s, want_grad, eps=1e-6):
    groups, after = s["case"]["groups"], s["case"]["after"]
    x, w = s["x"].double(), s["weight"].double()
    sig = torch.sigmoid(s["gate"].double()) if s["gate"] is not None else None
    gate = s["gate"].double() * sig if sig is not None else torch.ones_like(x)
    has = s["residual"] is not None
    res, scale = (s["residual"].double(), s["scale"].double()) if has else (torch.zeros_like(x), torch.ones_like(w))
    before = has and not after
    v = res + scale * x * gate if before else x * gate

    def parts(m):
        return m.reshape(m.shape[0], groups, -1)

    inv = (parts(v).square().mean(-1, keepdim=True) + eps).rsqrt()
    unit = (parts(v) * inv).reshape(v.shape)
    if not want_grad:
        if has and after:
            return {"out": res + scale * unit * w, "v": None}
        return {"out": unit * w, "v": v if has else None}
    dout = s["dout"].double()
    got, dn = {}, dout
    if has and after:
        got["residual"], got["scale"] = dout, (dout * unit * w).sum(0)
        dn = dout * scale
    got["weight"] = (dn * unit).sum(0)
    du = dn * w
    dv = (inv * (parts(du) - parts(unit) * (parts(du) * parts(unit)).mean(-1, keepdim=True))).reshape(v.shape)
    if before:
        if s["dv"] is not None:
            dv = dv + s["dv"].double()
        got["residual"], got["scale"] = dv, (dv * x * gate).sum(0)
        dv = dv * scale
    got["x"] = dv * gate
    if sig is not None:
        got["gate"] = dv * x * (sig + gate * (1 - sig))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    grad = op.endswith("_grad")
    if op in ("conv", "conv_grad", "scan", "scan_grad"):
        flat, sequences = _laid_flat(s)
        got = _exact_conv(flat, sequences, grad) if op.startswith("conv") else _exact_scan(flat, grad)
        if s["starts"] is None:
            got = {k: v.unflatten(0, (s["n"], s["longest"])) if k in ("x", "y", "dt", "B", "C") else v for k, v in got.items()}
        return got
    if op.startswith("norm"):
        return _exact_norm(s, grad)
    slots, state = s["slots"].long(), s["state"].double()
    if op == "conv_step":
        line = torch.cat([state[slots], s["x"].double()[:, None]], 1)
        u = s["bias"].double() + (line.transpose(1, 2) * s["weight"].double()).sum(-1)
        state[slots] = line[:, 1:]
        return {"y": u * torch.sigmoid(u) if s["activation"] else u, "state": state}
    x, dt, A, B, C, D, bias = (s[k].double() for k in SCAN[:-1])
    share = x.shape[1] // B.shape[1]
    step = torch.nn.functional.softplus(dt + bias, threshold=60)
    new = torch.exp(step * A)[..., None, None] * state[slots]
    new += (step[..., None] * x)[..., None] * B.repeat_interleave(share, 1)[:, :, None]
    state[slots] = new
    return {"y": (new @ C.repeat_interleave(share, 1)[..., None])[..., 0] + D[:, None] * x, "state": state}
