"""Short causal convolution, selective scan and gated norm against their definitions in 64 bits,
token by token, and what their entry points refuse.

Tolerances.  u = 2**-24, 2**-9, 2**-12 is the largest relative error of rounding to float32, bfloat16, float16.
Results of 16 bits are rounded once, and what is rounded to 16 bits on the way (weights and
states as operands of a product) counts once each: at most three roundings, 3 u of the
result's norm.  Results of 32 bits come from sums of up to some hundred terms, each with a few
roundings: 128 u = 7.6e-6 of the norm, where the terms' signs are random.
"""

import itertools

import numpy as np
import pytest
import torch

from helpers import host_queue

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ROUNDING = {F32: 128 * 2.0 ** -24, BF16: 3 * 2.0 ** -9, F16: 3 * 2.0 ** -12}


@pytest.fixture(scope="module")
def ops():
    from nengo_ocl_amd import hipra_selective

    return hipra_selective


def near(got, want, name=""):
    """Within the tolerance of the result's type: of the norm, and of the largest element."""
    got64, want = got.detach().cpu().double(), want.detach().cpu().double()
    assert got64.shape == want.shape, (name, got64.shape, want.shape)
    if not want.numel():
        return
    assert torch.equal(torch.isfinite(got64), torch.isfinite(want)), name
    ok = torch.isfinite(want)
    err, scale = (got64 - want)[ok], want[ok]
    tol = ROUNDING[got.dtype]
    assert err.norm() <= tol * scale.norm() + 1e-30, (name, float(err.norm() / scale.norm()))
    assert err.abs().max() <= 4 * tol * scale.abs().max() + 1e-30, (name, float(err.abs().max()))


def wide(*tensors):
    return [None if t is None else t.detach().cpu().double() for t in tensors]


# ------------------------------------------------------------------------------ definitions
def spans(x, starts):
    """(tokens back to back, [(begin, end), ...])"""
    if starts is None:
        s, n = x.shape[:2]
        return x.reshape((s * n,) + x.shape[2:]), [(k * n, k * n + n) for k in range(s)]
    at = [int(v) for v in starts]
    return x, list(zip(at[:-1], at[1:]))


def silu(v):
    return v * torch.sigmoid(v)


def conv_definition(x, weight, bias, silu_, initial, starts):
    flat, seqs = spans(x, starts)
    k, d = weight.shape[1], weight.shape[0]
    y, final = [], []
    for s, (a, b) in enumerate(seqs):
        line = torch.cat([initial[s] if initial is not None else flat.new_zeros(k - 1, d), flat[a:b]])
        u = sum(line[j:j + b - a] * weight[:, j] for j in range(k))
        u = u if bias is None else u + bias
        y.append(silu(u) if silu_ else u)
        final.append(line[b - a:])
    return torch.cat(y).reshape(x.shape), torch.stack(final)


def scan_definition(x, dt, A, B, C, D, dt_bias, softplus, initial, starts):
    flat, seqs = spans(x, starts)
    (dt, _), (B, _), (C, _) = spans(dt, starts), spans(B, starts), spans(C, starts)
    h, p = flat.shape[1:]
    share, n = h // B.shape[1], B.shape[2]
    step = dt if dt_bias is None else dt + dt_bias
    step = torch.logaddexp(step, torch.zeros_like(step)) if softplus else step
    ys, finals = [], []
    for s, (a, b) in enumerate(seqs):
        S = initial[s] if initial is not None else flat.new_zeros(h, p, n)
        for t in range(a, b):
            S = torch.exp(step[t] * A)[:, None, None] * S \
                + (step[t][:, None] * flat[t])[:, :, None] * B[t].repeat_interleave(share, 0)[:, None]
            y = (S * C[t].repeat_interleave(share, 0)[:, None]).sum(-1)
            ys.append(y if D is None else y + D[:, None] * flat[t])
        finals.append(S)
    y = torch.stack(ys) if ys else flat.new_zeros(0, h, p)
    return y.reshape(x.shape), torch.stack(finals)


def norm_definition(x, weight, gate, residual, scale, groups, eps, after):
    u = x if gate is None else x * silu(gate)
    scale = 1.0 if scale is None else scale
    if residual is not None and not after:
        u = residual + scale * u
    parts = u.reshape(u.shape[:-1] + (groups, u.shape[-1] // groups))
    out = (parts / torch.sqrt((parts ** 2).mean(-1, keepdim=True) + eps)).reshape(u.shape) * weight
    if residual is not None and after:
        return residual + scale * out, None
    return out, u if residual is not None else None


def gradients(function, inputs, outputs):
    """{name: gradient} of the definition in 64 bits."""
    leaves = {k: v.detach().cpu().double().requires_grad_() for k, v in inputs.items() if v is not None}
    pairs = [(y, g.cpu().double()) for y, g in zip(function(**leaves), outputs) if g is not None and y.requires_grad]
    got = torch.autograd.grad([y for y, _ in pairs], list(leaves.values()), [g for _, g in pairs], allow_unused=True)
    return {k: torch.zeros_like(leaves[k]) if g is None else g for k, g in zip(leaves, got)}


def along_differences(function, inputs, outputs, got, seed):
    """The gradient along a random direction against the difference of the definition's values there."""
    gen = torch.Generator().manual_seed(seed)
    base = {k: v.detach().cpu().double() for k, v in inputs.items() if v is not None}
    way = {k: torch.randn(v.shape, generator=gen, dtype=torch.float64) for k, v in base.items()}

    def value(eps):
        ys = function(**{k: v + eps * way[k] for k, v in base.items()})
        return sum((y * g.cpu().double()).sum() for y, g in zip(ys, outputs) if g is not None)

    eps = 1e-5  # central differences: their own error is of the order of eps**2
    want = float((value(eps) - value(-eps)) / (2 * eps))
    terms = [(got[k].cpu().double() * way[k]).sum() for k in base]
    size = sum(float(got[k].cpu().double().norm()) for k in base)
    tol = max(ROUNDING[got[k].dtype] for k in base)
    assert abs(float(sum(terms)) - want) <= (4 * tol + 1e-6) * size, (float(sum(terms)), want, size)


# ---------------------------------------------------------------------------------- inputs
class Maker:
    def __init__(self, seed):
        self.gen = torch.Generator().manual_seed(seed)

    def normal(self, *shape, dtype=F32, scale=1.0):
        return (torch.randn(*shape, generator=self.gen) * scale).to(dtype).cuda()

    def uniform(self, low, high, *shape):
        return (torch.rand(*shape, generator=self.gen) * (high - low) + low).cuda()


def starts_of(lengths):
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32).cuda()


RAGGED = [[5], [1, 0, 70, 64, 3], [0, 0], [129, 1, 1, 1, 63, 65], list(range(70))]


def conv_inputs(seed, dtype, lengths, channels, width, initial, dense=None):
    m = Maker(seed)
    lead = dense or (sum(lengths),)
    s = dense[0] if dense else len(lengths)
    return {"x": m.normal(*lead, channels, dtype=dtype), "weight": m.normal(channels, width, scale=width ** -0.5),
            "bias": m.normal(channels), "initial": m.normal(s, width - 1, channels, dtype=dtype) if initial else None}, \
        None if dense else starts_of(lengths), m


def scan_inputs(seed, dtype, lengths, heads, dim, groups, states, initial, dense=None):
    m = Maker(seed)
    lead = dense or (sum(lengths),)
    s = dense[0] if dense else len(lengths)
    return {"x": m.normal(*lead, heads, dim, dtype=dtype), "dt": m.normal(*lead, heads, dtype=dtype, scale=0.7),
            "A": -m.uniform(1.0, 8.0, heads), "B": m.normal(*lead, groups, states, dtype=dtype),
            "C": m.normal(*lead, groups, states, dtype=dtype, scale=states ** -0.5), "D": m.uniform(0.5, 1.5, heads),
            "dt_bias": m.uniform(-5.0, -1.0, heads),
            "initial": m.normal(s, heads, dim, states) if initial else None}, \
        None if dense else starts_of(lengths), m


# ----------------------------------------------------------------------------- convolution
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("channels, width, silu_, lengths", [
    (64, 4, True, RAGGED[1]), (37, 3, False, RAGGED[3]), (8, 1, True, RAGGED[0]), (520, 8, True, RAGGED[4]),
    (16, 2, False, RAGGED[2]), (1, 5, True, [200])])
def test_conv(queue, ops, dtype, channels, width, silu_, lengths):
    for initial in (False, True):
        given, starts, _ = conv_inputs(1, dtype, lengths, channels, width, initial)
        y, final = ops.causal_conv(queue, activation="silu" if silu_ else None, starts=starts, **given)
        y64, final64 = conv_definition(*wide(given["x"], given["weight"], given["bias"]), silu_,
                                       *wide(given["initial"]), starts)
        near(y, y64, "y")
        assert torch.equal(final.cpu().double(), final64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("channels, width, silu_, lengths", [
    (64, 4, True, RAGGED[1]), (37, 3, False, RAGGED[3]), (8, 1, True, RAGGED[0]), (72, 8, True, RAGGED[4]),
    (16, 2, False, RAGGED[2])])
def test_conv_gradient(queue, ops, dtype, channels, width, silu_, lengths):
    given, starts, m = conv_inputs(2, dtype, lengths, channels, width, True)
    dy = m.normal(sum(lengths), channels, dtype=dtype)
    dfinal = m.normal(len(lengths), width - 1, channels, dtype=dtype)
    got = ops.causal_conv_grad(queue, dy, activation="silu" if silu_ else None, starts=starts, dfinal=dfinal, **given)

    def function(x, weight, bias, initial):
        return conv_definition(x, weight, bias, silu_, initial, starts)

    want = gradients(function, given, (dy, dfinal))
    for k in want:
        near(getattr(got, k), want[k], k)
    along_differences(function, given, (dy, dfinal), got._asdict(), 3)


@pytest.mark.gpu
def test_conv_rows_with_strides(queue, ops):
    """Channels of a wider projection, side by side, with and without 16-byte rows; no bias."""
    for first, dtype in itertools.product((8, 3), (F32, BF16)):
        given, _, m = conv_inputs(4, dtype, None, 24, 4, False, dense=(3, 70))
        whole = m.normal(3, 70, 51, dtype=dtype)
        x = whole[:, :, first:first + 24]
        y, _ = ops.causal_conv(queue, x, given["weight"])
        near(y, conv_definition(*wide(x, given["weight"]), None, False, None, None)[0], "y")
        got = ops.causal_conv_grad(queue, whole[:, :, 27:51], x, given["weight"])
        want = gradients(lambda x, weight: conv_definition(x, weight, None, False, None, None)[:1],
                         {"x": x, "weight": given["weight"]}, (whole[:, :, 27:51],))
        near(got.x, want["x"], "x")
        near(got.weight, want["weight"], "weight")
        assert got.bias is None and got.initial is None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, channels, width", [(F32, 40, 4), (BF16, 40, 4), (F16, 33, 3), (BF16, 16, 1)])
def test_conv_token_by_token(queue, ops, dtype, channels, width):
    """Prompts, then single tokens that go on from their final state, in slots of a larger pool; a request
    without a slot gets zeros and changes nothing."""
    given, _, m = conv_inputs(5, dtype, None, channels, width, False, dense=(3, 12))
    y, _ = ops.causal_conv(queue, activation="silu", **given)
    _, final = ops.causal_conv(queue, given["x"][:, :7], given["weight"], given["bias"], "silu")
    pool = m.normal(6, width - 1, channels, dtype=dtype)
    slots = torch.tensor([4, 0, 5, -1, 6], dtype=torch.int32).cuda()
    pool[slots[:3].long()] = final
    before = pool.clone()
    for t in range(7, 12):
        x = torch.cat([given["x"][:, t], m.normal(2, channels, dtype=dtype)])
        out = ops.causal_conv_step(queue, pool, x, given["weight"], given["bias"], "silu", slots=slots)
        assert torch.equal(out[:3], y[:, t])
        assert not out[3:].any()
    if width > 1:
        assert torch.equal(pool[[1, 2, 3]], before[[1, 2, 3]])
        _, final = ops.causal_conv(queue, activation="silu", **given)
        assert torch.equal(pool[slots[:3].long()], final)


# ------------------------------------------------------------------------------------ scan
SIZES = [(2, 64, 1, 128), (4, 16, 2, 16), (3, 61, 1, 33), (2, 130, 2, 7), (6, 8, 3, 200), (1, 1, 1, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads, dim, groups, states", SIZES)
@pytest.mark.parametrize("lengths", [RAGGED[1], RAGGED[3], RAGGED[2]])
def test_scan(queue, ops, dtype, heads, dim, groups, states, lengths):
    for initial in (False, True):
        given, starts, _ = scan_inputs(6, dtype, lengths, heads, dim, groups, states, initial)
        y, final = ops.selective_scan(queue, softplus=True, starts=starts, **given)
        y64, final64 = scan_definition(**dict(zip(given, wide(*given.values()))), softplus=True, starts=starts)
        near(y, y64, "y")
        near(final, final64, "final")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_of_batches_without_the_optional(queue, ops, dtype):
    """[S, L, ...] with strides of a wider projection, steps as they are, no D and no bias."""
    for length in (1, 2, 64, 100):
        given, _, m = scan_inputs(7, dtype, None, 4, 24, 2, 20, False, dense=(3, length))
        whole = m.normal(3, length, 4 * 24 + 2 * 2 * 20 + 5, dtype=dtype)
        x = whole[..., :96].unflatten(-1, (4, 24))
        B, C = (whole[..., 96 + 40 * k:136 + 40 * k].unflatten(-1, (2, 20)) for k in range(2))
        dt = given["dt"].float().abs()[..., :1].expand(3, length, 4)  # one step for all heads
        y, final = ops.selective_scan(queue, x, dt, given["A"], B, C)
        y64, final64 = scan_definition(*wide(x, dt, given["A"], B, C), None, None, False, None, None)
        near(y, y64, "y")
        near(final, final64, "final")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_over_many_chunks(queue, ops, dtype):
    """Few rows of work over a long axis: the same results as chunk by chunk, for one sequence and for several."""
    for lengths in ([3001], [2000, 5, 0, 1100]):
        given, starts, _ = scan_inputs(8, dtype, lengths, 2, 16, 1, 16, True)
        y, final = ops.selective_scan(queue, softplus=True, starts=starts, **given)
        y64, final64 = scan_definition(**dict(zip(given, wide(*given.values()))), softplus=True, starts=starts)
        near(y, y64, "y")
        near(final, final64, "final")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_forgets_all(queue, ops, dtype):
    """Steps so large that nothing of the state is left, between small ones: what follows is as exact as ever."""
    given, starts, _ = scan_inputs(9, dtype, [150], 2, 16, 1, 16, True)
    given["dt"][[10, 40, 64, 127]] = 3.0e4
    y, final = ops.selective_scan(queue, softplus=True, starts=starts, **given)
    y64, final64 = scan_definition(**dict(zip(given, wide(*given.values()))), softplus=True, starts=starts)
    for a, b in ((0, 10), (11, 40), (41, 64), (65, 127), (128, 150)):
        near(y[a:b], y64[a:b], "y")
    near(final, final64, "final")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_scan_keeps_sequences_and_the_past_apart(queue, ops, dtype, bad):
    """A value that is none reaches the tokens behind it in its own sequence, and no others."""
    for name in ("x", "B", "dt"):
        given, starts, _ = scan_inputs(10, dtype, [40, 90, 30], 2, 16, 1, 16, False)
        clean, _ = ops.selective_scan(queue, softplus=True, starts=starts, **given)
        given[name] = given[name].clone()
        given[name][60] = bad
        y, final = ops.selective_scan(queue, softplus=True, starts=starts, **given)
        assert torch.equal(y[:60], clean[:60]) and torch.equal(y[130:], clean[130:]), name
        assert torch.isfinite(final[[0, 2]]).all(), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads, dim, groups, states", SIZES)
def test_scan_gradient(queue, ops, dtype, heads, dim, groups, states):
    for lengths in ([1, 0, 70, 64, 3], [0, 0]):
        given, starts, m = scan_inputs(11, dtype, lengths, heads, dim, groups, states, True)
        dy = m.normal(sum(lengths), heads, dim, dtype=dtype)
        dfinal = m.normal(len(lengths), heads, dim, states)
        got = ops.selective_scan_grad(queue, dy, softplus=True, starts=starts, dfinal=dfinal, **given)

        def function(**v):
            return scan_definition(softplus=True, starts=starts, **v)

        want = gradients(function, given, (dy, dfinal))
        for k in want:
            near(getattr(got, k), want[k], k)
        along_differences(function, given, (dy, dfinal), got._asdict(), 12)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths", [[230], [700, 3, 0, 420]])
def test_scan_gradient_over_many_chunks(queue, ops, dtype, lengths):
    """States and their gradients go through several segments, few and many."""
    given, starts, m = scan_inputs(24, dtype, lengths, 2, 16, 1, 16, True)
    dy, dfinal = m.normal(sum(lengths), 2, 16, dtype=dtype), m.normal(len(lengths), 2, 16, 16)
    got = ops.selective_scan_grad(queue, dy, softplus=True, starts=starts, dfinal=dfinal, **given)
    want = gradients(lambda **v: scan_definition(softplus=True, starts=starts, **v), given, (dy, dfinal))
    for k in want:
        near(getattr(got, k), want[k], k)


@pytest.mark.gpu
def test_scan_gradient_without_the_optional(queue, ops):
    given, _, m = scan_inputs(13, BF16, None, 8, 32, 2, 32, False, dense=(2, 200))
    dy = m.normal(2, 200, 8, 32, dtype=BF16)
    inputs = {"x": given["x"], "dt": given["dt"].abs().float(), "A": given["A"], "B": given["B"], "C": given["C"]}
    got = ops.selective_scan_grad(queue, dy, **inputs)
    want = gradients(lambda **v: scan_definition(D=None, dt_bias=None, softplus=False, initial=None, starts=None, **v)[:1],
                     inputs, (dy,))
    for k in want:
        near(getattr(got, k), want[k], k)
    assert got.D is None and got.dt_bias is None and got.initial is None
    again = ops.selective_scan_grad(queue, dy, **inputs)
    assert all(torch.equal(getattr(got, k), getattr(again, k)) for k in want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, heads, dim, groups, states", [
    (F32, 4, 16, 2, 16), (BF16, 2, 64, 1, 128), (F16, 3, 5, 3, 9), (BF16, 2, 24, 1, 200)])
def test_scan_token_by_token(queue, ops, dtype, heads, dim, groups, states):
    """Single tokens that go on from a prompt's final state give what the whole prompt gives."""
    given, _, m = scan_inputs(14, dtype, None, heads, dim, groups, states, False, dense=(3, 12))
    rows = ("x", "dt", "B", "C")
    rest = {k: v for k, v in given.items() if k not in rows and k != "initial"}
    y64, _ = scan_definition(**dict(zip(given, wide(*given.values()))), softplus=True, starts=None)
    _, final = ops.selective_scan(queue, softplus=True, **{k: given[k][:, :7] for k in rows}, **rest)
    pool = m.normal(6, heads, dim, states)
    slots = torch.tensor([4, 0, 5, -1, 6], dtype=torch.int32).cuda()
    pool[slots[:3].long()] = final
    before = pool.clone()
    for t in range(7, 12):
        now = {k: torch.cat([given[k][:, t], given[k][:2, 0]]) for k in rows}
        out = ops.selective_step(queue, pool, softplus=True, slots=slots, **now, **rest)
        near(out[:3], y64[:, t], t)
        assert not out[3:].any()
    assert torch.equal(pool[[1, 2, 3]], before[[1, 2, 3]])
    _, final = ops.selective_scan(queue, softplus=True, **{k: given[k] for k in rows}, **rest)
    near(pool[slots[:3].long()], final, "state")


# ------------------------------------------------------------------------------------ norm
def norm_inputs(seed, dtype, rows, channels, gate, residual, scale):
    m = Maker(seed)
    return {"x": m.normal(rows, channels, dtype=dtype), "weight": m.uniform(0.5, 1.5, channels),
            "gate": m.normal(rows, channels, dtype=dtype) if gate else None,
            "residual": m.normal(rows, channels, dtype=dtype) if residual else None,
            "scale": m.uniform(0.2, 1.0, channels) if scale else None}, m


NORMS = [(7, 64, 1), (33, 96, 4), (5, 1000, 8), (3, 2048, 2), (9, 777, 7), (2, 4104, 1), (40, 3, 1), (3, 9000, 1),
         (0, 16, 1), (2, 1030, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, channels, groups", NORMS)
def test_norm_and_gradient(queue, ops, dtype, rows, channels, groups):
    for gate, residual, scale, after in ((0, 0, 0, 0), (1, 0, 0, 1), (0, 1, 1, 0), (1, 1, 0, 0), (1, 1, 1, 1), (0, 1, 0, 1)):
        given, m = norm_inputs(15, dtype, rows, channels, gate, residual, scale)
        same = dict(groups=groups, eps=1e-5, after=bool(after))
        out, v = ops.block_norm(queue, **given, **same)
        out64, v64 = norm_definition(**dict(zip(given, wide(*given.values()))), **same)
        near(out, out64, "out")
        assert (v is None) == (v64 is None)
        if v is not None:
            near(v, v64, "v")
        dout = m.normal(rows, channels, dtype=dtype)
        dv = m.normal(rows, channels, dtype=dtype) if v is not None else None
        got = ops.block_norm_grad(queue, dout, dv=dv, **given, **same)

        def function(x, weight, gate=None, residual=None, scale=None):
            return norm_definition(x, weight, gate, residual, scale, **same)

        want = gradients(function, given, (dout, dv))
        for k in want:
            near(getattr(got, k), want[k], (k, gate, residual, scale, after))
        if rows and channels < 1000:
            along_differences(function, given, (dout, dv), got._asdict(), 16)


@pytest.mark.gpu
def test_norm_of_rows_with_strides_and_of_zeros(queue, ops):
    given, m = norm_inputs(17, BF16, 6, 48, True, True, True)
    whole = m.normal(6, 3, 50, dtype=BF16)
    given.update(x=whole[:, 0, :48], gate=whole[:, 1, 1:49], residual=whole[:, 2, 2:50])
    out, v = ops.block_norm(queue, **given)
    out64, v64 = norm_definition(**dict(zip(given, wide(*given.values()))), groups=1, eps=1e-6, after=False)
    near(out, out64, "out")
    near(v, v64, "v")
    zeros = torch.zeros(4, 32, device="cuda")
    out, _ = ops.block_norm(queue, zeros, torch.ones(32, device="cuda"))
    assert not out.any()


# ------------------------------------------------------------- streams, graphs, bad offsets
@pytest.mark.gpu
def test_queue_on_the_programs_own_stream(queue, ops):
    from nengo_ocl_amd.hipraggedarray import Queue

    given, _, _ = scan_inputs(18, BF16, None, 4, 32, 1, 32, False, dense=(2, 300))
    want = ops.selective_scan(queue, softplus=True, **given)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.selective_scan(Queue(0, stream=stream), softplus=True, **{k: None if v is None else v * 1
                                                                            for k, v in given.items()})
        other = ops.selective_scan(queue, softplus=True, **{k: None if v is None else v * 1 for k, v in given.items()})
    stream.synchronize()
    for a in (got, other):
        assert torch.equal(a[0], want[0]) and torch.equal(a[1], want[1])


@pytest.mark.gpu
def test_recorded_steps(queue, ops):
    """A decoding step as a list of plans, recorded once and replayed, against the same calls made one by one."""
    from nengo_ocl_amd.plan import Plans

    n, h, p, s, width = 3, 2, 16, 16, 4
    m = Maker(19)
    d = h * p
    weight, bias, gain = m.normal(d, width), m.normal(d), m.uniform(0.5, 1.5, d)
    A, B, C, dt = -m.uniform(1.0, 4.0, h), m.normal(n, 1, s), m.normal(n, 1, s), m.uniform(0.1, 0.5, n, h)
    x = m.normal(n, d)
    states = [(m.normal(n, width - 1, d), m.normal(n, h, p, s))]
    states.append(tuple(v.clone() for v in states[0]))
    torch.cuda.synchronize()
    conv = ops.plan_causal_conv_step(queue, states[0][0], x, weight, bias, "silu")
    scan = ops.plan_selective_step(queue, states[0][1], conv.y.view(n, h, p), dt, A, B, C)
    norm = ops.plan_block_norm(queue, scan.y.view(n, d), gain, gate=x)
    plans = Plans([conv, scan, norm], profiling=False)
    plans.prepare()
    for steps in (1, 2, 5):
        plans.call_n_times(steps)
        for _ in range(steps):
            y = ops.causal_conv_step(queue, states[1][0], x, weight, bias, "silu")
            y = ops.selective_step(queue, states[1][1], y.view(n, h, p), dt, A, B, C)
            out, _ = ops.block_norm(queue, y.view(n, d), gain, gate=x)
        torch.cuda.synchronize()
        assert torch.equal(norm.out, out)
        assert all(torch.equal(a, b) for a, b in zip(*states))
    plans.close()


@pytest.mark.gpu
def test_offsets_beyond_the_tokens(queue, ops):
    """Offsets are cut to the tokens that there are, a sequence that ends in front of its start is empty."""
    given, _, _ = scan_inputs(20, F32, [30, 40], 2, 8, 1, 8, False)
    odd = torch.tensor([-5, 30, 20, 99], dtype=torch.int32).cuda()
    y, final = ops.selective_scan(queue, softplus=True, starts=odd, **given)
    want, ends = ops.selective_scan(queue, softplus=True, starts=starts_of([30, 0]), **given)
    assert torch.equal(y[:20], want[:20]) and torch.equal(final[0], ends[0]) and not final[1].any()
    conv, _, _ = conv_inputs(21, F32, [30, 40], 8, 3, False)
    y, _ = ops.causal_conv(queue, starts=odd, **conv)
    want, _ = ops.causal_conv(queue, starts=starts_of([30]), **conv)
    assert torch.equal(y[:20], want[:20])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,copies", [(700, 3), (9000, 5)])
def test_offsets_that_go_back(queue, ops, tokens, copies):
    """Sequences that overlap make more chunks than there are places: those that have one hold."""
    given, _, _ = scan_inputs(22, F32, [tokens], 2, 8, 1, 8, False)
    given.pop("initial", None)
    starts = torch.tensor([0, tokens] * copies, dtype=torch.int32).cuda()
    s = 2 * copies - 1
    plans = [ops.plan_selective_scan(queue, softplus=True, starts=starts, **given),
             ops.plan_selective_scan_grad(queue, given["x"], softplus=True, starts=starts, **given)]
    torch.cuda.synchronize()
    for plan in plans:
        plan()
    want, end = ops.selective_scan(queue, softplus=True, starts=starts[:2].contiguous(), **given)
    assert plans[0].final.shape[0] == s and torch.isfinite(plans[0].y[:64]).all()
    assert torch.equal(plans[0].y[:64], want[:64])
    conv, _, _ = conv_inputs(23, F32, [tokens], 8, 3, False)
    conv.pop("initial", None)
    y, _ = ops.causal_conv(queue, starts=starts, **conv)
    want, _ = ops.causal_conv(queue, starts=starts[:2].contiguous(), **conv)
    assert torch.equal(y, want)


@pytest.mark.gpu
def test_norm_of_more_parts_than_an_axis_of_a_grid_has(queue, ops):
    """2**26 + 3 rows of one channel: 64 threads each."""
    n = 2 ** 26 + 3
    x = torch.full((n, 1), 3.0, dtype=BF16, device="cuda")
    x[-1] = -3.0
    out, _ = ops.block_norm(queue, x, torch.full((1,), 2.0, device="cuda"), eps=0.0)
    assert float(out[0]) == 2.0 and float(out[-1]) == -2.0 and int((out == 2.0).sum()) == n - 1


# -------------------------------------------------------------------------------- refusals
@pytest.fixture
def host(monkeypatch):
    """A queue without a device: plans can be made, launches do nothing."""
    return host_queue(monkeypatch)


def refused(error, function, *args, **kw):
    with pytest.raises(error):
        function(*args, **kw)


def test_refusals_of_the_convolution(host, ops):
    x, w, b = torch.zeros(2, 5, 8), torch.zeros(8, 4), torch.zeros(8)
    f = ops.plan_causal_conv
    assert f(host, x, w, b).y.shape == x.shape
    refused(TypeError, f, host, x.double(), w)
    refused(TypeError, f, host, x, w.bfloat16())
    refused(ValueError, f, host, x, torch.zeros(8, 9))
    refused(ValueError, f, host, x, torch.zeros(8, 0))
    refused(ValueError, f, host, x, torch.zeros(7, 4))
    refused(ValueError, f, host, x, w, torch.zeros(7))
    refused(ValueError, f, host, x, w, activation="relu")
    refused(ValueError, f, host, x[0], w)                                      # no starts
    refused(ValueError, f, host, x, w, starts=torch.zeros(2, dtype=torch.int32))
    refused(TypeError, f, host, x[0], w, starts=torch.tensor([0, 5]))
    refused(ValueError, f, host, x, w, initial=torch.zeros(2, 4, 8))
    refused(TypeError, f, host, x.bfloat16(), w, initial=torch.zeros(2, 3, 8))
    refused(ValueError, f, host, torch.zeros(2, 8, 5).transpose(1, 2), w)      # channels apart
    refused(ValueError, f, host, x, w, y=torch.zeros(2, 5, 9))
    refused(ValueError, ops.plan_causal_conv_grad, host, x[:, :4], x, w)
    refused(TypeError, ops.plan_causal_conv_grad, host, x.half(), x, w)
    g = ops.plan_causal_conv_step
    assert g(host, torch.zeros(4, 3, 8), x[0, :4], w, b).y.shape == (4, 8)
    refused(ValueError, g, host, torch.zeros(4, 3, 8), x[0], w)                # five requests, four slots
    refused(ValueError, g, host, torch.zeros(4, 4, 8), x[0, :4], w)
    refused(TypeError, g, host, torch.zeros(4, 3, 8).half(), x[0, :4], w)
    refused(TypeError, g, host, torch.zeros(4, 3, 8), x[0, :4], w, slots=torch.zeros(4))
    refused(ValueError, g, host, torch.zeros(4, 3, 16)[:, :, :8], x[0, :4], w)  # a slot in pieces


def test_refusals_of_the_scan(host, ops):
    x, dt, A, B = torch.zeros(2, 5, 4, 8), torch.zeros(2, 5, 4), torch.zeros(4), torch.zeros(2, 5, 2, 6)
    f = ops.plan_selective_scan
    plan = f(host, x, dt, A, B, B)
    assert plan.y.shape == x.shape and plan.final.shape == (2, 4, 8, 6)
    refused(TypeError, f, host, x.double(), dt, A, B, B)
    refused(TypeError, f, host, x, dt, None, B, B)
    refused(TypeError, f, host, x, dt, A.double(), B, B)
    refused(TypeError, f, host, x, dt, A, B.half(), B)
    refused(ValueError, f, host, x, dt[:, :, :3], A, B, B)
    refused(ValueError, f, host, x, dt, A[:3], B, B)
    refused(ValueError, f, host, x, dt, A, torch.zeros(2, 5, 3, 6), torch.zeros(2, 5, 3, 6))
    refused(ValueError, f, host, x, dt, A, torch.zeros(2, 5, 2, 257), torch.zeros(2, 5, 2, 257))
    refused(ValueError, f, host, x, dt, A, B, B[:, :4])
    refused(ValueError, f, host, x, dt, A, B, B, D=torch.zeros(3))
    refused(ValueError, f, host, x, dt, A, B, B, initial=torch.zeros(1, 4, 8, 6))
    refused(ValueError, f, host, x, dt, A, B, B, final=torch.zeros(2, 4, 8, 12)[..., ::2])
    refused(ValueError, f, host, x[0], dt[0], A, B[0], B[0])
    refused(ValueError, ops.plan_selective_scan_grad, host, x[:1], x, dt, A, B, B)
    refused(TypeError, ops.plan_selective_scan_grad, host, x, x, dt, A, B, B, dfinal=torch.zeros(2, 4, 8, 6).half())
    g = ops.plan_selective_step
    state = torch.zeros(5, 4, 8, 6)
    assert g(host, state, x[0], dt[0], A, B[0], B[0]).y.shape == (5, 4, 8)
    refused(TypeError, g, host, state.half(), x[0], dt[0], A, B[0], B[0])
    refused(ValueError, g, host, state[:4], x[0], dt[0], A, B[0], B[0])
    refused(ValueError, g, host, state, x[0], dt[0], A, B[0], B[0], slots=torch.zeros(4, dtype=torch.int32))
    refused(ValueError, g, host, state.transpose(1, 2), x[0], dt[0], A, B[0], B[0])


def test_refusals_of_the_norm(host, ops):
    x, w = torch.zeros(3, 5, 12), torch.zeros(12)
    f = ops.plan_block_norm
    assert f(host, x, w).v is None and f(host, x, w, residual=x).v.shape == x.shape
    refused(TypeError, f, host, x.double(), w)
    refused(TypeError, f, host, x, None)
    refused(TypeError, f, host, x, w.half())
    refused(TypeError, f, host, x, w, gate=x.half())
    refused(ValueError, f, host, x, w, groups=5)
    refused(ValueError, f, host, x, w, groups=0)
    refused(ValueError, f, host, x, w, scale=w)                                # no residual
    refused(ValueError, f, host, x, w, residual=x[:2])
    refused(ValueError, f, host, x, w, eps=-1.0)
    refused(ValueError, f, host, x, w, residual=x, after=True, v=x)
    refused(ValueError, f, host, x.transpose(0, 1), w)                         # rows at two distances
    refused(ValueError, ops.plan_block_norm_grad, host, x, x, w, dv=x)         # no residual
    refused(ValueError, ops.plan_block_norm_grad, host, x[:2], x, w)


def test_the_library_refuses_what_python_does_not_see(ops):
    """Null pointers, sizes out of range and a workspace too small come back as codes, without a launch."""
    import ctypes

    from nengo_ocl_amd import _lib

    lib, bad, too_big = _lib.lib(), -1, -4
    args = ops._ScanArgs(n_heads=2, dim=8, n_groups=1, states=8)
    args.tokens.n_seqs, args.tokens.length, args.tokens.n_tokens = 1, 4, 4
    ref = ctypes.byref
    for entry in (lib.nhip_selective_scan, lib.nhip_selective_scan_grad):
        assert entry(None, None) == bad
        assert entry(None, ref(args)) == bad                                   # no A, no x
    for key, value in (("n_groups", 0), ("n_heads", 3), ("states", 257), ("states", 0), ("type", 7), ("dim", 0)):
        given = ops._ScanArgs.from_buffer_copy(args)
        one = 1 << 20
        given.A = given.x.p = given.dt.p = given.B.p = given.C.p = one
        need = ctypes.c_longlong(-1)
        assert lib.nhip_selective_scan_grad_workspace(ref(given), ref(need)) == 0 and need.value > 0
        given.dA = given.dD = given.ddt_bias = given.dy.p = given.dx = given.ddt = given.dB = given.dC = one
        given.workspace, given.workspace_bytes = one, need.value - 1
        assert lib.nhip_selective_scan_grad(None, ref(given)) == too_big
        given.n_groups = 2 if key == "n_heads" else 1
        setattr(given, key, value)
        assert lib.nhip_selective_scan(None, ref(given)) == bad, key
    conv = ops._ConvArgs(channels=4, width=9, weight=1 << 20)
    assert lib.nhip_causal_conv(None, ref(conv)) == bad
    norm = ops._NormArgs(channels=6, groups=4, weight=1 << 20)
    assert lib.nhip_block_norm(None, ref(norm)) == bad
