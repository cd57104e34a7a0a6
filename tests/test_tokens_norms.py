"""How far results of 16 bits are off as a whole: the norm of the error, which the bounds of test_tokens.py, element by element and
for the worst signs, leave open by far.

u is half a step of a type at one.  A value of binade 2**e is rounded by an error that is evenly spread over +- u 2**e, its mean
square u**2 4**e / 3.  Values that are sums of many terms are spread like a normal distribution, of which the mean of
4**floor(log2|v|) is 0.54 of the mean square: one rounding is off by 0.42 u of the norm.  The gradients of products have two,
each independent of the other: that of the result, and that of what stands between the products, whose errors add up like
its values: 0.42 sqrt(2) = 0.60 u.  The sums in 32 bits are off by 2**-24 times the root of their length, below 0.03 u.  So
the norm of the error is 0.5 u and 0.75 u at most of the result's: a fifth more than expected, of thousands of roundings.
Values that are cut instead of rounded are off by twice as much, 0.85 u, and all to the same side.
"""

import pytest
import torch

import test_tokens
from test_tokens import (BF16, F16, U, Maker, act, gated_inputs, loss_inputs, norm_definition, norm_inputs, ops,  # noqa: F401
                         shares, teacher_inputs, wide)

ONCE, TWICE = 0.5, 0.75


@pytest.fixture(autouse=True)
def where_there_is_a_device(monkeypatch):
    if torch.cuda.is_available():
        monkeypatch.setattr(test_tokens, "PLACE", "cuda")
    yield
    if torch.cuda.is_available():
        torch.cuda.empty_cache()


def norm_is(got, want, roundings, name=""):
    off = float((wide(got) - want).norm() / want.norm()) / U[got.dtype]
    assert off <= roundings, (name, off)


# ------------------------------------------------------------------------------------ definitions
def gated_gradients(x, gate, up, dy, name, between=lambda t: t):
    """(x, gate, up) in 64 bits; `between` is what becomes of dg and du."""
    g, u = x @ gate.t(), x @ up.t()
    leaf = g.clone().requires_grad_()
    f = act(name, leaf)
    slope, = torch.autograd.grad(f.sum(), leaf)
    dg, du = between(dy * u * slope), between(dy * f.detach())
    return dg @ gate + du @ up, dg.t() @ x, du.t() @ x


def loss_gradients(given, temperature, dloss, between=lambda t: t):
    x, w = wide(given["x"]), wide(given["weight"])
    q, _, counts = shares(given, temperature)
    G = torch.softmax(x @ w.t() / temperature, -1).sub_(q)
    G *= torch.where(counts, wide(dloss) / temperature, 0.0)[:, None]
    G = between(G)
    return G @ w, G.t() @ torch.where(counts[:, None], x, 0.0)


# ------------------------------------------------------------------------- what the bound can tell
def cut(t, bits):
    """Numbers of `bits` bits, what lies behind cut off."""
    m, e = torch.frexp(t)
    return torch.ldexp(torch.trunc(torch.ldexp(m, torch.tensor(bits))), e - bits)


def host_cases():
    """Every gradient as (its exact results, its results with `between` in the middle)."""
    gen = torch.Generator().manual_seed(91)
    normal = lambda *shape, scale=1.0: (torch.randn(*shape, generator=gen) * scale).to(BF16).double()
    x, gate, up, dy = normal(1000, 64), normal(200, 64, scale=0.125), normal(200, 64, scale=0.125), normal(1000, 200)
    yield lambda between: gated_gradients(x, gate, up, dy, "silu", between)
    labels = torch.randint(-50, 500, (1000,), generator=gen)
    given = {"x": x, "weight": normal(500, 64, scale=0.25), "labels": labels}
    dloss = torch.rand(1000, generator=gen)
    yield lambda between: loss_gradients(given, 1.0, dloss, between)


@pytest.mark.parametrize("case", [0, 1])
def test_the_bound_tells_mistakes_from_roundings(monkeypatch, case):
    """What the kernels' results should be passes; G cut instead of rounded, of fewer bits, and results that are a little
    too large do not.  (Planted in the definition, on the host.)"""
    monkeypatch.setattr(test_tokens, "PLACE", "cpu")
    made = list(host_cases())[case]
    want = made(lambda t: t)

    def off(between, scale=1.0):
        return [float(((t * scale).to(BF16).double() - w).norm() / w.norm()) / U[BF16] for t, w in zip(made(between), want)]

    rounded = lambda t: t.to(BF16).double()
    assert max(off(rounded)) <= TWICE and max(off(lambda t: t)) <= ONCE
    assert min(off(lambda t: cut(t, 8))) > TWICE                     # as many bits, but cut
    assert min(off(lambda t: cut(t, 6))) > 2 * TWICE
    for scale in (1.02, 0.98, 1.005):
        assert min(off(rounded, scale)) > TWICE


# ------------------------------------------------------------------------------------- the kernels
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lead, d", [(2000, 130), (500, 2048), (100, 8192), (300, 1023)])
def test_layer_norm(queue, ops, dtype, lead, d):  # noqa: F811
    given, m = norm_inputs(92, dtype, (lead,), d, True, True)
    dout = m.normal(lead, d, dtype=dtype)
    out, v = ops.layer_norm(queue, **given)
    got = ops.layer_norm_grad(queue, dout, dv=dout, **given)
    leaves = {k: wide(t).requires_grad_() for k, t in given.items()}
    want, v64 = norm_definition(*(leaves[k] for k in ("x", "weight", "bias", "residual")), 1e-5)
    dx, = torch.autograd.grad([want, v64], [leaves["x"]], [wide(dout)] * 2)
    for name, a, b in (("out", out, want.detach()), ("v", v, v64.detach()), ("x", got.x, dx)):
        norm_is(a, b, ONCE, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n, d, f, name", [
    (300, 520, 4601, "silu"), (300, 523, 4601, "gelu"), (3100, 1032, 7201, "silu"), (8300, 136, 20001, "gelu"),
    (4000, 264, 130, "silu"), (1000, 1024, 1024, "silu"), (40, 264, 3000, "gelu"), (200, 8192, 2100, "silu")])
def test_gated_projection(queue, ops, dtype, n, d, f, name):  # noqa: F811
    given, m = gated_inputs(93, dtype, n, d, f)
    dy = m.normal(n, f, dtype=dtype)
    x, gate, up = (wide(t) for t in given.values())
    norm_is(ops.gated_projection(queue, activation=name, **given), act(name, x @ gate.t()) * (x @ up.t()), ONCE, "y")
    got = ops.gated_projection_grad(queue, dy, activation=name, **given)
    for key, a, b in zip(("x", "gate", "up"), got, gated_gradients(x, gate, up, wide(dy), name)):
        norm_is(a, b, TWICE, key)


LOSSES = [(300, 520, 9001, 0.3), (261, 523, 9001, 0.0), (3100, 1032, 14500, 0.1), (8300, 136, 40000, 0.2), (5000, 200, 600, 0.0),
          (1500, 64, 300, 0.5), (300, 8192, 3001, 0.1), (300, 1040, 130001, 0.1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n, d, v, masked", LOSSES)
@pytest.mark.parametrize("top", [0, 70])
def test_losses(queue, ops, dtype, n, d, v, masked, top):  # noqa: F811
    if top:
        given, m = teacher_inputs(95, dtype, n, d, v, masked, top)
        temperature, kept = 2.0, {"temperature": 2.0}
        forward, backward = ops.teacher_loss, ops.teacher_loss_grad
    else:
        given, m = loss_inputs(94, dtype, n, d, v, masked)
        temperature, kept = 1.0, {}
        forward, backward = ops.vocabulary_loss, ops.vocabulary_loss_grad
    _, lse = forward(queue, **given, **kept)
    dloss = (torch.rand(n, generator=m.gen) + 0.5).cuda()
    got = backward(queue, dloss, lse=lse, **given, **kept)
    for key, a, b in zip(("x", "weight"), got, loss_gradients(given, temperature, dloss)):
        norm_is(a, b, TWICE, key)
