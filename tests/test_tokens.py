"""Layer norm, gated projection, and the losses over a vocabulary against their definitions in 64 bits, and what their
entry points refuse.

Tolerances, element by element.  u = 2**-24, 2**-8, 2**-11: half a step of float32, bfloat16, float16.  A sum of K terms
in 32 bits is off by at most (K + 8) 2**-24 of the sum of their magnitudes (`sums`); a result is rounded once more, u
of itself.  The gradients of products sum products of what stands between, G: G is off by u of itself
(its rounding), and by what the error of the logits makes of it.  Where all is 32 bits the worst case of such sums is
far from what random signs give: there the norm of the error is 128 u of the result's, too.
"""

import math

import pytest
import torch

from helpers import host_queue

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
E = 2.0 ** -24
TINY = {F32: 1e-37, BF16: 1e-37, F16: 2.0 ** -24}  # a step of the type's smallest numbers


@pytest.fixture(scope="module")
def ops():
    from nengo_ocl_amd import hipra_tokens

    return hipra_tokens


@pytest.fixture
def host(monkeypatch):
    return host_queue(monkeypatch)


PLACE = "cpu"  # where the definitions are computed


def wide(t):
    return None if t is None else t.detach().to(PLACE).double()


def within(got, want, bound, name="", apart=0.0):
    """|got - want| <= bound + the rounding of the result, element by element; in 32 bits the norm, too: 128 u of the result's,
    and `apart` where the result is a difference of what is larger."""
    got64, want = wide(got), wide(want)
    assert got64.shape == want.shape, (name, got64.shape, want.shape)
    if not want.numel():
        return
    assert torch.isfinite(got64).all(), name
    off = (got64 - want).abs()
    most = bound + U[got.dtype] * want.abs() + TINY[got.dtype]
    worst = float((off / most).max())
    assert worst <= 1.0, (name, worst)
    if got.dtype == F32:
        assert off.norm() <= 128 * E * want.norm() + apart + 1e-30, (name, float(off.norm() / want.norm()))


class Maker:
    def __init__(self, seed):
        self.gen = torch.Generator().manual_seed(seed)

    def normal(self, *shape, dtype=F32, scale=1.0):
        return (torch.randn(*shape, generator=self.gen) * scale).to(dtype).cuda()

    def whole(self, high, *shape):
        return torch.randint(high, shape, generator=self.gen)


# -------------------------------------------------------------------------------- layer norm
def norm_definition(x, weight, bias, residual, eps):
    v = x if residual is None else residual + x
    off = v - v.mean(-1, keepdim=True)
    u = off / torch.sqrt((off ** 2).mean(-1, keepdim=True) + eps)
    out = u * weight
    return out if bias is None else out + bias, v


def norm_inputs(seed, dtype, lead, d, with_bias, with_residual):
    m = Maker(seed)
    return {"x": m.normal(*lead, d, dtype=dtype) + 0.5, "weight": m.normal(d), "bias": m.normal(d) if with_bias else None,
            "residual": m.normal(*lead, d, dtype=dtype, scale=3.0) if with_residual else None}, m


def norm_bounds(given, eps):
    """How far the normed values may be off: the mean and the deviation of a row are sums over it, d + 8 roundings each."""
    x, w, b, r = (wide(given[k]) for k in ("x", "weight", "bias", "residual"))
    v = x if r is None else x + r
    d = v.shape[-1]
    inv = 1 / torch.sqrt(v.var(-1, unbiased=False, keepdim=True) + eps)
    size = v.abs().amax(-1, keepdim=True) * inv + (v - v.mean(-1, keepdim=True)).abs() * inv + 1
    return (d + 16) * E * size, inv


NORMS = [((5,), 7), ((3, 4), 64), ((1,), 1), ((33,), 130), ((2, 3), 2048), ((9,), 1023), ((4,), 5000), ((2,), 8192 + 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lead, d", NORMS)
def test_layer_norm(queue, ops, dtype, lead, d):
    for with_bias, with_residual in ((True, True), (False, False), (True, False)):
        given, _ = norm_inputs(1, dtype, lead, d, with_bias, with_residual)
        out, v = ops.layer_norm(queue, eps=1e-5, **given)
        want, v64 = norm_definition(*(wide(given[k]) for k in ("x", "weight", "bias", "residual")), 1e-5)
        off, _ = norm_bounds(given, 1e-5)
        w = wide(given["weight"]).abs()
        within(out, want, off * w + 4 * E * (want.abs() + w), "out")
        assert (v is None) == (not with_residual)
        if v is not None:
            within(v, v64, 2 * E * v64.abs(), "v")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lead, d", NORMS + [((1000,), 96), ((2500,), 520)])
def test_layer_norm_gradient(queue, ops, dtype, lead, d):
    for with_bias, with_residual in ((True, True), (False, False)):
        given, m = norm_inputs(2, dtype, lead, d, with_bias, with_residual)
        dout = m.normal(*lead, d, dtype=dtype)
        dv = m.normal(*lead, d, dtype=dtype) if with_residual else None
        got = ops.layer_norm_grad(queue, dout, dv=dv, **given)
        leaves = {k: wide(t).requires_grad_() for k, t in given.items() if t is not None}
        out, v = norm_definition(*(leaves.get(k) for k in ("x", "weight", "bias", "residual")), 1e-5)
        outputs, grads = [out], [wide(dout)]
        if with_residual:
            outputs, grads = outputs + [v], grads + [wide(dv)]
        want = dict(zip(leaves, torch.autograd.grad(outputs, list(leaves.values()), grads)))
        off, inv = norm_bounds(given, 1e-5)
        n = len(want["x"].reshape(-1, d))
        e, w = wide(dout).abs(), wide(given["weight"]).abs()
        u = (norm_definition(*(wide(given[k]) for k in ("x", "weight", "bias", "residual")), 1e-5)[1])
        u = ((u - u.mean(-1, keepdim=True)) * inv).abs()
        ew = (e * w)
        size = ew + ew.mean(-1, keepdim=True) + (u + off) * (ew * (u + 1)).mean(-1, keepdim=True)
        slack = (d + 32) * E * size + 3 * off * (ew.mean(-1, keepdim=True) + (ew * u).mean(-1, keepdim=True))
        within(got.x, want["x"], slack * inv * (1 + u) + 4 * E * (0 if dv is None else wide(dv).abs()), "x")
        rows = lambda t: t.reshape(-1, d).sum(0)
        within(got.weight, want["weight"], (n + 8) * E * rows(e * (u + off)) + rows(e * off), "weight")
        if with_bias:
            within(got.bias, want["bias"], (n + 8) * E * rows(e), "bias")
        else:
            assert got.bias is None
        assert got.residual is (got.x if with_residual else None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_of_a_mean_far_from_zero(queue, ops, dtype):
    """The squares are those of what the mean leaves: 1000 above a deviation of one."""
    x = (Maker(3).normal(4, 600) + 1000.0).to(dtype)
    w = torch.ones(600, device="cuda")
    out, _ = ops.layer_norm(queue, x, w)
    want, _ = norm_definition(wide(x), wide(w), None, None, 1e-5)
    off, _ = norm_bounds({"x": x, "weight": w, "bias": None, "residual": None}, 1e-5)
    got = wide(out)
    assert ((got - want).abs() <= off + U[dtype] * want.abs() + 1e-30).all()


# -------------------------------------------------------------------------- gated projection
def act(name, g):
    # (erfc(-t) for 1 + erf(t), the same value: the sum loses its digits where g is far below zero, 2**-53 of 1e-12 at -7)
    return g * torch.sigmoid(g) if name == "silu" else 0.5 * g * torch.special.erfc(g * -math.sqrt(0.5))


GATED = [(1, 64, 64, "silu"), (3, 40, 33, "gelu"), (17, 130, 70, "silu"), (64, 256, 200, "gelu"), (65, 128, 300, "silu"),
         (130, 72, 129, "silu"), (300, 65, 131, "gelu"), (257, 192, 8192 + 4, "silu"), (1, 1, 1, "gelu")]


def gated_inputs(seed, dtype, n, d, f):
    m = Maker(seed)
    return {"x": m.normal(n, d, dtype=dtype), "gate": m.normal(f, d, dtype=dtype, scale=d ** -0.5),
            "up": m.normal(f, d, dtype=dtype, scale=d ** -0.5)}, m


def gated_bounds(x, gate, up, name):
    """(act, its slope, g, u and how far each may be off): |act'| and |act''| are below 1.2 and 1 for both."""
    d = x.shape[1]
    g, u = x @ gate.t(), x @ up.t()
    eg, eu = ((d + 8) * E * (x.abs() @ w.abs().t()) for w in (gate, up))
    leaf = g.clone().requires_grad_()
    f = act(name, leaf)
    slope, = torch.autograd.grad(f.sum(), leaf)
    return f.detach(), slope, g, u, 1.2 * eg + 32 * E * (1 + g.abs()), eg + 32 * E * (1 + g.abs()), eu


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n, d, f, name", GATED)
def test_gated_projection(queue, ops, dtype, n, d, f, name):
    given, _ = gated_inputs(4, dtype, n, d, f)
    y = ops.gated_projection(queue, activation=name, **given)
    a, _, g, u, ea, _, eu = gated_bounds(*(wide(t) for t in given.values()), name)
    within(y, a * u, ea * u.abs() + eu * a.abs() + ea * eu, "y")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n, d, f, name", GATED)
def test_gated_projection_gradient(queue, ops, dtype, n, d, f, name):
    given, m = gated_inputs(5, dtype, n, d, f)
    dy = m.normal(n, f, dtype=dtype)
    got = ops.gated_projection_grad(queue, dy, activation=name, **given)
    x, gate, up = (wide(t) for t in given.values())
    a, slope, g, u, ea, es, eu = gated_bounds(x, gate, up, name)
    e = wide(dy)
    dg, du = e * u * slope, e * a
    # what the rounding to the inputs' type (u of it), and the errors of g and u, make of both
    r = 0.0 if dtype == F32 else U[dtype]
    tiny = TINY[dtype]
    og = r * dg.abs() + tiny + (1 + r) * e.abs() * (es * u.abs() + eu * slope.abs() + es * eu) + 4 * E * dg.abs()
    ou = r * du.abs() + tiny + (1 + r) * e.abs() * ea + 4 * E * du.abs()
    sg, su = dg.abs() + og, du.abs() + ou
    within(got.x, dg @ gate + du @ up,
           og @ gate.abs() + ou @ up.abs() + (2 * f + 8) * E * (sg @ gate.abs() + su @ up.abs()), "x")
    within(got.gate, dg.t() @ x, og.t() @ x.abs() + (n + 8) * E * (sg.t() @ x.abs()), "gate")
    within(got.up, du.t() @ x, ou.t() @ x.abs() + (n + 8) * E * (su.t() @ x.abs()), "up")


# ----------------------------------------------------------------------- losses over a vocabulary
LOSSES = [(1, 64, 50, 0.0), (5, 33, 7, 0.4), (16, 128, 300, 0.0), (40, 200, 1000, 0.3), (70, 72, 257, 0.5), (200, 96, 513, 0.1),
          (300, 130, 300, 0.6), (520, 64, 9000, 0.2), (3, 1, 1, 0.0)]


def loss_inputs(seed, dtype, n, d, v, masked):
    m = Maker(seed)
    labels = m.whole(v, n)
    labels[torch.rand(n, generator=m.gen) < masked] = -100
    return {"x": m.normal(n, d, dtype=dtype), "weight": m.normal(v, d, dtype=dtype, scale=2.0 * d ** -0.5),
            "labels": labels.cuda()}, m


def teacher_inputs(seed, dtype, n, d, v, masked, top):
    given, m = loss_inputs(seed, dtype, n, d, v, 0.0)
    given.pop("labels")
    k = min(top, v)
    words = torch.stack([torch.randperm(v, generator=m.gen)[:k] for _ in range(n)]).int()
    words[torch.rand(n, k, generator=m.gen) < masked / 2] = -1
    words[torch.rand(n, generator=m.gen) < masked] = v
    return dict(given, indices=words.cuda(), logits=m.normal(n, k, scale=2.0, dtype=dtype)), m


def shares(given, temperature):
    """[n, words] shares of the targets, sum q log q, which rows count."""
    n, v = given["x"].shape[0], given["weight"].shape[0]
    q = torch.zeros(n, v, dtype=torch.float64, device=PLACE)
    if "labels" in given:
        words, logits = given["labels"].to(PLACE).long()[:, None], torch.zeros(n, 1, dtype=torch.float64, device=PLACE)
    else:
        words, logits = given["indices"].to(PLACE).long(), wide(given["logits"]) / temperature
    ok = (words >= 0) & (words < v) & (logits > -math.inf)
    counts = ok.any(1)
    p = torch.softmax(torch.where(ok, logits, -math.inf), 1)
    p = torch.where(ok, p, 0.0)  # (of a row without any, too)
    q.scatter_add_(1, words.clamp(0, v - 1), p)
    return q, torch.special.xlogy(p, p).sum(1), counts


def loss_definition(given, temperature):
    """(loss, lse, p, q, how far z may be off, which rows count)"""
    x, w = wide(given["x"]), wide(given["weight"])
    q, self, counts = shares(given, temperature)
    z = x @ w.t() / temperature
    lse = torch.logsumexp(z, -1)
    loss = self + lse * q.sum(1) - (q * z).sum(1)
    ez = (x.shape[1] + 16) * E * (x.abs() @ w.abs().t()) / temperature + 4 * E * z.abs()
    return torch.where(counts, loss, 0.0), torch.where(counts, lse, 0.0), torch.exp(z - lse[:, None]), q, ez, z, counts


def check_losses(loss, lse, given, temperature):
    want, lse64, p, q, ez, z, counts = loss_definition(given, temperature)
    # the logarithm of the sum is off by what its terms are, weighted by their shares, and by its own roundings
    e_lse = (p * ez).sum(1) + (16 + 2 * math.ceil(p.shape[1] ** 0.5)) * E * (1 + lse64.abs()) + 4 * E * z.abs().amax(1)
    e_loss = e_lse + (q * ez).sum(1) + 64 * E * (1 + (q * z.abs()).sum(1) + lse64.abs() + (8 if q.shape[1] > 1 else 0))
    for got, exact, most in ((lse, lse64, e_lse), (loss, want, e_loss)):
        off = (wide(got) - exact).abs()
        assert torch.isfinite(off).all() and (off <= most).all(), float((off / most).max())
        assert not wide(got)[~counts].any()
    return want, lse64


def check_loss_gradients(got, given, temperature, dloss, lse):
    """G, its error and the products' as the module's docstring says; `lse` may be off by what the forward pass leaves."""
    _, lse64, p, q, ez, z, counts = loss_definition(given, temperature)
    dtype = given["x"].dtype
    x, w = wide(given["x"]), wide(given["weight"])
    x = torch.where(counts[:, None], x, 0.0)
    scale = torch.where(counts, wide(dloss) / temperature, 0.0)[:, None]
    G = (p - q) * scale
    e_lse = torch.where(counts, (wide(lse) - lse64).abs(), 0.0)[:, None]
    r = 0.0 if dtype == F32 else U[dtype]
    # (float16: G is scaled to 2**13, its smallest step 2**-24 is 2**-37 of the largest)
    tiny = float(scale.abs().max()) * 2.0 ** -37 if dtype == F16 else 1e-37
    off = r * G.abs() + tiny + scale.abs() * (p * (ez + e_lse + 16 * E * (1 + z.abs() + lse64.abs()[:, None])) + 8 * E * q)
    size = G.abs() + off
    n, v = G.shape
    # p and q are each off by some roundings of themselves, 8 E, also where their difference is smaller (a vocabulary of one
    # word: p = q = 1, G = 0 and off by 8 E scale); and exp(z - lse) by those of z and lse, numbers of 32 bits whose
    # own steps are E of them (2000: 1e-4, and p as much of itself).  The products carry that on.
    both = 8 * E * scale.abs() * (p * (1 + z.abs() + lse64.abs()[:, None]) + q)
    within(got.x, G @ w, off @ w.abs() + (v + 8) * E * (size @ w.abs()), "x", (both @ w.abs()).norm())
    within(got.weight, G.t() @ x, off.t() @ x.abs() + (n + 8) * E * (size.t() @ x.abs()), "weight", (both.t() @ x.abs()).norm())
    return G


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n, d, v, masked", LOSSES)
def test_vocabulary_loss_and_gradient(queue, ops, dtype, n, d, v, masked):
    given, m = loss_inputs(6, dtype, n, d, v, masked)
    for kind in (torch.int64, torch.int32):
        given["labels"] = given["labels"].to(kind)
        loss, lse = ops.vocabulary_loss(queue, **given)
        check_losses(loss, lse, given, 1.0)
    dloss = (torch.rand(n, generator=m.gen) / n).cuda()
    got = ops.vocabulary_loss_grad(queue, dloss, lse=lse, **given)
    check_loss_gradients(got, given, 1.0, dloss, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n, d, v, masked", LOSSES)
@pytest.mark.parametrize("top, temperature", [(1, 1.0), (5, 2.0), (70, 0.5), (200, 4.0)])
def test_teacher_loss_and_gradient(queue, ops, dtype, n, d, v, masked, top, temperature):
    given, m = teacher_inputs(7, dtype, n, d, v, masked, top)
    loss, lse = ops.teacher_loss(queue, temperature=temperature, **given)
    check_losses(loss, lse, given, temperature)
    dloss = (torch.rand(n, generator=m.gen) / n).cuda()
    got = ops.teacher_loss_grad(queue, dloss, lse=lse, temperature=temperature, **given)
    check_loss_gradients(got, given, temperature, dloss, lse)
