"""Float16: gradients of the gated projection whose parts between the products the type does not hold, although it holds the
result; a teacher's logits that a temperature takes beyond 32 bits.  Definitions and tolerances are those of test_tokens.py.

What stands between the products, dg and du, is stored by a power of two where its largest magnitude is beyond the type or below
2**-8: then the largest is 2**14 at least, half of the type's smallest step 2**-25 is 2**-39 of it.  Where it is stored as it
is, 2**-25 is 2**-17 of the largest at most.  So each is off by a 2**-11 of itself or by 2**-17 of the largest.
"""

import pytest
import torch

import test_tokens
from test_tokens import (E, F16, F32, U, check_loss_gradients, check_losses, gated_bounds, gated_inputs, ops,  # noqa: F401
                         teacher_inputs, wide, within)


@pytest.fixture(autouse=True)
def on_the_device(monkeypatch):
    monkeypatch.setattr(test_tokens, "PLACE", "cuda")
    yield
    torch.cuda.empty_cache()


def check_gated_gradients(got, dy, given, name):
    x, gate, up = (wide(t) for t in given.values())
    n, f = dy.shape
    a, slope, g, u, ea, es, eu = gated_bounds(x, gate, up, name)
    e = wide(dy)
    dg, du = e * u * slope, e * a
    r, tiny = U[F16], 2.0 ** -17 * float(torch.maximum(dg.abs().max(), du.abs().max()))
    og = r * dg.abs() + tiny + (1 + r) * e.abs() * (es * u.abs() + eu * slope.abs() + es * eu) + 4 * E * dg.abs()
    ou = r * du.abs() + tiny + (1 + r) * e.abs() * ea + 4 * E * du.abs()
    sg, su = dg.abs() + og, du.abs() + ou
    within(got.x, dg @ gate + du @ up,
           og @ gate.abs() + ou @ up.abs() + (2 * f + 8) * E * (sg @ gate.abs() + su @ up.abs()), "x")
    within(got.gate, dg.t() @ x, og.t() @ x.abs() + (n + 8) * E * (sg.t() @ x.abs()), "gate")
    within(got.up, du.t() @ x, ou.t() @ x.abs() + (n + 8) * E * (su.t() @ x.abs()), "up")
    return dg, du


# small tiles; rows of weights that are copied; matrices read as they lie, k in parts; two pieces of the features
SIZES = [(1, 64, 80), (50, 64, 80), (130, 70, 129), (300, 520, 4601), (8300, 136, 20001)]


@pytest.mark.gpu
@pytest.mark.parametrize("n, d, f", SIZES)
@pytest.mark.parametrize("name", ["silu", "gelu"])
@pytest.mark.parametrize("where", ["first", "last"])
def test_gated_gradient_beyond_float16(queue, ops, n, d, f, name, where):  # noqa: F811
    """A row and a feature whose activation is 38 (in exact numbers), and a gradient of 2000 there: 76000 between the products."""
    given, m = gated_inputs(81, F16, n, d, f)
    row, feature = (0, 5) if where == "first" else (n - 1, f - 1)
    sign = torch.where(torch.arange(d, device="cuda") % 3 == 0, 1.0, -1.0)
    given["gate"][feature] = (608.0 / d * sign).half()
    given["x"][row] = (sign * 0.0625).half()
    dy = m.normal(n, f, dtype=F16)
    dy[row, feature] = 2000.0
    got = ops.gated_projection_grad(queue, dy, activation=name, **given)
    dg, du = check_gated_gradients(got, dy, given, name)
    assert float(du.abs().max()) > 70000.0
    assert all(float(wide(t).abs().max()) < 60000.0 for t in got)


@pytest.mark.gpu
@pytest.mark.parametrize("n, d, f", SIZES)
@pytest.mark.parametrize("scale", [2.0 ** -20, 2.0 ** -14, 2.0 ** -8, 1.0, 2.0 ** 6])
def test_gated_gradient_of_any_magnitude(queue, ops, n, d, f, scale):  # noqa: F811
    """Gradients down to the type's smallest numbers: the weights', sums over many rows, are large again."""
    given, m = gated_inputs(82, F16, n, d, f)
    dy = (m.normal(n, f) * scale).half()
    got = ops.gated_projection_grad(queue, dy, **given)
    check_gated_gradients(got, dy, given, "silu")


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_gated_gradient_of_what_is_no_number(queue, ops, bad):  # noqa: F811
    """It stays in its row of x's gradient, and does not take part in the largest."""
    given, m = gated_inputs(83, F16, 40, 64, 80)
    for scale in (2.0 ** -12, 1.0):
        dy = (m.normal(40, 80) * scale).half()
        clean = ops.gated_projection_grad(queue, dy, **given)
        dy[7, 3] = bad
        got = ops.gated_projection_grad(queue, dy, **given)
        others = torch.arange(40, device="cuda") != 7
        assert not torch.isfinite(got.x[7]).any() and torch.isfinite(got.x[others]).all()
        # (the row's own elements were among those that the scale came from)
        assert (wide(got.x[others]) - wide(clean.x[others])).abs().max() <= 2 * U[F16] * wide(clean.x).abs().max()


@pytest.mark.gpu
def test_gated_gradient_recorded(queue, ops):  # noqa: F811
    """A replay decides by its own inputs whether they are formed once more."""
    from nengo_ocl_amd.plan import Plans

    given, m = gated_inputs(84, F16, 70, 64, 80)
    dy = m.normal(70, 80, dtype=F16)
    plan = ops.plan_gated_projection_grad(queue, dy, **given)
    group = Plans([plan], False)
    for scale in (1.0, 2.0 ** -13, 3000.0, 1.0, 2.0 ** -13):
        dy.copy_((m.normal(70, 80).clamp(-3.0, 3.0) * scale).half())
        torch.cuda.synchronize()
        group.enqueue_n_times(2)
        queue.finish()
        got = [t.clone() for t in plan.gradients]
        torch.zeros(1 << 20, device="cuda").sum().item()
        want = ops.gated_projection_grad(queue, dy, **given)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        if scale <= 1.0:
            check_gated_gradients(plan.gradients, dy, given, "silu")


@pytest.mark.gpu
@pytest.mark.parametrize("n, top", [(6, 9), (70, 40), (300, 200)])
@pytest.mark.parametrize("dtype", [F32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [0.1, 0.5, 1.0, 4.0])
def test_teacher_logits_beyond_32_bits_over_a_temperature(queue, ops, n, top, dtype, temperature):  # noqa: F811
    """A type's lowest value is a value at any temperature: in a row of them, and beside others; only -inf is left out."""
    given, m = teacher_inputs(85, F32, n, 40, 500, 0.0, top)
    low = torch.finfo(dtype).min
    logits = given["logits"].to(dtype)
    logits[0] = low
    logits[1, ::2] = low
    logits[2] = -2e38
    logits[3, 0], logits[3, 1:] = low, float("-inf")
    logits[4] = 2e38
    logits[5] = float("-inf")
    given["logits"] = logits
    loss, lse = ops.teacher_loss(queue, temperature=temperature, **given)
    check_losses(loss, lse, given, temperature)
    assert loss[:5].all() and not loss[5]
    dloss = (torch.rand(n, generator=m.gen) / n).cuda()
    check_loss_gradients(ops.teacher_loss_grad(queue, dloss, lse=lse, temperature=temperature, **given), given, temperature, dloss, lse)
