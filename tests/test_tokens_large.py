"""Products of many tiles: matrices that are read as they lie, rows that are copied because they begin at odd places, k in parts,
last rounds that are not full, several pieces.  Definitions and tolerances are those of test_tokens.py, computed on the device.
"""

import pytest
import torch

import test_tokens
from test_tokens import (BF16, E, F16, F32, TINY, U, Maker, act, check_loss_gradients, check_losses, gated_bounds,  # noqa: F401
                         gated_inputs, loss_inputs, ops, teacher_inputs, wide, within)


@pytest.fixture(autouse=True)
def on_the_device(monkeypatch):
    monkeypatch.setattr(test_tokens, "PLACE", "cuda")
    yield
    torch.cuda.empty_cache()


LOSSES = [
    (BF16, 300, 520, 9001, 0.3),    # G, x and W read as they lie; k of dx in parts
    (F16, 261, 523, 9001, 0.0),     # rows of W at odd places: copied first
    (BF16, 3100, 1032, 14500, 0.1),  # the last round of dW's tiles in parts
    (BF16, 8300, 136, 40000, 0.2),  # two pieces of the vocabulary
    (F32, 5000, 64, 9000, 0.5),     # large tiles of 32 bits
    (BF16, 5000, 200, 600, 0.0),    # few words: k of dW in parts
    (F32, 3000, 40, 70, 0.1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, n, d, v, masked", LOSSES)
def test_vocabulary_loss(queue, ops, dtype, n, d, v, masked):  # noqa: F811
    given, m = loss_inputs(21, dtype, n, d, v, masked)
    loss, lse = ops.vocabulary_loss(queue, **given)
    check_losses(loss, lse, given, 1.0)
    dloss = (torch.rand(n, generator=m.gen) / n).cuda()
    got = ops.vocabulary_loss_grad(queue, dloss, lse=lse, **given)
    check_loss_gradients(got, given, 1.0, dloss, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, n, d, v, masked", [LOSSES[0], LOSSES[2], LOSSES[4]])
@pytest.mark.parametrize("top, temperature", [(70, 2.0), (256, 1.0)])
def test_teacher_loss(queue, ops, dtype, n, d, v, masked, top, temperature):  # noqa: F811
    given, m = teacher_inputs(22, dtype, n, d, v, masked, top)
    given["indices"][:, ::3] %= 500  # many in the same tiles, some of them twice
    loss, lse = ops.teacher_loss(queue, temperature=temperature, **given)
    check_losses(loss, lse, given, temperature)
    dloss = (torch.rand(n, generator=m.gen) / n).cuda()
    got = ops.teacher_loss_grad(queue, dloss, lse=lse, temperature=temperature, **given)
    check_loss_gradients(got, given, temperature, dloss, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, n, d, f, name", [
    (BF16, 300, 520, 4601, "silu"), (F16, 300, 523, 4601, "gelu"), (BF16, 3100, 1032, 7201, "silu"), (BF16, 8300, 136, 20001, "gelu"),
    (F32, 2100, 70, 9000, "silu"), (BF16, 4000, 264, 130, "silu"), (BF16, 1000, 1024, 1024, "silu")])
def test_gated_projection(queue, ops, dtype, n, d, f, name):  # noqa: F811
    given, m = gated_inputs(23, dtype, n, d, f)
    x, gate, up = (wide(t) for t in given.values())
    a, slope, g, u, ea, es, eu = gated_bounds(x, gate, up, name)
    y = ops.gated_projection(queue, activation=name, **given)
    within(y, a * u, ea * u.abs() + eu * a.abs() + ea * eu, "y")
    dy = m.normal(n, f, dtype=dtype)
    got = ops.gated_projection_grad(queue, dy, activation=name, **given)
    e = wide(dy)
    dg, du = e * u * slope, e * a
    r = 0.0 if dtype == F32 else U[dtype]
    og = r * dg.abs() + TINY[dtype] + (1 + r) * e.abs() * (es * u.abs() + eu * slope.abs() + es * eu) + 4 * E * dg.abs()
    ou = r * du.abs() + TINY[dtype] + (1 + r) * e.abs() * ea + 4 * E * du.abs()
    sg, su = dg.abs() + og, du.abs() + ou
    within(got.x, dg @ gate + du @ up,
           og @ gate.abs() + ou @ up.abs() + (2 * f + 8) * E * (sg @ gate.abs() + su @ up.abs()), "x")
    within(got.gate, dg.t() @ x, og.t() @ x.abs() + (n + 8) * E * (sg.t() @ x.abs()), "gate")
    within(got.up, du.t() @ x, ou.t() @ x.abs() + (n + 8) * E * (su.t() @ x.abs()), "up")


@pytest.mark.gpu
@pytest.mark.parametrize("n", [8193, 65537, 70001])
def test_many_tokens_of_which_some_count(queue, ops, n):  # noqa: F811
    """Tokens are brought together in groups of 64 and of 1024."""
    given, m = loss_inputs(24, BF16, n, 8, 40, 0.4)
    loss, lse = ops.vocabulary_loss(queue, **given)
    check_losses(loss, lse, given, 1.0)
    dloss = (torch.rand(n, generator=m.gen) / n).cuda()
    check_loss_gradients(ops.vocabulary_loss_grad(queue, dloss, lse=lse, **given), given, 1.0, dloss, lse)
    given, m = teacher_inputs(25, BF16, n, 8, 40, 0.4, 3)
    loss, lse = ops.teacher_loss(queue, **given)
    check_losses(loss, lse, given, 1.0)
    check_loss_gradients(ops.teacher_loss_grad(queue, dloss, lse=lse, **given), given, 1.0, dloss, lse)


@pytest.mark.gpu
def test_offsets_behind_32_bits(queue, ops):  # noqa: F811
    """Rows of x and of weights that lie more than 2**31 elements behind the first: the same as where they are near."""
    n, d, v = 5, 64, 300
    room = torch.empty(n, 1 << 30, device="cuda", dtype=BF16)  # the last row 2**32 elements behind the first
    given, m = loss_inputs(26, BF16, n, d, v, 0.0)
    x, weight = room[:, :d], room[:, d:2 * d]
    x.copy_(given["x"])
    want = ops.vocabulary_loss(queue, **given)
    got = ops.vocabulary_loss(queue, x, given["weight"], given["labels"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    dloss = torch.rand(n, generator=m.gen).cuda()
    a, b = (ops.vocabulary_loss_grad(queue, dloss, t, given["weight"], given["labels"], want[1]) for t in (x, given["x"]))
    assert torch.equal(a.x, b.x) and torch.equal(a.weight, b.weight)
    near, words = given["weight"][:n].contiguous(), given["labels"] % n
    weight.copy_(near)
    for t in (given["x"], x):
        got, want = (ops.vocabulary_loss(queue, t, w, words) for w in (weight, near))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(ops.gated_projection(queue, t, weight, weight), ops.gated_projection(queue, t, near, near))
        gain = torch.ones(d, device="cuda")
        assert torch.equal(ops.layer_norm(queue, t, gain)[0], ops.layer_norm(queue, given["x"], gain)[0])
