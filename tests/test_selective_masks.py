"""Steps of the selective scan that are masked (softplus of -inf or of the lowest value is zero) or larger than any
exponential holds, in the scan, its gradient and its step for single tokens.  Definitions and tolerances are those of
test_selective.py.
"""

import pytest
import torch

from test_selective import (BF16, F16, F32, along_differences, gradients, near, ops, scan_definition,  # noqa: F401
                            scan_inputs, wide)

MASKS = [-float("inf"), "lowest", -1e10, -65000.0]


def masked(value, dtype):
    return torch.finfo(dtype).min if value == "lowest" else value


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("value", MASKS)
@pytest.mark.parametrize("dt_type", ["same", F32, BF16])
def test_scan_of_masked_tokens(queue, ops, dtype, value, dt_type):  # noqa: F811
    """A masked token changes nothing behind it: first ones, last ones, whole chunks and a whole sequence of them."""
    given, starts, m = scan_inputs(31, dtype, [150, 70, 3], 2, 16, 1, 16, True)
    if dt_type != "same":
        given["dt"] = given["dt"].to(dt_type)
    low = masked(value, given["dt"].dtype)
    for a, b in ((0, 2), (9, 10), (60, 130), (147, 150), (160, 165), (220, 223)):
        given["dt"][a:b] = low
    y, final = ops.selective_scan(queue, softplus=True, starts=starts, **given)
    y64, final64 = scan_definition(**dict(zip(given, wide(*given.values()))), softplus=True, starts=starts)
    assert torch.isfinite(y64).all() and torch.isfinite(final64).all()
    near(y, y64, "y")
    near(final, final64, "final")
    assert torch.equal(final[2], given["initial"][2])

    dy, dfinal = m.normal(223, 2, 16, dtype=dtype), m.normal(3, 2, 16, 16)
    got = ops.selective_scan_grad(queue, dy, softplus=True, starts=starts, dfinal=dfinal, **given)

    def function(**v):
        return scan_definition(softplus=True, starts=starts, **v)

    want = gradients(function, given, (dy, dfinal))
    assert all(torch.isfinite(v).all() for v in want.values())
    for k in want:
        near(getattr(got, k), want[k], k)
    assert not got.dt[60:130].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [1e10, 1e30])
def test_scan_of_steps_beyond_all_exponentials(queue, ops, dtype, value):  # noqa: F811
    """softplus(v) is v there and the decay zero; each span is compared by its own size."""
    given, starts, _ = scan_inputs(32, dtype, [150, 40], 2, 16, 1, 16, True)
    given["dt"][[10, 64, 170]] = value
    y, final = ops.selective_scan(queue, softplus=True, starts=starts, **given)
    y64, final64 = scan_definition(**dict(zip(given, wide(*given.values()))), softplus=True, starts=starts)
    for a, b in ((0, 10), (10, 11), (11, 64), (64, 65), (65, 150), (150, 170), (170, 190)):
        near(y[a:b], y64[a:b], (a, b))
    for s in range(2):
        near(final[s], final64[s], s)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_step_of_masked_tokens_and_of_large_ones(queue, ops, dtype):  # noqa: F811
    values = [-float("inf"), torch.finfo(dtype).min, -1e10, 1e10, 1e30, 0.3]
    n = len(values)
    given, _, m = scan_inputs(33, dtype, [n], 2, 16, 1, 16, False)
    given.pop("initial")
    given["dt"] = torch.tensor(values, dtype=dtype, device="cuda")[:, None].expand(n, 2)
    state = m.normal(n, 2, 16, 16)
    before = state.clone()
    y = ops.selective_step(queue, state, softplus=True, **given)
    for r in range(n):
        one = {k: v[r:r + 1][None] if k in ("x", "dt", "B", "C") else v for k, v in given.items()}
        y64, final64 = scan_definition(**dict(zip(one, wide(*one.values()))), softplus=True,
                                       initial=before[r:r + 1].cpu().double(), starts=None)
        near(y[r], y64[0, 0], values[r])
        near(state[r], final64[0], values[r])
    assert torch.equal(state[:3], before[:3])
    # no softplus: the decay of a step far beyond any exponential is zero, and of one so far below it is one
    rate = -torch.full((2,), 8.0, device="cuda")
    for value in (3e38, 1e30, 1e10):
        state = before.clone()
        x = torch.full((n, 2, 16), 1.0 / value, device="cuda").to(dtype)
        dt = torch.full((n, 2), value, dtype=dtype, device="cuda")
        ops.selective_step(queue, state, x, dt, rate, given["B"], given["C"])
        want = (dt.double()[..., None] * x.double())[..., None] * given["B"].double()[:, :, None]
        near(state, want.cpu(), value)


@pytest.mark.gpu
def test_gradient_along_differences_with_masked_tokens(queue, ops):  # noqa: F811
    given, starts, m = scan_inputs(34, F32, [90], 2, 8, 1, 8, True)
    hidden = torch.arange(90, device="cuda") % 3 == 1
    given["dt"][hidden] = -1e30
    dy, dfinal = m.normal(90, 2, 8), m.normal(1, 2, 8, 8)
    got = ops.selective_scan_grad(queue, dy, softplus=True, starts=starts, dfinal=dfinal, **given)
    along_differences(lambda **v: scan_definition(softplus=True, starts=starts, **v), given, (dy, dfinal),
                      got._asdict(), 35)
