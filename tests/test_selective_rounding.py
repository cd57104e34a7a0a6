"""The scan's 16-bit results are rounded once: element by element, however much the terms of a sum cancel.

Tolerance.  A result v = want + d is rounded to want's type: an error of at most r |v|, where r is half the distance
from 1 to the next number: 2**-8 for bfloat16 (seven bits behind the leading one), 2**-11 for float16 (ten), or, below
float16's smallest normal number, of half the distance of the numbers there, 2**-25.  d comes
from the terms of the sums, whose magnitudes add up to `size` (the definition itself, applied to the magnitudes of all
inputs): sums in 32 bits are off by at most 128 u = 2**-17 of it (as in test_selective.py), and operands held in two
bfloat16 parts by r r = 2**-16.  Together less than 2**-15 `size`, r of it included.
"""

import pytest
import torch

from test_selective import BF16, F16, gradients, ops, scan_definition, scan_inputs, wide  # noqa: F401

ROUNDED = {BF16: 2.0 ** -8, F16: 2.0 ** -11}
SMALLEST = {BF16: 2.0 ** -134, F16: 2.0 ** -25}
CASES = [([1, 0, 70, 64, 3], 2, 64, 1, 128), ([150], 4, 16, 2, 16), ([33, 90], 3, 61, 1, 33), ([100], 2, 130, 2, 7),
         ([70, 40], 6, 8, 3, 200)]


def magnitudes(given):
    return {k: v if v is None or k in ("dt", "A", "dt_bias") else v.abs() for k, v in given.items()}


def rounded_once(got, want, size, name):
    got64 = got.detach().cpu().double()
    assert got64.shape == want.shape, name
    bound = ROUNDED[got.dtype] * want.abs() + 2.0 ** -15 * size + SMALLEST[got.dtype]
    worst = ((got64 - want).abs() / bound).max() if want.numel() else 0.0
    assert float(worst) <= 1.0, (name, float(worst))


def scan64(given, starts):
    return scan_definition(**dict(zip(given, wide(*given.values()))), softplus=True, starts=starts)[0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths, heads, dim, groups, states", CASES)
def test_scan_is_rounded_once(queue, ops, dtype, lengths, heads, dim, groups, states):  # noqa: F811
    given, starts, _ = scan_inputs(51, dtype, lengths, heads, dim, groups, states, True)
    y, _ = ops.selective_scan(queue, softplus=True, starts=starts, **given)
    rounded_once(y, scan64(given, starts), scan64(magnitudes(given), starts), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scan_of_a_large_state_that_the_output_does_not_see(queue, ops, dtype):  # noqa: F811
    """A state of hundreds whose rows are all but orthogonal to C, which is the same for all tokens."""
    given, starts, m = scan_inputs(52, dtype, [50, 80], 2, 32, 1, 64, True)
    C = m.normal(1, 1, 64, dtype=dtype, scale=0.125)
    given["C"] = C.expand(130, 1, 64).contiguous()
    S, c = given["initial"] * 300.0, C.float()[0, 0]
    given["initial"] = (S - (S @ c)[..., None] * c / (c @ c)).contiguous()
    given["x"] = (given["x"].float() * 0.1).to(dtype)
    y, _ = ops.selective_scan(queue, softplus=True, starts=starts, **given)
    want, size = scan64(given, starts), scan64(magnitudes(given), starts)
    assert float((size[:5] / want[:5].abs()).median()) > 100.0  # (what the case is for: terms that cancel)
    rounded_once(y, want, size, "y")


def gradients64(given, starts, dy, dfinal):
    return gradients(lambda **v: scan_definition(softplus=True, starts=starts, **v), given, (dy, dfinal))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths, heads, dim, groups, states", CASES)
def test_gradient_of_the_scan_is_rounded_once(queue, ops, dtype, lengths, heads, dim, groups, states):  # noqa: F811
    given, starts, m = scan_inputs(53, dtype, lengths, heads, dim, groups, states, True)
    dy, dfinal = m.normal(sum(lengths), heads, dim, dtype=dtype), m.normal(len(lengths), heads, dim, states)
    got = ops.selective_scan_grad(queue, dy, softplus=True, starts=starts, dfinal=dfinal, **given)
    want = gradients64(given, starts, dy, dfinal)
    size = gradients64(magnitudes(given), starts, dy.abs(), dfinal.abs())
    for k in ("x", "B", "C"):
        rounded_once(getattr(got, k), want[k], size[k], k)
