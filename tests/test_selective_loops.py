"""The loops of the selective operators that short inputs do not enter: walks over several chunks of a segment, sequences left
whole, several heads and tiles to a work-group of the gradient, many requests to a step, norms whose rows
several packs of a lane hold.  Definitions and tolerances are those of test_selective.py.
"""

import pytest
import torch

from test_selective import (BF16, F16, F32, gradients, near, norm_definition, norm_inputs, ops,  # noqa: F401
                            scan_definition, scan_inputs, wide)

# (sequences, heads, dim, groups, states): what the kernels make of it on this device, whose launches aim at
# 256 walks at least (512 in bfloat16 with up to 128 states), each over two units of 64 of a head's dimension
WALKS = [
    # sequences that stay whole: six chunks, the last of them of ten tokens; six heads to a work-group of the gradient,
    # whose blocks are added up by a launch of their own
    ([330] * 8, 64, 8, 1, 16),
    # five chunks; four heads of each of 16 groups to a work-group, and no other blocks
    ([300] * 8, 64, 16, 16, 16),
    # 21 chunks of one sequence in segments of three to eleven; a head to each group
    ([1300], 64, 8, 64, 8),
    # six heads to a work-group of the gradient over few segments
    ([1300], 128, 8, 1, 16),
    # ragged: segments of several chunks that begin and end within them, an empty sequence and one of a token
    ([1700, 0, 1, 600], 128, 8, 2, 16),
    # heads of two whole tiles of 64, two of them to a work-group
    ([200] * 8, 24, 128, 1, 16),
    # chunks of 32 tokens
    ([200] * 4, 64, 8, 1, 200),
    # an odd number of heads to a group, units without a second, rows that are no multiple of 16 bytes
    ([130] * 16, 15, 21, 3, 13),
]


def given_for(seed, dtype, lengths, *sizes):
    dense = None if len(set(lengths)) > 1 else (len(lengths), lengths[0])
    given, starts, m = scan_inputs(seed, dtype, lengths, *sizes, True, dense=dense)
    # rates at which something is left of a state for some chunks, and nothing of it for some heads
    given["A"] = -m.uniform(0.05, 1.0, sizes[0])
    return given, starts, m


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lengths, heads, dim, groups, states", WALKS)
def test_scan_over_several_chunks_of_a_segment(queue, ops, dtype, lengths, heads, dim, groups, states):  # noqa: F811
    given, starts, _ = given_for(41, dtype, lengths, heads, dim, groups, states)
    y, final = ops.selective_scan(queue, softplus=True, starts=starts, **given)
    y64, final64 = scan_definition(**dict(zip(given, wide(*given.values()))), softplus=True, starts=starts)
    near(y, y64, "y")
    near(final, final64, "final")
    # (a wrong chunk of one sequence is little of the whole norm)
    tokens = y.flatten(0, 1) if starts is None else y
    y64 = y64.flatten(0, 1) if starts is None else y64
    for t in range(0, tokens.shape[0], 64):
        near(tokens[t:t + 64], y64[t:t + 64], t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, lengths, heads, dim, groups, states",
                         [(t,) + w for w in WALKS for t in (F32, BF16)] + [(F16,) + w for w in (WALKS[3], WALKS[7])])
def test_scan_gradient_over_several_chunks_and_heads(queue, ops, dtype, lengths, heads, dim, groups,  # noqa: F811
                                                     states):
    given, starts, m = given_for(42, dtype, lengths, heads, dim, groups, states)
    dy = m.normal(*given["x"].shape, dtype=dtype)
    dfinal = m.normal(len(lengths), heads, dim, states)
    got = ops.selective_scan_grad(queue, dy, softplus=True, starts=starts, dfinal=dfinal, **given)
    want = gradients(lambda **v: scan_definition(softplus=True, starts=starts, **v), given, (dy, dfinal))
    for k in want:
        near(getattr(got, k), want[k], k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n, heads, dim, groups, states", [
    (16, 64, 20, 4, 33), (20, 56, 64, 1, 128), (40, 32, 9, 2, 5), (17, 64, 70, 64, 200)])
def test_step_of_many_requests(queue, ops, dtype, n, heads, dim, groups, states):  # noqa: F811
    """Eight rows to a lane: 1024 work-groups and more, rows that end within a lane's eight."""
    given, _, m = scan_inputs(43, dtype, [n], heads, dim, groups, states, False)
    given.pop("initial")
    pool = m.normal(n + 3, heads, dim, states)
    slots = torch.randperm(n + 3, generator=m.gen)[:n].to(torch.int32).cuda()
    slots[3] = n + 3
    before = pool.clone()
    y = ops.selective_step(queue, pool, softplus=True, slots=slots, **given)
    here = [r for r in range(n) if r != 3]
    at = slots.long()[here]
    one = {k: v[here][:, None] if k in ("x", "dt", "B", "C") else v for k, v in given.items()}
    y64, final64 = scan_definition(**dict(zip(one, wide(*one.values()))), softplus=True, initial=before[at].cpu().double(),
                                   starts=None)
    near(y[here], y64[:, 0], "y")
    near(pool[at], final64, "state")
    assert not y[3].any()
    rest = [s for s in range(n + 3) if s not in set(at.tolist())]
    assert torch.equal(pool[rest], before[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, channels, groups", [
    (45, 2048, 1), (45, 4096, 1), (21, 3000, 1), (45, 512, 1), (19, 8192, 4), (45, 700, 1), (23, 1000, 2), (9, 1025, 1)])
def test_norm_gradient_of_rows_in_several_packs(queue, ops, dtype, rows, channels, groups):  # noqa: F811
    for gate, residual, scale, after in ((0, 1, 1, 0), (1, 0, 0, 0), (1, 1, 1, 1)):
        given, m = norm_inputs(44, dtype, rows, channels, gate, residual, scale)
        same = dict(groups=groups, eps=1e-5, after=bool(after))
        out, v = ops.block_norm(queue, **given, **same)
        out64, v64 = norm_definition(**dict(zip(given, wide(*given.values()))), **same)
        near(out, out64, "out")
        dout = m.normal(rows, channels, dtype=dtype)
        dv = m.normal(rows, channels, dtype=dtype) if v is not None else None
        got = ops.block_norm_grad(queue, dout, dv=dv, **given, **same)

        def function(x, weight, gate=None, residual=None, scale=None):
            return norm_definition(x, weight, gate, residual, scale, **same)

        want = gradients(function, given, (dout, dv))
        for k in want:
            near(getattr(got, k), want[k], (k, gate, residual, scale, after))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_no_number_over_several_chunks(queue, ops, dtype, bad):  # noqa: F811
    """In a walk over six chunks it reaches no earlier token and no other sequence, from C its own token alone; in the
    gradient, the other sequences' parts stay as they are."""
    given, _, m = given_for(45, dtype, *WALKS[0])
    dy = m.normal(*given["x"].shape, dtype=dtype)
    clean, _ = ops.selective_scan(queue, softplus=True, **given)
    grads = ops.selective_scan_grad(queue, dy, softplus=True, **given)
    others = [0, 1, 2, 4, 5, 6, 7]
    for name in ("x", "B", "C"):
        odd = dict(given)
        odd[name] = given[name].clone()
        odd[name][3, 200, 0, 3] = bad
        y, final = ops.selective_scan(queue, softplus=True, **odd)
        assert torch.equal(y[others], clean[others]) and torch.equal(y[3, :200], clean[3, :200]), name
        assert torch.isfinite(final[others]).all()
        assert not torch.isfinite(y[3, 200]).all(), name
        if name == "C":
            assert torch.equal(y[3, 201:], clean[3, 201:]) and torch.isfinite(final).all()
        if name == "x":  # head 0, element 3 of its dimension
            rest = [0, 1, 2, 4, 5, 6, 7]
            assert torch.equal(y[3, :, 1:], clean[3, :, 1:]) and torch.equal(y[3, :, 0][:, rest], clean[3, :, 0][:, rest])
        got = ops.selective_scan_grad(queue, dy, softplus=True, **odd)
        for k in ("x", "dt", "B", "C", "initial"):
            assert torch.equal(getattr(got, k)[others], getattr(grads, k)[others]), (name, k)
