"""Tokens that no sequence holds, calls without any sequence, calls of more work than a launch takes, queues and streams of two
devices: what is left as it was, what does nothing, and what is refused.  Definitions and tolerances are those of
test_selective.py.
"""

import pytest
import torch

from test_selective import (BF16, F32, conv_definition, conv_inputs, gradients, near, ops, scan_definition,  # noqa: F401
                            scan_inputs, wide)

LEFT = 7.0  # what outputs hold before the call


def spread(plan, *outputs):
    """Outputs filled, the workspace without a number in it; then the plan runs."""
    for v in outputs:
        v.fill_(LEFT)
    for v in plan.full_args[0].keep:
        if isinstance(v, torch.Tensor) and v.dtype == torch.uint8:
            v.fill_(255)
    torch.cuda.synchronize()
    plan()
    plan.queue.finish()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads, groups, lengths", [
    (4, 1, [5, 70, 0, 64]),  # the heads of a group in blocks, whose sums are added up by a launch of their own
    (4, 4, [5, 70, 0, 64]),  # one work-group to a group
    (6, 2, [900])])          # several segments
def test_scan_leaves_tokens_of_no_sequence(queue, ops, dtype, heads, groups, lengths):  # noqa: F811
    front, back = 37, 90
    n = sum(lengths)
    padded, _, m = scan_inputs(61, dtype, [front + n + back], heads, 16, groups, 16, False)
    padded.pop("initial")
    starts = torch.tensor([front] + lengths, dtype=torch.int32).cumsum(0).int().cuda()
    held = slice(front, front + n)
    given = {k: v[held] if k in ("x", "dt", "B", "C") else v for k, v in padded.items()}
    at = (starts - front).cpu()

    def function(**v):
        return scan_definition(softplus=True, initial=None, starts=at, **v)

    plan = ops.plan_selective_scan(queue, softplus=True, starts=starts, **padded)
    spread(plan, plan.y)
    near(plan.y[held], function(**dict(zip(given, wide(*given.values()))))[0], "y")
    assert (plan.y[:front] == LEFT).all() and (plan.y[front + n:] == LEFT).all()

    dy = m.normal(*padded["x"].shape, dtype=dtype)
    plan = ops.plan_selective_scan_grad(queue, dy, softplus=True, starts=starts, **padded)
    got = plan.gradients
    rows = ("x", "dt", "B", "C")
    spread(plan, *(getattr(got, k) for k in rows))
    want = gradients(function, given, (dy[held], None))
    for k in want:
        v = getattr(got, k)
        near(v[held] if k in rows else v, want[k], k)
    for k in rows:
        assert (getattr(got, k)[:front] == LEFT).all() and (getattr(got, k)[front + n:] == LEFT).all(), k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, channels", [(F32, 20), (BF16, 64)])
def test_convolution_leaves_tokens_of_no_sequence(queue, ops, dtype, channels):  # noqa: F811
    front, lengths, back = 20, [3, 0, 130], 70
    n = sum(lengths)
    padded, _, m = conv_inputs(62, dtype, [front + n + back], channels, 4, False)
    padded.pop("initial")
    starts = torch.tensor([front] + lengths, dtype=torch.int32).cumsum(0).int().cuda()
    held = slice(front, front + n)
    given = dict(padded, x=padded["x"][held])

    def function(**v):
        return conv_definition(silu_=True, initial=None, starts=(starts - front).cpu(), **v)

    plan = ops.plan_causal_conv(queue, activation="silu", starts=starts, **padded)
    spread(plan, plan.y)
    near(plan.y[held], function(**dict(zip(given, wide(*given.values()))))[0], "y")
    dy = m.normal(front + n + back, channels, dtype=dtype)
    grad = ops.plan_causal_conv_grad(queue, dy, activation="silu", starts=starts, **padded)
    spread(grad, grad.gradients.x)
    want = gradients(function, given, (dy[held], None))
    near(grad.gradients.x[held], want["x"], "x")
    near(grad.gradients.weight, want["weight"], "weight")
    near(grad.gradients.bias, want["bias"], "bias")
    for v in (plan.y, grad.gradients.x):
        assert (v[:front] == LEFT).all() and (v[front + n:] == LEFT).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens", [0, 100, 3000])
def test_calls_without_sequences(queue, ops, dtype, tokens):  # noqa: F811
    """One offset, no sequence, any number of tokens: nothing is written, the parameters' gradients are zero."""
    starts = torch.zeros(1, dtype=torch.int32, device="cuda")
    given, _, m = scan_inputs(63, dtype, [tokens], 4, 16, 2, 16, False)
    given.pop("initial")
    plan = ops.plan_selective_scan(queue, softplus=True, starts=starts, **given)
    grad = ops.plan_selective_scan_grad(queue, given["x"], softplus=True, starts=starts, **given)
    got = grad.gradients
    rows = [plan.y] + [getattr(got, k) for k in ("x", "dt", "B", "C")]
    spread(plan, *rows)
    spread(grad, got.A, got.D, got.dt_bias)
    assert plan.final.shape == (0, 4, 16, 16)
    assert all((v == LEFT).all() for v in rows)
    assert not got.A.any() and not got.D.any() and not got.dt_bias.any()
    given, _, _ = conv_inputs(64, dtype, [tokens], 24, 4, False)
    given.pop("initial")
    plan = ops.plan_causal_conv(queue, starts=starts, **given)
    grad = ops.plan_causal_conv_grad(queue, given["x"], starts=starts, **given)
    spread(plan, plan.y)
    spread(grad, *grad.gradients[:3])
    assert (plan.y == LEFT).all() and (grad.gradients.x == LEFT).all()
    assert not grad.gradients.weight.any() and not grad.gradients.bias.any()


def test_more_work_than_a_launch_takes_is_refused_before_any(ops):  # noqa: F811
    """2**24 work-groups of 256 threads are one more than an axis of a grid has; a workspace is told up to there."""
    import ctypes

    from nengo_ocl_amd import _lib

    lib, bad, ref, need, one = _lib.lib(), -1, ctypes.byref, ctypes.c_longlong(), 1 << 20

    def told(entry, args):
        return entry(ref(args), ref(need))

    conv = ops._ConvArgs(channels=1, width=2, weight=one, y=one, dx=one, dweight=one, dbias=one, workspace=one,
                         workspace_bytes=1 << 60)
    conv.x.p = conv.dy.p = one
    conv.tokens.n_seqs = 1
    conv.tokens.length = conv.tokens.n_tokens = 2 ** 30 - 64
    assert told(lib.nhip_causal_conv_grad_workspace, conv) == 0
    conv.tokens.length = conv.tokens.n_tokens = 2 ** 30
    assert told(lib.nhip_causal_conv_grad_workspace, conv) == bad
    assert lib.nhip_causal_conv(None, ref(conv)) == bad and lib.nhip_causal_conv_grad(None, ref(conv)) == bad

    scan = ops._ScanArgs(n_heads=1, dim=1, n_groups=1, states=1, A=one, y=one, dx=one, ddt=one, dB=one, dC=one, dA=one,
                         dD=one, ddt_bias=one, workspace=one, workspace_bytes=1 << 60)
    scan.x.p = scan.dt.p = scan.B.p = scan.C.p = scan.dy.p = one
    for seqs, forward, gradient in ((2 ** 23 - 1, 0, 0), (2 ** 23, 0, bad), (2 ** 24 - 1, 0, bad), (2 ** 24, bad, bad)):
        scan.tokens.n_seqs, scan.tokens.length, scan.tokens.n_tokens = seqs, 1, seqs
        assert told(lib.nhip_selective_scan_workspace, scan) == forward
        assert told(lib.nhip_selective_scan_grad_workspace, scan) == gradient
    assert lib.nhip_selective_scan(None, ref(scan)) == bad and lib.nhip_selective_scan_grad(None, ref(scan)) == bad
    # sequences back to back, cut into segments: a lane to four elements of each one's state
    scan.n_heads, scan.dim, scan.states, scan.tokens.starts = 8, 64, 128, one
    scan.tokens.length, scan.tokens.n_tokens = 0, 2 ** 26
    for seqs, code in ((2 ** 18 - 1, 0), (2 ** 18, bad)):
        scan.tokens.n_seqs = seqs
        assert told(lib.nhip_selective_scan_workspace, scan) == code
    assert lib.nhip_selective_scan(None, ref(scan)) == bad

    step = ops._ScanStepArgs(n_heads=1, dim=1, n_groups=1, states=1, n=2 ** 24, n_slots=2 ** 24, A=one, state=one, y=one)
    step.x.p = step.dt.p = step.B.p = step.C.p = one
    assert lib.nhip_selective_step(None, ref(step)) == bad
    step = ops._ConvStepArgs(channels=256, width=1, n=2 ** 24, n_slots=2 ** 24, x=one, x_stride=257, weight=one, y=one)
    assert lib.nhip_causal_conv_step(None, ref(step)) == bad
    norm = ops._NormArgs(channels=2 ** 27, groups=1, rows=1, weight=one, x=one, dout=one, dx=one, dweight=one,
                         workspace=one, workspace_bytes=1 << 60)
    assert lib.nhip_block_norm_grad(None, ref(norm)) == bad


def test_a_queue_takes_no_stream_of_another_device(monkeypatch):
    import types

    from nengo_ocl_amd import hipraggedarray

    monkeypatch.setattr(hipraggedarray, "_TORCH", torch)
    other = types.SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=0)
    with pytest.raises(ValueError, match="cuda:1"):
        hipraggedarray.Queue(0, stream=other)


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_scan_on_a_device_that_is_not_the_current_one(ops):  # noqa: F811
    """Its launches take more LDS than a kernel has without being asked for, on the queue's device."""
    from nengo_ocl_amd.hipraggedarray import Queue

    given, starts, m = scan_inputs(65, BF16, [70, 200], 2, 64, 1, 128, False)
    given.pop("initial")
    there = {k: v.to("cuda:1") for k, v in dict(given, starts=starts).items()}
    queue = Queue(1)
    assert torch.cuda.current_device() == 0
    y, _ = ops.selective_scan(queue, softplus=True, **there)
    got = ops.selective_scan_grad(queue, there["x"], softplus=True, **there)
    assert torch.cuda.current_device() == 0
    want, _ = ops.selective_scan(Queue(0), softplus=True, starts=starts, **given)
    assert torch.equal(y.cpu(), want.cpu()) and torch.isfinite(got.A).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_recorded_scans(queue, ops, dtype):  # noqa: F811
    """A scan, its gradient and a convolution's as a list of plans, recorded once and replayed."""
    from nengo_ocl_amd.plan import Plans

    given, starts, m = scan_inputs(66, dtype, [300, 0, 700, 1], 8, 32, 2, 128, True)
    conv, _, _ = conv_inputs(67, dtype, [300, 0, 700, 1], 256, 4, False)
    conv.pop("initial")
    dy = m.normal(1001, 8, 32, dtype=dtype)
    want = ops.selective_scan(queue, softplus=True, starts=starts, **given)
    grad = ops.selective_scan_grad(queue, dy, softplus=True, starts=starts, **given)
    of_conv = ops.causal_conv_grad(queue, grad.x.flatten(1), activation="silu", starts=starts, **conv)
    torch.cuda.synchronize()
    scan = ops.plan_selective_scan(queue, softplus=True, starts=starts, **given)
    back = ops.plan_selective_scan_grad(queue, dy, softplus=True, starts=starts, **given)
    last = ops.plan_causal_conv_grad(queue, back.gradients.x.flatten(1), activation="silu", starts=starts, **conv)
    plans = Plans([scan, back, last], profiling=False)
    plans.prepare()
    for steps in (1, 2, 3):
        for v in (scan.y, scan.final, back.gradients.x, back.gradients.A, last.gradients.x, last.gradients.weight):
            v.fill_(LEFT)
        torch.cuda.synchronize()
        plans.call_n_times(steps)
        torch.cuda.synchronize()
        assert torch.equal(scan.y, want[0]) and torch.equal(scan.final, want[1])
        assert all(torch.equal(a, b) for a, b in zip(back.gradients, grad))
        assert all(torch.equal(a, b) for a, b in zip(last.gradients[:3], of_conv[:3]))
    plans.close()
