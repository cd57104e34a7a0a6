"""What the operators over tokens do where it is easy to go wrong: rows that do not count whatever they hold, values that are no
numbers, workspaces that hold anything, rows with strides and at odd places, plans recorded and replayed, empty calls;
and what their entry points refuse.  Definitions and tolerances are those of test_tokens.py.
"""

import ctypes
import itertools
import math

import pytest
import torch

from test_tokens import (BF16, E, F16, F32, U, Maker, act, check_loss_gradients, check_losses, gated_bounds,  # noqa: F401
                         gated_inputs, host, loss_inputs, norm_definition, norm_inputs, ops, teacher_inputs, wide, within)

NAN, INF = float("nan"), float("inf")
# small tiles; tiles through the large kernels, whose products read matrices as they lie
SIZES = [(F32, 70, 40, 130), (BF16, 40, 72, 257), (BF16, 300, 520, 9001), (F16, 300, 520, 9001), (F32, 300, 130, 310)]


def same(a, b):
    """Equal bit for bit, NaN among them."""
    return torch.equal(torch.nan_to_num(a, nan=77.0), torch.nan_to_num(b, nan=77.0)) and torch.equal(torch.isnan(a), torch.isnan(b))


def calls(ops, queue, seed, dtype, n, d, v):  # noqa: F811
    """Every operator's call on inputs of these sizes: {name: (the arrays by name, a function of these to outputs)}."""
    loss, m = loss_inputs(seed, dtype, n, d, v, 0.3)
    teach, _ = teacher_inputs(seed + 1, dtype, n, d, v, 0.3, 20)
    gated, _ = gated_inputs(seed + 2, dtype, n, d, v)
    norm, _ = norm_inputs(seed + 3, dtype, (n,), d, True, True)
    dloss = (torch.rand(n, generator=m.gen) / n).cuda()
    dy, dout = m.normal(n, v, dtype=dtype), m.normal(n, d, dtype=dtype)
    lse = ops.vocabulary_loss(queue, **loss)[1]
    lse_t = ops.teacher_loss(queue, temperature=2.0, **teach)[1]
    return {
        "norm": (norm, lambda **k: ops.plan_layer_norm(queue, **k)),
        "norm_grad": (dict(norm, dout=dout, dv=dout), lambda **k: ops.plan_layer_norm_grad(queue, **k)),
        "gated": (gated, lambda **k: ops.plan_gated_projection(queue, **k)),
        "gated_grad": (dict(gated, dy=dy), lambda **k: ops.plan_gated_projection_grad(queue, **k)),
        "loss": (loss, lambda **k: ops.plan_vocabulary_loss(queue, **k)),
        "loss_grad": (dict(loss, dloss=dloss, lse=lse), lambda **k: ops.plan_vocabulary_loss_grad(queue, **k)),
        "teacher": (teach, lambda **k: ops.plan_teacher_loss(queue, temperature=2.0, **k)),
        "teacher_grad": (dict(teach, dloss=dloss, lse=lse_t), lambda **k: ops.plan_teacher_loss_grad(queue, temperature=2.0, **k)),
    }


def outputs(plan):
    got = [getattr(plan, k) for k in ("out", "v", "y", "loss", "lse") if getattr(plan, k, None) is not None]
    return got + [v for v in getattr(plan, "gradients", ()) if v is not None]


def run(plan):
    torch.cuda.synchronize()
    plan()
    plan.queue.finish()
    return [v.clone() for v in outputs(plan)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, n, d, v", SIZES)
def test_workspaces_and_outputs_may_hold_anything(queue, ops, dtype, n, d, v):  # noqa: F811
    """The same results, bit for bit, on every call, whatever lies in the workspace and in the outputs."""
    for name, (given, make) in calls(ops, queue, 31, dtype, n, d, v).items():
        plan = make(**given)
        first = run(plan)
        for fill in (255, 0, 127):
            for t in plan.full_args[0].keep:
                if isinstance(t, torch.Tensor) and t.dtype == torch.uint8:
                    t.fill_(fill)
            for t in outputs(plan):
                t.fill_(NAN)
            assert all(same(a, b) for a, b in zip(first, run(plan))), (name, fill)
        assert all(torch.isfinite(t).all() for t in first), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, n, d, v", SIZES)
def test_plans_recorded_and_replayed(queue, ops, dtype, n, d, v):  # noqa: F811
    """All operators in one graph, replayed with new inputs in the same arrays and other work between the replays."""
    from nengo_ocl_amd.plan import Plans

    made = calls(ops, queue, 32, dtype, n, d, v)
    plans = {name: make(**given) for name, (given, make) in made.items()}
    group = Plans(list(plans.values()), False)
    for turn in range(3):
        for given, _ in made.values():
            for k in ("x", "dy", "dout"):
                if k in given:
                    given[k].copy_((given[k].float() * -0.9).to(given[k].dtype))
        torch.cuda.synchronize()
        group.enqueue_n_times(2)
        queue.finish()
        got = {name: [t.clone() for t in outputs(p)] for name, p in plans.items()}
        torch.zeros(1 << 20, device="cuda").sum().item()
        for name, plan in plans.items():
            assert all(same(a, b) for a, b in zip(got[name], run(plan))), (name, turn)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, n, d, v", SIZES)
def test_the_current_stream_and_others(ops, dtype, n, d, v):  # noqa: F811
    """A queue with a stream of its own and one with torch's give the same, in order with torch's work on both sides."""
    from nengo_ocl_amd.hipraggedarray import Queue

    own, current = Queue(0), Queue(0, stream=torch.cuda.current_stream())
    given, _ = loss_inputs(33, dtype, n, d, v, 0.2)
    scaled = given["x"] * 0.5
    want = ops.vocabulary_loss(current, scaled, given["weight"], given["labels"])
    for _ in range(3):
        got = ops.vocabulary_loss(own, given["x"] * 0.5, given["weight"], given["labels"])
        assert same(got[0] + 0, want[0]) and same(got[1] + 0, want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.vocabulary_loss(own, given["x"] * 0.5, given["weight"], given["labels"])
        assert same(got[0] + 0, want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, n, d, v", SIZES)
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_rows_that_do_not_count(queue, ops, dtype, n, d, v, bad):  # noqa: F811
    """Whatever they hold, everything else is the same bit for bit, and they have zeros."""
    made = calls(ops, queue, 34, dtype, n, d, v)
    for name in ("loss", "loss_grad", "teacher", "teacher_grad"):
        given, make = made[name]
        left = given["labels"] < 0 if "labels" in given else ~((given["indices"] >= 0) & (given["indices"] < v)).any(1)
        assert left.any() and not left.all()
        clean = run(make(**given))
        dirty = {k: t.clone() for k, t in given.items()}
        for k in ("x", "dloss", "lse", "logits"):
            if k in dirty:
                dirty[k][left] = bad
        got = run(make(**dirty))
        assert all(same(a, b) for a, b in zip(clean, got)), name
        assert all(not t[left].any() for t in got if t.shape[0] == n), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, n, d, v", SIZES)
def test_values_that_are_no_numbers_stay_in_their_row(queue, ops, dtype, n, d, v):  # noqa: F811
    for name, (given, make) in calls(ops, queue, 35, dtype, n, d, v).items():
        row = 1
        if "labels" in given:
            given["labels"][row] = 0
        if "indices" in given:
            given["indices"][row, 0] = 0
        clean = run(make(**given))
        given = dict(given, x=given["x"].clone())
        given["x"][row, 3] = NAN
        got = run(make(**given))
        others = torch.arange(n, device="cuda") != row
        for a, b in zip(clean, got):
            if b.shape[0] == n and b.dim() <= 2 and not (n == d and name == "norm_grad"):
                assert same(a[others], b[others]), name
                assert torch.isnan(b[row]).any(), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n, d, v", [(5, 40, 70), (300, 130, 600), (300, 520, 9001)])
def test_rows_with_strides_and_at_odd_places(queue, ops, dtype, n, d, v):  # noqa: F811
    """Slices of wider arrays give what contiguous copies of them give."""
    m = Maker(36)
    x_all, w_all = m.normal(n, d + 11, dtype=dtype), m.normal(2 * v, d + 9, dtype=dtype, scale=d ** -0.5)
    dy_all = m.normal(n, v + 5, dtype=dtype)
    labels = m.whole(v, n).cuda()
    for at in (0, 1, 8):
        x, gate, up, dy = x_all[:, at:at + d], w_all[:v, at:at + d], w_all[v:, at:at + d], dy_all[:, at // 4:at // 4 + v]
        flat = [t.contiguous() for t in (x, gate, up, dy)]
        y = ops.gated_projection(queue, x, gate, up)
        want = ops.gated_projection(queue, *flat[:3])
        tol = 2 * U[dtype] if dtype != F32 else 64 * E
        near = lambda a, b: (a.double() - b.double()).abs().max() <= tol * b.double().abs().max()
        assert near(y, want)
        for a, b in zip(ops.gated_projection_grad(queue, dy, x, gate, up), ops.gated_projection_grad(queue, flat[3], *flat[:3])):
            assert near(a, b)
        loss, lse = ops.vocabulary_loss(queue, x, gate, labels)
        check_losses(loss, lse, {"x": x, "weight": gate, "labels": labels}, 1.0)
        dloss = torch.full((n,), 1.0 / n, device="cuda")
        got = ops.vocabulary_loss_grad(queue, dloss, x, gate, labels, lse)
        check_loss_gradients(got, {"x": x, "weight": gate, "labels": labels}, 1.0, dloss, lse)
        weight, bias = m.normal(d), m.normal(d)
        out, _ = ops.layer_norm(queue, x, weight, bias)
        assert near(out, ops.layer_norm(queue, flat[0], weight, bias)[0])
        for a, b in zip(ops.layer_norm_grad(queue, x, x, weight, bias), ops.layer_norm_grad(queue, flat[0], flat[0], weight, bias)):
            assert a is b is None or near(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_nothing_to_do(queue, ops, dtype):  # noqa: F811
    """No rows; rows of which none counts."""
    z = lambda *s, t=dtype: torch.zeros(*s, dtype=t, device="cuda")
    w = torch.ones(70, 40, dtype=dtype, device="cuda")
    assert ops.layer_norm(queue, z(0, 40), z(40, t=F32))[0].shape == (0, 40)
    got = ops.layer_norm_grad(queue, z(0, 40), z(0, 40), z(40, t=F32), z(40, t=F32))
    assert got.x.shape == (0, 40) and not got.weight.any() and not got.bias.any()
    assert ops.gated_projection(queue, z(2, 0, 40), w, w).shape == (2, 0, 70)
    got = ops.gated_projection_grad(queue, z(0, 70), z(0, 40), w, w)
    assert got.x.shape == (0, 40) and not got.gate.any() and not got.up.any()
    for n in (0, 3, 200):
        x = torch.full((n, 40), NAN, dtype=dtype, device="cuda")
        for labels in (torch.full((n,), -1, device="cuda"), torch.full((n,), 70, dtype=torch.int32, device="cuda"),
                       torch.full((n,), 1 << 40, device="cuda"), torch.full((n,), -(1 << 31), dtype=torch.int32, device="cuda")):
            loss, lse = ops.vocabulary_loss(queue, x, w, labels)
            assert loss.shape == (n,) and not loss.any() and not lse.any()
            got = ops.vocabulary_loss_grad(queue, z(n, t=F32) + 1, x, w, labels, lse)
            assert got.x.shape == (n, 40) and not got.x.any() and not got.weight.any()
        none = torch.full((n, 5), -INF, device="cuda")
        loss, lse = ops.teacher_loss(queue, x, w, torch.zeros(n, 5, dtype=torch.int32, device="cuda"), none)
        assert not loss.any() and not lse.any()
        got = ops.teacher_loss_grad(queue, z(n, t=F32) + 1, x, w, torch.zeros(n, 5, dtype=torch.int32, device="cuda"), none, lse)
        assert not got.x.any() and not got.weight.any()


@pytest.mark.gpu
def test_targets_twice_masked_and_of_the_lowest_value(queue, ops):  # noqa: F811
    """A word named twice is two targets; -inf is left out; a type's lowest value is a value; infinite ones are no numbers."""
    given, m = teacher_inputs(37, F32, 6, 40, 300, 0.0, 9)
    given["indices"][0] = 5
    given["indices"][1, 4:] = given["indices"][1, 3]
    given["logits"][2, 1:] = -INF
    given["logits"][3] = torch.finfo(F32).min
    given["logits"][4, 2] = torch.finfo(F32).min
    loss, lse = ops.teacher_loss(queue, **given)
    check_losses(loss, lse, given, 1.0)
    dloss = torch.rand(6, generator=m.gen).cuda()
    check_loss_gradients(ops.teacher_loss_grad(queue, dloss, lse=lse, **given), given, 1.0, dloss, lse)
    for bad in (NAN, INF):
        given["logits"][5, 0] = bad
        loss, _ = ops.teacher_loss(queue, **given)
        assert torch.isnan(loss[5]) and torch.isfinite(loss[:5]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [3, 50, 300])
def test_logits_far_apart(queue, ops, dtype, n):  # noqa: F811
    """Logits of thousands: the sum is of the largest; and a word of infinite logit, or all words of minus infinity."""
    given, m = loss_inputs(38, dtype, n, 64, 500, 0.0)
    given["x"] = given["x"] * 1000
    loss, lse = ops.vocabulary_loss(queue, **given)
    check_losses(loss, lse, given, 1.0)
    dloss = torch.rand(n, generator=m.gen).cuda()
    check_loss_gradients(ops.vocabulary_loss_grad(queue, dloss, lse=lse, **given), given, 1.0, dloss, lse)
    given["x"] = given["x"].abs() + 1
    given["labels"][0] = 8
    for value, word in ((INF, 7), (-INF, slice(None))):
        weight = given["weight"].clone()
        weight[word] = value
        loss, lse = ops.vocabulary_loss(queue, given["x"], weight, given["labels"])
        assert (lse == value).all()
        if value > 0:
            assert loss[0] == INF


@pytest.mark.gpu
@pytest.mark.parametrize("n, d, v", [(300, 520, 9001), (20, 64, 500)])
def test_float16_gradients_of_a_mean_over_many_tokens(queue, ops, n, d, v):  # noqa: F811
    """Shares of 1e-4 times 2**-20 are below the type's smallest number; the products' results are not."""
    given, m = loss_inputs(39, F16, n, d, v, 0.1)
    loss, lse = ops.vocabulary_loss(queue, **given)
    for scale in (2.0 ** -20, 1.0, 2.0 ** 12):
        dloss = (torch.rand(n, generator=m.gen) * scale / 64).cuda()
        got = ops.vocabulary_loss_grad(queue, dloss, lse=lse, **given)
        check_loss_gradients(got, given, 1.0, dloss, lse)


@pytest.mark.gpu
def test_gradients_that_are_none(queue, ops):  # noqa: F811
    """A gradient of zero makes zeros; one that is no number reaches its row and the weights."""
    given, m = loss_inputs(40, BF16, 50, 64, 300, 0.2)
    given["labels"][2] = 1
    _, lse = ops.vocabulary_loss(queue, **given)
    dloss = torch.zeros(50, device="cuda")
    got = ops.vocabulary_loss_grad(queue, dloss, lse=lse, **given)
    assert not got.x.any() and not got.weight.any()
    dloss[2] = NAN
    got = ops.vocabulary_loss_grad(queue, dloss, lse=lse, **given)
    assert torch.isnan(got.x[2]).all() and torch.isfinite(got.x[torch.arange(50) != 2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["silu", "gelu"])
@pytest.mark.parametrize("n", [2, 300])
def test_activations_of_large_values(queue, ops, name, n):  # noqa: F811
    x = torch.linspace(-300.0, 300.0, n, device="cuda")[:, None]
    gate, up = torch.ones(140, 1, device="cuda"), torch.ones(140, 1, device="cuda")
    y = ops.gated_projection(queue, x, gate, up, name)
    want = act(name, wide(x)) * wide(x)
    assert ((wide(y) - want).abs() <= 1e-5 * want.abs() + 1e-30).all()
    got = ops.gated_projection_grad(queue, torch.ones(n, 140, device="cuda"), x, gate, up, name)
    assert all(torch.isfinite(t).all() for t in got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_leading_axes_and_given_outputs(queue, ops, dtype):  # noqa: F811
    """[batch, tokens, channels] as [tokens, channels]; arrays to write, also at odd places."""
    m = Maker(41)
    x, gate, up = m.normal(2, 9, 40, dtype=dtype), m.normal(24, 40, dtype=dtype), m.normal(24, 40, dtype=dtype)
    labels, words = m.whole(24, 2, 9).cuda(), m.whole(24, 2, 9, 3).cuda()
    values = m.normal(2, 9, 3, dtype=dtype)
    y = ops.gated_projection(queue, x, gate, up)
    assert y.shape == (2, 9, 24) and torch.equal(y.view(18, 24), ops.gated_projection(queue, x.view(18, 40), gate, up))
    to = torch.empty(2 * 9 * 24 + 1, dtype=dtype, device="cuda")[1:].view(2, 9, 24)
    plan = ops.plan_gated_projection(queue, x, gate, up, y=to)
    run(plan)
    assert plan.y is to and torch.equal(to, y)
    loss, lse = ops.vocabulary_loss(queue, x, gate, labels)
    assert loss.shape == lse.shape == (2, 9)
    flat = ops.vocabulary_loss(queue, x.view(18, 40), gate, labels.view(18))
    assert torch.equal(loss.view(18), flat[0]) and torch.equal(lse.view(18), flat[1])
    loss, lse = ops.teacher_loss(queue, x, gate, words, values, 2.0)
    flat = ops.teacher_loss(queue, x.view(18, 40), gate, words.view(18, 3), values.view(18, 3), 2.0)
    assert torch.equal(loss.view(18), flat[0]) and torch.equal(lse.view(18), flat[1])
    got = ops.teacher_loss_grad(queue, loss, x, gate, words, values, lse, 2.0)
    assert got.x.shape == x.shape and got.weight.shape == gate.shape
    dy = m.normal(2, 9, 24, dtype=dtype)
    got = ops.gated_projection_grad(queue, dy, x, gate, up)
    assert got.x.shape == x.shape and got.gate.shape == got.up.shape == gate.shape


# ---------------------------------------------------------------------------------- refusals
def refused(kind, f, *args, **kwargs):
    with pytest.raises(kind):
        f(*args, **kwargs)


def test_refusals_of_the_layer_norm(host, ops):  # noqa: F811
    x, w = torch.zeros(3, 5, 12), torch.zeros(12)
    f = ops.plan_layer_norm
    assert f(host, x, w).v is None and f(host, x, w, w, residual=x).v.shape == x.shape
    refused(TypeError, f, host, x.double(), w)
    refused(TypeError, f, host, x, None)
    refused(TypeError, f, host, x, w.half())
    refused(TypeError, f, host, x, w, w.half())
    refused(TypeError, f, host, x, w, residual=x.half())
    refused(ValueError, f, host, x, w[:5])
    refused(ValueError, f, host, x, w, w[:5])
    refused(ValueError, f, host, x, w, residual=x[:2])
    refused(ValueError, f, host, x, w, eps=-1.0)
    refused(ValueError, f, host, x, w, eps=NAN)
    refused(ValueError, f, host, x, w, v=x)                                    # no residual
    refused(ValueError, f, host, x.transpose(0, 1), w)                         # rows at two distances
    refused(ValueError, f, host, torch.zeros(3, 0), torch.zeros(0))
    refused(ValueError, f, host, x, w, out=torch.zeros(3, 5, 13))
    g = ops.plan_layer_norm_grad
    refused(ValueError, g, host, x, x, w, dv=x)
    refused(ValueError, g, host, x[:2], x, w)
    refused(TypeError, g, host, x.half(), x, w)


def test_refusals_of_the_gated_projection(host, ops):  # noqa: F811
    x, w = torch.zeros(3, 5, 12), torch.zeros(7, 12)
    f = ops.plan_gated_projection
    assert f(host, x, w, w).y.shape == (3, 5, 7)
    refused(TypeError, f, host, x.double(), w, w)
    refused(TypeError, f, host, x, w.half(), w)
    refused(TypeError, f, host, x, w, w.half())
    refused(ValueError, f, host, x, w, w, "relu")
    refused(ValueError, f, host, x, w[:, :5], w)
    refused(ValueError, f, host, x, w, w[:5])
    refused(ValueError, f, host, x, w[0], w)
    refused(ValueError, f, host, x, w[:0], w[:0])
    refused(ValueError, f, host, x, torch.zeros(12, 7).t(), w)                 # channels apart
    refused(ValueError, f, host, x.transpose(0, 1), w, w)
    refused(ValueError, f, host, torch.zeros(1, 1).expand((1 << 20) + 1, 1), torch.zeros(2, 1), torch.zeros(2, 1))
    refused(ValueError, f, host, x, w, w, y=torch.zeros(3, 5, 8))
    g = ops.plan_gated_projection_grad
    assert g(host, torch.zeros(3, 5, 7), x, w, w).gradients.gate.shape == (7, 12)
    refused(ValueError, g, host, torch.zeros(3, 5, 8), x, w, w)
    refused(TypeError, g, host, torch.zeros(3, 5, 7).half(), x, w, w)


def test_refusals_of_the_losses(host, ops):  # noqa: F811
    x, w, labels = torch.zeros(3, 5, 12), torch.zeros(70, 12), torch.zeros(3, 5, dtype=torch.int64)
    f = ops.plan_vocabulary_loss
    assert f(host, x, w, labels).loss.shape == (3, 5)
    refused(TypeError, f, host, x.double(), w, labels)
    refused(TypeError, f, host, x, w.half(), labels)
    refused(TypeError, f, host, x, w, labels.float())
    refused(TypeError, f, host, x, w, labels.short())
    refused(ValueError, f, host, x, w, labels[:2])
    refused(ValueError, f, host, x, w, labels.t())
    refused(ValueError, f, host, x, w[:, :5], labels)
    refused(ValueError, f, host, x, w[:0], labels)
    refused(TypeError, f, host, x, w, labels, loss=torch.zeros(3, 5).half())
    g, one = ops.plan_vocabulary_loss_grad, torch.zeros(3, 5)
    assert g(host, one, x, w, labels, one).gradients.weight.shape == (70, 12)
    refused(ValueError, g, host, one[:2], x, w, labels, one)
    refused(TypeError, g, host, one.half(), x, w, labels, one)
    refused(TypeError, g, host, one, x, w, labels, one.half())
    words, values = torch.zeros(3, 5, 4, dtype=torch.int32), torch.zeros(3, 5, 4)
    t = ops.plan_teacher_loss
    assert t(host, x, w, words, values, 2.0).lse.shape == (3, 5)
    refused(TypeError, t, host, x, w, words, None)
    refused(TypeError, t, host, x, w, words, values.double())
    refused(TypeError, t, host, x, w, words.float(), values)
    refused(ValueError, t, host, x, w, words, values[..., :3])
    refused(ValueError, t, host, x, w, labels, one)
    refused(ValueError, t, host, x, w, words[..., :0], values[..., :0])
    refused(ValueError, t, host, x, w, torch.zeros(3, 5, 257, dtype=torch.int32), torch.zeros(3, 5, 257))
    for bad in (0.0, -1.0, NAN, INF):
        refused(ValueError, t, host, x, w, words, values, bad)
    refused(ValueError, ops.plan_teacher_loss_grad, host, one, x, w, words, values, one[:2])


def test_the_library_refuses_what_python_does_not_see(ops):  # noqa: F811
    """Null pointers, sizes out of range and a workspace too small come back as codes, without a launch."""
    from nengo_ocl_amd import _lib

    lib, bad, too_big, one = _lib.lib(), -1, -4, 1 << 20
    ref, need = ctypes.byref, ctypes.c_longlong(-1)
    for entry in (lib.nhip_layer_norm, lib.nhip_layer_norm_grad, lib.nhip_gated_projection, lib.nhip_gated_projection_grad,
                  lib.nhip_vocabulary_loss, lib.nhip_vocabulary_loss_grad):
        assert entry(None, None) == bad

    def loss(**more):
        given = dict(channels=8, words=70, rows=5, temperature=1.0, x=one, weight=one, x_stride=8, weight_stride=8, targets=one,
                     loss=one, lse=one, dloss=one, dx=one, dweight=one, workspace=one, workspace_bytes=1 << 40)
        return ops._LossArgs(**dict(given, **more))

    for entry in (lib.nhip_vocabulary_loss, lib.nhip_vocabulary_loss_grad):
        for more in (dict(type=3), dict(channels=0), dict(words=0), dict(rows=-1), dict(rows=(1 << 20) + 1), dict(top=257),
                     dict(top=-1), dict(temperature=0.0), dict(temperature=NAN), dict(x=0), dict(weight=0), dict(targets=0),
                     dict(lse=0), dict(top=2), dict(workspace=0), dict(workspace=one + 8), dict(words=(1 << 31) - 1)):
            assert entry(None, ref(loss(**more))) == bad, more
        assert entry(None, ref(loss(workspace_bytes=1))) == too_big
    assert lib.nhip_vocabulary_loss(None, ref(loss(loss=0))) == bad
    for key in ("dloss", "dx", "dweight"):
        assert lib.nhip_vocabulary_loss_grad(None, ref(loss(**{key: 0}))) == bad, key
    assert lib.nhip_vocabulary_loss_workspace(ref(loss()), None) == bad
    assert lib.nhip_vocabulary_loss_grad_workspace(ref(loss()), ref(need)) == 0 and need.value > 0

    def gated(**more):
        given = dict(channels=8, features=70, rows=5, x=one, gate=one, up=one, x_stride=8, gate_stride=8, up_stride=8, y=one, dy=one,
                     dy_stride=70, dx=one, dgate=one, dup=one, workspace=one, workspace_bytes=1 << 40)
        return ops._GatedArgs(**dict(given, **more))

    for entry in (lib.nhip_gated_projection, lib.nhip_gated_projection_grad):
        for more in (dict(type=-1), dict(activation=2), dict(channels=0), dict(features=0), dict(rows=-1), dict(rows=(1 << 20) + 1),
                     dict(x=0), dict(gate=0), dict(up=0)):
            assert entry(None, ref(gated(**more))) == bad, more
    assert lib.nhip_gated_projection(None, ref(gated(y=0))) == bad
    for key in ("dy", "dx", "dgate", "dup", "workspace"):
        assert lib.nhip_gated_projection_grad(None, ref(gated(**{key: 0}))) == bad, key
    assert lib.nhip_gated_projection_grad(None, ref(gated(workspace_bytes=1))) == too_big

    def norm(**more):
        given = dict(channels=8, rows=5, eps=1e-5, x=one, x_stride=8, weight=one, out=one, dout=one, dout_stride=8, dx=one,
                     dweight=one, dbias=one, workspace=one, workspace_bytes=1 << 30)
        return ops._LayerNormArgs(**dict(given, **more))

    for entry in (lib.nhip_layer_norm, lib.nhip_layer_norm_grad):
        for more in (dict(type=9), dict(channels=0), dict(rows=-1), dict(eps=-1.0), dict(eps=NAN), dict(x=0), dict(weight=0)):
            assert entry(None, ref(norm(**more))) == bad, more
    assert lib.nhip_layer_norm(None, ref(norm(out=0))) == bad
    assert lib.nhip_layer_norm(None, ref(norm(residual=one))) == bad             # no v_out
    for more in (dict(dout=0), dict(dx=0), dict(dweight=0), dict(dv=one), dict(bias=one, dbias=0), dict(workspace=0)):
        assert lib.nhip_layer_norm_grad(None, ref(norm(**more))) == bad, more
    assert lib.nhip_layer_norm_grad(None, ref(norm(workspace_bytes=1))) == too_big


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 16, 17, 64, 65])
@pytest.mark.parametrize("bad", [NAN, INF])
def test_few_rows_of_which_not_all_count(queue, ops, n, bad):  # noqa: F811
    """Few rows are computed all, also those that do not count: none, all, and some of them, whatever they hold."""
    for given, entry in ((loss_inputs(71, BF16, n, 72, 257, 0.5)[0], ops.plan_vocabulary_loss),
                         (teacher_inputs(72, BF16, n, 72, 257, 0.5, 9)[0], ops.plan_teacher_loss)):
        key = "labels" if "labels" in given else "indices"
        for left in (torch.arange(n) % 2 == 0, torch.ones(n, dtype=torch.bool), torch.zeros(n, dtype=torch.bool)):
            words = given[key].clone()
            words[words < 0] = 3
            words[words >= 257] = 4
            clean = run(entry(queue, **dict(given, **{key: words})))
            words[left.cuda()] = 257 if n % 2 else -1
            x = given["x"].clone()
            x[left.cuda()] = bad
            got = run(entry(queue, **dict(given, **{key: words, "x": x})))
            for a, b in zip(clean, got):
                assert torch.isfinite(a).all() and not b[left].any() and same(a[~left], b[~left])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [0, 3, 70, 300])
def test_events_span_all_launches(queue, ops, n):  # noqa: F811
    """A timed plan's events enclose all that its entry point launches; none are left for the next one."""
    for name, (given, make) in calls(ops, queue, 73, BF16, max(n, 1), 520, 9001).items():
        given = {k: t[:n] if t is not None and t.dim() and t.shape[0] == max(n, 1) and k not in ("weight", "bias", "gate", "up")
                 else t for k, t in given.items()}
        plan = make(**given)
        for _ in range(2):
            plan(profiling=True)
        plan.update_profiling()
        assert not queue.lib.nhip_launch_events_pending(), name
        assert plan.n_calls in (0, 2) if n == 0 else plan.n_calls == 2, name
        assert all(t >= 0.0 for t in plan.ctimes), name
        if n == 300 and name == "loss_grad":  # at least its 6 M N K operations at the highest rate there is
            assert min(plan.ctimes) > 6 * 0.6 * n * 520 * 9001 / 2.6e15, plan.ctimes


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, n, d, v", [(BF16, 40, 72, 257), (BF16, 300, 520, 9001), (F32, 300, 130, 310)])
def test_rows_that_are_one(queue, ops, dtype, n, d, v):  # noqa: F811
    """Inputs whose rows all lie at the same place (a stride of zero): the same as their copies, bit for bit."""
    for name, (given, make) in calls(ops, queue, 74, dtype, n, d, v).items():
        one = {k: given[k][:1].expand(n, -1) if k in ("x", "residual", "dy", "dout", "dv") and given.get(k) is not None else given[k]
               for k in given}
        if "labels" in one:
            one["labels"] = one["labels"].clone()
            one["labels"][0] = 1
        copies = {k: t.contiguous() if t is not None else None for k, t in one.items()}
        assert all(same(a, b) for a, b in zip(run(make(**one)), run(make(**copies)))), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_row_without_leading_axes(queue, ops, dtype):  # noqa: F811
    m = Maker(75)
    x, w = m.normal(72, dtype=dtype), m.normal(257, 72, dtype=dtype, scale=0.1)
    label = torch.tensor(5, device="cuda")
    for a, b in ((ops.vocabulary_loss(queue, x, w, label), ops.vocabulary_loss(queue, x[None], w, label[None])),
                 ((ops.gated_projection(queue, x, w, w),), (ops.gated_projection(queue, x[None], w, w),)),
                 (ops.layer_norm(queue, x, torch.ones(72, device="cuda"))[:1],
                  ops.layer_norm(queue, x[None], torch.ones(72, device="cuda"))[:1])):
        for s, t in zip(a, b):
            assert s.shape == t.shape[1:] and same(s, t[0])


@pytest.mark.gpu
def test_two_streams_at_once(ops):  # noqa: F811
    """Plans on two streams, under way together, give what they give alone."""
    from nengo_ocl_amd.hipraggedarray import Queue

    queues = [Queue(0), Queue(0)]
    plans = []
    for k, q in enumerate(queues):
        made = calls(ops, q, 76 + k, BF16, 300, 520, 9001)
        q.finish()
        torch.cuda.synchronize()
        plans.append([make(**given) for given, make in made.values()])
    alone = [[run(p) for p in of] for of in plans]
    for _ in range(3):
        for of in plans:
            for p in of:
                for t in outputs(p):
                    t.fill_(NAN)
        torch.cuda.synchronize()
        for a, b in zip(*plans):
            a.enqueue()
            b.enqueue()
        for q in queues:
            q.finish()
        for of, want in zip(plans, alone):
            for p, w in zip(of, want):
                assert all(same(s, t) for s, t in zip(outputs(p), w))
