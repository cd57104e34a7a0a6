"""Operators beside and behind blocks over tokens: layer norm, gated projection, losses over a vocabulary.

What a model of the blocks of `hipra_selective` needs to learn tokens: the norm with a mean, the
first half of a gated feed-forward block, and the losses at its end, cross entropy and the distance from a
teacher's largest logits, which form no logits in memory.  No counterpart in the reference.

=======================  ===========================  ====================================
immediate                bound to its arrays          C entry
=======================  ===========================  ====================================
layer_norm               plan_layer_norm              nhip_layer_norm
layer_norm_grad          plan_layer_norm_grad         nhip_layer_norm_grad
gated_projection         plan_gated_projection        nhip_gated_projection
gated_projection_grad    plan_gated_projection_grad   nhip_gated_projection_grad
vocabulary_loss          plan_vocabulary_loss         nhip_vocabulary_loss
vocabulary_loss_grad     plan_vocabulary_loss_grad    nhip_vocabulary_loss_grad
teacher_loss             plan_teacher_loss            nhip_vocabulary_loss
teacher_loss_grad        plan_teacher_loss_grad       nhip_vocabulary_loss_grad
=======================  ===========================  ====================================

Plans, queues, streams and arrays are as in `hipra_selective`: a ``plan_*`` function checks its arguments
and returns a `Plan` bound to them, the function without the prefix enqueues it once, in order with torch's
current stream.  Arrays are torch tensors or `DeviceArray`, float32, bfloat16 or float16, ``[..., channels]`` with
leading axes whose rows lie at one distance.  The norm's parameters are float32; the weights of products have
the type of what they multiply, ``[rows, channels]``.  Every plan has a workspace of its own, of the bytes that the
C library's ``*_workspace`` function names.  Outputs may not overlap inputs.  At most 2**20 rows go into a product, and 256 targets of a teacher to a row.

Sums, statistics, losses and the gradients of the norm's parameters are float32, added up in the same order on
every call.  A result of 16 bits is rounded once; the gradients of products go through one more rounding, that of
what stands between the two products (the gradient of the logits, of both projections) to the type of the
inputs.  In 16 bits the gradient of the logits is scaled by the largest magnitude of `dloss` first (in float16 to the
type's range) and the products' results back again; that of the projections is in float16, by a power of two, where
its largest magnitude is beyond the type or below 2**-8 (which takes their product once more).

Rows of the losses that do not count (a label outside the vocabulary, no target of a teacher) have a loss and a
logarithm of zero, no gradient, and take no part in any sum, whatever they hold; they cost nothing in the products.

Nothing is recorded for torch's autograd, also where an input has `requires_grad`: gradients come from the
``*_grad`` functions.
"""

import collections
import ctypes

from .hipra_selective import (_array, _Call, _flat, _like, _output, _packer, _parameter, _plain, _ptr, _type_code,
                              _workspace, c_float, c_int, c_ll, c_p)
from .hipraggedarray import _torch

MAX_ROWS = 1 << 20      # of a product
MAX_CHANNELS = 1 << 20  # of a product; features, too
MAX_TOP = 256           # targets of a row

LayerNormGradients = collections.namedtuple("LayerNormGradients", "x weight bias residual")
GatedGradients = collections.namedtuple("GatedGradients", "x gate up")
LossGradients = collections.namedtuple("LossGradients", "x weight")
_Like = collections.namedtuple("_Like", "shape dtype")


# ---------------------------------------------------------- structs of nengo_hip_tokens.h
class _LayerNormArgs(ctypes.Structure):
    _fields_ = [("type", c_int), ("channels", c_int), ("rows", c_ll), ("eps", c_float), ("x", c_p), ("residual", c_p),
                ("x_stride", c_ll), ("residual_stride", c_ll), ("weight", c_p), ("bias", c_p), ("out", c_p),
                ("v_out", c_p), ("dout", c_p), ("dv", c_p), ("dout_stride", c_ll), ("dv_stride", c_ll), ("dx", c_p),
                ("dweight", c_p), ("dbias", c_p), ("workspace", c_p), ("workspace_bytes", c_ll)]


class _GatedArgs(ctypes.Structure):
    _fields_ = [("type", c_int), ("activation", c_int), ("channels", c_int), ("features", c_int), ("rows", c_ll),
                ("x", c_p), ("gate", c_p), ("up", c_p), ("x_stride", c_ll), ("gate_stride", c_ll), ("up_stride", c_ll),
                ("y", c_p), ("dy", c_p), ("dy_stride", c_ll), ("dx", c_p), ("dgate", c_p), ("dup", c_p),
                ("workspace", c_p), ("workspace_bytes", c_ll)]


class _LossArgs(ctypes.Structure):
    _fields_ = [("type", c_int), ("channels", c_int), ("words", c_int), ("top", c_int), ("wide_targets", c_int),
                ("logits_type", c_int), ("rows", c_ll), ("temperature", c_float), ("x", c_p), ("weight", c_p),
                ("x_stride", c_ll), ("weight_stride", c_ll), ("targets", c_p), ("target_logits", c_p), ("loss", c_p),
                ("lse", c_p), ("dloss", c_p), ("dx", c_p), ("dweight", c_p), ("workspace", c_p),
                ("workspace_bytes", c_ll)]


# -------------------------------------------------------------------------------- layer norm
def _norm(queue, x, weight, bias, residual, eps):
    x = _plain(x)
    code = _type_code("x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x has shape %s: [..., channels] is wanted" % (tuple(x.shape),))
    if not eps >= 0.0:
        raise ValueError("eps is %r" % (eps,))
    d = x.shape[-1]
    if weight is None:
        raise TypeError("weight is None")
    weight, bias = _parameter(queue, "weight", weight, (d,)), _parameter(queue, "bias", bias, (d,))
    args = _LayerNormArgs(type=code, channels=d, rows=x.numel() // d, eps=float(eps), weight=_ptr(weight), bias=_ptr(bias))
    rows, args.x_stride = _flat(queue, "x", x, x)
    args.x = _ptr(rows)
    keep = [weight, bias, rows]
    if residual is not None:
        residual, args.residual_stride = _flat(queue, "residual", residual, x)
        args.residual = _ptr(residual)
        keep.append(residual)
    return args, x, keep


def _layer_norm(queue, x, weight, bias=None, residual=None, eps=1e-5, out=None, v=None):
    args, x, keep = _norm(queue, x, weight, bias, residual, eps)
    out = _like(x) if out is None else _output(queue, "out", out, x.shape, x.dtype)
    if v is not None and residual is None:
        raise ValueError("v is written with a residual only")
    v = None if residual is None else _output(queue, "v", v, x.shape, x.dtype)
    args.out, args.v_out = _ptr(out), _ptr(v)
    return _Call(queue.lib.nhip_layer_norm, args, keep + [out, v], "hip_layer_norm", out=out, v=v)


def plan_layer_norm(queue, x, weight, bias=None, residual=None, eps=1e-5, out=None, v=None, tag=None):
    """``out = (v - mean(v)) / sqrt(mean((v - mean(v))**2) + eps) * weight + bias`` over the last axis, with
    ``v = x``, or ``residual + x`` where there is a `residual` (like x).  `weight`, `bias` ``[channels]`` (float32).
    ``plan.out``, and ``plan.v`` with a residual."""
    return _layer_norm(queue, x, weight, bias, residual, eps, out, v).plan(queue, tag)


def layer_norm(queue, x, weight, bias=None, residual=None, eps=1e-5):
    """(out, v or None): see `plan_layer_norm`."""
    got = _layer_norm(queue, x, weight, bias, residual, eps).now(queue)
    return got["out"], got["v"]


def _layer_norm_grad(queue, dout, x, weight, bias=None, residual=None, eps=1e-5, dv=None):
    torch = _torch()
    args, x, keep = _norm(queue, x, weight, bias, residual, eps)
    dout, args.dout_stride = _flat(queue, "dout", dout, x)
    args.dout = _ptr(dout)
    if dv is not None:
        if residual is None:
            raise ValueError("dv goes with a residual")
        dv, args.dv_stride = _flat(queue, "dv", dv, x)
        args.dv = _ptr(dv)
    dx = _output(queue, "", None, x.shape, x.dtype)
    dweight, dbias = (_output(queue, "", None, (args.channels,), torch.float32) for _ in range(2))
    args.dx, args.dweight, args.dbias = _ptr(dx), _ptr(dweight), _ptr(dbias)
    space = _workspace(queue, args, queue.lib.nhip_layer_norm_grad_workspace)
    got = LayerNormGradients(dx, dweight, None if bias is None else dbias, None if residual is None else dx)
    return _Call(queue.lib.nhip_layer_norm_grad, args, keep + [dout, dv, dbias, space, got], "hip_layer_norm_grad",
                 gradients=got)


def plan_layer_norm_grad(queue, dout, x, weight, bias=None, residual=None, eps=1e-5, dv=None, tag=None):
    """The gradient of `plan_layer_norm`, from `dout` and (with a residual) `dv`; ``plan.gradients``: those of
    weight and bias are float32, that of the residual is the array of x's, which it equals."""
    return _layer_norm_grad(queue, dout, x, weight, bias, residual, eps, dv).plan(queue, tag)


def layer_norm_grad(queue, dout, x, weight, bias=None, residual=None, eps=1e-5, dv=None):
    """`LayerNormGradients` (x, weight, bias, residual): see `plan_layer_norm_grad`."""
    return _layer_norm_grad(queue, dout, x, weight, bias, residual, eps, dv).now(queue)["gradients"]


# -------------------------------------------------------------------------- gated projection
_activations = {"silu": 0, "gelu": 1}


def _product_rows(queue, x):
    """(tensor, its rows, their stride, their number, channels) of what a product multiplies, [..., channels]."""
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_CHANNELS:
        raise ValueError("x has shape %s: [..., channels] with 1 to %d channels is wanted" % (tuple(x.shape), MAX_CHANNELS))
    d = x.shape[-1]
    n = x.numel() // d
    if n > MAX_ROWS:
        raise ValueError("x has %d rows: at most %d in a call" % (n, MAX_ROWS))
    rows, stride = _flat(queue, "x", x, x)
    return rows, stride, n, d


def _weights(queue, name, t, d, dtype, rows=None):
    t = _plain(t)
    if t.dim() != 2 or t.shape[0] < 1:
        raise ValueError("%s has shape %s: [rows, channels] is wanted" % (name, tuple(t.shape)))
    t = _array(queue, name, t, (t.shape[0] if rows is None else rows, d), dtype)
    return t, t.stride(0)


def _gated(queue, x, gate, up, activation):
    x = _plain(x)
    code = _type_code("x", x)
    if activation not in _activations:
        raise ValueError("activation is %r: 'silu' and 'gelu' are known" % (activation,))
    rows, x_stride, n, d = _product_rows(queue, x)
    gate, gate_stride = _weights(queue, "gate", gate, d, x.dtype)
    f = gate.shape[0]
    if f > MAX_CHANNELS:
        raise ValueError("gate has %d features: at most %d in a call" % (f, MAX_CHANNELS))
    up, up_stride = _weights(queue, "up", up, d, x.dtype, f)
    args = _gated_args(code, _activations[activation], d, f, n, _ptr(rows), gate.data_ptr(), up.data_ptr(), x_stride,
                       gate_stride, up_stride, 0, 0, 0, 0, 0, 0, 0, 0)
    return args, x, x.shape[:-1] + (f,), [rows, gate, up]


_gated_args = _packer(_GatedArgs)


def _gated_projection(queue, x, gate, up, activation="silu", y=None):
    args, x, shape, keep = _gated(queue, x, gate, up, activation)
    y = _output(queue, "y", y, shape, x.dtype)
    args.y = _ptr(y)
    space = _workspace(queue, args, queue.lib.nhip_gated_projection_workspace)
    return _Call(queue.lib.nhip_gated_projection, args, keep + [y, space], "hip_gated_projection", y=y)


def plan_gated_projection(queue, x, gate, up, activation="silu", y=None, tag=None):
    """``y = f(x gate') * (x up')``, the first half of a gated feed-forward block: `x` ``[..., channels]``, `gate` and
    `up` ``[features, channels]`` (halves of one array, or two); f is v sigmoid(v) (``"silu"``) or v Phi(v)
    (``"gelu"``, with the normal distribution itself).  Few rows (single tokens) and many.  ``plan.y``
    ``[..., features]``."""
    return _gated_projection(queue, x, gate, up, activation, y).plan(queue, tag)


def gated_projection(queue, x, gate, up, activation="silu"):
    """y: see `plan_gated_projection`."""
    return _gated_projection(queue, x, gate, up, activation).now(queue)["y"]


def _gated_projection_grad(queue, dy, x, gate, up, activation="silu"):
    args, x, shape, keep = _gated(queue, x, gate, up, activation)
    dy, args.dy_stride = _flat(queue, "dy", _plain(dy), _Like(shape, x.dtype))
    dx = _output(queue, "", None, x.shape, x.dtype)
    dgate, dup = (_output(queue, "", None, (args.features, args.channels), x.dtype) for _ in range(2))
    args.dy, args.dx, args.dgate, args.dup = _ptr(dy), _ptr(dx), _ptr(dgate), _ptr(dup)
    space = _workspace(queue, args, queue.lib.nhip_gated_projection_grad_workspace)
    got = GatedGradients(dx, dgate, dup)
    return _Call(queue.lib.nhip_gated_projection_grad, args, keep + [dy, space, got], "hip_gated_projection_grad",
                 gradients=got)


def plan_gated_projection_grad(queue, dy, x, gate, up, activation="silu", tag=None):
    """The gradient of `plan_gated_projection`, from `dy`; it needs nothing that the forward pass computed.
    ``plan.gradients``, of the type of x."""
    return _gated_projection_grad(queue, dy, x, gate, up, activation).plan(queue, tag)


def gated_projection_grad(queue, dy, x, gate, up, activation="silu"):
    """`GatedGradients` (x, gate, up): see `plan_gated_projection_grad`."""
    return _gated_projection_grad(queue, dy, x, gate, up, activation).now(queue)["gradients"]


# -------------------------------------------------------------------- losses over a vocabulary
_loss_args = _packer(_LossArgs)


def _words(queue, name, t, shape):
    """(tensor, whether it has 64 bits) of numbers of words."""
    torch = _torch()
    t = _plain(t)
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError("%s is %s: int32 or int64 are known" % (name, t.dtype))
    return _array(queue, name, t, shape, None, contiguous=True), int(t.dtype == torch.int64)


def _loss(queue, x, weight, targets, logits=None, temperature=1.0):
    x = _plain(x)
    code = _type_code("x", x)
    rows, x_stride, n, d = _product_rows(queue, x)
    weight, w_stride = _weights(queue, "weight", weight, d, x.dtype)
    if weight.shape[0] > 1 << 30:
        raise ValueError("weight has %d words: at most %d" % (weight.shape[0], 1 << 30))
    lead, top, logits_code = x.shape[:-1], 0, 0
    if logits is None:
        targets, wide = _words(queue, "labels", targets, lead)
    else:
        if not 2.0 ** -126 <= temperature <= 2.0 ** 126:
            raise ValueError("temperature is %r: 2**-126 to 2**126, numbers of float32 and their reciprocals" % (temperature,))
        targets = _plain(targets)
        if targets.dim() != len(lead) + 1 or not 1 <= targets.shape[-1] <= MAX_TOP:
            raise ValueError("indices has shape %s: %s with 1 to %d targets is wanted"
                             % (tuple(targets.shape), tuple(lead) + ("targets",), MAX_TOP))
        top = targets.shape[-1]
        targets, wide = _words(queue, "indices", targets, lead + (top,))
        logits = _plain(logits)
        logits_code = _type_code("logits", logits)
        logits = _array(queue, "logits", logits, lead + (top,), None, contiguous=True)
    args = _loss_args(code, d, weight.shape[0], top, wide, logits_code, n, float(temperature), _ptr(rows),
                      weight.data_ptr(), x_stride, w_stride, _ptr(targets), _ptr(logits), 0, 0, 0, 0, 0, 0, 0)
    return args, x, weight, lead, [rows, weight, targets, logits]


def _loss_forward(queue, name, given, loss, lse):
    args, x, _, lead, keep = given
    loss, lse = (_output(queue, k, v, lead, _torch().float32) for k, v in (("loss", loss), ("lse", lse)))
    args.loss, args.lse = _ptr(loss), _ptr(lse)
    space = _workspace(queue, args, queue.lib.nhip_vocabulary_loss_workspace)
    return _Call(queue.lib.nhip_vocabulary_loss, args, keep + [loss, lse, space], name, loss=loss, lse=lse)


def _loss_gradient(queue, name, given, dloss, lse):
    args, x, weight, lead, keep = given
    f32 = _torch().float32
    dloss, lse = (_array(queue, k, _plain(v), lead, f32, contiguous=True) for k, v in (("dloss", dloss), ("lse", lse)))
    dx = _output(queue, "", None, x.shape, x.dtype)
    dweight = _output(queue, "", None, weight.shape, x.dtype)
    args.dloss, args.lse, args.dx, args.dweight = _ptr(dloss), _ptr(lse), _ptr(dx), _ptr(dweight)
    space = _workspace(queue, args, queue.lib.nhip_vocabulary_loss_grad_workspace)
    got = LossGradients(dx, dweight)
    return _Call(queue.lib.nhip_vocabulary_loss_grad, args, keep + [dloss, lse, space, got], name, gradients=got)


def plan_vocabulary_loss(queue, x, weight, labels, loss=None, lse=None, tag=None):
    """The cross entropy of ``softmax(x weight')`` against `labels`, token by token, without the logits in memory:
    `x` ``[..., channels]``, `weight` ``[words, channels]``, `labels` ``[...]`` (int32 or int64; one outside the
    vocabulary: the token does not count, and has zeros).  ``plan.loss`` and ``plan.lse``, the logarithm of the sum
    of the logits' exponentials, ``[...]`` (float32)."""
    return _loss_forward(queue, "hip_vocabulary_loss", _loss(queue, x, weight, labels), loss, lse).plan(queue, tag)


def vocabulary_loss(queue, x, weight, labels):
    """(loss, lse): see `plan_vocabulary_loss`."""
    got = _loss_forward(queue, "hip_vocabulary_loss", _loss(queue, x, weight, labels), None, None).now(queue)
    return got["loss"], got["lse"]


def plan_vocabulary_loss_grad(queue, dloss, x, weight, labels, lse, tag=None):
    """The gradient of `plan_vocabulary_loss`, from `dloss` ``[...]`` (float32: a mean over n tokens has 1 / n) and the
    `lse` that it wrote; ``plan.gradients``, of the type of x."""
    return _loss_gradient(queue, "hip_vocabulary_loss_grad", _loss(queue, x, weight, labels), dloss, lse).plan(queue, tag)


def vocabulary_loss_grad(queue, dloss, x, weight, labels, lse):
    """`LossGradients` (x, weight): see `plan_vocabulary_loss_grad`."""
    given = _loss(queue, x, weight, labels)
    return _loss_gradient(queue, "hip_vocabulary_loss_grad", given, dloss, lse).now(queue)["gradients"]


def _teacher(queue, x, weight, indices, logits, temperature):
    if logits is None:
        raise TypeError("logits is None")
    return _loss(queue, x, weight, indices, logits, temperature)


def plan_teacher_loss(queue, x, weight, indices, logits, temperature=1.0, loss=None, lse=None, tag=None):
    """How far ``p = softmax(x weight' / temperature)`` is from a teacher of whom the largest logits are known:
    ``sum_k q[k] (log q[k] - log p[indices[k]])`` with ``q = softmax(logits / temperature)`` over these alone.
    `indices` ``[..., k]`` (int32 or int64) are their words, `logits` ``[..., k]`` (float32, bfloat16 or float16) their
    values; `temperature` is 2**-126 to 2**126.  An index outside the vocabulary, or a value of -inf, is left out; a token without any does not
    count, and has zeros; an index named twice is two targets, whose shares of p's gradient add up.  ``plan.loss``,
    ``plan.lse`` as for `plan_vocabulary_loss`, the latter of the logits over the temperature."""
    given = _teacher(queue, x, weight, indices, logits, temperature)
    return _loss_forward(queue, "hip_teacher_loss", given, loss, lse).plan(queue, tag)


def teacher_loss(queue, x, weight, indices, logits, temperature=1.0):
    """(loss, lse): see `plan_teacher_loss`."""
    got = _loss_forward(queue, "hip_teacher_loss", _teacher(queue, x, weight, indices, logits, temperature), None,
                        None).now(queue)
    return got["loss"], got["lse"]


def plan_teacher_loss_grad(queue, dloss, x, weight, indices, logits, lse, temperature=1.0, tag=None):
    """The gradient of `plan_teacher_loss` with respect to x and weight, from `dloss` ``[...]`` (float32) and the `lse`
    that it wrote; ``plan.gradients``, of the type of x."""
    given = _teacher(queue, x, weight, indices, logits, temperature)
    return _loss_gradient(queue, "hip_teacher_loss_grad", given, dloss, lse).plan(queue, tag)


def teacher_loss_grad(queue, dloss, x, weight, indices, logits, lse, temperature=1.0):
    """`LossGradients` (x, weight): see `plan_teacher_loss_grad`."""
    given = _teacher(queue, x, weight, indices, logits, temperature)
    return _loss_gradient(queue, "hip_teacher_loss_grad", given, dloss, lse).now(queue)["gradients"]
