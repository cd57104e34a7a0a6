"""Operators of blocks that filter selectively: short causal convolution, selective scan, gated norm.

A synapse of the simulator is a linear filter whose matrices are constant
(`hipra_nonlinearities.plan_linearfilter`).  A selective scan is one whose step, input and
output matrices come from the signal itself; with the short convolution in front of it and
the gated norm around it, it makes a block that is trained on sequences and then answers
token by token.  No counterpart in the reference.

=====================  ===========================  ====================================
immediate              bound to its arrays          C entry
=====================  ===========================  ====================================
causal_conv            plan_causal_conv             nhip_causal_conv
causal_conv_grad       plan_causal_conv_grad        nhip_causal_conv_grad
causal_conv_step       plan_causal_conv_step        nhip_causal_conv_step
selective_scan         plan_selective_scan          nhip_selective_scan
selective_scan_grad    plan_selective_scan_grad     nhip_selective_scan_grad
selective_step         plan_selective_step          nhip_selective_step
block_norm             plan_block_norm              nhip_block_norm
block_norm_grad        plan_block_norm_grad         nhip_block_norm_grad
=====================  ===========================  ====================================

A ``plan_*`` function checks its arguments and returns a `Plan` bound to them, with the
arrays that it writes as attributes; such plans go into a `Plans` list (a decoding step is
recorded once and replayed).  The function without the prefix makes the plan and enqueues
it once, in order with torch's current stream whatever stream the queue has.

Arrays are torch tensors or `DeviceArray`, on the queue's device: float32, bfloat16 or
float16 (parameters and states: float32).  Sequences lie side by side, ``[S, L, ...]``, or,
with ``starts`` (int32, S + 1 offsets on the device, the layout of a ragged array's
``starts``), back to back, ``[T, ...]``; sequences may be empty.  Rows may have any
strides, the last axis has stride one.  ValueError and TypeError say what does not fit.

What the offsets on the device hold is not checked: they are cut to the tokens that there are,
results of tokens that no sequence holds are not written, and those of sequences that overlap
are undefined.  Outputs may not overlap inputs.  What would take a launch of 2**24 work-groups is
refused (`HipError`) before any.

Sums, states and parameters' gradients are float32 and added up in the same order on every call.
A result of 16 bits is rounded once: besides that rounding it is off by less than 2**-15 of the
magnitudes of the terms that it is the sum of (bfloat16 scans, whose states and weights go into
the matrix products as two bfloat16 parts; the state itself gains float32 values).

An input that is no finite number reaches what depends on it, no earlier token and no other
sequence; in the scan's gradient, all tokens of its chunk of 64 (32 with more than 128 states).
With `softplus`, a `dt` of -inf or of the lowest value of its type masks a token: its step is zero,
and the state passes it unchanged.

Nothing is recorded for torch's autograd, also where an input has `requires_grad`: gradients come
from the ``*_grad`` functions.
"""

import collections
import ctypes
import struct

from . import _lib
from .hipraggedarray import DeviceArray, _torch
from .plan import Plan

c_int, c_ll, c_float, c_p = ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_void_p

MAX_WIDTH = 8     # taps of the convolution
MAX_STATES = 256  # states per row of a head
MAX_TOKENS = 0x7fff0000  # of a call

ConvGradients = collections.namedtuple("ConvGradients", "x weight bias initial")
ScanGradients = collections.namedtuple("ScanGradients", "x dt A B C D dt_bias initial")
NormGradients = collections.namedtuple("NormGradients", "x weight gate residual scale")


# ------------------------------------------------------- structs of nengo_hip_selective.h
class _Rows(ctypes.Structure):
    _fields_ = [("p", c_p), ("seq", c_ll), ("token", c_ll), ("head", c_ll)]


class _Tokens(ctypes.Structure):
    _fields_ = [("starts", c_p), ("n_tokens", c_ll), ("n_seqs", c_int), ("length", c_int)]


class _ConvArgs(ctypes.Structure):
    _fields_ = [("tokens", _Tokens), ("type", c_int), ("channels", c_int), ("width", c_int), ("silu", c_int),
                ("x", _Rows), ("dy", _Rows), ("weight", c_p), ("bias", c_p), ("initial", c_p), ("y", c_p),
                ("final", c_p), ("dfinal", c_p), ("dx", c_p), ("dinitial", c_p), ("dweight", c_p), ("dbias", c_p),
                ("workspace", c_p), ("workspace_bytes", c_ll)]


class _ConvStepArgs(ctypes.Structure):
    _fields_ = [("type", c_int), ("channels", c_int), ("width", c_int), ("silu", c_int), ("n", c_int),
                ("n_slots", c_int), ("slots", c_p), ("x", c_p), ("x_stride", c_ll), ("state_stride", c_ll),
                ("weight", c_p), ("bias", c_p), ("state", c_p), ("y", c_p)]


class _ScanArgs(ctypes.Structure):
    _fields_ = [("tokens", _Tokens), ("type", c_int), ("dt_type", c_int), ("softplus", c_int), ("n_heads", c_int),
                ("dim", c_int), ("n_groups", c_int), ("states", c_int), ("x", _Rows), ("dt", _Rows), ("B", _Rows),
                ("C", _Rows), ("dy", _Rows), ("A", c_p), ("D", c_p), ("dt_bias", c_p), ("initial", c_p),
                ("dfinal", c_p), ("y", c_p), ("final", c_p), ("dx", c_p), ("ddt", c_p), ("dB", c_p), ("dC", c_p),
                ("dA", c_p), ("dD", c_p), ("ddt_bias", c_p), ("dinitial", c_p), ("workspace", c_p),
                ("workspace_bytes", c_ll)]


class _ScanStepArgs(ctypes.Structure):
    _fields_ = [("type", c_int), ("dt_type", c_int), ("softplus", c_int), ("n_heads", c_int), ("dim", c_int),
                ("n_groups", c_int), ("states", c_int), ("n", c_int), ("n_slots", c_int), ("slots", c_p),
                ("x", _Rows), ("dt", _Rows), ("B", _Rows), ("C", _Rows), ("A", c_p), ("D", c_p), ("dt_bias", c_p),
                ("state", c_p), ("state_stride", c_ll), ("y", c_p)]


class _NormArgs(ctypes.Structure):
    _fields_ = [("type", c_int), ("channels", c_int), ("groups", c_int), ("after", c_int), ("rows", c_ll),
                ("eps", c_float), ("x", c_p), ("gate", c_p), ("residual", c_p), ("x_stride", c_ll),
                ("gate_stride", c_ll), ("residual_stride", c_ll), ("weight", c_p), ("scale", c_p), ("out", c_p),
                ("v_out", c_p), ("dout", c_p), ("dv", c_p), ("dout_stride", c_ll), ("dv_stride", c_ll), ("dx", c_p),
                ("dgate", c_p), ("dresidual", c_p), ("dweight", c_p), ("dscale", c_p), ("workspace", c_p),
                ("workspace_bytes", c_ll)]


def _packer(kind):
    """A function of all fields of a struct in their order, those of structs in it among them, to the struct: where
    a call takes ten microseconds, to set 20 fields by their names takes four of them."""
    form, at = "@", 0

    def add(fields, base):
        nonlocal form, at
        for name, t in fields._fields_:
            place = base + getattr(fields, name).offset
            if issubclass(t, ctypes.Structure):
                add(t, place)
            else:
                form += "%dx" % (place - at) * (place > at) + {c_int: "i", c_ll: "q", c_p: "P", c_float: "f"}[t]
                at = place + ctypes.sizeof(t)

    add(kind, 0)
    form = struct.Struct("=" + form[1:].replace("P", "Q") + "%dx" % (ctypes.sizeof(kind) - at))
    return lambda *values: kind.from_buffer_copy(form.pack(*values))


_conv_step_args, _scan_step_args = _packer(_ConvStepArgs), _packer(_ScanStepArgs)


# ------------------------------------------------------------------------ argument checks
_codes = {}


def _type_code(name, t):
    if not _codes:
        torch = _torch()
        _codes.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
    code = _codes.get(t.dtype)
    if code is None:
        raise TypeError("%s is %s: float32, bfloat16 or float16 are known" % (name, t.dtype))
    return code


def _array(queue, name, t, shape, dtype, contiguous=False):
    """The tensor behind an argument, after its checks: its shape, type, device and the stride of its last axis."""
    if isinstance(t, DeviceArray):
        t = t.tensor
    if dtype is not None and t.dtype != dtype:
        raise TypeError("%s is %s, not %s" % (name, t.dtype, dtype))
    if t.shape != shape:
        raise ValueError("%s has shape %s, not %s" % (name, tuple(t.shape), tuple(shape)))
    if t.device != queue.device:
        raise ValueError("%s is on %s, the queue on %s" % (name, t.device, queue.device))
    if contiguous:
        if not t.is_contiguous():
            raise ValueError("%s has to be contiguous" % name)
    elif not t.is_contiguous() and shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError("%s has stride %d along its last axis, not 1" % (name, t.stride(-1)))
    return t


def _parameter(queue, name, t, shape):
    return None if t is None else _array(queue, name, t, shape, _torch().float32, True)


def _output(queue, name, t, shape, dtype):
    """An array to write: the caller's, or a new one."""
    if t is None:
        return _torch().empty(shape, dtype=dtype, device=queue.device)
    return _array(queue, name, t, shape, dtype, contiguous=True)


def _like(x):
    """A new array of the shape and type of `x`, contiguous."""
    return _torch().empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _plain(t):
    return t.tensor if isinstance(t, DeviceArray) else t


def _tokens(queue, x, starts, axes):
    """(struct, leading sizes of row arrays, sequences, the tensor of starts) of `x` with `axes` axes behind the tokens."""
    lead = x.dim() - axes
    if starts is None:
        if lead != 2:
            raise ValueError("x has %d axes: [S, L, ...] needs %d, back-to-back sequences need `starts`"
                             % (x.dim(), 2 + axes))
        s, n = x.shape[0], x.shape[1]
        if s * n > MAX_TOKENS:
            raise ValueError("%d tokens: at most %d in a call" % (s * n, MAX_TOKENS))
        return _Tokens(None, s * n, s, n), (s, n), s, None
    if lead != 1:
        raise ValueError("x has %d axes: with `starts` it has %d, [T, ...]" % (x.dim(), 1 + axes))
    starts = _plain(starts)
    if starts.dim() != 1 or starts.shape[0] < 1:
        raise ValueError("starts has shape %s: S + 1 offsets are wanted" % (tuple(starts.shape),))
    starts = _array(queue, "starts", starts, starts.shape, _torch().int32, contiguous=True)
    t, s = x.shape[0], starts.shape[0] - 1
    if t > MAX_TOKENS:
        raise ValueError("%d tokens: at most %d in a call" % (t, MAX_TOKENS))
    return _Tokens(starts.data_ptr(), t, s, 0), (t,), s, starts


def _rows(t, lead, heads=False):
    """How the rows of `t` lie, as a `_Rows`: [S, L, (heads,) ...] or [T, (heads,) ...]."""
    st = t.stride()
    if lead == 2:
        return t.data_ptr(), st[0], st[1], st[2] if heads else 0
    return t.data_ptr(), 0, st[0], st[1] if heads else 0


def _activation(name):
    if name not in (None, "silu"):
        raise ValueError("activation is %r: None and 'silu' are known" % (name,))
    return int(name == "silu")


def _slots(queue, slots, n, n_slots):
    if slots is None:
        if n > n_slots:
            raise ValueError("%d requests for a state with %d slots" % (n, n_slots))
        return None
    return _array(queue, "slots", slots, (n,), _torch().int32, contiguous=True)


def _workspace(queue, args, entry):
    need = c_ll()
    _lib.check(entry(ctypes.byref(args), ctypes.byref(need)), "workspace")
    if not need.value:
        return None
    space = _torch().empty(need.value, dtype=_torch().uint8, device=queue.device)
    args.workspace, args.workspace_bytes = space.data_ptr(), need.value
    return space


def _current_stream(device):
    """The handle of torch's current stream.  (Where torch has the function that gives the handle alone: an object for
    the stream costs two microseconds, as much as half a launch.)"""
    torch = _torch()
    try:
        return torch._C._cuda_getCurrentRawStream(device)
    except AttributeError:
        return torch.cuda.current_stream(device).cuda_stream


class _Call:
    """An entry point with its arguments, what they point into, and the arrays that it writes by name."""

    __slots__ = ("entry", "args", "keep", "name", "results")

    def __init__(self, entry, args, keep, name, **results):
        self.entry, self.args, self.keep, self.name, self.results = entry, args, keep, name, results

    def plan(self, queue, tag):
        plan = Plan(queue, self.entry, (ctypes.byref(self.args),), gsize=(64,), full_args=(self,), name=self.name,
                    tag=tag)
        for key, value in self.results.items():
            setattr(plan, key, value)
        return plan

    def now(self, queue):
        """Enqueued once, in order with torch's current stream: the arrays were made there, and are used there next."""
        if _current_stream(queue.device.index) == queue.stream.cuda_stream:
            _lib.check(self.entry(queue.handle, ctypes.byref(self.args)), self.name)
        else:
            current = _torch().cuda.current_stream(queue.device)
            queue.stream.wait_stream(current)
            _lib.check(self.entry(queue.handle, ctypes.byref(self.args)), self.name)
            current.wait_stream(queue.stream)
        return self.results


# ----------------------------------------------------------------- short causal convolution
def _conv(queue, x, weight, bias, activation, initial, starts):
    x, weight = _plain(x), _plain(weight)
    code = _type_code("x", x)
    if weight.dim() != 2 or not 1 <= weight.shape[1] <= MAX_WIDTH:
        raise ValueError("weight has shape %s: [channels, width] with a width of 1 to %d is wanted"
                         % (tuple(weight.shape), MAX_WIDTH))
    d, k = weight.shape
    tokens, lead, s, starts = _tokens(queue, x, starts, 1)
    x = _array(queue, "x", x, lead + (d,), None)
    weight, bias = _parameter(queue, "weight", weight, (d, k)), _parameter(queue, "bias", bias, (d,))
    if initial is not None:
        initial = _array(queue, "initial", initial, (s, k - 1, d), x.dtype, contiguous=True)
    if d < 1:
        raise ValueError("x has no channels")
    args = _ConvArgs(tokens=tokens, type=code, channels=d, width=k, silu=_activation(activation),
                     x=_rows(x, len(lead)), weight=_ptr(weight), bias=_ptr(bias), initial=_ptr(initial))
    return args, x, lead, (s, k - 1, d), [x, weight, bias, initial, starts]


def _causal_conv(queue, x, weight, bias=None, activation=None, initial=None, starts=None, y=None, final=None):
    args, x, lead, ends, keep = _conv(queue, x, weight, bias, activation, initial, starts)
    y = _output(queue, "y", y, x.shape, x.dtype)
    final = _output(queue, "final", final, ends, x.dtype)
    args.y, args.final = _ptr(y), _ptr(final)
    return _Call(queue.lib.nhip_causal_conv, args, keep + [y, final],
                 "hip_causal_conv", y=y, final=final)


def plan_causal_conv(queue, x, weight, bias=None, activation=None, initial=None, starts=None, y=None, final=None,
                     tag=None):
    """``y[t] = f(bias + sum_k weight[:, k] * x[t - width + 1 + k])``, channel by channel; f is the
    identity or (``activation="silu"``) v sigmoid(v).  In front of a sequence's first token lies
    `initial` ``[S, width - 1, channels]``, or zeros.  ``plan.y``, and ``plan.final``: the last
    width - 1 inputs of each sequence, what `causal_conv_step` goes on with."""
    return _causal_conv(queue, x, weight, bias, activation, initial, starts, y, final).plan(queue, tag)


def causal_conv(queue, x, weight, bias=None, activation=None, initial=None, starts=None):
    """(y, final): see `plan_causal_conv`."""
    got = _causal_conv(queue, x, weight, bias, activation, initial, starts).now(queue)
    return got["y"], got["final"]


def _causal_conv_grad(queue, dy, x, weight, bias=None, activation=None, initial=None, starts=None, dfinal=None):
    torch = _torch()
    args, x, lead, ends, keep = _conv(queue, x, weight, bias, activation, initial, starts)
    dy = _array(queue, "dy", dy, x.shape, x.dtype)
    if dfinal is not None:
        dfinal = _array(queue, "dfinal", dfinal, ends, x.dtype, contiguous=True)
    d, k = args.channels, args.width
    dx, dweight = _output(queue, "dx", None, x.shape, x.dtype), _output(queue, "dweight", None, (d, k), torch.float32)
    dbias = _output(queue, "dbias", None, (d,), torch.float32)
    dinitial = None if initial is None else _output(queue, "dinitial", None, ends, x.dtype)
    args.dy, args.dfinal = _rows(dy, len(lead)), _ptr(dfinal)
    args.dx, args.dinitial, args.dweight, args.dbias = _ptr(dx), _ptr(dinitial), _ptr(dweight), _ptr(dbias)
    space = _workspace(queue, args, queue.lib.nhip_causal_conv_grad_workspace)
    got = ConvGradients(dx, dweight, None if bias is None else dbias, dinitial)
    return _Call(queue.lib.nhip_causal_conv_grad, args, keep + [dy, dfinal, dbias, space, got],
                 "hip_causal_conv_grad", gradients=got)


def plan_causal_conv_grad(queue, dy, x, weight, bias=None, activation=None, initial=None, starts=None, dfinal=None,
                          tag=None):
    """The gradient of `plan_causal_conv`, from `dy` and (where it went on) `dfinal`; ``plan.gradients``."""
    return _causal_conv_grad(queue, dy, x, weight, bias, activation, initial, starts, dfinal).plan(queue, tag)


def causal_conv_grad(queue, dy, x, weight, bias=None, activation=None, initial=None, starts=None, dfinal=None):
    """`ConvGradients` (x, weight, bias, initial): see `plan_causal_conv_grad`."""
    got = _causal_conv_grad(queue, dy, x, weight, bias, activation, initial, starts, dfinal).now(queue)
    return got["gradients"]


def _causal_conv_step(queue, state, x, weight, bias=None, activation=None, slots=None, y=None):
    state, x, weight = _plain(state), _plain(x), _plain(weight)
    code = _type_code("x", x)
    if weight.dim() != 2 or not 1 <= weight.shape[1] <= MAX_WIDTH:
        raise ValueError("weight has shape %s: [channels, width] with a width of 1 to %d is wanted"
                         % (tuple(weight.shape), MAX_WIDTH))
    if state.dim() != 3 or x.dim() != 2:
        raise ValueError("state and x have %d and %d axes, not 3 and 2" % (state.dim(), x.dim()))
    (d, k), n, n_slots = weight.shape, x.shape[0], state.shape[0]
    x = _array(queue, "x", x, (n, d), None)
    state = _array(queue, "state", state, (n_slots, k - 1, d), x.dtype)
    if k > 2 and state.stride(1) != d:
        raise ValueError("a slot of the state has to be contiguous")
    weight, bias = _parameter(queue, "weight", weight, (d, k)), _parameter(queue, "bias", bias, (d,))
    slots = _slots(queue, slots, n, n_slots)
    y = _like(x) if y is None else _output(queue, "y", y, (n, d), x.dtype)
    if d < 1:
        raise ValueError("x has no channels")
    args = _conv_step_args(code, d, k, _activation(activation), n, n_slots, _ptr(slots), x.data_ptr(), x.stride(0),
                           state.stride(0), weight.data_ptr(), _ptr(bias), state.data_ptr(), y.data_ptr())
    return _Call(queue.lib.nhip_causal_conv_step, args, (state, x, weight, bias, slots, y),
                 "hip_causal_conv_step", y=y)


def plan_causal_conv_step(queue, state, x, weight, bias=None, activation=None, slots=None, y=None, tag=None):
    """One token each of n requests, `x` ``[n, channels]``: `state` ``[slots, width - 1, channels]`` holds
    the inputs before it, oldest first, and moves on by one.  Request r has the slot ``slots[r]`` (int32;
    each at most once), or r; one outside the state gets zeros.  ``plan.y``."""
    return _causal_conv_step(queue, state, x, weight, bias, activation, slots, y).plan(queue, tag)


def causal_conv_step(queue, state, x, weight, bias=None, activation=None, slots=None):
    """y: see `plan_causal_conv_step`."""
    got = _causal_conv_step(queue, state, x, weight, bias, activation, slots).now(queue)
    return got["y"]


# ------------------------------------------------------------------------- selective scan
def _scan(queue, x, dt, A, B, C, D, dt_bias, softplus, initial, starts):
    x, B = _plain(x), _plain(B)
    code = _type_code("x", x)
    tokens, lead, s, starts = _tokens(queue, x, starts, 2)
    h, p = x.shape[-2:]
    if B.dim() != len(lead) + 2:
        raise ValueError("B has %d axes, x has %d" % (B.dim(), x.dim()))
    g, n = B.shape[-2:]
    if h < 1 or p < 1 or g < 1 or h % g:
        raise ValueError("%d heads of %d in %d groups: every group has the same heads" % (h, p, g))
    if not 1 <= n <= MAX_STATES:
        raise ValueError("%d states: 1 to %d are known" % (n, MAX_STATES))
    x = _array(queue, "x", x, lead + (h, p), None)
    B, C = _array(queue, "B", B, lead + (g, n), x.dtype), _array(queue, "C", C, lead + (g, n), x.dtype)
    dt = _plain(dt)
    dt_code = _type_code("dt", dt)
    if dt.shape != lead + (h,) or dt.device != queue.device:
        raise ValueError("dt has shape %s on %s, not %s on %s" % (tuple(dt.shape), dt.device, lead + (h,), queue.device))
    if A is None:
        raise TypeError("A is None")
    A, D, dt_bias = (_parameter(queue, k, v, (h,)) for k, v in (("A", A), ("D", D), ("dt_bias", dt_bias)))
    initial = _parameter(queue, "initial", initial, (s, h, p, n))
    args = _ScanArgs(tokens=tokens, type=code, dt_type=dt_code, softplus=int(bool(softplus)), n_heads=h, dim=p,
                     n_groups=g, states=n, x=_rows(x, len(lead), True), dt=_rows(dt, len(lead), True),
                     B=_rows(B, len(lead), True), C=_rows(C, len(lead), True), A=_ptr(A), D=_ptr(D),
                     dt_bias=_ptr(dt_bias), initial=_ptr(initial))
    return args, x, dt, B, lead, (s, h, p, n), [x, dt, A, B, C, D, dt_bias, initial, starts]


def _selective_scan(queue, x, dt, A, B, C, D=None, dt_bias=None, softplus=False, initial=None, starts=None, y=None,
                    final=None):
    torch = _torch()
    args, x, _, _, _, ends, keep = _scan(queue, x, dt, A, B, C, D, dt_bias, softplus, initial, starts)
    y = _output(queue, "y", y, x.shape, x.dtype)
    final = _output(queue, "final", final, ends, torch.float32)
    args.y, args.final = _ptr(y), _ptr(final)
    space = _workspace(queue, args, queue.lib.nhip_selective_scan_workspace)
    return _Call(queue.lib.nhip_selective_scan, args, keep + [y, final, space],
                 "hip_selective_scan", y=y, final=final)


def plan_selective_scan(queue, x, dt, A, B, C, D=None, dt_bias=None, softplus=False, initial=None, starts=None,
                        y=None, final=None, tag=None):
    """The scan of `x` ``[..., heads, dim]``: with ``step = f(dt + dt_bias)`` (f: identity or softplus),

        S[t] = exp(step A) S[t - 1] + step x[t] (outer) B[t],     y[t] = S[t] C[t] + D x[t]

    per head, S of ``dim x states`` in float32.  `dt` ``[..., heads]``; `B`, `C` ``[..., groups, states]``,
    each for heads / groups heads; `A` (rates, below zero for a filter that forgets), `D`, `dt_bias`
    ``[heads]``.  `initial` ``[S, heads, dim, states]`` enters, or zeros.  ``plan.y``, ``plan.final``."""
    return _selective_scan(queue, x, dt, A, B, C, D, dt_bias, softplus, initial, starts, y, final).plan(queue, tag)


def selective_scan(queue, x, dt, A, B, C, D=None, dt_bias=None, softplus=False, initial=None, starts=None):
    """(y, final): see `plan_selective_scan`."""
    got = _selective_scan(queue, x, dt, A, B, C, D, dt_bias, softplus, initial, starts).now(queue)
    return got["y"], got["final"]


def _selective_scan_grad(queue, dy, x, dt, A, B, C, D=None, dt_bias=None, softplus=False, initial=None, starts=None,
                         dfinal=None):
    torch = _torch()
    args, x, dt, B, lead, ends, keep = _scan(queue, x, dt, A, B, C, D, dt_bias, softplus, initial, starts)
    dy = _array(queue, "dy", dy, x.shape, x.dtype)
    dfinal = _parameter(queue, "dfinal", dfinal, ends)
    h = args.n_heads
    dx, ddt = (_output(queue, "", None, v.shape, v.dtype) for v in (x, dt))
    dB, dC = (_output(queue, "", None, B.shape, B.dtype) for _ in range(2))
    dA, dD, dbias = (_output(queue, "", None, (h,), torch.float32) for _ in range(3))
    dinitial = None if initial is None else _output(queue, "", None, ends, torch.float32)
    args.dy, args.dfinal = _rows(dy, len(lead), True), _ptr(dfinal)
    args.dx, args.ddt, args.dB, args.dC = _ptr(dx), _ptr(ddt), _ptr(dB), _ptr(dC)
    args.dA, args.dD, args.ddt_bias, args.dinitial = _ptr(dA), _ptr(dD), _ptr(dbias), _ptr(dinitial)
    space = _workspace(queue, args, queue.lib.nhip_selective_scan_grad_workspace)
    got = ScanGradients(dx, ddt, dA, dB, dC, None if D is None else dD, None if dt_bias is None else dbias, dinitial)
    return _Call(queue.lib.nhip_selective_scan_grad, args, keep + [dy, dfinal, dD, dbias, space, got],
                 "hip_selective_scan_grad", gradients=got)


def plan_selective_scan_grad(queue, dy, x, dt, A, B, C, D=None, dt_bias=None, softplus=False, initial=None,
                             starts=None, dfinal=None, tag=None):
    """The gradient of `plan_selective_scan`, from `dy` and (where the state went on) `dfinal`; it needs
    nothing that the forward pass computed.  ``plan.gradients``: those of A, D and dt_bias are float32."""
    return _selective_scan_grad(queue, dy, x, dt, A, B, C, D, dt_bias, softplus, initial, starts,
                                dfinal).plan(queue, tag)


def selective_scan_grad(queue, dy, x, dt, A, B, C, D=None, dt_bias=None, softplus=False, initial=None, starts=None,
                        dfinal=None):
    """`ScanGradients` (x, dt, A, B, C, D, dt_bias, initial): see `plan_selective_scan_grad`."""
    got = _selective_scan_grad(queue, dy, x, dt, A, B, C, D, dt_bias, softplus, initial, starts, dfinal).now(queue)
    return got["gradients"]


def _selective_step(queue, state, x, dt, A, B, C, D=None, dt_bias=None, softplus=False, slots=None, y=None):
    torch = _torch()
    state, x, B, dt = _plain(state), _plain(x), _plain(B), _plain(dt)
    code, dt_code = _type_code("x", x), _type_code("dt", dt)
    if x.dim() != 3 or B.dim() != 3 or state.dim() != 4:
        raise ValueError("x, B and state have %d, %d and %d axes, not 3, 3 and 4" % (x.dim(), B.dim(), state.dim()))
    n, h, p = x.shape
    g, k = B.shape[1:]
    if h < 1 or p < 1 or g < 1 or h % g:
        raise ValueError("%d heads of %d in %d groups: every group has the same heads" % (h, p, g))
    if not 1 <= k <= MAX_STATES:
        raise ValueError("%d states: 1 to %d are known" % (k, MAX_STATES))
    n_slots = state.shape[0]
    x = _array(queue, "x", x, (n, h, p), None)
    B, C = _array(queue, "B", B, (n, g, k), x.dtype), _array(queue, "C", C, (n, g, k), x.dtype)
    if dt.shape != (n, h) or dt.device != queue.device:
        raise ValueError("dt has shape %s on %s, not %s on %s" % (tuple(dt.shape), dt.device, (n, h), queue.device))
    if A is None:
        raise TypeError("A is None")
    A = _array(queue, "A", A, (h,), torch.float32, True)
    D, dt_bias = _parameter(queue, "D", D, (h,)), _parameter(queue, "dt_bias", dt_bias, (h,))
    state = _array(queue, "state", state, (n_slots, h, p, k), torch.float32)
    if not state.is_contiguous() and n_slots and not state[0].is_contiguous():
        raise ValueError("a slot of the state has to be contiguous")
    slots = _slots(queue, slots, n, n_slots)
    y = _like(x) if y is None else _output(queue, "y", y, (n, h, p), x.dtype)
    args = _scan_step_args(code, dt_code, bool(softplus), h, p, g, k, n, n_slots, _ptr(slots), *_rows(x, 1, True),
                           *_rows(dt, 1, True), *_rows(B, 1, True), *_rows(C, 1, True), A.data_ptr(), _ptr(D),
                           _ptr(dt_bias), state.data_ptr(), state.stride(0), y.data_ptr())
    return _Call(queue.lib.nhip_selective_step, args, (state, x, dt, A, B, C, D, dt_bias, slots, y),
                 "hip_selective_step", y=y)


def plan_selective_step(queue, state, x, dt, A, B, C, D=None, dt_bias=None, softplus=False, slots=None, y=None,
                        tag=None):
    """One token each of n requests: `x` ``[n, heads, dim]``, `dt` ``[n, heads]``, `B`, `C`
    ``[n, groups, states]``; `state` ``[slots, heads, dim, states]`` (float32) is moved on by a token.  Slots
    as for `plan_causal_conv_step`.  ``plan.y``."""
    return _selective_step(queue, state, x, dt, A, B, C, D, dt_bias, softplus, slots, y).plan(queue, tag)


def selective_step(queue, state, x, dt, A, B, C, D=None, dt_bias=None, softplus=False, slots=None):
    """y: see `plan_selective_step`."""
    got = _selective_step(queue, state, x, dt, A, B, C, D, dt_bias, softplus, slots).now(queue)
    return got["y"]


# ----------------------------------------------------------------------------- gated norm
def _flat(queue, name, t, like):
    """(tensor, row stride) of an array [..., channels] whose leading axes make rows of one stride."""
    t = _array(queue, name, t, like.shape, like.dtype)
    if t.dim() == 2:
        return t, t.stride(0)
    try:
        rows = t.view(-1, t.shape[-1])
    except RuntimeError:
        raise ValueError("the rows of %s do not lie at one distance" % name)
    return rows, rows.stride(0)


def _norm(queue, x, weight, gate, residual, scale, groups, eps, after):
    x = _plain(x)
    code = _type_code("x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x has shape %s: [..., channels] is wanted" % (tuple(x.shape),))
    d, groups = x.shape[-1], int(groups)
    if groups < 1 or d % groups:
        raise ValueError("%d channels in %d groups: every group has as many" % (d, groups))
    if scale is not None and residual is None:
        raise ValueError("scale goes with a residual")
    if not eps >= 0.0:
        raise ValueError("eps is %r" % (eps,))
    weight, scale = _parameter(queue, "weight", weight, (d,)), _parameter(queue, "scale", scale, (d,))
    if weight is None:
        raise TypeError("weight is None")
    args = _NormArgs(type=code, channels=d, groups=groups, after=int(bool(after)), rows=x.numel() // d,
                     eps=float(eps), weight=_ptr(weight), scale=_ptr(scale))
    keep = [weight, scale]
    for name, t in (("x", x), ("gate", gate), ("residual", residual)):
        if t is not None:
            t, stride = _flat(queue, name, t, x)
            setattr(args, name, _ptr(t))
            setattr(args, name + "_stride", stride)
            keep.append(t)
    return args, x, residual is not None and not after, keep


def _block_norm(queue, x, weight, gate=None, residual=None, scale=None, groups=1, eps=1e-6, after=False, out=None,
                v=None):
    args, x, before, keep = _norm(queue, x, weight, gate, residual, scale, groups, eps, after)
    out = _like(x) if out is None else _output(queue, "out", out, x.shape, x.dtype)
    if v is not None and not before:
        raise ValueError("v is written with a residual in front of a block only")
    v = _output(queue, "v", v, x.shape, x.dtype) if before else None
    args.out, args.v_out = _ptr(out), _ptr(v)
    return _Call(queue.lib.nhip_block_norm, args, keep + [out, v],
                 "hip_block_norm", out=out, v=v)


def plan_block_norm(queue, x, weight, gate=None, residual=None, scale=None, groups=1, eps=1e-6, after=False, out=None,
                    v=None, tag=None):
    """The norm of ``u = x`` or ``x * gate * sigmoid(gate)``, in front of a block or (`after`) behind it:

        before:  v = residual + scale * u,   out = v / sqrt(mean(v**2) + eps) * weight
        after:   out = residual + scale * (u / sqrt(mean(u**2) + eps) * weight)

    with means over each of `groups` equal parts of the last axis.  `residual` (like x) and `scale`
    (``[channels]``, ones) are optional.  ``plan.out``, and ``plan.v`` where there is a residual in front."""
    return _block_norm(queue, x, weight, gate, residual, scale, groups, eps, after, out, v).plan(queue, tag)


def block_norm(queue, x, weight, gate=None, residual=None, scale=None, groups=1, eps=1e-6, after=False):
    """(out, v or None): see `plan_block_norm`."""
    got = _block_norm(queue, x, weight, gate, residual, scale, groups, eps, after).now(queue)
    return got["out"], got["v"]


def _block_norm_grad(queue, dout, x, weight, gate=None, residual=None, scale=None, groups=1, eps=1e-6, after=False,
                     dv=None):
    torch = _torch()
    args, x, before, keep = _norm(queue, x, weight, gate, residual, scale, groups, eps, after)
    d = args.channels
    plain_dout = dout = _plain(dout)
    dout, args.dout_stride = _flat(queue, "dout", dout, x)
    args.dout = _ptr(dout)
    if dv is not None:
        if not before:
            raise ValueError("dv goes with a residual in front of a block")
        dv, args.dv_stride = _flat(queue, "dv", dv, x)
        args.dv = _ptr(dv)
    dx = _output(queue, "", None, x.shape, x.dtype)
    dgate = None if gate is None else _output(queue, "", None, x.shape, x.dtype)
    dresidual = _output(queue, "", None, x.shape, x.dtype) if before else None
    dweight, dscale = (_output(queue, "", None, (d,), torch.float32) for _ in range(2))
    args.dx, args.dgate, args.dresidual = _ptr(dx), _ptr(dgate), _ptr(dresidual)
    args.dweight, args.dscale = _ptr(dweight), _ptr(dscale)
    space = _workspace(queue, args, queue.lib.nhip_block_norm_grad_workspace)
    got = NormGradients(dx, dweight, dgate, None if residual is None else dresidual if before else plain_dout,
                        None if scale is None else dscale)
    return _Call(queue.lib.nhip_block_norm_grad, args, keep + [dout, dv, dscale, space, got],
                 "hip_block_norm_grad", gradients=got)


def plan_block_norm_grad(queue, dout, x, weight, gate=None, residual=None, scale=None, groups=1, eps=1e-6,
                         after=False, dv=None, tag=None):
    """The gradient of `plan_block_norm`, from `dout` and (with a residual in front) `dv`;
    ``plan.gradients``: those of weight and scale are float32.  Behind a block (`after`) the residual's is
    `dout` itself, the caller's array and no copy."""
    return _block_norm_grad(queue, dout, x, weight, gate, residual, scale, groups, eps, after, dv).plan(queue, tag)


def block_norm_grad(queue, dout, x, weight, gate=None, residual=None, scale=None, groups=1, eps=1e-6, after=False,
                    dv=None):
    """`NormGradients` (x, weight, gate, residual, scale): see `plan_block_norm_grad`."""
    got = _block_norm_grad(queue, dout, x, weight, gate, residual, scale, groups, eps, after, dv).now(queue)
    return got["gradients"]