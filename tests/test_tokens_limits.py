"""Arguments at the ends of their ranges: what lies beyond is refused before any launch, by Python and by the library.
"""

import ctypes

import pytest
import torch

from test_tokens import host, ops  # noqa: F401

ONE = 1 << 20  # where an array might lie: refused calls read none


def loss_arguments(ops, **more):  # noqa: F811
    given = dict(channels=8, words=70, rows=5, temperature=1.0, x=ONE, weight=ONE, x_stride=8, weight_stride=8, targets=ONE, loss=ONE,
                 lse=ONE, dloss=ONE, dx=ONE, dweight=ONE, top=2, target_logits=ONE, workspace=ONE, workspace_bytes=1)
    return ctypes.byref(ops._LossArgs(**dict(given, **more)))


def test_temperatures(host, ops):  # noqa: F811
    """Those whose reciprocal 32 bits do not hold are no temperatures: 1e-39 divided by made no numbers."""
    from nengo_ocl_amd import _lib

    x, w = torch.zeros(3, 12), torch.zeros(70, 12)
    words, values = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 4)
    for t in (2.0 ** -126, 1e-30, 1.0, 1e30, 2.0 ** 126):
        assert ops.plan_teacher_loss(host, x, w, words, values, t).loss.shape == (3,)
    lib, bad, too_big = _lib.lib(), -1, -4
    for t in (1e-39, 1e-46, 1e-300, 1e38, 3e38, 1e39, 1e300):
        with pytest.raises(ValueError):
            ops.plan_teacher_loss(host, x, w, words, values, t)
        with pytest.raises(ValueError):
            ops.plan_teacher_loss_grad(host, values[:, 0].contiguous(), x, w, words, values, values[:, 0].contiguous(), t)
    for entry in (lib.nhip_vocabulary_loss, lib.nhip_vocabulary_loss_grad):
        for t in (1e-39, 1e38, 3e38):
            assert entry(None, loss_arguments(ops, temperature=t)) == bad, t
        for t in (2.0 ** -126, 2.0 ** 126):
            assert entry(None, loss_arguments(ops, temperature=t)) == too_big, t  # (of the workspace)


def test_channels_of_the_norms_gradients(ops):  # noqa: F811
    """The launch that adds up the sums for weight and bias takes 2**28 - 64 columns, two to a channel: more are refused before
    the first launch (the workspace of one byte, checked behind them, tells that they were not)."""
    from nengo_ocl_amd import _lib, hipra_selective

    lib, bad, too_big, need = _lib.lib(), -1, -4, ctypes.c_longlong()

    def layer(channels):
        return ctypes.byref(ops._LayerNormArgs(channels=channels, rows=1, eps=1e-5, x=ONE, x_stride=channels, weight=ONE, out=ONE,
                                               dout=ONE, dout_stride=channels, dx=ONE, dweight=ONE, workspace=ONE, workspace_bytes=1))

    def block(channels):
        return ctypes.byref(hipra_selective._NormArgs(channels=channels, groups=1, rows=1, eps=1e-5, x=ONE, x_stride=channels,
                                                      weight=ONE, out=ONE, dout=ONE, dout_stride=channels, dx=ONE, dweight=ONE,
                                                      workspace=ONE, workspace_bytes=1))

    most = 2 ** 27 - 32
    for entry, given in ((lib.nhip_layer_norm_grad, layer), (lib.nhip_block_norm_grad, block)):
        assert entry(None, given(most)) == too_big
        for channels in (most + 1, 2 ** 27 - 1):
            assert entry(None, given(channels)) == bad, channels
    assert lib.nhip_layer_norm_grad_workspace(layer(most), ctypes.byref(need)) == 0 and need.value == 2 * 4 * most
    assert lib.nhip_layer_norm_grad_workspace(layer(most + 1), ctypes.byref(need)) == bad
