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
