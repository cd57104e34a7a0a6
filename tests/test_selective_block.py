"""The operators of selective blocks run together: `examples/selective_block.py`, its gradients and its two ways to answer.

Tolerances.  A pass goes through about ten operators and products one after the other, each of whose results
in 32 bits is off by at most 128 u = 7.6e-6 of its norm (u = 2**-24): 1e-4.  A parameter's gradient sums its
terms over all tokens, where they cancel in part: 1e-3 of its norm.
"""

import os
import runpy
import types

import pytest
import torch

from test_selective import conv_definition, norm_definition, scan_definition

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "selective_block.py")


@pytest.fixture(scope="module")
def example():
    return types.SimpleNamespace(**runpy.run_path(PATH, run_name="selective_block"))


def defined(example, model, values, inputs, starts=None):
    """The model's answers from the operators' definitions, in 64 bits; `values` as model.parameters()."""
    embed, read, last = values[:3]
    h, residual, at = inputs @ embed.t(), None, 3
    for block in model.blocks:
        p = dict(zip(block.p, values[at:at + len(block.p)]))
        at += len(block.p)
        normed, v = norm_definition(h, p["norm"], None, residual, None, 1, 1e-6, False)
        residual = h if v is None else v
        gate, xbc, dt = (normed @ p["w_in"].t()).split(example.PARTS, dim=-1)
        conv, _ = conv_definition(xbc, p["conv"], p["conv_bias"], True, None, starts)
        n = example.GROUPS * example.STATES
        x, B, C = conv.split([example.INNER, n, n], dim=-1)
        parts = (example.GROUPS, example.STATES)
        y, _ = scan_definition(x.unflatten(-1, (example.HEADS, example.DIM)), dt, -torch.exp(p["log_rate"]),
                               B.unflatten(-1, parts), C.unflatten(-1, parts), p["D"], p["dt_bias"], True, None, starts)
        mixed, _ = norm_definition(y.flatten(-2), p["gain"], gate, None, None, 1, 1e-6, False)
        h = mixed @ p["w_out"].t()
    return norm_definition(h, last, None, residual, None, 1, 1e-6, False)[0] @ read.t()


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [None, [70, 0, 1, 25]])
def test_gradients_of_the_model(queue, example, lengths):
    model = example.Model(queue, seed=3)
    starts = None if lengths is None else torch.tensor([0] + lengths).cumsum(0).int()
    inputs, wanted = example.task((2, 96) if lengths is None else (sum(lengths),), 5, queue.device)
    answers, kept, _ = model.forward(inputs, None if starts is None else starts.cuda())
    got = model.backward((answers - wanted) * 2.0, kept)
    values = [v.detach().cpu().double().requires_grad_() for v in model.parameters()]
    want = defined(example, model, values, inputs.cpu().double(), starts)
    assert (answers.cpu().double() - want).norm() <= 1e-4 * want.norm()
    grads = torch.autograd.grad(((want - wanted.cpu().double()) ** 2).sum(), values)
    assert len(got) == len(grads)
    for k, (a, b) in enumerate(zip(got, grads)):
        assert a.shape == b.shape
        assert (a.cpu().double() - b).norm() <= 1e-3 * b.norm(), (k, float((a.cpu().double() - b).norm() / b.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tolerance", [(torch.float32, 1e-4), (torch.bfloat16, 10 * 3 * 2.0 ** -9)])
def test_token_by_token_as_the_whole_sequences(queue, example, dtype, tolerance):
    model = example.Model(queue, dtype=dtype, seed=4)
    inputs, _ = example.task((3, 90), 6, queue.device)
    lengths = [1, 64, 77]
    whole, _, _ = model.forward(inputs)
    got = example.answer(model, [inputs[k, :n] for k, n in enumerate(lengths)],
                         torch.stack([inputs[k, n:n + 13] for k, n in enumerate(lengths)]))
    want = torch.stack([whole[k, n:n + 13] for k, n in enumerate(lengths)])
    assert got.shape == want.shape and (got - want).norm() <= tolerance * want.norm()


@pytest.mark.gpu
def test_training_learns(queue, example):
    losses = example.train(example.Model(queue), 40, batch=8, length=64)
    assert all(x == x for x in losses) and sum(losses[-5:]) < 0.75 * sum(losses[:5])
