"""The operators over tokens together, as `examples/token_model.py` uses them: the gradients of a whole model, and that it runs.

Tolerances as for the selective blocks: a pass goes through some twenty operators and products one after the other,
each of whose results in 32 bits is off by at most 128 u = 7.6e-6 of its norm: 2e-4 of the loss, 1e-3 of the norm of a parameter's
gradient, which sums its terms over all tokens, where they cancel in part.
"""

import os
import runpy
import types

import pytest
import torch

from test_selective import conv_definition, norm_definition, scan_definition
from test_tokens import norm_definition as layer_norm_definition

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "token_model.py")


@pytest.fixture(scope="module")
def example():
    return types.SimpleNamespace(**runpy.run_path(PATH, run_name="token_model"))


def defined(example, model, values, tokens):
    """The logits from the operators' definitions, in 64 bits; `values` as model.parameters()."""
    block_of = example.selective
    embed, read, last, bias = values[:4]
    h, residual, at = embed[tokens], None, 4
    for block in model.blocks:
        p = dict(zip(block.p, values[at:at + len(block.p)]))
        at += len(block.p)
        if "gate" in p:
            normed, residual = layer_norm_definition(h, p["norm"], p["norm_bias"], residual, 1e-5)
            g = normed @ p["gate"].t()
            h = (g * torch.sigmoid(g) * (normed @ p["up"].t())) @ p["down"].t()
            continue
        normed, v = norm_definition(h, p["norm"], None, residual, None, 1, 1e-6, False)
        residual = h if v is None else v
        gate, xbc, dt = (normed @ p["w_in"].t()).split(block_of.PARTS, dim=-1)
        conv, _ = conv_definition(xbc, p["conv"], p["conv_bias"], True, None, None)
        n = block_of.GROUPS * block_of.STATES
        x, B, C = conv.split([block_of.INNER, n, n], dim=-1)
        parts = (block_of.GROUPS, block_of.STATES)
        y, _ = scan_definition(x.unflatten(-1, (block_of.HEADS, block_of.DIM)), dt, -torch.exp(p["log_rate"]),
                               B.unflatten(-1, parts), C.unflatten(-1, parts), p["D"], p["dt_bias"], True, None, None)
        mixed, _ = norm_definition(y.flatten(-2), p["gain"], gate, None, None, 1, 1e-6, False)
        h = mixed @ p["w_out"].t()
    return layer_norm_definition(h, last, bias, residual, 1e-5)[0] @ read.t()


def compare(loss, grads, want, values):
    assert abs(float(loss) - float(want.detach())) <= 2e-4 * abs(float(want.detach()))
    exact = torch.autograd.grad(want, values, allow_unused=True)
    assert len(grads) == len(exact)
    for k, (a, b) in enumerate(zip(grads, exact)):
        assert a.shape == b.shape
        assert (a.cpu().double() - b).norm() <= 1e-3 * b.norm(), (k, float((a.cpu().double() - b).norm() / b.norm()))


@pytest.mark.gpu
def test_gradients_of_the_model(queue, example):
    model = example.Model(queue, 211, seed=3)
    tokens, labels = example.task(211, 2, 70, 5, queue.device)
    loss, grads = model.loss(tokens, labels)
    values = [v.detach().cpu().double().requires_grad_() for v in model.parameters()]
    z = defined(example, model, values, tokens.cpu())
    want = torch.nn.functional.cross_entropy(z.flatten(0, 1), labels.cpu().flatten(), ignore_index=-100)
    compare(loss, grads, want, values)


@pytest.mark.gpu
def test_gradients_of_the_distance(queue, example):
    model, temperature = example.Model(queue, 97, n_blocks=1, seed=4), 2.0
    tokens, _ = example.task(97, 3, 33, 6, queue.device)
    gen = torch.Generator().manual_seed(7)
    best = torch.randn(3, 33, 97, generator=gen).mul(2.0).topk(8)
    loss, grads = model.distance(tokens, best.indices.cuda(), best.values.cuda(), temperature)
    values = [v.detach().cpu().double().requires_grad_() for v in model.parameters()]
    logp = torch.log_softmax(defined(example, model, values, tokens.cpu()) / temperature, -1)
    q = torch.softmax(best.values.double() / temperature, -1)
    want = (q * (q.log() - torch.gather(logp, -1, best.indices))).sum(-1).mean()
    compare(loss, grads, want, values)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_teacher_and_student_run(queue, example, dtype):
    teacher = example.Model(queue, 60, dtype=dtype)
    losses = example.train(teacher, 3, batch=4, length=32)
    student = example.Model(queue, 60, 1, dtype, seed=9)
    losses += example.train(student, 3, batch=4, length=32, step_of=example.from_teacher(teacher, student))
    assert len(losses) == 6 and all(x == x and x > 0 for x in losses)
