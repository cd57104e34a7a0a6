"""Calls that go over the vocabulary, or the features, in several pieces: by the length of rows that are copied, by the tiles that
a launch reaches, and by what a gradient keeps of G.  Definitions and tolerances are those of test_tokens.py, on the device; of
results with 2**20 rows some are compared.
"""

import pytest
import torch

import test_tokens
from test_tokens import (BF16, F16, F32, Maker, check_loss_gradients, check_losses, gated_bounds, loss_inputs,  # noqa: F401
                         ops, teacher_inputs, wide, within)


@pytest.fixture(autouse=True)
def on_the_device(monkeypatch):
    monkeypatch.setattr(test_tokens, "PLACE", "cuda")
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


COPIED = 1 << 21  # words of a piece whose rows of five channels are copied to rows of 256 bytes, 512 MB


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 20, 70])
@pytest.mark.parametrize("kind", ["labels", "targets"])
def test_words_that_are_copied_in_pieces(queue, ops, n, kind):  # noqa: F811
    d, v = 5, COPIED + 70001
    m = Maker(101)
    x, weight = m.normal(n, d), m.normal(v, d, scale=0.5)
    edges = torch.tensor([0, COPIED - 1, COPIED, COPIED + 1, v - 1, COPIED // 2, COPIED - 128, COPIED + 128])
    given = {"x": x, "weight": weight}
    if kind == "labels":
        given["labels"] = edges.repeat(9)[:n].cuda()
        loss, lse = ops.vocabulary_loss(queue, **given)
        check_losses(loss, lse, given, 1.0)
        return
    words = m.whole(v, n, 20)
    words[:, :8] = edges
    given.update(indices=words.int().cuda(), logits=m.normal(n, 20))
    loss, lse = ops.teacher_loss(queue, temperature=2.0, **given)
    check_losses(loss, lse, given, 2.0)


ROWS, REACH = 1 << 20, 1 << 16  # 2**21 tiles of 128 x 256 to a launch: 65536 words of so many rows


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["labels", "targets"])
def test_more_words_than_a_launch_reaches(queue, ops, kind):  # noqa: F811
    d, v = 8, REACH + 4321
    m = Maker(102)
    gen = torch.Generator(device="cuda").manual_seed(103)
    x = torch.randn(ROWS, d, generator=gen, device="cuda").to(BF16)
    weight = m.normal(v, d, dtype=BF16, scale=0.5)
    some = torch.cat([torch.arange(200), m.whole(ROWS, 200), torch.arange(ROWS - 200, ROWS)]).cuda()
    edges = torch.tensor([0, REACH - 1, REACH, REACH + 1, v - 1], device="cuda")
    words = torch.randint(v, (ROWS, 6), generator=gen, device="cuda")
    words[some, :5] = edges[torch.arange(len(some), device="cuda")[:, None].add(torch.arange(5, device="cuda")) % 5]
    words[some[::7]] = -1  # rows that do not count
    if kind == "labels":
        labels = words[:, 0].contiguous()
        loss, lse = ops.vocabulary_loss(queue, x, weight, labels)
        check_losses(loss[some], lse[some], {"x": x[some], "weight": weight, "labels": labels[some]}, 1.0)
        return
    logits = torch.randn(ROWS, 6, generator=gen, device="cuda")
    loss, lse = ops.teacher_loss(queue, x, weight, words, logits, 2.0)
    check_losses(loss[some], lse[some], {"x": x[some], "weight": weight, "indices": words[some], "logits": logits[some]}, 2.0)


END = 20224  # of the first of two pieces of 40000 words, whose halves are rounded to 256


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, n, d, v, top", [(BF16, 8300, 136, 40000, 70), (F16, 8300, 136, 40000, 9), (F32, 4200, 40, 40000, 70)])
def test_gradient_of_the_teachers_loss(queue, ops, dtype, n, d, v, top):  # noqa: F811
    """Targets on both sides of a piece's end, some of them twice, rows that do not count among the others."""
    given, m = teacher_inputs(104, dtype, n, d, v, 0.2, top)
    edges = torch.tensor([0, END - 1, END, END + 255, v - 1], dtype=torch.int32)
    given["indices"][::3, :5] = edges.cuda()
    loss, lse = ops.teacher_loss(queue, temperature=2.0, **given)
    check_losses(loss, lse, given, 2.0)
    dloss = (torch.rand(n, generator=m.gen) / n).cuda()
    got = ops.teacher_loss_grad(queue, dloss, lse=lse, temperature=2.0, **given)
    check_loss_gradients(got, given, 2.0, dloss, lse)


@pytest.mark.gpu
def test_more_features_than_a_launch_reaches(queue, ops):  # noqa: F811
    """2**20 rows: 32768 features to a launch, y has 68 GB."""
    d, f = 8, (1 << 15) + 203
    m = Maker(105)
    gen = torch.Generator(device="cuda").manual_seed(106)
    x = torch.randn(ROWS, d, generator=gen, device="cuda").to(BF16)
    gate, up = (m.normal(f, d, dtype=BF16, scale=d ** -0.5) for _ in range(2))
    y = ops.gated_projection(queue, x, gate, up)
    some = torch.cat([torch.arange(100), m.whole(ROWS, 200), torch.arange(ROWS - 100, ROWS)]).cuda()
    a, _, g, u, ea, _, eu = gated_bounds(wide(x[some]), wide(gate), wide(up), "silu")
    within(y[some], a * u, ea * u.abs() + eu * a.abs() + ea * eu, "y")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, n, d, v, masked", [
    (BF16, 130, 8192, 3001, 0.2), (F16, 66, 5120, 4000, 0.0), (BF16, 40, 4096, 128001, 0.1), (F32, 70, 4100, 3000, 0.3),
    (BF16, 600, 128, 131072, 0.1)])
def test_many_channels_and_many_words(queue, ops, dtype, n, d, v, masked):  # noqa: F811
    given, m = loss_inputs(107, dtype, n, d, v, masked)
    loss, lse = ops.vocabulary_loss(queue, **given)
    check_losses(loss, lse, given, 1.0)
    dloss = (torch.rand(n, generator=m.gen) / n).cuda()
    check_loss_gradients(ops.vocabulary_loss_grad(queue, dloss, lse=lse, **given), given, 1.0, dloss, lse)
