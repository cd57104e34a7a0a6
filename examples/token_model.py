"""A model over tokens as it is used: a teacher learns sequences, a smaller student learns from its largest logits.

    python examples/token_model.py [--steps 200] [--type float32|bfloat16] [--length 128]

Each word is followed by one of four, by a table that the models do not see; the first quarter of a sequence
is a prompt and does not count.  A model is an embedding, selective
blocks (`selective_block.py`), behind each a feed-forward block (layer norm, gated projection, projection),
a last layer norm and the loss over the vocabulary; no logits are ever in memory.  The gradients are those of
`nengo_ocl_amd.hipra_tokens` and `hipra_selective`, the other products are torch's.
"""

import argparse
import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [os.path.dirname(HERE), HERE]

import torch  # noqa: E402

import selective_block as selective  # noqa: E402
from nengo_ocl_amd import hipra_tokens as ops  # noqa: E402
from nengo_ocl_amd.hipraggedarray import Queue  # noqa: E402

WIDTH, FEATURES = selective.WIDTH, 176


class FeedForward:
    """A layer norm with the residual in front of it, the gated projection, and a projection back."""

    def __init__(self, queue, seed, features=FEATURES):
        gen = torch.Generator().manual_seed(seed)

        def normal(*shape, scale):
            return (torch.randn(*shape, generator=gen) * scale).to(queue.device)

        self.queue = queue
        self.p = {
            "norm": normal(WIDTH, scale=0.0) + 1.0,
            "norm_bias": normal(WIDTH, scale=0.0),
            "gate": normal(features, WIDTH, scale=WIDTH ** -0.5),
            "up": normal(features, WIDTH, scale=WIDTH ** -0.5),
            "down": normal(WIDTH, features, scale=features ** -0.5),
        }

    def _weights(self, dtype):
        return [self.p[k].to(dtype) for k in ("gate", "up", "down")]

    def forward(self, h, residual):
        """(output, residual for the next block, what `backward` needs)"""
        normed, v = ops.layer_norm(self.queue, h, self.p["norm"], self.p["norm_bias"], residual=residual)
        gate, up, down = self._weights(h.dtype)
        y = ops.gated_projection(self.queue, normed, gate, up, "silu")
        return y @ down.t(), v, (h, residual, normed, y)

    def backward(self, dout, dv, saved):
        """Gradients of h, of the residual, and of the parameters by name."""
        h, residual, normed, y = saved
        gate, up, down = self._weights(h.dtype)
        of_y = ops.gated_projection_grad(self.queue, dout @ down, normed, gate, up, "silu")
        of_norm = ops.layer_norm_grad(self.queue, of_y.x, h, self.p["norm"], self.p["norm_bias"], residual=residual, dv=dv)
        grads = {"norm": of_norm.weight, "norm_bias": of_norm.bias, "gate": of_y.gate.float(), "up": of_y.up.float(),
                 "down": dout.flatten(0, -2).t().float() @ y.flatten(0, -2).float()}
        return of_norm.x, of_norm.residual, grads


class Model:
    def __init__(self, queue, words, n_blocks=2, dtype=torch.float32, seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.queue, self.dtype, self.words = queue, dtype, words
        self.embed = (torch.randn(words, WIDTH, generator=gen)).to(queue.device)
        self.read = (torch.randn(words, WIDTH, generator=gen) * WIDTH ** -0.5).to(queue.device)
        self.norm, self.bias = torch.ones(WIDTH, device=queue.device), torch.zeros(WIDTH, device=queue.device)
        self.blocks = [kind(queue, seed + 1 + 2 * k + j) for k in range(n_blocks)
                       for j, kind in enumerate((selective.Block, FeedForward))]

    def parameters(self):
        return [self.embed, self.read, self.norm, self.bias] + [v for b in self.blocks for v in b.p.values()]

    def forward(self, tokens):
        """(what the last norm leaves, the weights of the vocabulary, what `backward` needs)"""
        h, residual, saved = self.embed[tokens].to(self.dtype), None, []
        for block in self.blocks:
            h, residual, s = block.forward(h, residual)[:3]
            saved.append(s)
        normed, _ = ops.layer_norm(self.queue, h, self.norm, self.bias, residual=residual)
        return normed, self.read.to(self.dtype), (tokens, h, residual, saved)

    def backward(self, of_loss, kept):
        """The gradients, in the order of `parameters`, from those of the loss with respect to the last norm and the weights."""
        tokens, h, residual, saved = kept
        of_norm = ops.layer_norm_grad(self.queue, of_loss.x, h, self.norm, self.bias, residual=residual)
        dh, dres, grads = of_norm.x, of_norm.residual, []
        for block, s in zip(self.blocks[::-1], saved[::-1]):
            dh, dres, g = block.backward(dh, dres, s)
            grads.insert(0, g)
        dembed = torch.zeros_like(self.embed).index_add_(0, tokens.flatten(), dh.flatten(0, -2).float())
        return [dembed, of_loss.weight.float(), of_norm.weight, of_norm.bias] \
            + [g[k] for b, g in zip(self.blocks, grads) for k in b.p]

    def loss(self, tokens, labels):
        """(the mean over the tokens that count, the gradients)"""
        normed, read, kept = self.forward(tokens)
        loss, lse = ops.vocabulary_loss(self.queue, normed, read, labels)
        counts = (labels >= 0).sum().clamp(min=1)
        share = (torch.ones_like(loss) / counts).contiguous()
        of_loss = ops.vocabulary_loss_grad(self.queue, share, normed, read, labels, lse)
        return loss.sum() / counts, self.backward(of_loss, kept)

    def distance(self, tokens, indices, logits, temperature):
        """(the mean distance from a teacher's largest logits, the gradients)"""
        normed, read, kept = self.forward(tokens)
        loss, lse = ops.teacher_loss(self.queue, normed, read, indices, logits, temperature)
        share = torch.full_like(loss, 1.0 / loss.numel())
        of_loss = ops.teacher_loss_grad(self.queue, share, normed, read, indices, logits, lse, temperature)
        return loss.mean(), self.backward(of_loss, kept)


def task(words, batch, length, seed, device, successors=4):
    """(tokens, labels): every word is followed by one of `successors`; the first quarter's labels do not count."""
    table = torch.randint(words, (words, successors), generator=torch.Generator().manual_seed(words))
    gen = torch.Generator().manual_seed(seed)
    line = [torch.randint(words, (batch,), generator=gen)]
    for _ in range(length):
        line.append(table[line[-1], torch.randint(successors, (batch,), generator=gen)])
    line = torch.stack(line, 1)
    labels = line[:, 1:].clone()
    labels[:, :length // 4] = -100
    return line[:, :-1].contiguous().to(device), labels.contiguous().to(device)


def train(model, steps, batch=16, length=128, report=None, step_of=None):
    """The losses; `step_of` (tokens, labels) -> (loss, gradients), or the cross entropy."""
    optimizer = torch.optim.Adam(model.parameters(), lr=4e-3)
    losses = []
    for k in range(steps):
        tokens, labels = task(model.words, batch, length, k, model.queue.device)
        loss, grads = (step_of or model.loss)(tokens, labels)
        for p, g in zip(model.parameters(), grads):
            p.grad = g
        optimizer.step()
        losses.append(float(loss))
        if report and (k % 50 == 0 or k == steps - 1):
            report("step %4d  %.4f" % (k, losses[-1]))
    return losses


def from_teacher(teacher, student, top=8, temperature=2.0):
    """A step of the student towards the teacher's `top` largest logits."""
    def step(tokens, labels):
        normed, read, _ = teacher.forward(tokens)
        best = (normed.float() @ read.float().t()).topk(top)
        return student.distance(tokens, best.indices.contiguous(), best.values.contiguous(), temperature)
    return step


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--length", type=int, default=128)
    parser.add_argument("--words", type=int, default=300)
    parser.add_argument("--type", choices=("float32", "bfloat16"), default="float32")
    args = parser.parse_args()
    queue, dtype = Queue(0, stream=torch.cuda.current_stream()), getattr(torch, args.type)
    say = lambda line: print(line, flush=True)
    teacher = Model(queue, args.words, 2, dtype)
    say("teacher, cross entropy")
    train(teacher, args.steps, length=args.length, report=say)
    student = Model(queue, args.words, 1, dtype, seed=50)
    say("student, distance from the teacher")
    train(student, args.steps, length=args.length, report=say, step_of=from_teacher(teacher, student))


if __name__ == "__main__":
    main()
