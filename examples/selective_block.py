"""Selective blocks as they are used: trained on sequences, then answering token by token.

    python examples/selective_block.py [--steps 300] [--type float32|bfloat16] [--length 256]

The task needs a filter that chooses: a signal arrives with marks, and the answer at every token
is the signal's value at the last mark (0 before the first).  Blocks of norm, projection, short
convolution, selective scan, gated norm and projection learn it; the gradients are those of
`nengo_ocl_amd.hipra_selective`, the projections are torch's products.  Then prompts of several
lengths, back to back, fill the states of a few slots, and the answers go on from there one
token per request, which has to give what the whole sequences give.
"""

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from nengo_ocl_amd import hipra_selective as ops  # noqa: E402
from nengo_ocl_amd.hipraggedarray import Queue  # noqa: E402

WIDTH, HEADS, DIM, GROUPS, STATES, TAPS = 64, 4, 32, 1, 16, 4
INNER = HEADS * DIM
PARTS = [INNER, INNER + 2 * GROUPS * STATES, HEADS]  # gate; x, B and C; dt


class Block:
    """One block: its parameters (float32), the forward pass, its gradient, and the step of a token."""

    def __init__(self, queue, seed):
        gen = torch.Generator().manual_seed(seed)

        def normal(*shape, scale):
            return (torch.randn(*shape, generator=gen) * scale).to(queue.device)

        steps = torch.logspace(-3, -1, HEADS)
        self.queue = queue
        self.p = {
            "norm": normal(WIDTH, scale=0.0) + 1.0,
            "w_in": normal(sum(PARTS), WIDTH, scale=WIDTH ** -0.5),
            "conv": normal(PARTS[1], TAPS, scale=TAPS ** -0.5),
            "conv_bias": normal(PARTS[1], scale=0.0),
            "log_rate": torch.log(torch.linspace(1.0, 8.0, HEADS)).to(queue.device),
            "D": normal(HEADS, scale=0.0) + 1.0,
            "dt_bias": torch.log(torch.expm1(steps)).to(queue.device),  # softplus of it: the steps
            "gain": normal(INNER, scale=0.0) + 1.0,
            "w_out": normal(WIDTH, INNER, scale=INNER ** -0.5),
        }

    def _project(self, h, name):
        return h @ self.p[name].to(h.dtype).t()

    def _scan_inputs(self, conv, dt):
        x, B, C = conv.split([INNER, GROUPS * STATES, GROUPS * STATES], dim=-1)
        return dict(x=x.unflatten(-1, (HEADS, DIM)), dt=dt, A=-torch.exp(self.p["log_rate"]),
                    B=B.unflatten(-1, (GROUPS, STATES)), C=C.unflatten(-1, (GROUPS, STATES)),
                    D=self.p["D"], dt_bias=self.p["dt_bias"], softplus=True)

    def forward(self, h, residual, starts=None):
        """(output, residual for the next block, what `backward` needs, the state behind each sequence)."""
        q, p = self.queue, self.p
        normed, v = ops.block_norm(q, h, p["norm"], residual=residual)
        gate, xbc, dt = self._project(normed, "w_in").split(PARTS, dim=-1)
        conv, line = ops.causal_conv(q, xbc, p["conv"], p["conv_bias"], "silu", starts=starts)
        inputs = self._scan_inputs(conv, dt)
        y, state = ops.selective_scan(q, starts=starts, **inputs)
        y = y.flatten(-2)
        mixed, _ = ops.block_norm(q, y, p["gain"], gate=gate)
        saved = (h, residual, normed, gate, xbc, inputs, y, mixed, starts)
        return self._project(mixed, "w_out"), h if v is None else v, saved, (line, state)

    def backward(self, dout, dv, saved):
        """Gradients of h, of the residual, and of the parameters by name, from those of `forward`'s results."""
        q, p = self.queue, self.p
        h, residual, normed, gate, xbc, inputs, y, mixed, starts = saved

        def product(d, inp):
            return d.flatten(0, -2).t().float() @ inp.flatten(0, -2).float()

        g = {"w_out": product(dout, mixed)}
        of_mixed = ops.block_norm_grad(q, dout @ p["w_out"].to(dout.dtype), y, p["gain"], gate=gate)
        of_scan = ops.selective_scan_grad(q, of_mixed.x.unflatten(-1, (HEADS, DIM)), starts=starts, **inputs)
        dconv = torch.cat([of_scan.x.flatten(-2), of_scan.B.flatten(-2), of_scan.C.flatten(-2)], dim=-1)
        of_conv = ops.causal_conv_grad(q, dconv, xbc, p["conv"], p["conv_bias"], "silu", starts=starts)
        dproj = torch.cat([of_mixed.gate, of_conv.x, of_scan.dt], dim=-1)
        g.update(w_in=product(dproj, normed), conv=of_conv.weight, conv_bias=of_conv.bias,
                 log_rate=of_scan.A * inputs["A"], D=of_scan.D, dt_bias=of_scan.dt_bias, gain=of_mixed.weight)
        # without a residual v is h itself, and its gradient comes back beside the norm's
        of_norm = ops.block_norm_grad(q, dproj @ p["w_in"].to(dproj.dtype), h, p["norm"], residual=residual,
                                      dv=dv if residual is not None else None)
        g["norm"] = of_norm.weight
        return (of_norm.x, of_norm.residual, g) if residual is not None else (of_norm.x + dv, None, g)

    def new_states(self, n_slots, dtype):
        """The convolution's last inputs and the scan's states of `n_slots` requests."""
        return (torch.zeros(n_slots, TAPS - 1, PARTS[1], dtype=dtype, device=self.queue.device),
                torch.zeros(n_slots, HEADS, DIM, STATES, device=self.queue.device))

    def step(self, h, residual, states, slots):
        """One token each of the requests in `slots`; `states` moves on."""
        q, p = self.queue, self.p
        normed, v = ops.block_norm(q, h, p["norm"], residual=residual)
        gate, xbc, dt = self._project(normed, "w_in").split(PARTS, dim=-1)
        conv = ops.causal_conv_step(q, states[0], xbc, p["conv"], p["conv_bias"], "silu", slots)
        y = ops.selective_step(q, states[1], slots=slots, **self._scan_inputs(conv, dt))
        mixed, _ = ops.block_norm(q, y.flatten(-2), p["gain"], gate=gate)
        return self._project(mixed, "w_out"), h if v is None else v


class Model:
    def __init__(self, queue, n_blocks=2, dtype=torch.float32, seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.queue, self.dtype = queue, dtype
        self.embed = torch.randn(WIDTH, 2, generator=gen).to(queue.device)
        self.read = (torch.randn(1, WIDTH, generator=gen) * WIDTH ** -0.5).to(queue.device)
        self.norm = torch.ones(WIDTH, device=queue.device)
        self.blocks = [Block(queue, seed + 1 + k) for k in range(n_blocks)]

    def parameters(self):
        return [self.embed, self.read, self.norm] + [v for b in self.blocks for v in b.p.values()]

    def forward(self, inputs, starts=None):
        """(answers, what `backward` needs, the states behind each sequence)."""
        h, residual, saved, states = (inputs @ self.embed.t()).to(self.dtype), None, [], []
        for block in self.blocks:
            h, residual, s, state = block.forward(h, residual, starts)
            saved.append(s)
            states.append(state)
        normed, _ = ops.block_norm(self.queue, h, self.norm, residual=residual)
        return normed.float() @ self.read.t(), (inputs, h, residual, normed, saved), states

    def backward(self, danswers, kept):
        """The gradients, in the order of `parameters`."""
        inputs, h, residual, normed, saved = kept
        dread = danswers.flatten(0, -2).t() @ normed.flatten(0, -2).float()
        of_norm = ops.block_norm_grad(self.queue, (danswers @ self.read).to(self.dtype), h, self.norm, residual=residual)
        dh, dres, grads = of_norm.x, of_norm.residual, []
        for block, s in zip(self.blocks[::-1], saved[::-1]):
            dh, dres, g = block.backward(dh, dres, s)
            grads.insert(0, g)
        dembed = dh.flatten(0, -2).t().float() @ inputs.flatten(0, -2)
        return [dembed, dread, of_norm.weight] + [g[k] for b, g in zip(self.blocks, grads) for k in b.p]

    def step(self, inputs, states, slots):
        h, residual = (inputs @ self.embed.t()).to(self.dtype), None
        for block, state in zip(self.blocks, states):
            h, residual = block.step(h, residual, state, slots)
        normed, _ = ops.block_norm(self.queue, h, self.norm, residual=residual)
        return normed.float() @ self.read.t()


def task(shape, seed, device):
    """(signal and marks, the signal at the last mark), for sequences that lie along the last axis of `shape`."""
    gen = torch.Generator().manual_seed(seed)
    signal = torch.randn(*shape, generator=gen)
    marks = torch.rand(*shape, generator=gen) < 0.1
    at = torch.where(marks, torch.arange(shape[-1]), -1).cummax(-1).values
    wanted = torch.where(at >= 0, signal.gather(-1, at.clamp(min=0)), 0.0)
    return torch.stack([signal, marks.float()], -1).to(device), wanted[..., None].to(device)


def train(model, steps, batch=16, length=256, report=None):
    """The mean squared error at each step."""
    optimizer = torch.optim.Adam(model.parameters(), lr=4e-3)
    losses = []
    for k in range(steps):
        inputs, wanted = task((batch, length), k, model.queue.device)
        answers, kept, _ = model.forward(inputs)
        off = answers - wanted
        losses.append(float((off ** 2).mean()))
        for p, g in zip(model.parameters(), model.backward(off * (2.0 / off.numel()), kept)):
            p.grad = g
        optimizer.step()
        if report and (k % 50 == 0 or k == steps - 1):
            report("step %4d  mean squared error %.4f" % (k, losses[-1]))
    return losses


def answer(model, prompts, rest):
    """The answers to `rest` ``[requests, tokens, 2]``, token by token behind prompts (a list of ``[tokens, 2]``)."""
    n, device = len(prompts), model.queue.device
    starts = torch.tensor([0] + [len(p) for p in prompts]).cumsum(0).to(device, torch.int32)
    _, _, ends = model.forward(torch.cat(prompts), starts)
    # requests lie in any slots: here from the last one down, and one slot is nobody's
    slots = torch.arange(n, 0, -1, dtype=torch.int32, device=device)
    states = [block.new_states(n + 1, model.dtype) for block in model.blocks]
    for state, end in zip(states, ends):
        for cache, values in zip(state, end):
            cache[slots.long()] = values
    return torch.stack([model.step(rest[:, t], states, slots) for t in range(rest.shape[1])], 1)


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=300)
    parser.add_argument("--length", type=int, default=256)
    parser.add_argument("--type", choices=("float32", "bfloat16"), default="float32")
    args = parser.parse_args()
    # the program's own stream: nothing has to wait for another one
    model = Model(Queue(0, stream=torch.cuda.current_stream()), dtype=getattr(torch, args.type))
    train(model, args.steps, length=args.length, report=lambda line: print(line, flush=True))
    inputs, wanted = task((4, args.length + 32), 65535, model.queue.device)
    lengths = [args.length - k for k in (0, 1, 17, args.length - 1)]
    prompts = [inputs[k, :n] for k, n in enumerate(lengths)]
    rest = torch.stack([inputs[k, n:n + 32] for k, n in enumerate(lengths)])
    answers = answer(model, prompts, rest)
    whole, _, _ = model.forward(inputs)
    whole = torch.stack([whole[k, n:n + 32] for k, n in enumerate(lengths)])
    wanted = torch.stack([wanted[k, n:n + 32] for k, n in enumerate(lengths)])
    print("token by token: mean squared error %.4f; largest distance from the whole sequences' answers %.1e"
          % (float(((answers - wanted) ** 2).mean()), float((answers - whole).abs().max())))


if __name__ == "__main__":
    main()
