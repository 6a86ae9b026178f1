"""A dense net trained with its level pairs in few bits, then answered by the
edge arena.

The net's full level pairs are matrices with 32-bit master weights. Each
training step quantises them to 4 bits, answers the batch, keeps 8 bits of
every activation for the backward, and moves the master weights along the
gradient of the 4-bit net. The trained net, its weights the values that their
4 bits stand for, is then built as edges and run by ``make_step``, one sample
at a time, and single samples are answered from the 4-bit matrices too: the
same numbers up to the rounding of float32 sums.

Run on the GPU: ``python examples/lowbit_mlp.py``.
"""

from __future__ import annotations

import pathlib
import sys

import numpy as np
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))

import plastax_amd as px  # noqa: E402
from plastax_amd import lowbit  # noqa: E402

SIZES = (96, 256, 160, 10)


class Tanh(px.ForwardPass):
    combine = px.monoid.sum_

    def map(self, u, dst, src, c, cid, g):
        return c[px.WEIGHT, cid] * u[px.ACTIVATION, src]

    def apply(self, u, i, g, acc):
        return px.UnitWrite.of((px.ACTIVATION, px.numpy.tanh(acc)))


class Mlp(px.Network):
    forward_pass = Tanh()


def train(sizes, batches, rate: float, seed: int = 0):
    """(master weights, the loss of every batch) of (inputs, targets) batches."""
    rng = torch.Generator(device="cuda").manual_seed(seed)
    weights = [torch.randn((o, i), generator=rng, device="cuda") / i**0.5 for i, o in zip(sizes, sizes[1:])]
    losses = []
    for x, target in batches:
        pairs, inputs, kept = [lowbit.quantise4(w) for w in weights], [], []
        for pair in pairs:
            inputs.append(lowbit.quantise8(x))
            x, k = lowbit.activate(lowbit.product(x, pair), "tanh")
            kept.append(k)
        error = x.float() - target
        losses.append((error * error).sum(1).mean() / 2)
        grad = (error / error.shape[0]).to(x.dtype)
        for j in reversed(range(len(pairs))):
            grad = lowbit.activate_grad(grad, kept[j], "tanh")
            weights[j] -= rate * lowbit.weight_grad(grad, inputs[j])
            if j:
                grad = lowbit.product_grad(grad, pairs[j])
    return weights, torch.stack(losses).tolist()


def answer(pairs, x: torch.Tensor) -> torch.Tensor:
    """The net's answer to a batch (or one sample) from its 4-bit pairs."""
    for pair in pairs:
        x, _ = lowbit.activate(lowbit.product(x, pair), "tanh")
    return x


def edge_net(pairs):
    """The same net as edges: every unit of a level to every unit of the next."""
    sizes = [pairs[0].shape[1]] + [p.shape[0] for p in pairs]
    first = np.concatenate([[0], np.cumsum(sizes)])
    src, dst, weight = [], [], []
    for j, pair in enumerate(pairs):
        o, i = pair.shape
        src.append(np.tile(first[j] + np.arange(i), o))
        dst.append(np.repeat(first[j + 1] + np.arange(o), i))
        weight.append(pair.values().cpu().numpy().ravel())
    return px.NetworkBuilder.from_edges(
        Mlp, int(first[-1]), np.concatenate(src), np.concatenate(dst), weights=np.concatenate(weight),
        input_ids=list(range(sizes[0])), output_ids=list(range(int(first[-2]), int(first[-1]))), globals_=None,
        device="cuda")


def data(sizes, count: int, batch: int, dtype: torch.dtype, seed: int = 1):
    """Batches of a fixed random map of the inputs to learn."""
    rng = torch.Generator(device="cuda").manual_seed(seed)
    teacher = torch.randn((sizes[0], sizes[-1]), generator=rng, device="cuda") / sizes[0] ** 0.5
    for _ in range(count):
        x = torch.randn((batch, sizes[0]), generator=rng, device="cuda")
        yield x.to(dtype), torch.tanh(x @ teacher)


def main(steps: int = 200, batch: int = 256, dtype: torch.dtype = torch.bfloat16, samples: int = 4):
    """(first losses' mean, last losses' mean, largest difference of the arena's answers from the 4-bit pairs')."""
    weights, losses = train(SIZES, data(SIZES, steps, batch, dtype), rate=0.5)
    pairs = [lowbit.quantise4(w) for w in weights]
    static, state = edge_net(pairs)
    step, worst = px.make_step(Mlp, static), 0.0
    outputs = torch.tensor(static.output_ids, device="cuda")
    for x, _ in data(SIZES, samples, 1, torch.float32, seed=2):
        state = step(state, px.StepInputs(x[0].cpu().numpy())).state
        arena = state.units["activation"][outputs]
        worst = max(worst, float((arena - answer(pairs, x)[0]).abs().max()))
    n = max(1, steps // 10)
    return sum(losses[:n]) / n, sum(losses[-n:]) / n, worst


if __name__ == "__main__":
    first, last, worst = main()
    print(f"loss {first:.4f} -> {last:.4f} with 4-bit weights and 8-bit kept activations; "
          f"the edge arena's answers differ by {worst:.1e} at most")
