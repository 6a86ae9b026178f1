"""A net that reads tokens, taught by another one's answers.

One unit of the input level is on for each token; its level pair's rows are
looked up by id, normalised, and go through a level pair in 4 bits into a level
that is carried along the sequence. That one is normalised and answered by a
second 4-bit pair, one output for each token that may follow. The net learns
from a teacher that names a few outputs of each token (of sequences of
different lengths, packed into one batch, with states carried from batch to
batch), and is then run one token at a time: the same answers, up to the
rounding of float32 sums.

Run on the GPU: ``python examples/token_net.py``.
"""

from __future__ import annotations

import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))

from plastax_amd import dense, lowbit  # noqa: E402

TOKENS, WIDTH, CARRIED, NAMED = 300, 64, 96, 8  # ids, units of the levels, outputs that the teacher names
SCALE = 8.0  # of looked-up rows


def make(seed: int = 0) -> dict[str, torch.Tensor]:
    """The net's parameters in float32."""
    rng = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape: int) -> torch.Tensor:
        return torch.randn(shape, generator=rng, device="cuda")

    return {
        "table": randn(TOKENS, WIDTH) / SCALE,
        "weight1": torch.ones(WIDTH, device="cuda"), "bias1": torch.zeros(WIDTH, device="cuda"),
        "into": randn(2 * CARRIED, WIDTH) / WIDTH**0.5,  # x beside the gates' z
        "weight2": torch.ones(CARRIED, device="cuda"), "bias2": torch.zeros(CARRIED, device="cuda"),
        "out": randn(TOKENS, CARRIED) / CARRIED**0.5,
    }


def learn(net, batch, state):
    """(the tokens' losses, the parameters' gradients, the carried states) of the 4-bit net on a batch: ids, the
    sequences' starts, the named outputs and their logits."""
    ids, starts, named, top = batch
    into, out = lowbit.quantise4(net["into"]), lowbit.quantise4(net["out"])
    x = dense.look_up(ids, net["table"], SCALE)
    n1, kept1 = dense.normalise(x, net["weight1"], net["bias1"])
    n1_8 = lowbit.quantise8(n1)
    xz = lowbit.product(n1, into)
    h, last, walked = dense.recur(xz, starts, state)
    n2, kept2 = dense.normalise(h, net["weight2"], net["bias2"])
    n2_8 = lowbit.quantise8(n2)
    mean = torch.full((ids.shape[0],), 1.0 / ids.shape[0], device="cuda")
    loss, d = dense.distil_grad(mean, lowbit.product(n2, out), named, top, temperature=2.0)

    grads = {"out": lowbit.weight_grad(d, n2_8)}
    d, grads["weight2"], grads["bias2"] = dense.normalise_grad(lowbit.product_grad(d, out), h, net["weight2"], kept2)
    d, _ = dense.recur_grad(d, xz, walked, starts, state)
    grads["into"] = lowbit.weight_grad(d, n1_8)
    d, grads["weight1"], grads["bias1"] = dense.normalise_grad(lowbit.product_grad(d, into), x, net["weight1"], kept1)
    grads["table"] = dense.look_up_grad(d, ids, TOKENS, SCALE)
    return loss, grads, last


def answer(net, pairs, ids, state):
    """The outputs for one new token of each sequence; the states go on in place."""
    into, out = pairs
    n, _ = dense.normalise(dense.look_up(ids, net["table"], SCALE), net["weight1"], net["bias1"])
    h = dense.recur_step(lowbit.product(n, into), state)
    n, _ = dense.normalise(h, net["weight2"], net["bias2"])
    return lowbit.product(n, out)


def batches(count: int, sequences: int = 6, tokens: int = 256, seed: int = 1):
    """Packed sequences, and what a fixed random teacher says may follow each token."""
    rng = torch.Generator(device="cuda").manual_seed(seed)
    teacher = 3 * torch.randn((TOKENS, TOKENS), generator=rng, device="cuda")
    for _ in range(count):
        ids = torch.randint(TOKENS, (tokens,), generator=rng, device="cuda")
        cuts = torch.sort(torch.randint(tokens + 1, (sequences - 1,), generator=rng, device="cuda")).values
        starts = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), tokens)])
        top, named = torch.topk(teacher[ids], NAMED)
        yield ids, starts, named, top


def main(steps: int = 300, rate: float = 0.5):
    """(first losses' mean, last losses' mean, largest difference of single tokens' answers from the batch's)."""
    net, losses, state = make(), [], None
    for batch in batches(steps):
        loss, grads, state = learn(net, batch, state)
        for name, grad in grads.items():
            net[name] -= rate * grad
        losses.append(loss.mean())
    losses = torch.stack(losses).tolist()

    pairs = [lowbit.quantise4(net["into"]), lowbit.quantise4(net["out"])]
    ids = torch.arange(20, device="cuda") % TOKENS
    n, _ = dense.normalise(dense.look_up(ids, net["table"], SCALE), net["weight1"], net["bias1"])
    n, _ = dense.normalise(dense.recur(lowbit.product(n, pairs[0]))[0], net["weight2"], net["bias2"])
    whole = lowbit.product(n, pairs[1])
    now = torch.zeros((1, CARRIED), device="cuda")
    worst = max(float((answer(net, pairs, ids[t : t + 1], now)[0] - whole[t]).abs().max()) for t in range(ids.shape[0]))
    n = max(1, steps // 10)
    return sum(losses[:n]) / n, sum(losses[-n:]) / n, worst


if __name__ == "__main__":
    first, last, worst = main()
    print(f"loss {first:.4f} -> {last:.4f} with 4-bit level pairs; one token at a time the answers differ by {worst:.1e} "
          "at most")
