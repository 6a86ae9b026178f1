"""examples/token_net.py: the run of the operators around 4-bit level pairs, its gradients against autograd in 64 bits,
and single tokens' answers against the batch's."""

from __future__ import annotations

import pathlib
import sys

import pytest
import torch

from plastax_amd import dense, lowbit

pytestmark = pytest.mark.gpu

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "examples"))


def _norm(x, w, b):
    x = x - x.mean(1, keepdim=True)
    return x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-5) * w + b


def test_the_examples_gradients_are_autograds() -> None:
    """In 64 bits with the pairs' 4-bit values and, for the pairs' own gradients, their inputs' 8-bit values. The
    float32 net's roundings are some 2^-24 an operation over sums of up to 300 terms: 1e-4 of a gradient's norm is
    over ten times what they add up to. (Inputs that lie next to a border of the 8-bit codes may round the other way
    in float32: the codes are taken from the float32 net's own inputs, which differ from the 64-bit ones by 1e-6.)"""
    import token_net as ex

    net = ex.make(3)
    batch = next(iter(ex.batches(1, seed=4)))
    ids, starts, named, top = batch
    rng = torch.Generator(device="cuda").manual_seed(5)
    state = torch.randn((starts.shape[0] - 1, ex.CARRIED), generator=rng, device="cuda")
    loss, grads, last = ex.learn(net, batch, state)

    w = {k: v.double().requires_grad_() for k, v in net.items()}
    into, out = (lowbit.quantise4(net[k]).values().double().requires_grad_() for k in ("into", "out"))
    x = w["table"][ids] * ex.SCALE
    n1 = _norm(x, w["weight1"], w["bias1"])
    xz = n1 @ into.t()
    xz.retain_grad()
    a, b, v = torch.sigmoid(xz[:, ex.CARRIED :]), torch.sigmoid(-xz[:, ex.CARRIED :]), xz[:, : ex.CARRIED]
    rows, ends = [], []
    cuts = starts.tolist()
    for s in range(len(cuts) - 1):
        now = state[s].double()
        for t in range(cuts[s], cuts[s + 1]):
            now = a[t] * now + b[t] * v[t]
            rows.append(now)
        ends.append(now)
    h = torch.stack(rows)
    n2 = _norm(h, w["weight2"], w["bias2"])
    logits = n2 @ out.t()
    logits.retain_grad()
    p = torch.softmax(top.double() / 2, 1)
    want = 4 * (p * (torch.log(p) - torch.log_softmax(logits / 2, 1).gather(1, named))).sum(1)
    want.mean().backward()

    assert float((loss.double() - want.detach()).abs().max()) <= 1e-4 * float(want.detach().abs().max())
    assert float((last.double() - torch.stack(ends).detach()).abs().max()) <= 1e-5 * float(torch.stack(ends).detach().abs().max())
    y, _ = dense.normalise(dense.look_up(ids, net["table"], ex.SCALE), net["weight1"], net["bias1"])
    n1_8 = lowbit.quantise8(y).values().double()
    f, _, _ = dense.recur(lowbit.product(y, lowbit.quantise4(net["into"])), starts, state)
    n2_8 = lowbit.quantise8(dense.normalise(f, net["weight2"], net["bias2"])[0]).values().double()
    expected = {"into": xz.grad.t() @ n1_8, "out": logits.grad.t() @ n2_8,
                **{k: w[k].grad for k in ("table", "weight1", "bias1", "weight2", "bias2")}}
    for name, grad in grads.items():
        assert float((grad.double() - expected[name]).norm()) <= 1e-4 * float(expected[name].norm()), name


def test_the_example_runs_and_single_tokens_are_answered_as_batches_are() -> None:
    import token_net as ex

    first, last, worst = ex.main(steps=20)
    assert first == first and last == last
    # (differences of sums in another order through three levels: some 1e-6 of answers of a few units)
    assert worst < 1e-4
