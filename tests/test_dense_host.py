"""plastax_amd.dense's refusals, its entry points' checks, and the plain 64-bit
forms against differences (CPU only: no kernel is launched)."""

from __future__ import annotations

import contextlib
import types

import pytest
import torch
from torch.autograd import forward_ad

import dense_plain as plain
from plastax_amd import _lib, dense

P = 4096  # a pointer that is never followed: each call below is refused, or has nothing to do


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from plastax_amd import build

        build.build()
    return _lib.load()


def _calls():
    """Every function that takes a batch, as a call of it (5 tokens of 8 units)."""
    ids, w, named = torch.zeros(5, dtype=torch.int64), torch.ones(8), torch.zeros((5, 2), dtype=torch.int32)
    top, g, kept = torch.zeros((5, 2)), torch.ones(5), torch.zeros((5, 2))
    return {
        "look_up": lambda t: dense.look_up(ids, t),
        "look_up_grad": lambda t: dense.look_up_grad(t, ids, 7),
        "normalise": lambda t: dense.normalise(t, w),
        "normalise_grad": lambda t: dense.normalise_grad(t, t, w, kept),
        "recur": lambda t: dense.recur(t),
        "recur_grad": lambda t: dense.recur_grad(t[:, :4], t, torch.zeros((1, 4))),
        "recur_step": lambda t: dense.recur_step(t, torch.zeros((5, 4))),
        "distil": lambda t: dense.distil(t, named, top),
        "distil_grad": lambda t: dense.distil_grad(g, t, named, top),
    }


@pytest.mark.parametrize("name", list(_calls()))
def test_batches_are_checked(name) -> None:
    call, x = _calls()[name], torch.zeros(5, 8)
    with pytest.raises(TypeError):
        call(x.double())
    with pytest.raises(TypeError):
        call(x.int())
    with pytest.raises((ValueError, IndexError)):
        call(x[0])
    with pytest.raises(ValueError, match="GPU"):  # there is no CPU fallback
        call(x)
    with pytest.raises(ValueError, match="GPU"):
        call(x.t().contiguous().t())
    with pytest.raises(ValueError, match="autograd"):
        call(x.clone().requires_grad_())
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
        call(x.clone().requires_grad_())
    with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        call(forward_ad.make_dual(x, torch.ones_like(x)))


def test_ids_and_tables_are_checked() -> None:
    table, ids = torch.zeros(7, 8), torch.zeros(5, dtype=torch.int64)
    for bad in (ids.float(), ids.to(torch.int16), ids.to(torch.uint8), ids.bool()):
        with pytest.raises(TypeError, match="int32 or int64"):
            dense.look_up(bad, table)
        with pytest.raises(TypeError, match="int32 or int64"):
            dense.look_up_grad(table[:5], bad, 7)
    with pytest.raises(ValueError, match="1 dimensions"):
        dense.look_up(ids[None], table)
    with pytest.raises(ValueError, match="ids expected"):
        dense.look_up_grad(table, ids, 7)
    for rows in (-1, (1 << 24) + 1):
        with pytest.raises(ValueError, match="rows expected"):
            dense.look_up_grad(table[:5], ids, rows)
    with pytest.raises(ValueError, match="2\\^24 rows"):
        dense.look_up(ids, torch.zeros(1, 8).expand((1 << 24) + 1, 8))
    with pytest.raises(ValueError, match="2\\^30 tokens"):
        dense.normalise(torch.zeros(1, 8).expand((1 << 30) + 1, 8), torch.ones(8))


def test_parameters_are_checked() -> None:
    x, w = torch.zeros(5, 8, dtype=torch.bfloat16), torch.ones(8)
    for bad in (w.double(), w.half()):
        with pytest.raises(TypeError, match="weight and bias"):
            dense.normalise(x, bad)
    with pytest.raises(TypeError, match="weight and bias"):
        dense.normalise(x, w, w.bfloat16())
    with pytest.raises(ValueError, match="8 units"):
        dense.normalise(x, w[1:])
    with pytest.raises(ValueError, match="8 units"):
        dense.normalise(x, w, w[None])
    for eps in (-1e-9, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            dense.normalise(x, w, eps=eps)
    with pytest.raises(ValueError, match="autograd"):
        dense.normalise(x, w.clone().requires_grad_())
    kept = torch.zeros(5, 2)
    with pytest.raises(TypeError, match="gradient of x's type"):
        dense.normalise_grad(x.float(), x, w, kept)
    with pytest.raises(ValueError, match="gradient of"):
        dense.normalise_grad(x[1:], x, w, kept)
    with pytest.raises(ValueError, match="kept of"):
        dense.normalise_grad(x, x, w, kept[1:])
    with pytest.raises(TypeError, match="kept of float32"):
        dense.normalise_grad(x, x, w, kept.double())


def test_sequences_are_checked() -> None:
    xz, starts = torch.zeros(5, 8), torch.tensor([0, 2, 5])
    with pytest.raises(ValueError, match="even"):
        dense.recur(xz[:, 1:])
    with pytest.raises(TypeError, match="starts of int32"):
        dense.recur(xz, starts.float())
    with pytest.raises(ValueError, match="starts of 1"):
        dense.recur(xz, starts[:0])
    for state in (torch.zeros(3, 4), torch.zeros(2, 8), torch.zeros(4)):
        with pytest.raises(ValueError, match="state of"):
            dense.recur(xz, starts, state)
    with pytest.raises(TypeError, match="state of float32"):
        dense.recur(xz, starts, torch.zeros(2, 4, dtype=torch.bfloat16))
    g, kept = torch.zeros(5, 4), torch.zeros(1, 4)
    with pytest.raises(TypeError, match="gradient of xz's type"):
        dense.recur_grad(g.half(), xz, kept)
    with pytest.raises(ValueError, match="a gradient of"):
        dense.recur_grad(xz, xz, kept)
    with pytest.raises(ValueError, match="kept of"):
        dense.recur_grad(g, xz, kept[:0])
    with pytest.raises(ValueError, match="GPU"):
        dense.recur_grad(g, xz, kept, g_last=torch.zeros(1, 4))


def test_states_in_place_are_checked() -> None:
    xz = torch.zeros(5, 8)
    with pytest.raises(ValueError, match="even"):
        dense.recur_step(xz[:, 1:], torch.zeros(5, 3))
    with pytest.raises(TypeError, match="float32"):
        dense.recur_step(xz, torch.zeros(5, 4, dtype=torch.float64))
    with pytest.raises(ValueError, match="a state of"):
        dense.recur_step(xz, torch.zeros(4, 4))
    for state in (torch.zeros(4, 5).t(), torch.zeros(1, 4).expand(5, 4), torch.zeros(5, 8)[:, ::2]):
        with pytest.raises(ValueError, match="in place"):
            dense.recur_step(xz, state)
    with pytest.raises(ValueError, match="in place"):
        dense.recur_step(xz, torch.complex(torch.zeros(5, 4), torch.zeros(5, 4)).conj().imag)
    with pytest.raises(ValueError, match="autograd"):
        dense.recur_step(xz, torch.zeros(5, 4).requires_grad_())


def test_teachers_are_checked() -> None:
    x, ids, top = torch.zeros(5, 8), torch.zeros((5, 2), dtype=torch.int64), torch.zeros(5, 2)
    with pytest.raises(TypeError, match="ids of int32"):
        dense.distil(x, ids.float(), top)
    with pytest.raises(ValueError, match="ids of"):
        dense.distil(x, ids[1:], top)
    with pytest.raises(ValueError, match="at most 1024"):
        dense.distil(x, ids.expand(5, 2).repeat(1, 513), top.repeat(1, 513))
    with pytest.raises(ValueError, match="top of"):
        dense.distil(x, ids, top[:, :1])
    with pytest.raises(TypeError):
        dense.distil(x, ids, top.double())
    for t in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            dense.distil(x, ids, top, t)
    with pytest.raises(TypeError, match="g of float32"):
        dense.distil_grad(torch.ones(5).half(), x, ids, top)
    with pytest.raises(ValueError, match="g of"):
        dense.distil_grad(torch.ones(5, 1), x, ids, top)


@pytest.mark.parametrize("t", [1e-37, 2.0**-121, 2.0**121, 3e38])
def test_temperatures_whose_inverse_float32_has_not_are_refused(lib, t) -> None:
    x, ids, top = torch.zeros(5, 8), torch.zeros((5, 2), dtype=torch.int64), torch.zeros(5, 2)
    with pytest.raises(ValueError, match="temperature"):
        dense.distil(x, ids, top, t)
    assert lib.plx_distil(5, 8, 2, 0, P, 8, P, 1, 0, P, t, P, None) == 1
    assert lib.plx_distil_grad(5, 8, 2, P, 0, P, 8, P, 1, 0, P, t, P, P, None) == 1


def test_plans_and_launches_run_with_the_arguments_device_current(monkeypatch) -> None:
    """A plan counts the current device's CUs, as the launch does that its workspace is for."""
    current, seen = [0], []

    @contextlib.contextmanager
    def device(index):
        was, current[0] = current[0], index
        yield
        current[0] = was

    names = ("plx_look_up_workspace", "plx_normalise_workspace", "plx_recur_workspace", "plx_recur")
    entries = {n: (lambda *args, n=n: seen.append((n, current[0])) or 0) for n in names}
    monkeypatch.setattr(_lib, "load", lambda: types.SimpleNamespace(**entries))
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    for index in (0, 1):
        at = torch.device("cuda", index)
        for name in names[:3]:
            assert dense._space(at, name, 5, 8, 8) == (None, None, 0)
        dense._launch(at, names[3])
        assert seen == [(n, index) for n in names] and current == [0]
        seen.clear()


def test_sizes_out_of_range_have_no_workspace(lib) -> None:
    assert lib.plx_look_up_workspace((1 << 25) + 1, 7, 8) == -1
    assert lib.plx_look_up_workspace(1 << 25, 7, 8) > 0
    assert lib.plx_recur_workspace(1 << 28, 128, 1, 0) > 0
    assert lib.plx_recur_workspace((1 << 28) + 1, 128, 1, 0) == -1
    assert lib.plx_recur_workspace(1 << 28, 129, 1, 0) == -1


def test_entry_points_check_before_they_launch(lib) -> None:
    bad, unknown = 1, 3
    big = (1 << 24) + 1
    assert lib.plx_look_up(-1, 7, 8, P, 0, 0, P, 8, 1.0, P, None) == bad
    assert lib.plx_look_up(5, big, 8, P, 0, 0, P, 8, 1.0, P, None) == bad
    assert lib.plx_look_up(5, 7, 8, P, 2, 0, P, 8, 1.0, P, None) == bad
    assert lib.plx_look_up(5, 7, 8, P, 0, 3, P, 8, 1.0, P, None) == unknown
    assert lib.plx_look_up(5, 7, 8, None, 0, 0, P, 8, 1.0, P, None) == bad
    assert lib.plx_look_up(0, 7, 8, None, 0, 0, None, 8, 1.0, None, None) == 0
    assert lib.plx_look_up_grad(5, 7, 8, P, 0, 0, P, 8, 1.0, P, None, 0, None) == bad
    assert b"plx_look_up_workspace" in lib.plx_last_error()
    assert lib.plx_look_up_grad(5, 7, 8, P, 0, 0, P, 8, 1.0, None, P, 1 << 30, None) == bad
    assert lib.plx_look_up_grad(5, 0, 8, P, 0, 0, P, 8, 1.0, P, None, 0, None) == 0
    assert lib.plx_look_up_grad((1 << 25) + 1, 7, 8, P, 0, 0, P, 8, 1.0, P, P, 1 << 62, None) == bad
    assert lib.plx_look_up_workspace(-1, 7, 8) == -1 and lib.plx_look_up_workspace((1 << 25) + 1, 7, 8) == -1
    assert lib.plx_look_up_workspace(5, big, 8) == -1
    assert lib.plx_normalise(5, big, 0, P, 8, 0, P, P, 1e-5, P, P, None) == bad
    assert lib.plx_normalise(5, 8, 1, P, 8, 2, P, P, 1e-5, P, P, None) == unknown
    assert lib.plx_normalise(5, 8, 0, P, 8, 0, P, P, -1.0, P, P, None) == bad
    assert lib.plx_normalise(5, 8, 0, P, 8, 0, None, P, 1e-5, P, P, None) == bad
    assert lib.plx_normalise(5, 0, 0, None, 8, 0, None, None, 1e-5, None, None, None) == 0
    assert lib.plx_normalise_grad(5, 8, 0, P, 8, P, 8, 0, P, P, P, P, None, 0, None) == bad
    assert b"plx_normalise_workspace" in lib.plx_last_error()
    assert lib.plx_normalise_grad(5, 8, 0, None, 8, P, 8, 0, P, P, P, P, P, 1 << 30, None) == bad
    assert lib.plx_normalise_workspace(5, 8, 7) == -1 and lib.plx_normalise_workspace(-5, 8, 0) == -1
    assert lib.plx_recur(5, 4, 2, 0, P, 8, None, 0, None, P, P, P, None, 0, None) == bad  # no starts, two sequences
    assert lib.plx_recur(5, 4, 1, 5, P, 8, None, 0, None, P, P, P, None, 0, None) == unknown
    assert lib.plx_recur(5, 4, 1, 0, P, 8, None, 0, None, P, None, P, None, 0, None) == bad
    assert lib.plx_recur(5, (1 << 23) + 1, 1, 0, P, 8, None, 0, None, P, P, P, None, 0, None) == bad
    assert lib.plx_recur(5, 4, 2, 0, P, 8, P, 0, None, P, P, P, None, 0, None) == bad
    assert b"plx_recur_workspace" in lib.plx_last_error()
    assert lib.plx_recur(0, 4, 0, 0, None, 8, P, 0, None, None, None, None, None, 0, None) == 0
    assert lib.plx_recur_grad(5, 4, 1, 0, None, 4, P, 8, None, 0, None, None, P, P, P, None, 0, None) == bad
    assert lib.plx_recur_grad(5, 4, 2, 0, P, 4, P, 8, P, 0, None, None, P, P, P, None, 0, None) == bad
    assert lib.plx_recur_workspace(5, -4, 1, 0) == -1 and lib.plx_recur_workspace(5, 4, -1, 1) == -1
    assert lib.plx_recur_step(5, 4, 0, P, 8, None, 4, P, None) == bad
    assert lib.plx_recur_step(5, 4, 4, P, 8, P, 4, P, None) == unknown
    assert lib.plx_recur_step(0, 4, 0, None, 8, None, 4, None, None) == 0
    assert lib.plx_distil(5, 8, 1025, 0, P, 8, P, 0, 0, P, 1.0, P, None) == bad
    assert lib.plx_distil(5, 8, 2, 0, P, 8, P, 0, 3, P, 1.0, P, None) == unknown
    assert lib.plx_distil(5, 8, 2, 0, P, 8, P, 0, 0, P, 0.0, P, None) == bad
    assert lib.plx_distil(5, 8, 2, 0, P, 8, None, 0, 0, P, 1.0, P, None) == bad
    assert lib.plx_distil(0, 8, 2, 0, None, 8, None, 0, 0, None, 1.0, None, None) == 0
    assert lib.plx_distil_grad(5, 8, 2, None, 0, P, 8, P, 0, 0, P, 1.0, P, P, None) == bad
    assert lib.plx_distil_grad(5, 8, 2, P, 0, P, 8, P, 0, 0, P, 1.0, P, None, None) == bad


# --------------------------------------------------------------------------
# The plain forms' gradients against differences of their results in 64 bits: with a step of 1e-5 a central difference
# is off by some 1e-10 of the third derivative and 1e-11 of the value; 1e-6 of the sums' magnitudes is far above both.
# --------------------------------------------------------------------------
def _difference(f, x: torch.Tensor, v: torch.Tensor) -> float:
    return float(f(x + 1e-5 * v) - f(x - 1e-5 * v)) / 2e-5


def _rand(*shape: int, seed: int) -> torch.Tensor:
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def _agree(slope: float, grad: torch.Tensor, v: torch.Tensor) -> None:
    assert abs(slope - float((grad * v).sum())) <= 1e-6 * float((grad * v).abs().sum()) + 1e-9


def test_plain_gradients_are_the_differences() -> None:
    g, v = _rand(6, 10, seed=1), _rand(6, 10, seed=2)
    ids = torch.tensor([0, 3, -1, 3, 9, 1])
    grad, _ = plain.look_up_grad(g, ids, 5, 1.5)
    _agree(_difference(lambda w: (plain.look_up(ids, w, 1.5) * g).sum(), _rand(5, 10, seed=3), v[:5]), grad, v[:5])

    x, w, b = _rand(6, 10, seed=4), _rand(10, seed=5), _rand(10, seed=6)
    _, (dx, _), (dw, _), (db, _) = plain.normalise(x, w, b, 1e-3, g)
    _agree(_difference(lambda t: (plain.normalise(t, w, b, 1e-3)[0][0] * g).sum(), x, v), dx, v)
    _agree(_difference(lambda t: (plain.normalise(x, t, b, 1e-3)[0][0] * g).sum(), w, v[0]), dw, v[0])
    _agree(_difference(lambda t: (plain.normalise(x, w, t, 1e-3)[0][0] * g).sum(), b, v[0]), db, v[0])

    starts, state, g_last = [1, 4, 4, 6], _rand(3, 5, seed=7), _rand(3, 5, seed=8)
    h_grad = g[:, :5]
    _, _, (dxz, _), (ds, _) = plain.recur(x, starts, state, h_grad, g_last)

    def value(xz, s):
        (h, _), (last, _) = plain.recur(xz, starts, s)
        return (h * h_grad).sum() + (last * g_last).sum()

    _agree(_difference(lambda t: value(t, state), x, v), dxz, v)
    _agree(_difference(lambda t: value(x, t), state, v[:3, :5]), ds, v[:3, :5])

    ids = torch.tensor([[0, 3], [4, -1], [-1, 10], [9, 9], [1, 2], [5, 0]])
    top, weight = _rand(6, 2, seed=9), _rand(6, seed=10)
    top[4, 1] = -torch.inf
    (loss, _), (d, _) = plain.distil(x, ids, top, 1.5, weight)
    assert float(loss[2]) == 0.0 and float(d[2].abs().max()) == 0.0 and float(loss.min()) >= 0.0
    _agree(_difference(lambda t: (plain.distil(t, ids, top, 1.5)[0][0] * weight).sum(), x, v), d, v)


@pytest.mark.parametrize("eps", [1e-46, 1e-40, 2.0**-127, 1e39, 2.0**128])
def test_eps_that_float32_has_not_is_refused(eps) -> None:
    """1e-46 is 0 in float32: a row of one value would be NaN, where the formula gives the bias."""
    x, w = torch.zeros(5, 8), torch.ones(8)
    with pytest.raises(ValueError, match="eps"):
        dense.normalise(x, w, eps=eps)
    for fine in (0, 0.0, 2.0**-126, 2.0**127):
        with pytest.raises(ValueError, match="GPU"):
            dense.normalise(x, w, eps=fine)


@pytest.mark.parametrize("scale", [1e39, -1e39, 2.0**128, 1e-40, -(2.0**-127), 1e-300])
def test_scales_that_float32_has_not_are_refused(scale) -> None:
    """1e39 is an infinity in float32, and 0 times it a NaN."""
    table, ids = torch.zeros(7, 8), torch.zeros(5, dtype=torch.int64)
    with pytest.raises(ValueError, match="scale"):
        dense.look_up(ids, table, scale)
    with pytest.raises(ValueError, match="scale"):
        dense.look_up_grad(table[:5], ids, 7, scale)
    for fine in (0, 1, -2.5, 2.0**-126, 2.0**127, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="GPU"):
            dense.look_up(ids, table, fine)
        with pytest.raises(ValueError, match="GPU"):
            dense.look_up_grad(table[:5], ids, 7, fine)
