"""plastax_amd.lowbit's plans and argument checks at their limits (CPU only:
no kernel is launched)."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from plastax_amd import _lib, lowbit

P = 4096  # a pointer that is never followed
F32, BF16, F16 = range(3)
PRODUCT, PRODUCT_GRAD, WEIGHT_GRAD, WEIGHT_GRAD_COLUMNS = range(4)


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from plastax_amd import build

        build.build()
    return _lib.load()


@pytest.mark.parametrize("kind", [PRODUCT, PRODUCT_GRAD, WEIGHT_GRAD, WEIGHT_GRAD_COLUMNS])
def test_lines_that_run_backwards_are_copied_before_a_large_product(lib, kind) -> None:
    """A large product reads lines of bf16 where they are by 32-bit offsets, which go forwards only."""
    n = 4096
    weights = 2 * n * n  # the codes as bf16
    for strides in ((n, 1), (1, n), (0, 1), (2 * n, 1)):
        assert lib.plx_mx_workspace(kind, n, n, n, BF16, P, *strides) == weights
    for strides in ((-n, 1), (1, -n), (-2 * n, 1), (-8, 1), (n, -1), (-1, n)):
        assert lib.plx_mx_workspace(kind, n, n, n, BF16, P, *strides) == 2 * weights, strides


def _mx4(lines: int, n: int) -> lowbit.Mx4:
    b = -(-n // 128) * 4
    return lowbit.Mx4(torch.zeros((lines, 16 * b), dtype=torch.uint8), torch.full((lines, b), 127, dtype=torch.uint8), n)


def _mx8(shape: tuple[int, int]) -> lowbit.Mx8:
    b = -(-shape[1] // 32)
    return lowbit.Mx8(torch.zeros((shape[0], 32 * b), dtype=torch.uint8),
                      torch.full((shape[0], b), 127, dtype=torch.uint8), shape, 1)


def _calls():
    """Every function that takes a tensor [5, 70]."""
    w, wt, kept = _mx4(9, 70), _mx4(70, 9), _mx8((5, 70))
    return [lowbit.quantise4, lowbit.quantise8, lambda t: lowbit.activate(t, "tanh"),
            lambda t: lowbit.activate_grad(t, kept, "tanh"), lambda t: lowbit.product(t, w),
            lambda t: lowbit.product_grad(t, wt), lambda t: lowbit.weight_grad(t, kept)]


def test_views_are_given_as_the_values_that_they_stand_for(monkeypatch) -> None:
    """What a kernel finds where each call points it: the imaginary part of a conjugate is kept with the other sign."""
    seen = []

    def launch(device, name, *args):
        at = next(i for i, a in enumerate(args) if a > 1 << 20)  # the argument's address; its strides follow
        seen.append(torch.tensor([[ctypes.c_float.from_address(args[at] + 4 * (r * args[at + 1] + c * args[at + 2])).value
                                   for c in range(70)] for r in range(5)]))

    monkeypatch.setattr(lowbit, "_launch", launch)
    monkeypatch.setattr(lowbit, "_on_gpu", lambda *a: None)
    z = torch.complex(torch.randn(5, 70), torch.randn(5, 70))
    for x in (z.conj().imag, z.conj().imag[:, :], z.imag, z.real):
        for call in _calls():
            seen.clear()
            call(x)
            assert torch.equal(seen[0], x.clone())


def test_tangents_are_refused() -> None:
    """A result without the tangent would be a derivative of zero."""
    x = torch.randn(5, 70)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in _calls():
            with pytest.raises(ValueError, match="forward-mode"):
                call(dual)
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                call(dual)
            with pytest.raises(ValueError, match="GPU"):  # none of its own: as outside of the level
                call(forward_ad.unpack_dual(dual).primal)
            with pytest.raises(ValueError, match="GPU"):
                call(x)
