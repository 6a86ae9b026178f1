"""plastax_amd.lowbit's plans and argument checks at their limits (CPU only:
no kernel is launched)."""

from __future__ import annotations

import contextlib
import ctypes
import types

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
    monkeypatch.setattr(lowbit, "_workspace", lambda *a: None)
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


def test_plans_and_launches_run_with_the_arguments_device_current(monkeypatch) -> None:
    """Both count the current device's CUs: a size query on another one's plan is a workspace too small."""
    current, seen = [0], []

    @contextlib.contextmanager
    def device(index):
        was, current[0] = current[0], index
        yield
        current[0] = was

    def entry(name, result):
        return lambda *args: seen.append((name, current[0])) or result

    lib = types.SimpleNamespace(**{n: entry(n, 0) for n in ("plx_mx_workspace", "plx_mx_product", "plx_mx4_workspace",
                                                            "plx_mx4_product")})
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    for index in (0, 1):
        at = torch.device("cuda", index)
        for name in ("plx_mx_workspace", "plx_mx4_workspace"):
            assert lowbit._workspace(at, name) is None
        for name in ("plx_mx_product", "plx_mx4_product"):
            lowbit._launch(at, name)
        assert [i for _, i in seen] == [index] * 4 and current == [0]
        seen.clear()


def test_the_shapes_of_the_large_products_tests_are_large(lib) -> None:
    """Each holds its codes as bf16, for each of the four products, types and layouts; some run in ranges of k."""
    from test_gpu_lowbit import LARGE

    ranges = set()
    for tokens, inputs, outputs in LARGE:
        for kind in (PRODUCT, PRODUCT_GRAD, WEIGHT_GRAD, WEIGHT_GRAD_COLUMNS):
            m, n, k = ((tokens, outputs, inputs), (tokens, inputs, outputs), (outputs, inputs, tokens))[min(kind, 2)]
            units = inputs if kind == PRODUCT else outputs
            for dtype in (F32, BF16, F16):
                for at, strides in ((P, (units, 1)), (P, (1, tokens)), (P + 2, (units + 3, 1))):
                    need = lib.plx_mx_workspace(kind, tokens, inputs, outputs, dtype, at, *strides)
                    assert need >= 2 * -(-k // 64) * 64 * n, (kind, tokens, inputs, outputs, dtype)
                    ranges.add(need >= 2 * -(-k // 64) * 64 * (n + 3 * m) + 8 * m * n)
    assert ranges == {False, True}
    for tokens, inputs, outputs in ((2056, 2120, 6000), (1100, 5000, 4608), (264, 9600, 10000), (3001, 1300, 6500),
                                    (256, 131072, 768)):
        scales = (-(-tokens // 256) + -(-outputs // 256)) * -(-inputs // 256) * 2048
        parts = lib.plx_mx4_workspace(tokens, inputs, outputs) - scales
        assert parts >= 0 and parts % (4 * tokens * outputs) == 0
