"""plastax_amd.lowbit's refusals, and the plain 64-bit forms its GPU tests
compare with (CPU only: no kernel is launched)."""

from __future__ import annotations

import pytest
import torch

import lowbit_plain as plain
from plastax_amd import _lib, lowbit


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from plastax_amd import build

        build.build()
    return _lib.load()


def _mx4(lines: int, n: int) -> lowbit.Mx4:
    b = -(-n // 128) * 4
    return lowbit.Mx4(torch.zeros((lines, 16 * b), dtype=torch.uint8), torch.full((lines, b), 127, dtype=torch.uint8), n)


def _mx8(shape: tuple[int, int], axis: int) -> lowbit.Mx8:
    b = -(-shape[axis] // 32)
    return lowbit.Mx8(torch.zeros((shape[1 - axis], 32 * b), dtype=torch.uint8),
                      torch.full((shape[1 - axis], b), 127, dtype=torch.uint8), shape, axis)


def test_plain_codes_are_torchs_and_the_tables() -> None:
    x = torch.randn(7, 96) * 3
    codes, scales = plain.quantise8(x)
    e = scales.double() - 127
    m = (x.double().view(7, 3, 32) * torch.exp2(-e)[:, :, None]).float()
    assert torch.equal(codes.view(7, 3, 32), m.to(torch.float8_e4m3fn).view(torch.uint8))
    assert torch.equal(plain.values8(codes, scales, 96).view(7, 3, 32),
                       m.to(torch.float8_e4m3fn).double() * torch.exp2(e)[:, :, None])
    grid = torch.tensor(plain.TABLE4 * 4)[None]  # the magnitudes themselves, under the scale 1
    codes, scales = plain.quantise4(grid)
    assert scales.tolist() == [[127, 2, 2, 2]]
    assert torch.equal(plain.values4(codes, scales, 32), grid.double())
    ties = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]])
    assert plain.values4(*plain.quantise4(ties), 8).tolist() == [[0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]]


def test_formats_are_checked() -> None:
    codes, scales = torch.zeros((3, 64), dtype=torch.uint8), torch.zeros((3, 4), dtype=torch.uint8)
    assert lowbit.Mx4(codes, scales, 128).shape == (3, 128)
    for n in (0, 129, -1):
        with pytest.raises(ValueError):
            lowbit.Mx4(codes, scales, n)
    with pytest.raises(TypeError):
        lowbit.Mx4(codes.int(), scales, 128)
    with pytest.raises(ValueError):
        lowbit.Mx4(codes, scales[:, :3], 128)
    with pytest.raises(ValueError):
        lowbit.Mx4(codes[0], scales, 128)
    with pytest.raises(ValueError, match="contiguous"):
        lowbit.Mx4(torch.zeros((64, 3), dtype=torch.uint8).t(), scales, 128)
    with pytest.raises(ValueError, match="16 bytes"):
        lowbit.Mx4(torch.zeros(3 * 64 + 1, dtype=torch.uint8)[1:].view(3, 64), scales, 128)
    assert _mx8((5, 70), 1).codes.shape == (5, 96) and _mx8((5, 70), 0).codes.shape == (70, 32)
    with pytest.raises(ValueError):
        lowbit.Mx8(torch.zeros((5, 64), dtype=torch.uint8), torch.zeros((5, 2), dtype=torch.uint8), (5, 70), 1)
    with pytest.raises(ValueError):
        lowbit.Mx8(torch.zeros((5, 96), dtype=torch.uint8), torch.zeros((5, 3), dtype=torch.uint8), (5, 70), 2)


def test_arguments_are_checked() -> None:
    x, w, kept = torch.zeros(5, 70), _mx4(9, 70), _mx8((5, 70), 1)
    calls = [lambda t: lowbit.quantise4(t), lambda t: lowbit.quantise8(t), lambda t: lowbit.activate(t, "relu"),
             lambda t: lowbit.activate_grad(t, kept, "relu"), lambda t: lowbit.product(t, w),
             lambda t: lowbit.product_grad(t, _mx4(70, 9)), lambda t: lowbit.weight_grad(t, kept)]
    for call in calls:
        with pytest.raises(TypeError):
            call(x.double())
        with pytest.raises(TypeError):
            call(x.int())
        with pytest.raises(ValueError):
            call(x[0])
        with pytest.raises(ValueError, match="GPU"):  # there is no CPU fallback
            call(x)
        with pytest.raises(ValueError, match="autograd"):
            call(x.clone().requires_grad_())
        with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
            call(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="inputs expected"):
        lowbit.product(x[:, 1:], w)
    with pytest.raises(ValueError, match="inputs expected"):
        lowbit.product(_mx4(5, 69), w)
    with pytest.raises(ValueError, match="outputs expected"):
        lowbit.product_grad(x, w)
    with pytest.raises(ValueError, match="tokens expected"):
        lowbit.weight_grad(x[1:], kept)
    with pytest.raises(ValueError, match="gradient of"):
        lowbit.activate_grad(x[:, 1:], kept, "relu")
    for fn in ("gelu", "", "ReLU"):
        with pytest.raises(ValueError, match="expected"):
            lowbit.activate(x, fn)
        with pytest.raises(ValueError, match="expected"):
            lowbit.activate_grad(x, kept, fn)
    with pytest.raises(ValueError, match="axis"):
        lowbit.activate(x, "relu", axis=-1)
    with pytest.raises(ValueError, match="axis"):
        lowbit.quantise8(x, axis=2)
    with pytest.raises(TypeError):
        lowbit.product(x, w, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        lowbit.product(_mx4(5, 70), w, dtype=torch.float64)
    with pytest.raises(TypeError):
        w.values(torch.float64)
    with pytest.raises(ValueError, match="GPU"):
        w.values()
    with pytest.raises(ValueError, match="GPU"):
        kept.values()


def test_entry_points_check_before_they_launch(lib) -> None:
    p = 4096  # a pointer that is never followed: each call below is refused, or has nothing to do
    assert lib.plx_mx4_quantise(-1, 4, 0, p, 4, 1, p, p, None) == 1
    assert lib.plx_mx4_quantise(4, (1 << 30) + 1, 0, p, 4, 1, p, p, None) == 1
    assert lib.plx_mx4_quantise(4, 4, 3, p, 4, 1, p, p, None) == 3
    assert lib.plx_mx4_quantise(4, 4, 0, None, 4, 1, p, p, None) == 1
    assert lib.plx_mx4_quantise(4, 4, 0, p, 4, 1, p + 1, p, None) == 1
    assert b"16 bytes" in lib.plx_last_error()
    assert lib.plx_mx4_quantise(0, 4, 0, None, 4, 1, None, None, None) == 0
    assert lib.plx_mx_values(5, 4, 4, p, p, 0, p, None) == 3
    assert lib.plx_mx_values(4, 4, 4, p, None, 0, p, None) == 1
    assert lib.plx_mx_values(8, 4, 0, None, None, 0, None, None) == 0
    assert lib.plx_mx8_activate(4, 4, 0, 4, p, 4, 1, p, 4, 1, p, p, None) == 3
    assert lib.plx_mx8_activate(4, 4, 0, 0, None, 4, 1, p, 4, 1, p, p, None) == 1
    assert lib.plx_mx8_activate(4, 4, 0, 0, p, 4, 1, None, 4, 1, None, p, None) == 1
    assert lib.plx_mx8_activate(4, 0, 0, 0, None, 4, 1, None, 4, 1, None, None, None) == 0
    assert lib.plx_mx8_activate_grad(4, 4, 0, -1, p, 4, 1, p, p, p, 4, 1, None) == 3
    assert lib.plx_mx8_activate_grad(4, 4, 7, 0, p, 4, 1, p, p, p, 4, 1, None) == 3
    assert lib.plx_mx8_activate_grad(4, 4, 0, 0, p, 4, 1, p + 8, p, p, 4, 1, None) == 1
    assert lib.plx_mx_product(4, 4, 4, 4, 0, p, 4, 1, p, p, p, None, 0, None) == 3
    assert lib.plx_mx_product(0, 4, -4, 4, 0, p, 4, 1, p, p, p, None, 0, None) == 1
    assert lib.plx_mx_product(0, 4, 4, 4, 0, None, 4, 1, p, p, p, None, 0, None) == 1
    assert lib.plx_mx_product(0, 0, 4, 4, 0, None, 4, 1, p, p, None, None, 0, None) == 0
    assert lib.plx_mx_product(0, 4096, 4096, 4096, 1, p, 4096, 1, p, p, p, None, 0, None) == 1
    assert b"plx_mx_workspace" in lib.plx_last_error()
    assert lib.plx_mx4_product(4, 4, 4, p, p, p, p, 9, p, None, 0, None) == 3
    assert lib.plx_mx4_product(4, 4, 4, p, p, p, None, 0, p, None, 0, None) == 1
    assert lib.plx_mx4_product(4, 4, 0, None, None, None, None, 0, None, None, 0, None) == 0
    assert lib.plx_mx4_product(4096, 4096, 4096, p, p, p, p, 0, p, None, 0, None) == 1
    assert b"plx_mx4_workspace" in lib.plx_last_error()
    assert lib.plx_mx_workspace(0, -1, 4, 4, 0, p, 4, 1) == -1
    assert lib.plx_mx_workspace(9, 4, 4, 4, 0, p, 4, 1) == -1
    assert lib.plx_mx_workspace(0, 4, 4, 4, 5, p, 4, 1) == -1
    assert lib.plx_mx4_workspace(4, -1, 4) == -1
    assert lib.plx_mx4_workspace(4, 4, (1 << 24) + 1) == -1
    assert lib.plx_mx_product(0, 4, (1 << 24) + 1, 4, 0, p, 4, 1, p, p, p, None, 0, None) == 1
    assert lib.plx_mx4_product(4, 4, (1 << 24) + 1, p, p, p, p, 0, p, None, 0, None) == 1
