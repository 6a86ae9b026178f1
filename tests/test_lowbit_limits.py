"""plastax_amd.lowbit's plans and argument checks at their limits (CPU only:
no kernel is launched)."""

from __future__ import annotations

import pytest

from plastax_amd import _lib

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
