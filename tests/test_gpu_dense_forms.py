"""plastax_amd.dense on the GPU at sizes that take the kernels' other forms: long runs of tiles, many tokens, frequent
ids. Against the plain 64-bit forms, within the bounds that they count."""

from __future__ import annotations

import pytest
import torch

import dense_plain as plain
import test_gpu_dense as base

pytestmark = pytest.mark.gpu

DEV = base.DEV
F32, BF16, F16 = plain.DTYPES


# --------------------------------------------------------------------------
# A level carried along sequences
# --------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16], ids=str)
@pytest.mark.parametrize("units", [129, 1003])
def test_recur_over_rows_of_tiles_with_a_last_slab_in_part(units, dtype) -> None:
    """More than 64 tiles forwards (of 128 rows) and backwards (of 64), so that sums go through groups and rows of
    groups, in levels whose last slab of 128 units has lanes without any, or with one of two."""
    tokens = 8192 + 261
    base._say("recur long", tokens, units, dtype)
    g = base._gen(tokens, units)
    xz, d = base._xz(tokens, units, dtype, g), base._randn((tokens, units), g).to(dtype)
    state, g_last = base._randn((1, units), g), base._randn((1, units), g)
    base._check_recur(xz, [0, tokens], state, d, g_last, None)
    starts = [3, 130, 130, 8200, 8201, tokens - 2]
    state, g_last = base._randn((5, units), g), base._randn((5, units), g)
    base._check_recur(xz, starts, state, d, g_last, torch.int32)
