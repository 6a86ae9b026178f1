"""plastax_amd.dense on the GPU at sizes that take the kernels' other forms: long runs of tiles, many tokens, frequent
ids. Against the plain 64-bit forms, within the bounds that they count."""

from __future__ import annotations

import pytest
import torch

import dense_plain as plain
import test_gpu_dense as base
from plastax_amd import dense

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


# --------------------------------------------------------------------------
# Layer norm
# --------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("units", [1, 64, 128, 1024, 2048, 4096, 8192, 16384, 32768])
def test_rows_of_one_large_value(units, dtype) -> None:
    """Rows without variance have n = 0, r = 1 / sqrt(eps), y = bias and dx = r (u - mean(u)), however large their value:
    their sums are whole multiples of a power of two below 2^24 of it, and exact, as is the mean over 2^k units.
    (r times the value is past float32: what lies behind a row's end must not come to it.)"""
    base._say("one value", units, dtype)
    g = base._gen(units, 3)
    tokens, eps = 5, 2.0**-40
    x = torch.tensor([2.0**112, -(2.0**112), 3.0, 0.0, 2.0**100], device=DEV)[:, None].expand(tokens, units).to(dtype)
    d, w, b = base._randn((tokens, units), g).to(dtype), base._randn((units,), g), base._randn((units,), g)
    y, kept = dense.normalise(x, w, b, eps)
    assert torch.equal(y, b.to(dtype).expand(tokens, units))
    assert torch.equal(kept[:, 0], x[:, 0].float()) and torch.equal(kept[:, 1], torch.full((tokens,), 2.0**20, device=DEV))
    (_, _), (dx, dx_off), (dw, _), (db, db_off) = plain.normalise(torch.zeros_like(x), w, b, eps, d)
    got = dense.normalise_grad(d, x, w, kept)
    plain.near(got[0], dx, dx_off + plain.rounded(dx, dtype))
    assert not dw.any() and not got[1].any()
    plain.near(got[2], db, db_off)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("units", [3, 100, 1003, 1425, 3396, 9000, 20001])
def test_the_mean_is_the_sum_over_the_units(units, dtype) -> None:
    """A sum that is exact has a mean that is: a row of one value c (few bits, so that units * c is a float32 number)
    has it for mean, and is normalised to the bias, also where one rounding of the mean, squared, would pass float32."""
    base._say("mean", units, dtype)
    g = base._gen(units, 4)
    x = torch.tensor([2.0**110, -3 * 2.0**100, 5.0, 100.0, 0.0], device=DEV)[:, None].expand(5, units).to(dtype)
    d, w, b = base._randn((5, units), g).to(dtype), base._randn((units,), g), base._randn((units,), g)
    y, kept = dense.normalise(x, w, b, 2.0**-20)
    assert torch.equal(kept[:, 0], x[:, 0].float()) and torch.equal(kept[:, 1], torch.full((5,), 2.0**10, device=DEV))
    assert torch.equal(y, b.to(dtype).expand(5, units))
    (_, _), (dx, dx_off), _, _ = plain.normalise(torch.zeros_like(x), w, b, 2.0**-20, d)
    got = dense.normalise_grad(d, x, w, kept)
    plain.near(got[0], dx, dx_off + plain.rounded(dx, dtype))
    assert not got[1].any()
