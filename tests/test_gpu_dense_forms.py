"""plastax_amd.dense on the GPU at sizes that take the kernels' other forms: long runs of tiles, many tokens, frequent
ids, the widest levels. Against the plain 64-bit forms, within the bounds that they count."""

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


def _cus() -> int:
    return torch.cuda.get_device_properties(DEV).multi_processor_count


# units that take 1, 2, 4, 8 and 16 waves a row (a chunk of 4 float32 or 8 16-bit units a lane), then 2 chunks a lane
# (and 4 of float32), filled and with a rest
WAVES = {1: 1, 2: 2, 4: 4, 8: 8, 16: 16, 32: 16, 64: 16}


@pytest.mark.parametrize("chunks", list(WAVES))
@pytest.mark.parametrize("dtype", plain.DTYPES, ids=str)
def test_normalise_of_many_tokens(chunks, dtype) -> None:
    """Several rows at a time, once over the chip and in rounds, with a rest of rows, and gradients with two workgroups
    a CU: from twice as many tokens on as the chip's waves take at once."""
    if chunks == 64 and dtype != F32:
        pytest.skip("rows of 16-bit units past two chunks a lane are not held in registers")
    waves, full = WAVES[chunks], chunks * 64 * (4 if dtype == F32 else 8)
    once = _cus() * 32 // waves
    for tokens, units, params in ((2 * once + 3, full - 3, dtype), (2 * once + 1, full, F32), (4 * once + 6, full - full // 5, F32)):
        base._say("normalise many", tokens, units, dtype, params)
        g = base._gen(tokens, units)
        x, d = base._levels(tokens, units, dtype, g), base._randn((tokens, units), g).to(dtype)
        w, b = (1 + 0.3 * base._randn((units,), g)).to(params), base._randn((units,), g).to(params)
        (y, off), (dx, dx_off), (dw, dw_off), (db, db_off) = plain.normalise(x, w, b, 1e-3, d)
        got, kept = dense.normalise(x, w, b, 1e-3)
        plain.near(got, y, off + plain.rounded(y, dtype))
        got = dense.normalise_grad(d, x, w, kept)
        plain.near(got[0], dx, dx_off + plain.rounded(dx, dtype))
        plain.near(got[1], dw, dw_off)
        plain.near(got[2], db, db_off)


def test_normalise_of_the_widest_levels() -> None:
    """2^24 units, the most that there may be."""
    units, g = 1 << 24, base._gen(24)
    x, d, w = base._levels(2, units, BF16, g), base._randn((2, units), g).to(BF16), 1 + 0.3 * base._randn((units,), g)
    (y, off), (dx, dx_off), (dw, dw_off), (db, db_off) = plain.normalise(x, w, None, 1e-3, d)
    got, kept = dense.normalise(x, w, None, 1e-3)
    plain.near(got, y, off + plain.rounded(y, BF16))
    got = dense.normalise_grad(d, x, w, kept)
    plain.near(got[0], dx, dx_off + plain.rounded(dx, BF16))
    plain.near(got[1], dw, dw_off)
    plain.near(got[2], db, db_off)


def test_normalise_of_wide_levels_over_several_launches() -> None:
    """Levels that no registers hold, of more than 2^20 tokens: all rows the same, and what one row gives."""
    tokens, units, g = (1 << 20) + 3, 16392, base._gen(20)
    x, d, w = base._randn((1, units), g).to(BF16), base._randn((1, units), g).to(BF16), base._randn((units,), g)
    one, one_kept = dense.normalise(x, w)
    y, kept = dense.normalise(x.expand(tokens, units), w)
    assert torch.equal(kept, one_kept.expand(tokens, 2))
    assert torch.equal(y[-5:], one.expand(5, units)) and torch.equal(y[:5], one.expand(5, units))
    del y
    one_dx, _, one_db = dense.normalise_grad(d, x, w, one_kept)
    dx, _, db = dense.normalise_grad(d.expand(tokens, units), x.expand(tokens, units), w, kept)
    assert torch.equal(dx[-5:], one_dx.expand(5, units)) and torch.equal(dx[:5], one_dx.expand(5, units))
    want = one_db.double() * tokens
    plain.near(db, want, (tokens / 64 + 150) * plain.EPS * want.abs())


# --------------------------------------------------------------------------
# An input level by ids
# --------------------------------------------------------------------------
@pytest.mark.parametrize("units", [70, 300])
def test_rows_of_the_gradient_around_a_part(units) -> None:
    """A part is 16 places of the list: rows of 15, 16, 17 tokens and so on that begin at each of its places. (Rows of
    a class, ids 256 apart, lie behind each other in the list. Whole numbers: exact sums.)"""
    for first in range(16):
        runs = [first, 15, 16, 17, 1, 31, 32, 33, 14, 47, 48, 49, 2, 16, 16, 16]
        ids = torch.cat([torch.full((n,), 256 * i, device=DEV) for i, n in enumerate(runs)])
        g = base._gen(first, units)
        ids = ids[torch.randperm(ids.shape[0], generator=g, device=DEV)]
        grad = torch.randint(-8, 9, (ids.shape[0], units), generator=g, device=DEV).float()
        want = torch.zeros((256 * len(runs), units), dtype=torch.float64, device=DEV).index_add_(0, ids, grad.double())
        assert torch.equal(dense.look_up_grad(grad, ids, 256 * len(runs)).double(), want), first


@pytest.mark.parametrize("wide", [torch.int32, torch.int64], ids=str)
@pytest.mark.parametrize("rows", [1, 3, 10, 700])
def test_frequent_ids(rows, wide) -> None:
    """More tokens of a class than a wave of the sort has room for (512), of one row, of a few, and of one beside many
    rare ones. (Whole numbers: exact sums.)"""
    for tokens, units in ((20000, 70), (9001, 600)):
        base._say("frequent", tokens, rows, units, wide)
        g = base._gen(tokens, rows)
        ids = torch.randint(rows, (tokens,), generator=g, device=DEV)
        if rows == 700:
            ids[torch.rand((tokens,), generator=g, device=DEV) < 0.6] = 300
        ids[7::50] = -1
        grad = torch.randint(-8, 9, (tokens, units), generator=g, device=DEV).to(BF16)
        there = ids >= 0
        want = torch.zeros((rows, units), dtype=torch.float64, device=DEV).index_add_(0, ids[there], grad[there].double())
        assert torch.equal(dense.look_up_grad(grad, ids.to(wide), rows).double(), want)


def test_one_id_of_more_tokens_than_a_place_has_bits_for() -> None:
    """From 2^24 tokens on a wave's range of them is longer than 2^20. (A broadcast gradient of one: exact sums.)"""
    tokens = (1 << 24) + 4097
    ids = torch.zeros(tokens, dtype=torch.int32, device=DEV)
    ids[::3], ids[5::7] = 2, 259
    want = torch.bincount(ids, minlength=300)[:, None]
    one = torch.ones((1, 1), device=DEV).expand(tokens, 1)
    assert torch.equal(dense.look_up_grad(one, ids, 300), want.float())


def test_look_up_of_the_widest_levels() -> None:
    units, g = 1 << 24, base._gen(25)
    grad = torch.randint(-8, 9, (1, units), generator=g, device=DEV).to(BF16)
    ids = torch.tensor([1] * 18 + [0] * 3, device=DEV)
    got = dense.look_up_grad(grad.expand(21, units), ids, 2)
    assert torch.equal(got, grad.float() * torch.tensor([[3.0], [18.0]], device=DEV))
    assert torch.equal(dense.look_up(ids[17:19], got.to(BF16)), got[[1, 0]].to(BF16))


# --------------------------------------------------------------------------
# An output level learned from a teacher
# --------------------------------------------------------------------------
@pytest.mark.parametrize("chunks", [1, 64, 65, 100, 128, 129, 256, 257, 400, 512, 513, 1024, 1025, 2048])
@pytest.mark.parametrize("dtype", plain.DTYPES, ids=str)
def test_distil_of_many_tokens(chunks, dtype) -> None:
    """From two tokens a CU on rows go to few waves with several chunks of 16 bytes a lane."""
    tokens, w = 2 * _cus() + 61, 4 if dtype == F32 else 8
    for outputs, named, wide, layout in ((chunks * w, 5, torch.int64, "rows"), (chunks * w - w + 1, 70, torch.int32, "apart")):
        base._say("distil many", tokens, outputs, dtype)
        g = base._gen(tokens, outputs, named)
        logits = (3 * base._randn((tokens, outputs), g)).to(dtype)
        if outputs > 5:
            logits[:, 3::9] = -torch.inf
            logits[:, 4::9] = torch.finfo(dtype).min
        ids, top = base._teacher(tokens, outputs, named, wide, g)
        finite = torch.isfinite(torch.gather(logits, 1, ids.long().clamp(0, outputs - 1)))
        ids[1:][~finite[1:]] = -1  # (a named output of -inf has an infinite loss: the first token keeps its)
        weight = torch.rand((tokens,), generator=g, device=DEV)
        weight[::5] = 0
        (loss, off), (d, d_off) = plain.distil(logits, ids, top, 2.0, weight)
        x = base._layout(logits, layout)
        got = dense.distil_grad(weight, x, ids, top, 2.0)
        plain.near(got[0], loss, off)
        plain.near(got[1], d, d_off + plain.rounded(d, dtype))
        assert torch.equal(dense.distil(x, ids, top, 2.0), got[0])


def test_distil_of_the_widest_levels() -> None:
    outputs, g = 1 << 24, base._gen(26)
    logits = (3 * base._randn((2, outputs), g)).to(BF16)
    ids, top = torch.randint(outputs, (2, 40), generator=g, device=DEV), base._randn((2, 40), g)
    weight = torch.rand((2,), generator=g, device=DEV)
    (loss, off), (d, d_off) = plain.distil(logits, ids, top, 1.0, weight)
    got = dense.distil_grad(weight, logits, ids, top)
    plain.near(got[0], loss, off)
    plain.near(got[1], d, d_off + plain.rounded(d, BF16))


def test_recur_of_the_widest_levels() -> None:
    """2^23 units: a unit's results are those of a narrow level with it."""
    tokens, units, some, g = 130, 1 << 23, 300, base._gen(27)
    xz = base._randn((1, 2 * units), g).to(BF16).expand(tokens, 2 * units)
    turn = base._randn((tokens, 1), g).to(BF16)
    d = turn.expand(tokens, units)
    h, last, kept = dense.recur(xz)
    few = torch.cat([xz[:, units - some : units], xz[:, -some:]], 1)
    h2, last2, kept2 = dense.recur(few)
    assert torch.equal(h[:, -some:], h2) and torch.equal(last[:, -some:], last2) and torch.equal(kept[:, -some:], kept2)
    dxz, ds = dense.recur_grad(d, xz, kept)
    dxz2, ds2 = dense.recur_grad(d[:, :some], few, kept2)
    assert torch.equal(dxz[:, units - some : units], dxz2[:, :some]) and torch.equal(dxz[:, -some:], dxz2[:, some:])
    assert torch.equal(ds[:, -some:], ds2)


def test_states_in_place_are_known_to_autograd() -> None:
    """What a backward pass needs of a state is not what recur_step leaves there: the pass says so, as after torch's own
    operations in place, in place of a wrong gradient."""
    state, w = torch.ones((3, 8), device=DEV), torch.ones((3, 8), device=DEV, requires_grad=True)
    seen = (state * w).sum()
    with torch.no_grad():
        dense.recur_step(torch.ones((3, 16), device=DEV), state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        seen.backward()
    with torch.inference_mode():  # (such tensors have no versions)
        dense.recur_step(torch.ones((3, 16), device=DEV), torch.zeros((3, 8), device=DEV))
