"""The formats and operators of plastax_amd.lowbit in plain 64-bit torch."""

from __future__ import annotations

import torch

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0**-24  # half a step of float32, relative
TABLE4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def _blocks(x: torch.Tensor, per: int) -> torch.Tensor:
    r, n = x.shape
    b = -(-n // (32 * per)) * per
    v = torch.zeros((r, b * 32), dtype=torch.float64, device=x.device)
    v[:, :n] = x.double()
    return v.view(r, b, 32)


def _exponent(amax: torch.Tensor, largest: float, floor: int) -> torch.Tensor:
    """The least e >= floor with amax <= largest 2^e."""
    m, e = torch.frexp(amax / largest)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.where(amax == 0, floor, e).clamp_min(floor)


def quantise4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales): the nearest of the 8 magnitudes, a tie to the even code."""
    v = _blocks(x, 4)
    fine = torch.isfinite(v).all(2)
    v = torch.where(fine[:, :, None], v, 0.0)
    e = _exponent(v.abs().amax(2), 6.0, -125)
    m = v.abs() * torch.exp2(-e.double())[:, :, None]
    code = torch.zeros_like(m)
    for k in range(7):  # past the border between code k and k + 1 (on it: where k + 1 is even)
        border = (TABLE4[k] + TABLE4[k + 1]) / 2
        code += (m >= border) if k % 2 else (m > border)
    code = code.to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    code = code.view(v.shape[0], -1, 2)
    return code[:, :, 0] | (code[:, :, 1] << 4), torch.where(fine, e + 127, 255).to(torch.uint8)


def _scale(scales: torch.Tensor) -> torch.Tensor:
    return torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127))


def values4(codes: torch.Tensor, scales: torch.Tensor, n: int) -> torch.Tensor:
    table = torch.tensor(TABLE4 + [-t for t in TABLE4], dtype=torch.float64, device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], 2).flatten(1).long()
    return (table[c] * _scale(scales).repeat_interleave(32, 1))[:, :n]


def quantise8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of e4m3: 3 bits behind the leading one, exponents from -6."""
    v = _blocks(x, 1)
    fine = torch.isfinite(v)
    w = torch.where(fine, v, 0.0)
    e = _exponent(w.abs().amax(2), 448.0, -117)
    m = w.abs() * torch.exp2(-e.double())[:, :, None]
    _, own = torch.frexp(m)
    own = torch.where(m == 0, -6, own - 1).clamp_min(-6)
    units = torch.round(m * torch.exp2(3 - own.double())).long()  # of 2^(own - 3); 16 carries into the next exponent
    code = torch.where(units < 8, units, ((own + 7).long() << 3) + units - 8)
    code = torch.where(fine, code, 0x7F) | (torch.signbit(w) & fine).long() << 7
    return code.to(torch.uint8).view(v.shape[0], -1), (e + 127).to(torch.uint8)


def values8(codes: torch.Tensor, scales: torch.Tensor, n: int) -> torch.Tensor:
    c = codes.long()
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, m * 2.0**-9, torch.exp2(e.double() - 7) * (1 + m / 8))
    v = torch.where((c & 127) == 127, torch.nan, v)
    return (torch.where(c >= 128, -v, v) * _scale(scales).repeat_interleave(32, 1))[:, :n]


def act(fn: str, h: torch.Tensor) -> torch.Tensor:
    h = h.double()
    if fn == "relu":
        return torch.where(h <= 0, 0.0, h)
    if fn == "tanh":
        return torch.tanh(h)
    return torch.sigmoid(h) if fn == "sigmoid" else h * torch.sigmoid(h)


def act_grad(fn: str, q: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fn'(q), and the size of the terms that it is the sum of."""
    if fn == "relu":
        d = (q > 0).double()
    elif fn == "tanh":
        d = 1 / torch.cosh(q) ** 2
    else:
        d = 1 / (2 + torch.exp(q) + torch.exp(-q))
        if fn == "silu":
            s = torch.sigmoid(q)
            return s + q * d, s + q.abs() * d
    return d, d


def sum_bound(k: int) -> float:
    """Of a float32 sum of k exact products, relative to the sum of their sizes: a matrix instruction adds 32 of them
    with a step's rounding each at most, and their sums are added one after the other."""
    return (k / 32 + 32) * 2 * U


def assert_product(got: torch.Tensor, a: torch.Tensor, b: torch.Tensor) -> None:
    """got = a b^T, a [m, k] and b [n, k] in float64."""
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    # (the 1-norm bound holds per value; a result below the type's normal numbers is off by half its least step)
    tol = size * sum_bound(a.shape[1]) + want.abs() * half_step(got.dtype) + torch.finfo(got.dtype).tiny * half_step(got.dtype) * 2
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    bad = ~(off <= tol) & ~nan & ~(got.double() == want)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off / tol)[bad].max())} of the bound"


def layouts(x: torch.Tensor) -> dict[str, torch.Tensor]:
    """The same matrix in other strides, alignments and orders."""
    r, n = x.shape
    off = torch.zeros((r, n + 3), dtype=x.dtype, device=x.device)
    off[:, 1 : n + 1] = x
    step = torch.zeros((2 * r, 2 * n), dtype=x.dtype, device=x.device)
    step[::2, ::2] = x
    return {"rows": x.contiguous(), "columns": x.t().contiguous().t(), "offset": off[:, 1 : n + 1],
            "offset_columns": torch.cat([x[:1] * 0, x]).t().contiguous().t()[1:], "steps": step[::2, ::2]}
