"""plastax_amd.dense's operators in elementary operations in 64 bits, each with
a bound on how far float32 sums and the roundings of a type may be from it.

``EPS`` is float32's rounding, 2^-24, and ``half(dtype)`` a type's, relative to
the value; below a type's normal numbers the rounding is half its least step."""

from __future__ import annotations

import torch

EPS = 2.0**-24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def rounded(want: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """How far the nearest value of the type may be."""
    return want.abs() * half(dtype) + torch.finfo(dtype).tiny * half(dtype)


def near(got: torch.Tensor, want: torch.Tensor, tol: torch.Tensor) -> None:
    """``got`` within ``tol`` of ``want``; infinities and NaN in the same places.

    A type's largest value is (2 - eps) 2^e; from (2 - eps / 2) 2^e on the nearest is an infinity (a loss of 3.9e38 is
    one in float32)."""
    top = torch.finfo(got.dtype)
    border = top.max / (2 - top.eps) * (2 - top.eps / 2)
    want = torch.where(want.abs() >= border, torch.copysign(torch.full_like(want, torch.inf), want), want)
    got = got.double()
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    off = torch.where(fine, (got - want).abs() - tol, 0.0)
    assert float(off.max() if off.numel() else 0.0) <= 0.0, (float(off.max()), float((got - want).abs().max()))


# --------------------------------------------------------------------------
def look_up(ids, table, scale):
    there = (ids >= 0) & (ids < table.shape[0])
    if table.shape[0] == 0:
        return torch.zeros((ids.shape[0], table.shape[1]), dtype=torch.float64, device=table.device)
    return torch.where(there[:, None], table.double()[ids.clamp(0, table.shape[0] - 1).long()] * scale, 0.0)


def look_up_grad(g, ids, rows, scale):
    """(the sums, their bound): n float32 sums lose n - 1 roundings of the sum of magnitudes at most, the scale one
    more and its own one."""
    there = (ids >= 0) & (ids < rows)
    at, g = ids[there].long(), g[there].double() * scale
    zero = torch.zeros((rows, g.shape[1]), dtype=torch.float64, device=g.device)
    count = torch.zeros((rows,), dtype=torch.float64, device=g.device).index_add_(0, at, torch.ones_like(g[:, 0]))
    return zero.index_add(0, at, g), (count[:, None] + 2) * EPS * zero.index_add(0, at, g.abs())


# --------------------------------------------------------------------------
def normalise(x, weight, bias, eps, g=None):
    """((y, its bound), and with g (dx, bound), (dweight, bound), (dbias, bound)); the bounds without the results'
    own rounding. A row's sums are made of at most k roundings on a value's way: 16 and units / 1024 in its lane, 10
    over the lanes, 4 besides."""
    tokens, units = x.shape
    x, w = x.double(), weight.double()
    b = torch.zeros_like(w) if bias is None else bias.double()
    k = 30 + units / 1024
    mean = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    n = (x - mean) * r
    off = k * EPS * x.abs().mean(1, keepdim=True)  # of the mean
    dn = r * (off + EPS * (x.abs() + mean.abs())) + n.abs() * ((k + 8) * EPS + (off * r) ** 2)
    y = n * w + b
    out = [(y, dn * w.abs() + 3 * EPS * ((n * w).abs() + b.abs()))]
    if g is None:
        return out
    g = g.double()
    u = g * w
    m, mn = u.mean(1, keepdim=True), (u * n).mean(1, keepdim=True)
    dx = r * (u - m - n * mn)
    dr = (k + 8) * EPS + (off * r) ** 2
    dm = k * EPS * u.abs().mean(1, keepdim=True)
    dmn = k * EPS * (u * n).abs().mean(1, keepdim=True) + (u.abs() * dn).mean(1, keepdim=True)
    size = u.abs() + m.abs() + (n * mn).abs()
    out.append((dx, r * ((dr + 4 * EPS) * size + dm + dn * mn.abs() + n.abs() * dmn)))
    # over the tokens: at most one rounding a token and 4 besides; 64 a workgroup's and 84 over workgroups
    deep = min(tokens + 4, tokens / 64 + 150) * EPS
    out.append(((g * n).sum(0), (g.abs() * dn).sum(0) + deep * (g * n).abs().sum(0)))
    out.append((g.sum(0), deep * g.abs().sum(0)))
    return out


# --------------------------------------------------------------------------
def recur(xz, starts, state, g=None, g_last=None):
    """((h, bound), (last, bound)) and with g ((dxz, bound), (dstate, bound)), row by row; the bounds without the
    results' own rounding.

    Each term of h has come through a product for each row on its way, with a few roundings each: gates have at most
    4 (an exponential with its argument's error carried 2, a reciprocal 1, a product 1), a product and a sum 2, and
    they are made twice (summed up, then walked). So with m the same recurrence of magnitudes and
    e[t] = a (e[t-1] + m[t-1]) + m[t], the sum of the terms' magnitudes times their rows, h is off by 14 e EPS at
    most."""
    units = xz.shape[1] // 2
    x, z = xz[:, :units].double(), xz[:, units:].double()
    a, b = torch.sigmoid(z), torch.sigmoid(-z)
    tokens, sequences = xz.shape[0], len(starts) - 1
    zeros = torch.zeros((sequences, units), dtype=torch.float64, device=xz.device)
    state = zeros if state is None else state.double()
    h, before, m, e = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    m_before, e_before = torch.zeros_like(x), torch.zeros_like(x)
    last, last_e = state.clone(), zeros.clone()
    for s in range(sequences):
        now, size, err = state[s], state[s].abs(), zeros[s]
        for t in range(starts[s], starts[s + 1]):
            before[t], m_before[t], e_before[t] = now, size, err
            now = a[t] * now + b[t] * x[t]
            err = a[t] * (err + 2 * size) + b[t] * x[t].abs()
            size = a[t] * size + b[t] * x[t].abs()
            h[t], m[t], e[t] = now, size, err
        last[s], last_e[s] = now, err
    tiny = 1e-36
    out = [(h, 14 * EPS * e + tiny), (last, 14 * EPS * last_e + tiny)]
    if g is None:
        return out
    g_last = zeros if g_last is None else g_last.double()
    g = g.double()
    c, cm, ce = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    dstate, ds_e = g_last.clone(), zeros.clone()
    for s in range(sequences):
        back, size, err = g_last[s], g_last[s].abs(), zeros[s]
        for t in range(starts[s + 1] - 1, starts[s] - 1, -1):
            c[t], cm[t], ce[t] = g[t] + back, g[t].abs() + size, err + g[t].abs() + size
            back = a[t] * c[t]
            err = a[t] * (ce[t] + cm[t])
            size = a[t] * cm[t]
        dstate[s], ds_e[s] = back, err
    dx, dz = b * c, a * b * (before - x) * c
    size = m_before + x.abs()
    dx_off = 14 * EPS * b * (ce + cm)
    dz_off = 14 * EPS * a * b * ((e_before + size) * cm + size * (ce + cm))
    out += [(torch.cat([dx, dz], 1), torch.cat([dx_off, dz_off], 1) + tiny), (dstate, 14 * EPS * ds_e + tiny)]
    return out


# --------------------------------------------------------------------------
def distil(logits, ids, top, temperature, g=None):
    """((loss, bound)) and with g (dlogits, bound); the bounds without the results' own rounding.

    exp((x - m) / T) is off by the roundings of its argument, 4 |x - m| / T, and 2 more, and its sum over the row by
    at most k more: 128 in a lane, 10 over the lanes, 4 besides (or a lane's share of a longer row)."""
    tokens, outputs = logits.shape
    t = float(temperature)
    there = (ids >= 0) & (ids < outputs) & (top != -torch.inf)
    at = torch.where(there, ids, 0).long()
    v = torch.where(there, top.double() / t, -torch.inf)
    some = there.any(1, keepdim=True)
    v = v - torch.where(some, v.amax(1, keepdim=True), 0.0) if v.shape[1] else v
    total = torch.exp(v).sum(1, keepdim=True)
    p = torch.where(there, torch.exp(v) / total, 0.0)
    x = logits.double() / t
    d = (x - x.amax(1, keepdim=True)).abs()
    log_q = torch.log_softmax(x, 1)
    q = torch.exp(log_q)
    loss = torch.where(p != 0, p * (v - torch.log(total) - log_q.gather(1, at)), 0.0).sum(1) * t * t
    loss = torch.where(some[:, 0], loss, 0.0)
    k = 144 + outputs / 1024
    shift = torch.where(q > 0, 4 * d, 0.0)  # (a logit of -inf has no part in the sum)
    mean = (q * shift).sum(1, keepdim=True) + k + 8
    out = [(loss, t * t * EPS * mean[:, 0] + EPS * loss.abs())]
    if g is None:
        return out
    scale = t * g.double()[:, None]
    dx = torch.where(some, q, 0.0).scatter_add(1, at, -p) * scale
    size = torch.where(some, q, 0.0).scatter_add(1, at, p) * scale.abs()
    out.append((dx, scale.abs() * EPS * q * (shift + mean) + 4 * EPS * size + 1e-36))
    return out
