"""Level pairs as whole matrices in few bits: the measured operators.

A level pair of a net (every unit of one level against every unit of the next)
can be held as a matrix in blocks of 32 values that share a power of two. A
trained net answers batches and single samples from 4-bit matrices, and learns
with them: the batch's activations wait for the backward in 8 bits. Shapes
below are ``tokens`` (samples, positions) by ``inputs`` or ``outputs`` (units).

Formats. 32 consecutive values along a line share the scale ``2^(s - 127)``,
``s`` one byte: the least power of two under which the block's largest value
is not above the format's largest (6 in 4 bits, 448 in 8), and not less than
2^-125 or 2^-117, so that every value is a normal float32. Values go to the
nearest, ties to the even code.

- 4 bits (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign): two to a byte, the
  earlier one in the low half; a line holds ``ceil(n / 128) * 4`` blocks,
  those past its end with zero codes. A block with an infinity or a NaN has
  ``s = 255`` and stands for NaN.
- 8 bits (e4m3, no infinities): one to a byte; a line holds ``ceil(n / 32)``
  blocks. An infinity or a NaN is stored as NaN, in its own place alone.

Kinds of case (``case["kind"]``):

- ``quantise``: a matrix to 4 bits, and the values it then stands for (what
  is written back to the arena). ``order`` "rows": lines contiguous;
  "columns": contiguous across the lines, as a bucket's source-major weights;
- ``product``: ``y = x w^T`` with the weights in 4 bits; ``low`` has the
  activations quantised to 4 bits on the way, else they are taken as they are;
- ``input_grad``: its gradient for the input, ``dx = g w``;
- ``activate``: ``y = fn(h)`` with h kept in 8 bits, then ``dh = dy fn'(h)``
  from what was kept. ``order`` "rows": token-major, blocks along the units;
  "columns": unit-major columns, blocks along the tokens;
- ``weight_grad``: ``dw = g^T x`` from inputs kept in 8 bits, the same orders.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # The first level pair of a sparse MLP (784 to 4096), as the arena
        # holds it (source-major), quantised after a training chunk.
        {"name": "quantise_first", "kind": "quantise", "rows": 4096, "cols": 784, "dtype": "float32", "order": "columns"},
        # A large matrix in half precision, lines contiguous.
        {"name": "quantise_large", "kind": "quantise", "rows": 8192, "cols": 8192, "dtype": "bfloat16", "order": "rows"},
        # One sample answered by the middle level pair: all latency.
        {"name": "product_token", "kind": "product", "tokens": 1, "inputs": 4096, "outputs": 4096, "dtype": "bfloat16",
         "low": False},
        # A mini-batch in 32 bits through odd level sizes.
        {"name": "product_odd", "kind": "product", "tokens": 70, "inputs": 1003, "outputs": 777, "dtype": "float32",
         "low": False},
        # A mini-batch of 256 through the middle level pair, 4 bits by 4 bits.
        {"name": "product_batch", "kind": "product", "tokens": 256, "inputs": 4096, "outputs": 4096, "dtype": "bfloat16",
         "low": True},
        # The largest: a large batch through a wide level pair.
        {"name": "product_large", "kind": "product", "tokens": 8192, "inputs": 8192, "outputs": 8192,
         "dtype": "bfloat16", "low": True},
        # Back through the middle level pair, a large batch.
        {"name": "input_grad_large", "kind": "input_grad", "tokens": 8192, "inputs": 4096, "outputs": 4096,
         "dtype": "bfloat16"},
        # Back through odd level sizes in 32 bits.
        {"name": "input_grad_odd", "kind": "input_grad", "tokens": 256, "inputs": 1003, "outputs": 777,
         "dtype": "float32"},
        # A small odd level of a batched step (unit-major columns).
        {"name": "activate_odd", "kind": "activate", "tokens": 70, "units": 1003, "dtype": "float32", "fn": "relu",
         "order": "columns"},
        # A large batch, token-major.
        {"name": "activate_large", "kind": "activate", "tokens": 8192, "units": 8192, "dtype": "bfloat16", "fn": "silu",
         "order": "rows"},
        # The batched step's columns (256 samples), gradients in 32 bits.
        {"name": "weight_grad_columns", "kind": "weight_grad", "tokens": 256, "inputs": 4096, "outputs": 4096,
         "dtype": "float32", "order": "columns"},
        # A large batch, token-major.
        {"name": "weight_grad_large", "kind": "weight_grad", "tokens": 8192, "inputs": 4096, "outputs": 4096,
         "dtype": "bfloat16", "order": "rows"},
    ]


def _log(rng, lo, hi):
    """A whole number, uniform over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantise", "product", "product", "product", "input_grad", "activate", "weight_grad"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    order = rng.choice(["rows", "columns"])
    if kind == "quantise":
        return {"kind": kind, "rows": _log(rng, 10, 8192), "cols": _log(rng, 10, 8192), "dtype": dtype, "order": order}
    if kind == "activate":
        return {"kind": kind, "tokens": _log(rng, 1, 8192), "units": _log(rng, 10, 8192), "dtype": dtype,
                "fn": rng.choice(["relu", "tanh", "sigmoid", "silu"]), "order": order}
    case = {"kind": kind, "tokens": _log(rng, 1, 8192), "inputs": _log(rng, 10, 8192), "outputs": _log(rng, 10, 8192),
            "dtype": dtype}
    if kind == "product":
        case["low"] = rng.random() < 0.5
    elif kind == "weight_grad":
        case["order"] = order
    return case


# --------------------------------------------------------------------------
# The formats in elementary operations
# --------------------------------------------------------------------------
def _power(e):
    """2^e of whole numbers in [-126, 127], by the bits of a float32."""
    return ((e + 127) << 23).view(torch.float32)


def _blocks(x, per):
    """x [R, n] as float32 blocks [R, b, 32], b a multiple of ``per``; zeros past the line's end."""
    r, n = x.shape
    b = -(-n // (32 * per)) * per
    out = torch.zeros((r, b * 32), dtype=torch.float32, device=x.device)
    out[:, :n] = x
    return out.view(r, b, 32)


def _exponent(amax, mantissa, top, least):
    """The block's exponent: amax <= (1 + mantissa / 2^23) 2^top 2^e."""
    bits = amax.view(torch.int32)
    e = (bits >> 23) - 127 - top + ((bits & 0x7FFFFF) > mantissa).to(torch.int32)
    return e.clamp_min(least)


def _scale(s):
    """The scales that bytes stand for (255: NaN)."""
    s = s.to(torch.int32)
    return torch.where(s == 255, math.nan, (s << 23).view(torch.float32))


def _quantise4(x):
    """(codes uint8 [R, 16 b], scales uint8 [R, b]) of x [R, n]."""
    v = _blocks(x, 4)
    fine = torch.isfinite(v).all(2)
    v = torch.where(fine[:, :, None], v, 0.0)
    e = _exponent(v.abs().amax(2), 0x400000, 2, -125)
    m = v.abs() * _power(-e)[:, :, None]
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    m = torch.round(m / step) * step
    code = torch.where(m < 2, m * 2, torch.where(m < 4, m + 2, m / 2 + 4)).to(torch.uint8)
    code = (code | ((v.view(torch.int32) < 0).to(torch.uint8) << 3)).view(v.shape[0], -1, 2)
    return code[:, :, 0] | (code[:, :, 1] << 4), torch.where(fine, e + 127, 255).to(torch.uint8)


def _values4(codes, scales, n):
    """The float32 values [R, n] that 4-bit codes stand for."""
    c = torch.stack([codes & 15, codes >> 4], 2).view(codes.shape[0], -1, 32)
    m = (c & 7).to(torch.float32)
    m = torch.where(m < 4, m * 0.5, torch.where(m < 6, m - 2, 2 * m - 8))
    v = torch.where(c >= 8, -m, m) * _scale(scales)[:, :, None]
    return v.view(codes.shape[0], -1)[:, :n]


def _quantise8(x):
    """(codes uint8 [R, 32 b], scales uint8 [R, b]) of x [R, n]."""
    v = _blocks(x, 1)
    fine = torch.isfinite(v)
    e = _exponent(torch.where(fine, v, 0.0).abs().amax(2), 0x600000, 8, -117)
    c = (torch.where(fine, v, math.nan) * _power(-e)[:, :, None]).to(torch.float8_e4m3fn)
    return c.view(torch.uint8).view(v.shape[0], -1), (e + 127).to(torch.uint8)


def _values8(codes, scales, n):
    """The float32 values [R, n] that 8-bit codes stand for."""
    v = codes.view(torch.float8_e4m3fn).to(torch.float32).view(codes.shape[0], -1, 32) * _scale(scales)[:, :, None]
    return v.view(codes.shape[0], -1)[:, :n]


def _fn(fn, h):
    if fn == "relu":
        return torch.clamp_min(h, 0)
    if fn == "tanh":
        return torch.tanh(h)
    return torch.sigmoid(h) if fn == "sigmoid" else h * torch.sigmoid(h)


def _fn_grad(fn, h):
    if fn == "relu":
        return (h > 0).to(h.dtype)
    if fn == "tanh":
        u = torch.exp(-2 * h.abs())
        return 4 * u / ((1 + u) * (1 + u))
    t = torch.exp(-h.abs())
    d = t / ((1 + t) * (1 + t))
    return d if fn == "sigmoid" else torch.sigmoid(h) + h * d


# --------------------------------------------------------------------------
# The measured passes
# --------------------------------------------------------------------------
def _activations(rng, tokens, units, dtype):
    """What a level of rectifiers holds: about half zeros, some samples without an active unit, one scale a sample."""
    x = torch.randn((tokens, units), generator=rng, device="cuda").clamp_min_(0)
    scale = torch.rand((tokens, 1), generator=rng, device="cuda") * 2
    return (x * torch.where(scale < 0.02, 0.0, scale)).to(dtype)


def _weights(rng, outputs, inputs):
    """Weights of a trained level pair, about a tenth of them pruned."""
    w = torch.randn((outputs, inputs), generator=rng, device="cuda") / math.sqrt(inputs)
    return torch.where(torch.rand((outputs, inputs), generator=rng, device="cuda") < 0.1, 0.0, w)


def _gradients(rng, tokens, units, dtype):
    """Gradients of a mean over the batch, of different sizes for each sample."""
    scale = torch.exp(torch.randn((tokens, 1), generator=rng, device="cuda")) / 256
    return (torch.randn((tokens, units), generator=rng, device="cuda") * scale).to(dtype)


def prepare(case, seed):
    rng = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = {"kind": kind}
    if kind == "quantise":
        x = _weights(rng, case["rows"], case["cols"]).to(dtype)
        state["x"] = x if case["order"] == "rows" else x.t().contiguous().t()
        return state
    tokens = case["tokens"]
    if kind == "activate":
        h = (2 * torch.randn((tokens, case["units"]), generator=rng, device="cuda")).to(dtype)
        dy = _gradients(rng, tokens, case["units"], dtype)
        if case["order"] == "columns":
            h, dy = h.t().contiguous().t(), dy.t().contiguous().t()
        return {"kind": kind, "h": h, "dy": dy, "fn": case["fn"], "axis": 1 if case["order"] == "rows" else 0}
    inputs, outputs = case["inputs"], case["outputs"]
    if kind == "weight_grad":
        x, g = _activations(rng, tokens, inputs, torch.float32), _gradients(rng, tokens, outputs, dtype)
        rows = case["order"] == "rows"
        state["codes"], state["scales"] = _quantise8(x if rows else x.t())
        state["g"] = g if rows else g.t().contiguous().t()
        state["shape"], state["axis"] = (tokens, inputs), 1 if rows else 0
        return state
    state["codes"], state["scales"] = _quantise4(_weights(rng, outputs, inputs))
    state["inputs"] = inputs
    if kind == "product":
        state["x"], state["low"] = _activations(rng, tokens, inputs, dtype), case["low"]
    else:
        state["g"] = _gradients(rng, tokens, outputs, dtype)
    return state


def _own(s):
    from plastax_amd import lowbit

    kind = s["kind"]
    if kind == "quantise":
        return lowbit.quantise4(s["x"]).values(torch.float32)
    if kind == "activate":
        y, kept = lowbit.activate(s["h"], s["fn"], axis=s["axis"])
        return y, kept.values(torch.bfloat16), lowbit.activate_grad(s["dy"], kept, s["fn"])
    if kind == "weight_grad":
        return lowbit.weight_grad(s["g"], lowbit.Mx8(s["codes"], s["scales"], s["shape"], s["axis"]))
    w = lowbit.Mx4(s["codes"], s["scales"], s["inputs"])
    if kind == "input_grad":
        return lowbit.product_grad(s["g"], w)
    if s["low"]:
        return lowbit.product(lowbit.quantise4(s["x"]), w, dtype=s["x"].dtype)
    return lowbit.product(s["x"], w)


def run(s):
    if own:
        return _own(s)
    kind = s["kind"]
    if kind == "quantise":
        x = s["x"]
        return _values4(*_quantise4(x), x.shape[1])
    if kind == "activate":
        h, axis = s["h"], s["axis"]
        codes, scales = _quantise8(h if axis else h.t())
        kept = _values8(codes, scales, h.shape[axis])
        kept = kept if axis else kept.t()
        dh = s["dy"].to(torch.float32) * _fn_grad(s["fn"], kept)
        return _fn(s["fn"], h.to(torch.float32)).to(h.dtype), kept.to(torch.bfloat16), dh.to(h.dtype)
    if kind == "weight_grad":
        x = _values8(s["codes"], s["scales"], s["shape"][s["axis"]])
        return s["g"].to(torch.float32).t() @ (x if s["axis"] else x.t())
    w = _values4(s["codes"], s["scales"], s["inputs"])
    if kind == "input_grad":
        return (s["g"].to(torch.float32) @ w).to(s["g"].dtype)
    x = s["x"].to(torch.float32)
    if s["low"]:
        x = _values4(*_quantise4(x), s["inputs"])
    return (x @ w.t()).to(s["x"].dtype)


def work(case):
    """Every input read once, every output written once; what is kept in 4 or 8 bits is an output too."""
    size = 4 if case["dtype"] == "float32" else 2
    kind = case["kind"]
    if kind == "quantise":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (size + 17 / 32 + 4), "flops": 4 * n}
    if kind == "activate":
        n = case["tokens"] * case["units"]
        return {"bytes": n * (4 * size + 33 / 32 + 2), "flops": 16 * n}
    t, k, n = case["tokens"], case["inputs"], case["outputs"]
    if kind == "weight_grad":
        return {"bytes": t * k * 33 / 32 + t * n * size + 4 * n * k, "flops": 2 * t * n * k}
    return {"bytes": n * k * 17 / 32 + t * (n + k) * size, "flops": 2 * t * n * k}


# --------------------------------------------------------------------------
# The definitions in 64 bits
# --------------------------------------------------------------------------
def _power64(e):
    """2^e of whole numbers in float64, by its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest64(x, largest, digits, least, floor):
    """x [R, n] in float64 to the nearest multiples of its blocks' steps: values of ``digits`` bits behind the leading
    one, exponents from ``least``, at most ``largest``, times the block's scale, which is 2^floor at least."""
    r, n = x.shape
    v = torch.zeros((r, -(-n // 32) * 32), dtype=torch.float64, device=x.device)
    v[:, :n] = x
    v = v.view(r, -1, 32)
    amax = v.abs().amax(2, keepdim=True)
    m, e = torch.frexp(amax / largest)  # amax / largest = m 2^e, 0.5 <= m < 1
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(amax == 0, floor, e).clamp_min(floor)
    v = v * _power64(-e)
    _, own_e = torch.frexp(v)
    step = _power64(torch.where(v == 0, least, own_e - 1).clamp_min(least) - digits)
    v = torch.round(v / step) * step * _power64(e)
    return v.reshape(r, -1)[:, :n]


def _table64(codes, scales, n):
    """4-bit codes through a table of the sixteen values."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=codes.device)
    table = torch.cat([table, -table])
    pairs = table[torch.stack([codes % 16, codes // 16], -1).flatten(1).long()]
    return (pairs * _power64(scales.long() - 127).repeat_interleave(32, 1))[:, :n]


def _bits64(codes, scales, n):
    """8-bit codes by their fields: sign, 4 bits of exponent, 3 behind the point."""
    c = codes.long()
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, m * 2.0**-9, _power64(e - 7) * (1 + m / 8))
    return (torch.where(c >= 128, -v, v) * _power64(scales.long() - 127).repeat_interleave(32, 1))[:, :n]


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "quantise":
        return _nearest64(s["x"].double(), 6, 1, 0, -125)
    if kind == "activate":
        h = s["h"].double()
        lines = h if s["axis"] else h.t()
        kept = _nearest64(lines, 448, 3, -6, -117)
        kept = kept if s["axis"] else kept.t()
        fns = {"relu": (lambda v: v.clamp_min(0), lambda v: (v > 0).double()),
               "tanh": (torch.tanh, lambda v: 1 / torch.cosh(v) ** 2),
               "sigmoid": (lambda v: 1 / (1 + torch.exp(-v)), lambda v: 1 / (2 + torch.exp(v) + torch.exp(-v))),
               "silu": (lambda v: v / (1 + torch.exp(-v)),
                        lambda v: 1 / (1 + torch.exp(-v)) + v / (2 + torch.exp(v) + torch.exp(-v)))}
        f, df = fns[s["fn"]]
        return f(h), kept, s["dy"].double() * df(kept)
    if kind == "weight_grad":
        x = _bits64(s["codes"], s["scales"], s["shape"][s["axis"]])
        return s["g"].double().t() @ (x if s["axis"] else x.t())
    w = _table64(s["codes"], s["scales"], s["inputs"])
    if kind == "input_grad":
        return s["g"].double() @ w
    x = s["x"].double()
    return (_nearest64(x, 6, 1, 0, -125) if s["low"] else x) @ w.t()
