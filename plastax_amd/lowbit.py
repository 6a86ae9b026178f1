"""Level pairs as whole matrices in few bits, and learning with them.

A level pair of a net (every unit of one level against every unit of the
next) is a matrix ``[outputs, inputs]``. Here it is held in 4 bits
(:class:`Mx4`, :func:`quantise4`), answers batches or single samples
(:func:`product`), and gives its input's gradient (:func:`product_grad`); the
activation between two pairs keeps its argument in 8 bits for the backward
(:func:`activate`, :class:`Mx8`, :func:`activate_grad`), and so does the
weights' own gradient its pair's input (:func:`quantise8`, :func:`weight_grad`).

Formats. 32 consecutive values of a line share a scale ``2^(s - 127)``, ``s``
one byte: the least power of two under which the block's largest value is not
above the format's largest (6 or 448), and at least 2^-125 or 2^-117. Values
go to the nearest, ties to the even code.

- 4 bits (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign): two values to a byte, the
  earlier one in the low half; a line holds ``ceil(n / 128) * 4`` blocks, zero
  codes past its end (the scales of blocks past it count for nothing). A block
  with an infinity or a NaN has ``s = 255`` and stands for NaN.
- 8 bits (e4m3, no infinities): one value to a byte; a line holds
  ``ceil(n / 32)`` blocks, and codes past its end count for nothing. An
  infinity or a NaN is kept as NaN in its place, with the sign bit of a
  negative infinity alone.

Arguments are 2-dimensional GPU tensors of float32, bfloat16 or float16 with
any strides; batches are ``[tokens, units]``. Work goes to torch's current
stream of the arguments' device, results and workspaces are allocated there.
Products are exact over each type's whole range, sums are float32 (a value
rounded up past float32's largest is an infinity, and sums with one are not
finite). Results carry no autograd graph and no tangent: an argument
that asks for one is refused, the gradients are calls of their own. The reference has no
counterpart: its weights and activations are float32.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from plastax_amd import _lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # PLX_LB_F32, _BF16, _F16
FUNCTIONS = {"relu": 0, "tanh": 1, "sigmoid": 2, "silu": 3}  # PLX_LB_RELU ..
_PRODUCT, _PRODUCT_GRAD, _WEIGHT_GRAD, _WEIGHT_GRAD_COLUMNS = range(4)


def _check_codes(who: str, codes: torch.Tensor, scales: torch.Tensor, lines: int, blocks: int, size: int) -> None:
    if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8:
        raise TypeError(f"{who}: codes and scales are uint8, got {codes.dtype} and {scales.dtype}")
    if codes.shape != (lines, blocks * size) or scales.shape != (lines, blocks):
        raise ValueError(f"{who}: codes {(lines, blocks * size)} and scales {(lines, blocks)} expected, "
                         f"got {tuple(codes.shape)} and {tuple(scales.shape)}")
    if not (codes.is_contiguous() and scales.is_contiguous()):
        raise ValueError(f"{who}: codes and scales must be contiguous")
    if codes.device != scales.device:
        raise ValueError(f"{who}: codes and scales are on different devices")
    if codes.data_ptr() & 15:
        raise ValueError(f"{who}: codes must start on 16 bytes")


class Mx4:
    """A matrix ``[lines, n]`` in 4-bit blocks along its lines.

    ``codes`` uint8 ``[lines, 16 b]`` and ``scales`` uint8 ``[lines, b]``,
    ``b = ceil(n / 128) * 4``, scale bytes 2 to 253, or 255."""

    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, n: int) -> None:
        if n < 0 or codes.dim() != 2:
            raise ValueError("Mx4: codes of two dimensions and n >= 0 expected")
        _check_codes("Mx4", codes, scales, codes.shape[0], -(-n // 128) * 4, 16)
        self.codes, self.scales, self.shape = codes, scales, (codes.shape[0], n)

    @classmethod
    def _empty(cls, lines: int, n: int, device: torch.device) -> Mx4:
        m, b = object.__new__(cls), -(-n // 128) * 4
        m.codes = torch.empty((lines, 16 * b), dtype=torch.uint8, device=device)
        m.scales = m.codes.new_empty((lines, b))
        m.shape = lines, n
        return m

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def values(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values as a matrix (exact in float32 and bfloat16; one that was
        rounded up past their largest is an infinity)."""
        return _values(self, 4, self.shape, dtype)


class Mx8:
    """A batch ``[tokens, units]`` in 8-bit blocks along ``axis`` 1 (a line per
    token) or 0 (a line per unit, for batches kept unit-major).

    ``codes`` uint8 ``[lines, 32 b]`` and ``scales`` uint8 ``[lines, b]``,
    ``b = ceil(n / 32)`` of a line's n values, scale bytes 10 to 247."""

    __slots__ = ("codes", "scales", "shape", "axis")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape: tuple[int, int], axis: int) -> None:
        if axis not in (0, 1) or len(shape) != 2 or min(shape) < 0:
            raise ValueError(f"Mx8: axis 0 or 1 and a shape of two dimensions expected, got {axis} and {shape}")
        _check_codes("Mx8", codes, scales, shape[1 - axis], -(-shape[axis] // 32), 32)
        self.codes, self.scales, self.shape, self.axis = codes, scales, (shape[0], shape[1]), axis

    @classmethod
    def _empty(cls, shape: tuple[int, int], axis: int, device: torch.device) -> Mx8:
        m, lines, b = object.__new__(cls), shape[1 - axis], -(-shape[axis] // 32)
        m.codes = torch.empty((lines, 32 * b), dtype=torch.uint8, device=device)
        m.scales = m.codes.new_empty((lines, b))
        m.shape, m.axis = shape, axis
        return m

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def values(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values as a batch, its lines contiguous (exact in float32 and
        bfloat16; one that was rounded up past their largest is an infinity)."""
        if self.axis:
            return _values(self, 8, self.shape, dtype)
        return _values(self, 8, (self.shape[1], self.shape[0]), dtype).t()


def _check(who: str, t: torch.Tensor) -> torch.Tensor:
    """``t`` checked, with the values that it stands for in its memory (the
    imaginary part of a conjugate view holds them with the other sign)."""
    if t.dim() != 2:
        raise ValueError(f"{who}: a matrix expected, got {t.dim()} dimensions")
    if t.dtype not in DTYPES:
        raise TypeError(f"{who}: float32, bfloat16 or float16 expected, got {t.dtype}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{who}: no autograd here; detach the argument and call the gradients")
    # (the level is -1 outside of dual_level(), where no tensor has a tangent)
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{who}: no forward-mode autograd here; unpack the argument and its tangent")
    return t.resolve_neg() if t.is_neg() else t


def _on_gpu(who: str, device: torch.device, *others: torch.device) -> None:
    if device.type != "cuda":
        raise ValueError(f"{who}: arguments must be on the GPU, got {device}")
    for d in others:
        if d != device:
            raise ValueError(f"{who}: arguments are on different devices, {device} and {d}")


def _call(device: torch.device, name: str, *args: object) -> int:
    """The entry point with ``device`` as the current one: kernels launch on
    it, and plans go by its CUs."""
    fn = getattr(_lib.load(), name)
    # (a tensor is there, so the device is set up: current_device() without its check for that)
    if device.index == torch._C._cuda_getDevice():
        return fn(*args)
    with torch.cuda.device(device.index):
        return fn(*args)


def _launch(device: torch.device, name: str, *args: object) -> None:
    """The entry point on torch's current stream of ``device``."""
    # (current_stream(device).cuda_stream without its Stream object, 2 us of a 10 us call)
    rc = _call(device, name, *args, torch._C._cuda_getCurrentRawStream(device.index))
    if rc:
        _lib.check(rc, name)


def _values(m: Mx4 | Mx8, bits: int, shape: tuple[int, int], dtype: torch.dtype) -> torch.Tensor:
    if dtype not in DTYPES:
        raise TypeError(f"values: float32, bfloat16 or float16 expected, got {dtype}")
    _on_gpu("values", m.device)
    out = torch.empty(shape, dtype=dtype, device=m.device)
    _launch(m.device, "plx_mx_values", bits, shape[0], shape[1], m.codes.data_ptr(), m.scales.data_ptr(),
            DTYPES[dtype], out.data_ptr())
    return out


def quantise4(x: torch.Tensor) -> Mx4:
    """``x`` in 4-bit blocks along its second dimension."""
    x = _check("quantise4", x)
    _on_gpu("quantise4", x.device)
    lines, n = x.shape
    m = Mx4._empty(lines, n, x.device)
    _launch(x.device, "plx_mx4_quantise", lines, n, DTYPES[x.dtype], x.data_ptr(), x.stride(0), x.stride(1),
            m.codes.data_ptr(), m.scales.data_ptr())
    return m


def activate(h: torch.Tensor, fn: str, axis: int = 1) -> tuple[torch.Tensor, Mx8]:
    """``(fn(h), h in 8-bit blocks along axis)``: "relu", "tanh", "sigmoid" or
    "silu" of a batch ``[tokens, units]``, and what its gradient needs. Blocks
    along 1 suit a token-major batch, along 0 one kept unit-major; the result
    has h's layout."""
    h = _check("activate", h)
    if fn not in FUNCTIONS:
        raise ValueError(f"activate: one of {sorted(FUNCTIONS)} expected, got {fn!r}")
    if axis not in (0, 1):
        raise ValueError(f"activate: axis 0 or 1 expected, got {axis}")
    _on_gpu("activate", h.device)
    y, kept = torch.empty_like(h), Mx8._empty(tuple(h.shape), axis, h.device)
    _launch(h.device, "plx_mx8_activate", h.shape[1 - axis], h.shape[axis], DTYPES[h.dtype], FUNCTIONS[fn],
            h.data_ptr(), h.stride(1 - axis), h.stride(axis), y.data_ptr(), y.stride(1 - axis), y.stride(axis),
            kept.codes.data_ptr(), kept.scales.data_ptr())
    return y, kept


def quantise8(x: torch.Tensor, axis: int = 1) -> Mx8:
    """``x`` ``[tokens, units]`` in 8-bit blocks along ``axis``: a level pair's
    input, kept for :func:`weight_grad`."""
    x = _check("quantise8", x)
    if axis not in (0, 1):
        raise ValueError(f"quantise8: axis 0 or 1 expected, got {axis}")
    _on_gpu("quantise8", x.device)
    kept = Mx8._empty(tuple(x.shape), axis, x.device)
    _launch(x.device, "plx_mx8_activate", x.shape[1 - axis], x.shape[axis], DTYPES[x.dtype], FUNCTIONS["relu"],
            x.data_ptr(), x.stride(1 - axis), x.stride(axis), None, 1, 1, kept.codes.data_ptr(),
            kept.scales.data_ptr())
    return kept


def activate_grad(dy: torch.Tensor, kept: Mx8, fn: str) -> torch.Tensor:
    """``dy * fn'(q)``, q the values that :func:`activate` kept; dy's type and
    layout. At a kept infinity or NaN the rectifier's slope is 1 (0 at a
    negative infinity), the others' is NaN."""
    dy = _check("activate_grad", dy)
    if fn not in FUNCTIONS:
        raise ValueError(f"activate_grad: one of {sorted(FUNCTIONS)} expected, got {fn!r}")
    if tuple(dy.shape) != kept.shape:
        raise ValueError(f"activate_grad: a gradient of {kept.shape} expected, got {tuple(dy.shape)}")
    _on_gpu("activate_grad", dy.device, kept.device)
    axis = kept.axis
    dh = torch.empty_like(dy)
    _launch(dy.device, "plx_mx8_activate_grad", dy.shape[1 - axis], dy.shape[axis], DTYPES[dy.dtype], FUNCTIONS[fn],
            dy.data_ptr(), dy.stride(1 - axis), dy.stride(axis), kept.codes.data_ptr(), kept.scales.data_ptr(),
            dh.data_ptr(), dh.stride(1 - axis), dh.stride(axis))
    return dh


def _workspace(device: torch.device, name: str, *args: object) -> torch.Tensor | None:
    # (without _call's frame in the usual case: every product asks)
    if device.index == torch._C._cuda_getDevice():
        need = getattr(_lib.load(), name)(*args)
    else:
        need = _call(device, name, *args)
    if need > 0:
        return torch.empty(need, dtype=torch.uint8, device=device)
    if need < 0:
        raise ValueError(f"{name}: at most 2^24 units a level and 2^30 tokens")
    return None


def _product(kind: int, a: torch.Tensor, m: Mx4 | Mx8, inputs: int, outputs: int, out: torch.Tensor) -> torch.Tensor:
    device, tokens = a.device, a.shape[0]
    of_a = (DTYPES[a.dtype], a.data_ptr(), *a.stride())
    work = _workspace(device, "plx_mx_workspace", kind, tokens, inputs, outputs, *of_a)
    at, need = (None, 0) if work is None else (work.data_ptr(), work.numel())
    _launch(device, "plx_mx_product", kind, tokens, inputs, outputs, *of_a, m.codes.data_ptr(), m.scales.data_ptr(),
            out.data_ptr(), at, need)
    return out


def product(x: torch.Tensor | Mx4, w: Mx4, dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x w^T`` ``[tokens, outputs]`` of weights ``[outputs, inputs]``.

    x as a tensor is taken as it is, and ``dtype`` must be its type or None.
    x in 4 bits (``quantise4(x)``) is multiplied as it is kept; the result is
    then rounded to ``dtype`` (float32 if None)."""
    outputs, inputs = w.shape
    if isinstance(x, Mx4):
        if x.shape[1] != inputs:
            raise ValueError(f"product: {inputs} inputs expected, got {x.shape[1]}")
        dtype = torch.float32 if dtype is None else dtype
        if dtype not in DTYPES:
            raise TypeError(f"product: float32, bfloat16 or float16 expected, got {dtype}")
        _on_gpu("product", x.device, w.device)
        out = torch.empty((x.shape[0], outputs), dtype=dtype, device=x.device)
        work = _workspace(x.device, "plx_mx4_workspace", x.shape[0], inputs, outputs)
        at, need = (None, 0) if work is None else (work.data_ptr(), work.numel())
        _launch(x.device, "plx_mx4_product", x.shape[0], inputs, outputs, x.codes.data_ptr(), x.scales.data_ptr(),
                w.codes.data_ptr(), w.scales.data_ptr(), DTYPES[dtype], out.data_ptr(), at, need)
        return out
    x = _check("product", x)
    if dtype is not None and dtype != x.dtype:
        raise TypeError(f"product: the result has x's type, {x.dtype}, not {dtype}")
    if x.shape[1] != inputs:
        raise ValueError(f"product: {inputs} inputs expected, got {x.shape[1]}")
    _on_gpu("product", x.device, w.device)
    return _product(_PRODUCT, x, w, inputs, outputs, x.new_empty((x.shape[0], outputs)))


def product_grad(g: torch.Tensor, w: Mx4) -> torch.Tensor:
    """``g w`` ``[tokens, inputs]``: the gradient of :func:`product` for its
    input, from the gradient ``[tokens, outputs]`` of its result."""
    outputs, inputs = w.shape
    g = _check("product_grad", g)
    if g.shape[1] != outputs:
        raise ValueError(f"product_grad: {outputs} outputs expected, got {g.shape[1]}")
    _on_gpu("product_grad", g.device, w.device)
    return _product(_PRODUCT_GRAD, g, w, inputs, outputs, g.new_empty((g.shape[0], inputs)))


def weight_grad(g: torch.Tensor, kept: Mx8) -> torch.Tensor:
    """``g^T x`` ``[outputs, inputs]`` in float32: the gradient of a level
    pair's weights, from its result's gradient ``[tokens, outputs]`` and its
    input kept in 8 bits."""
    g = _check("weight_grad", g)
    tokens, inputs = kept.shape
    if g.shape[0] != tokens:
        raise ValueError(f"weight_grad: {tokens} tokens expected, got {g.shape[0]}")
    _on_gpu("weight_grad", g.device, kept.device)
    out = torch.empty((g.shape[1], inputs), dtype=torch.float32, device=g.device)
    return _product(_WEIGHT_GRAD if kept.axis else _WEIGHT_GRAD_COLUMNS, g, kept, inputs, g.shape[1], out)
