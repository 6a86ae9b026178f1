"""What a net of dense level pairs needs around them to read and learn tokens.

Level pairs held as matrices (:mod:`plastax_amd.lowbit`) answer batches
``[tokens, units]``. Here are the levels between them:

- an input level of which one unit is on for each token: :func:`look_up` takes
  its level pair's rows by id, :func:`look_up_grad` sums their gradients;
- layer norm: :func:`normalise`, :func:`normalise_grad`;
- a level carried along sequences by a gated linear recurrence: :func:`recur`,
  :func:`recur_grad`, and :func:`recur_step` for one token of each sequence;
- an output level that learns from a teacher which named a few outputs of each
  token: :func:`distil` (the loss), :func:`distil_grad` (with its gradient).

Arguments are GPU tensors. Batches are of float32, bfloat16 or float16, with any
strides (one whose tokens' units lie apart is copied first); results have the
batch's type, are contiguous, and are rounded once. Sums, states, norms and the
gradients of weights and tables are float32, summed in a fixed order: a call
gives the same bits each time. Ids are int32 or int64. Work goes to torch's
current stream of the arguments' device, results and workspaces are allocated
there. Results carry no autograd graph and no tangent: an argument that asks for
one is refused, the gradients are calls of their own. The reference has no
counterpart.
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from plastax_amd import _lib
from plastax_amd.lowbit import DTYPES, _call, _launch

_IDS = {torch.int32: 0, torch.int64: 1}
_KEEP = 64  # PLX_RECUR_KEEP
MAX_NAMED = 1024  # PLX_MAX_NAMED
_MAX_TOKENS, _MAX_UNITS = 1 << 30, 1 << 24
_LEAST, _MOST = 2.0**-126, 2.0**128 - 2.0**104  # float32's normal numbers


def _plain(who: str, t: torch.Tensor) -> torch.Tensor:
    """``t`` without autograd, with the values that it stands for in its memory."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{who}: no autograd here; detach the argument and call the gradients")
    # (the level is -1 outside of dual_level(), where no tensor has a tangent)
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{who}: no forward-mode autograd here; unpack the argument and its tangent")
    return t.resolve_neg() if t.is_neg() else t


def _batch(who: str, t: torch.Tensor) -> torch.Tensor:
    """``t`` checked, each token's units next to each other."""
    if t.dim() != 2:
        raise ValueError(f"{who}: a batch [tokens, units] expected, got {t.dim()} dimensions")
    if t.dtype not in DTYPES:
        raise TypeError(f"{who}: float32, bfloat16 or float16 expected, got {t.dtype}")
    tokens, units = t.shape
    if tokens > _MAX_TOKENS or units > _MAX_UNITS:
        raise ValueError(f"{who}: at most 2^30 tokens and 2^24 units, got {(tokens, units)}")
    t = _plain(who, t)
    return t if units <= 1 or t.stride(1) == 1 else t.contiguous()


def _ids(who: str, name: str, t: torch.Tensor, dims: int) -> torch.Tensor:
    if t.dtype not in _IDS:
        raise TypeError(f"{who}: {name} of int32 or int64 expected, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{who}: {name} of {dims} dimensions expected, got {t.dim()}")
    return t if t.is_contiguous() else t.contiguous()


def _floats(who: str, name: str, t: torch.Tensor, shape: tuple[int, ...]) -> torch.Tensor:
    """A contiguous float32 argument beside a batch."""
    if t.dtype is not torch.float32:
        raise TypeError(f"{who}: {name} of float32 expected, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{who}: {name} of {shape} expected, got {tuple(t.shape)}")
    t = _plain(who, t)
    return t if t.is_contiguous() else t.contiguous()


def _together(who: str, t: torch.Tensor, *others: torch.Tensor | None) -> None:
    device = t.device
    if device.type != "cuda":
        raise ValueError(f"{who}: arguments must be on the GPU, got {device}")
    for o in others:
        if o is not None and o.device != device:
            raise ValueError(f"{who}: arguments are on different devices, {device} and {o.device}")


def _space(device: torch.device, name: str, *args: object) -> tuple[torch.Tensor | None, int | None, int]:
    """The call's workspace: the tensor, its address and its bytes."""
    need = getattr(_lib.load(), name)(*args) if device.index == torch._C._cuda_getDevice() else _call(device, name, *args)
    if need < 0:
        raise ValueError(f"{name}: sizes out of range")
    if need == 0:
        return None, None, 0
    work = torch.empty(need, dtype=torch.uint8, device=device)
    return work, work.data_ptr(), need


# --------------------------------------------------------------------------
# An input level by ids
# --------------------------------------------------------------------------
def _scale(who: str, scale: float) -> None:
    if not (_LEAST <= abs(scale) <= _MOST or scale == 0 or not math.isfinite(scale)):
        raise ValueError(f"{who}: a scale that float32 has expected (0, or 2^-126 to 3.4e38), got {scale}")


def look_up(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[ids]`` ``[tokens, units]`` of a table ``[rows, units]``.

    scale is taken in float32. An id that the table has no row for (-1,
    padding) gives a row of zeros."""
    _scale("look_up", scale)
    table, ids = _batch("look_up", table), _ids("look_up", "ids", ids, 1)
    rows, units = table.shape
    if rows > _MAX_UNITS:
        raise ValueError(f"look_up: at most 2^24 rows, got {rows}")
    if ids.shape[0] > _MAX_TOKENS:
        raise ValueError(f"look_up: at most 2^30 tokens, got {ids.shape[0]}")
    _together("look_up", table, ids)
    out = table.new_empty((ids.shape[0], units))
    _launch(table.device, "plx_look_up", ids.shape[0], rows, units, ids.data_ptr(), _IDS[ids.dtype],
            DTYPES[table.dtype], table.data_ptr(), table.stride(0), scale, out.data_ptr())
    return out


def look_up_grad(g: torch.Tensor, ids: torch.Tensor, rows: int, scale: float = 1.0) -> torch.Tensor:
    """The table's gradient ``[rows, units]`` in float32: ``scale`` times the
    sums of the tokens' gradients g ``[tokens, units]`` by id, zeros for rows
    that no token named. Ids outside of the rows count for nothing. At most 2^25
    tokens."""
    _scale("look_up_grad", scale)
    g, ids = _batch("look_up_grad", g), _ids("look_up_grad", "ids", ids, 1)
    if not 0 <= rows <= _MAX_UNITS:
        raise ValueError(f"look_up_grad: 0 to 2^24 rows expected, got {rows}")
    if ids.shape[0] != g.shape[0]:
        raise ValueError(f"look_up_grad: {g.shape[0]} ids expected, got {ids.shape[0]}")
    _together("look_up_grad", g, ids)
    tokens, units = g.shape
    out = torch.empty((rows, units), dtype=torch.float32, device=g.device)
    _work, at, need = _space(g.device, "plx_look_up_workspace", tokens, rows, units)
    _launch(g.device, "plx_look_up_grad", tokens, rows, units, ids.data_ptr(), _IDS[ids.dtype], DTYPES[g.dtype],
            g.data_ptr(), g.stride(0), scale, out.data_ptr(), at, need)
    return out


# --------------------------------------------------------------------------
# Layer norm
# --------------------------------------------------------------------------
def _param(who: str, name: str, x: torch.Tensor, p: torch.Tensor) -> torch.Tensor:
    if p.dtype is not x.dtype and p.dtype is not torch.float32:
        raise TypeError(f"{who}: weight and bias both of {x.dtype} or of float32 expected, got {name} of {p.dtype}")
    if p.shape != x.shape[1:]:
        raise ValueError(f"{who}: {name} of {x.shape[1]} units expected, got {tuple(p.shape)}")
    p = _plain(who, p)
    return p if p.is_contiguous() else p.contiguous()


def normalise(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
              eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """``(y, kept)``: y = (x - mean) / sqrt(var + eps) * weight + bias, mean and
    variance over each token's units, and what the gradient needs (each token's
    mean and 1 / sqrt(var + eps), float32 ``[tokens, 2]``).

    weight and bias ``[units]`` are both float32, or both of x's type. eps is
    taken in float32, and a row's sums are float32, of x and of the squares of
    x - mean (mean with the rounding of its sum): where they pass its range, 3.4e38,
    or where the squares vanish, below 1e-38, beside an eps as small or 0, results
    are not what the formula gives."""
    x = _batch("normalise", x)
    if not (_LEAST <= eps <= _MOST or eps == 0):
        raise ValueError(f"normalise: an eps that float32 has expected (0, or 2^-126 to 3.4e38), got {eps}")
    weight = _param("normalise", "weight", x, weight)
    if bias is not None:
        if bias.dtype is not weight.dtype:
            raise TypeError(f"normalise: weight and bias of one type expected, got {weight.dtype} and {bias.dtype}")
        bias = _param("normalise", "bias", x, bias)
    _together("normalise", x, weight, bias)
    tokens, units = x.shape
    y = x.new_empty((tokens, units))
    kept = torch.empty((tokens, 2), dtype=torch.float32, device=x.device)
    _launch(x.device, "plx_normalise", tokens, units, DTYPES[x.dtype], x.data_ptr(), x.stride(0),
            DTYPES[weight.dtype], weight.data_ptr(), None if bias is None else bias.data_ptr(), eps, y.data_ptr(),
            kept.data_ptr())
    return y, kept


def normalise_grad(g: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                   kept: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(dx, dweight, dbias)`` from g, the gradient of :func:`normalise`'s y,
    its x and weight, and what it kept; dweight and dbias are float32."""
    g, x = _batch("normalise_grad", g), _batch("normalise_grad", x)
    if g.dtype != x.dtype:
        raise TypeError(f"normalise_grad: a gradient of x's type, {x.dtype}, expected, got {g.dtype}")
    if g.shape != x.shape:
        raise ValueError(f"normalise_grad: a gradient of {tuple(x.shape)} expected, got {tuple(g.shape)}")
    weight = _param("normalise_grad", "weight", x, weight)
    tokens, units = x.shape
    kept = _floats("normalise_grad", "kept", kept, (tokens, 2))
    _together("normalise_grad", x, g, weight, kept)
    dx = x.new_empty((tokens, units))
    dparams = torch.empty((2, units), dtype=torch.float32, device=x.device)
    _work, at, need = _space(x.device, "plx_normalise_workspace", tokens, units, DTYPES[x.dtype])
    _launch(x.device, "plx_normalise_grad", tokens, units, DTYPES[x.dtype], g.data_ptr(), g.stride(0), x.data_ptr(),
            x.stride(0), DTYPES[weight.dtype], weight.data_ptr(), kept.data_ptr(), dx.data_ptr(), dparams.data_ptr(),
            at, need)
    return dx, *dparams.unbind(0)


# --------------------------------------------------------------------------
# A level carried along sequences
# --------------------------------------------------------------------------
def _sequences(who: str, xz: torch.Tensor, starts: torch.Tensor | None,
               state: torch.Tensor | None) -> tuple[torch.Tensor, int, torch.Tensor | None, int, torch.Tensor | None]:
    """xz checked, its units, starts, the sequences, and the state."""
    xz = _batch(who, xz)
    if xz.shape[1] % 2:
        raise ValueError(f"{who}: x beside z, an even number of columns, expected, got {xz.shape[1]}")
    units, sequences = xz.shape[1] // 2, 1
    if starts is not None:
        starts = _ids(who, "starts", starts, 1)
        sequences = starts.shape[0] - 1
        if not 0 <= sequences <= _MAX_TOKENS:
            raise ValueError(f"{who}: starts of 1 to 2^30 + 1 rows expected, got {starts.shape[0]}")
    if state is not None:
        state = _floats(who, "state", state, (sequences, units))
    return xz, units, starts, sequences, state


def recur(xz: torch.Tensor, starts: torch.Tensor | None = None,
          state: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(h, last, kept)``: with x and z side by side in xz ``[tokens, 2 units]``
    and a = sigmoid(z), ``h[t] = a[t] h[t-1] + (1 - a[t]) x[t]`` along sequences.

    Sequence s is the rows from ``starts[s]`` to before ``starts[s + 1]``
    (rising, within the tokens; they are not read on the host); without starts
    all rows are one. It goes on from ``state[s]`` (float32 ``[sequences,
    units]``; zeros if None); last is its last h in float32, or its state if it
    has no rows. h ``[tokens, units]`` is 0 in rows of no sequence. kept is what
    the gradient needs (float32, one row in 64). At most 2^22 pieces of 64 rows
    by 128 units. An infinity or a NaN stays in
    its sequence and unit, where what follows is not finite."""
    xz, units, starts, sequences, state = _sequences("recur", xz, starts, state)
    _together("recur", xz, starts, state)
    tokens = xz.shape[0]
    h = xz.new_empty((tokens, units))
    last = torch.empty((sequences, units), dtype=torch.float32, device=xz.device)
    kept = last.new_empty((-(-tokens // _KEEP), units))
    at_starts, wide = (None, 0) if starts is None else (starts.data_ptr(), _IDS[starts.dtype])
    _work, at, need = _space(xz.device, "plx_recur_workspace", tokens, units, sequences, starts is not None)
    _launch(xz.device, "plx_recur", tokens, units, sequences, DTYPES[xz.dtype], xz.data_ptr(), xz.stride(0), at_starts,
            wide, None if state is None else state.data_ptr(), h.data_ptr(), last.data_ptr(), kept.data_ptr(), at, need)
    return h, last, kept


def recur_grad(g: torch.Tensor, xz: torch.Tensor, kept: torch.Tensor, starts: torch.Tensor | None = None,
               state: torch.Tensor | None = None,
               g_last: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(dxz, dstate)`` from g ``[tokens, units]``, the gradient of
    :func:`recur`'s h, and g_last (float32 ``[sequences, units]``; zeros if
    None), that of its last; the other arguments are recur's and what it kept.
    dxz ``[tokens, 2 units]`` has the gradients of x and z side by side, 0 in
    rows of no sequence; dstate is float32."""
    xz, units, starts, sequences, state = _sequences("recur_grad", xz, starts, state)
    g = _batch("recur_grad", g)
    tokens = xz.shape[0]
    if g.dtype != xz.dtype:
        raise TypeError(f"recur_grad: a gradient of xz's type, {xz.dtype}, expected, got {g.dtype}")
    if g.shape != (tokens, units):
        raise ValueError(f"recur_grad: a gradient of {(tokens, units)} expected, got {tuple(g.shape)}")
    kept = _floats("recur_grad", "kept", kept, (-(-tokens // _KEEP), units))
    if g_last is not None:
        g_last = _floats("recur_grad", "g_last", g_last, (sequences, units))
    _together("recur_grad", xz, g, kept, starts, state, g_last)
    dxz = xz.new_empty((tokens, 2 * units))
    dstate = torch.empty((sequences, units), dtype=torch.float32, device=xz.device)
    at_starts, wide = (None, 0) if starts is None else (starts.data_ptr(), _IDS[starts.dtype])
    _work, at, need = _space(xz.device, "plx_recur_workspace", tokens, units, sequences, starts is not None)
    _launch(xz.device, "plx_recur_grad", tokens, units, sequences, DTYPES[xz.dtype], g.data_ptr(), g.stride(0),
            xz.data_ptr(), xz.stride(0), at_starts, wide, None if state is None else state.data_ptr(),
            None if g_last is None else g_last.data_ptr(), kept.data_ptr(), dxz.data_ptr(), dstate.data_ptr(), at, need)
    return dxz, dstate


def recur_step(xz: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
    """One token of each sequence: xz ``[sequences, 2 units]``; the state
    (float32 ``[sequences, units]``, each sequence's units next to each other,
    no two sequences in the same memory, nor in xz's) is updated in place, and h
    is what it became in xz's type."""
    xz = _batch("recur_step", xz)
    sequences, units = xz.shape[0], xz.shape[1] // 2
    if xz.shape[1] % 2:
        raise ValueError(f"recur_step: x beside z, an even number of columns, expected, got {xz.shape[1]}")
    if state.dtype is not torch.float32:
        raise TypeError(f"recur_step: a state of float32 expected, got {state.dtype}")
    if state.shape != (sequences, units):
        raise ValueError(f"recur_step: a state of {(sequences, units)} expected, got {tuple(state.shape)}")
    if _plain("recur_step", state) is not state:
        raise ValueError("recur_step: the state is updated in place: a negated view is not")
    if (units > 1 and state.stride(1) != 1) or (sequences > 1 and state.stride(0) < units):
        raise ValueError("recur_step: the state is updated in place: units next to each other and sequences apart "
                         f"expected, got strides {state.stride()}")
    _together("recur_step", xz, state)
    h = xz.new_empty((sequences, units))
    _launch(xz.device, "plx_recur_step", sequences, units, DTYPES[xz.dtype], xz.data_ptr(), xz.stride(0),
            state.data_ptr(), state.stride(0), h.data_ptr())
    torch._C._increment_version((state,))  # (autograd.graph.increment_version without its check, 0.5 us)
    return h


# --------------------------------------------------------------------------
# An output level learned from a teacher
# --------------------------------------------------------------------------
def _named(who: str, logits: torch.Tensor, ids: torch.Tensor, top: torch.Tensor,
           temperature: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    logits, ids = _batch(who, logits), _ids(who, "ids", ids, 2)
    if ids.shape[0] != logits.shape[0] or ids.shape[1] > MAX_NAMED:
        raise ValueError(f"{who}: ids of {logits.shape[0]} tokens and at most {MAX_NAMED} outputs each expected, "
                         f"got {tuple(ids.shape)}")
    if top.dtype not in DTYPES:
        raise TypeError(f"{who}: top of float32, bfloat16 or float16 expected, got {top.dtype}")
    if top.shape != ids.shape:
        raise ValueError(f"{who}: top of {tuple(ids.shape)} expected, got {tuple(top.shape)}")
    top = _plain(who, top)
    top = top if top.is_contiguous() else top.contiguous()
    if not 2.0**-120 <= temperature <= 2.0**120:  # (its inverse is a normal number of float32 too)
        raise ValueError(f"{who}: a temperature from 2^-120 to 2^120 expected, got {temperature}")
    return logits, ids, top


def distil(logits: torch.Tensor, ids: torch.Tensor, top: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """The loss of each token ``[tokens]`` in float32, ``T^2 sum p (log p - log q)``.

    q = softmax(logits / T) over the outputs; p = softmax(top / T) over the
    outputs that ids ``[tokens, named]`` name, top the teacher's logits for
    them. A place whose id is no output (-1), or whose top is -inf, counts for
    nothing; a token without any other place has the loss 0 (and the gradient
    0). An output named twice counts twice. The temperature is taken in
    float32."""
    logits, ids, top = _named("distil", logits, ids, top, temperature)
    _together("distil", logits, ids, top)
    tokens, outputs = logits.shape
    loss = torch.empty((tokens,), dtype=torch.float32, device=logits.device)
    _launch(logits.device, "plx_distil", tokens, outputs, ids.shape[1], DTYPES[logits.dtype], logits.data_ptr(),
            logits.stride(0), ids.data_ptr(), _IDS[ids.dtype], DTYPES[top.dtype], top.data_ptr(), temperature,
            loss.data_ptr())
    return loss


def distil_grad(g: torch.Tensor, logits: torch.Tensor, ids: torch.Tensor, top: torch.Tensor,
                temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """``(loss, dlogits)``: :func:`distil`'s losses, and the gradient of their
    sum weighted by g (float32 ``[tokens]``; 1 / tokens for a mean, 0 for a
    token that is not learned from), in one pass over the logits. g times the
    temperature is float32."""
    logits, ids, top = _named("distil_grad", logits, ids, top, temperature)
    tokens, outputs = logits.shape
    g = _floats("distil_grad", "g", g, (tokens,))
    _together("distil_grad", logits, ids, top, g)
    loss = torch.empty((tokens,), dtype=torch.float32, device=logits.device)
    d = logits.new_empty((tokens, outputs))
    _launch(logits.device, "plx_distil_grad", tokens, outputs, ids.shape[1], g.data_ptr(), DTYPES[logits.dtype],
            logits.data_ptr(), logits.stride(0), ids.data_ptr(), _IDS[ids.dtype], DTYPES[top.dtype], top.data_ptr(),
            temperature, loss.data_ptr(), d.data_ptr())
    return loss, d
