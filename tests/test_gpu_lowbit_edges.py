"""plastax_amd.lowbit where its forms meet their limits: what lies behind a
line's end, views, the ends of float32's range, infinities, and the large
products (each case's form pinned by its workspace)."""

from __future__ import annotations

import pytest
import torch

import lowbit_plain as plain
from plastax_amd import _lib, lowbit

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(shape, g) -> torch.Tensor:
    return torch.randn(shape, generator=g, device=DEV)


def _say(*what) -> None:
    print(*what, flush=True)


def _ranges(kind: str, w: lowbit.Mx4 | lowbit.Mx8, a: torch.Tensor) -> int:
    """The ranges of k that a product of ``a`` runs in as a large one, 0 if it runs in small tiles: by its workspace,
    which holds the codes as bf16, a's pieces (a itself where it is bf16 already) and the ranges' sums."""
    lib = _lib.load()
    tokens = a.shape[0]
    if kind == "weight_grad":
        number, inputs, outputs = 2 if w.axis else 3, w.shape[1], a.shape[1]
        m, n, k = outputs, inputs, tokens
    else:
        number, (outputs, inputs) = ("product", "product_grad").index(kind), w.shape
        m, n, k = (tokens, outputs, inputs) if number == 0 else (tokens, inputs, outputs)
    need = lib.plx_mx_workspace(number, tokens, inputs, outputs, lowbit.DTYPES[a.dtype], a.data_ptr(), *a.stride())
    padded = -(-k // 64) * 64
    pieces = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}[a.dtype]
    along_m = (a.stride(1) if number >= 2 else a.stride(0)) == 1
    codes, copy = -(-2 * padded * n // 256) * 256, -(-2 * pieces * padded * (-(-m // 8) * 8 if along_m else m) // 256) * 256
    for size in (codes, codes + copy) if pieces == 1 else (codes + copy,):
        if need == size:
            return 1
        if need > size and (need - size) % (4 * m * n) == 0 and (need - size) // (4 * m * n) > 1:
            return (need - size) // (4 * m * n)
    return 0


# ---------------------------------------------------------------------------
# Behind a line's end
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("shape", [(1, 40, 24), (33, 130, 70), (70, 300, 200), (257, 770, 520), (1003, 64, 64),
                                   (8190, 1100, 1100)])
def test_codes_of_8_bits_behind_a_lines_end_count_for_nothing(shape, dtype) -> None:
    tokens, inputs, outputs = shape
    _say("padding8", shape, dtype)
    g = _gen(1)
    x, dy = _randn((tokens, inputs), g), _randn((tokens, outputs), g).to(dtype)
    for axis in (0, 1):
        n = (tokens, inputs)[axis]
        kept = lowbit.quantise8(x, axis=axis)
        want, values = lowbit.weight_grad(dy, kept), kept.values()
        slopes = lowbit.activate_grad(x, kept, "silu")
        for byte in (0x7F, 0xFF, 0x38):
            codes = kept.codes.clone()
            codes[:, n:] = byte
            other = lowbit.Mx8(codes, kept.scales, (tokens, inputs), axis)
            assert torch.equal(lowbit.weight_grad(dy, other), want)
            assert torch.equal(other.values(), values)
            assert torch.equal(lowbit.activate_grad(x, other, "silu"), slopes)


@pytest.mark.parametrize("shape", [(1, 1, 70), (3, 31, 70), (16, 1000, 100), (40, 33, 65), (300, 1003, 777),
                                   (1100, 2049, 4608), (1100, 5000, 4700)])
def test_scales_of_4_bits_behind_a_lines_end_count_for_nothing(shape) -> None:
    tokens, inputs, outputs = shape
    _say("padding4", shape)
    g = _gen(2)

    def with_nan_scales(m: lowbit.Mx4) -> lowbit.Mx4:
        scales = m.scales.clone()
        scales[:, -(-m.shape[1] // 32):] = 255
        return lowbit.Mx4(m.codes, scales, m.shape[1])

    w = lowbit.quantise4(_randn((outputs, inputs), g))
    other = with_nan_scales(w)
    assert torch.equal(other.values(), w.values())
    for dtype in plain.DTYPES:
        x, dy = _randn((tokens, inputs), g).to(dtype), _randn((tokens, outputs), g).to(dtype)
        assert torch.equal(lowbit.product(x, other), lowbit.product(x, w))
        assert torch.equal(lowbit.product_grad(dy, other), lowbit.product_grad(dy, w))
        x4 = lowbit.quantise4(x)
        assert torch.equal(lowbit.product(with_nan_scales(x4), other, dtype=dtype), lowbit.product(x4, w, dtype=dtype))


# ---------------------------------------------------------------------------
# Lines that run backwards (of C callers: torch has no such views)
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("shape", [(5, 256, 70), (70, 300, 200), (2304, 2112, 2304)])
def test_products_of_lines_that_run_backwards(shape, dtype) -> None:
    tokens, inputs, outputs = shape
    _say("backwards", shape, dtype)
    g = _gen(3)
    w = lowbit.quantise4(_randn((outputs, inputs), g))
    x = _randn((tokens, inputs), g).to(dtype)
    lib, size, stream = _lib.load(), x.element_size(), torch.cuda.current_stream().cuda_stream
    back, columns = x.flip(0).contiguous(), x.t().flip(0).contiguous()
    for at, strides in ((back.data_ptr() + (tokens - 1) * inputs * size, (-inputs, 1)),
                        (columns.data_ptr() + (inputs - 1) * tokens * size, (1, -tokens))):
        args = (0, tokens, inputs, outputs, lowbit.DTYPES[dtype], at, *strides)
        need = lib.plx_mx_workspace(*args)
        work = torch.empty(need, dtype=torch.uint8, device=DEV)
        out = torch.empty((tokens, outputs), dtype=dtype, device=DEV)
        _lib.check(lib.plx_mx_product(*args, w.codes.data_ptr(), w.scales.data_ptr(), out.data_ptr(),
                                      work.data_ptr(), need, stream), "plx_mx_product")
        assert torch.equal(out, lowbit.product(x, w))


# ---------------------------------------------------------------------------
# Views
# ---------------------------------------------------------------------------
def test_conjugate_parts_are_the_values_that_they_stand_for() -> None:
    """Their memory holds them with the other sign."""
    g = _gen(4)
    z = torch.complex(_randn((40, 70), g), _randn((40, 70), g))
    x = z.conj().imag
    assert x.is_neg()
    same = x.clone()
    w, wt = lowbit.quantise4(_randn((9, 70), g)), lowbit.quantise4(_randn((70, 9), g))
    assert torch.equal(lowbit.quantise4(x).codes, lowbit.quantise4(same).codes)
    assert torch.equal(lowbit.product(x, w), lowbit.product(same, w))
    assert torch.equal(lowbit.product_grad(x, wt), lowbit.product_grad(same, wt))
    for axis in (0, 1):
        y, kept = lowbit.activate(x, "silu", axis=axis)
        want, other = lowbit.activate(same, "silu", axis=axis)
        assert torch.equal(y, want) and torch.equal(kept.codes, other.codes)
        assert torch.equal(lowbit.quantise8(x, axis=axis).codes, kept.codes)
        assert torch.equal(lowbit.activate_grad(x, kept, "silu"), lowbit.activate_grad(same, kept, "silu"))
        assert torch.equal(lowbit.weight_grad(x, kept), lowbit.weight_grad(same, kept))


# ---------------------------------------------------------------------------
# Infinities and NaN in kept activations
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("layout", ["rows", "columns", "steps"])
@pytest.mark.parametrize("dtype", plain.DTYPES)
def test_the_rectifiers_gradient_passes_where_its_result_does(dtype, layout, axis) -> None:
    """At an infinity and a NaN, not at a negative infinity, as torch's own; the other slopes are NaN at all three."""
    g = _gen(5)
    h = _randn((70, 131), g) * 3
    places = torch.rand((70, 131), generator=g, device=DEV)
    h[places < 0.15] = torch.inf
    h[places < 0.10] = -torch.inf
    h[places < 0.05] = torch.nan
    h[places < 0.02] = -torch.tensor(torch.nan, device=DEV).abs()  # a NaN whose sign bit is set
    h[:, 64:96] = torch.where(places[:, 64:96] < 0.5, torch.inf, -torch.inf)  # blocks without a finite value
    h = h.to(dtype)
    dy = plain.layouts(_randn((70, 131), g).to(dtype))[layout]
    x = plain.layouts(h)[layout]
    y, kept = lowbit.activate(x, "relu", axis=axis)
    finite = torch.isfinite(h)
    assert torch.equal(torch.isposinf(y), torch.isposinf(h)) and torch.equal(torch.isnan(y), torch.isnan(h))
    q = kept.values(torch.float32)
    assert torch.equal(torch.isnan(q), ~finite)
    codes = (kept.codes[:, :131] if axis else kept.codes[:, :70].t())[~finite]
    assert torch.equal(codes == 0xFF, torch.isneginf(h)[~finite]) and bool(((codes & 0x7F) == 0x7F).all())
    passes = torch.where(finite, q > 0, ~torch.isneginf(h))
    assert torch.equal(lowbit.activate_grad(dy, kept, "relu"), torch.where(passes, dy, 0 * dy))
    for fn in ("tanh", "sigmoid", "silu"):
        assert torch.equal(torch.isnan(lowbit.activate_grad(dy, kept, fn)), ~finite)


# ---------------------------------------------------------------------------
# The pieces of float32
# ---------------------------------------------------------------------------
def _forms(tokens, inputs, outputs, x, dy):
    """(name, k, function, codes, tensor) of the products of x and dy with weights and kept inputs of ones."""
    w = lowbit.quantise4(torch.ones((outputs, inputs), device=DEV))
    yield "product", inputs, lowbit.product, w, x
    yield "product_grad", outputs, lowbit.product_grad, w, dy
    for axis in (0, 1):
        yield "weight_grad", tokens, lowbit.weight_grad, lowbit.quantise8(torch.ones((tokens, inputs), device=DEV), axis), dy


@pytest.mark.parametrize("layout", ["rows", "columns", "offset"])
@pytest.mark.parametrize("shape", [(4096, 4096, 4096), (8192, 4096, 2048)])
def test_large_sums_keep_what_float32_can_hold(shape, layout) -> None:
    """k times 1 + 2^-23 is one step above k, and its low pieces, half a step of the sum and less each, count together
    (in one range of k: two ranges may halve the step between them)."""
    tokens, inputs, outputs = shape
    _say("low pieces", shape, layout)
    x = plain.layouts(torch.full((tokens, inputs), 1 + 2.0**-23, device=DEV))[layout]
    dy = plain.layouts(torch.full((tokens, outputs), 1 + 2.0**-23, device=DEV))[layout]
    large = 0
    for kind, k, call, codes, a in _forms(*shape, x, dy):
        if _ranges(kind, codes, a) == 1:
            large += 1
            assert call(a, codes).eq(k * (1 + 2.0**-23)).all().item(), kind
    assert large == (4 if tokens == 4096 else 2)


def _numbers(n, dtype, g) -> torch.Tensor:
    """``n`` values of the type's whole range, subnormal ones among them, all of their bits drawn."""
    bits = {torch.float32: 32, torch.bfloat16: 16, torch.float16: 16}[dtype]
    as_int = {32: torch.int32, 16: torch.int16}[bits]
    v = torch.randint(-(1 << (bits - 1)), 1 << (bits - 1), (n,), generator=g, device=DEV).to(as_int).view(dtype)
    least = torch.arange(1, 9, device=DEV).to(as_int).view(dtype)  # the least ones of all, each kind once at least
    top = torch.finfo(dtype)
    ends = torch.tensor([top.tiny, top.max, -top.max, top.tiny * (2 - top.eps), top.tiny * (1 - top.eps)], device=DEV,
                        dtype=torch.float64).to(dtype)
    v = torch.where(torch.isfinite(v), v, torch.ones_like(v))
    some = torch.cat([least, ends])[:n]
    v[: some.numel()] = some
    return v


# few tokens; tiles of 32 and 64, k in one and four groups, in ranges; large ones, in ranges
ONES = [(1, 40, 33), (16, 300, 200), (70, 300, 200), (70, 4096, 130), (300, 1003, 777), (2048, 512, 512),
        (33, 2048, 2049), (4096, 2112, 2304), (512, 4200, 4608), (256, 32768, 1024), (8192, 256, 2048)]


@pytest.mark.parametrize("layout", ["rows", "columns", "offset", "steps"])
@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("shape", ONES)
def test_single_products_keep_every_bit(shape, dtype, layout) -> None:
    """One value a sum, anywhere along k, times powers of two from 2^-110 to 2^110: wherever the type holds the result,
    that is it, and one below its normal numbers is off by its least step at most."""
    tokens, inputs, outputs = shape
    _say("single", shape, dtype, layout)
    g = _gen(7)

    def check(got, want):
        size = torch.finfo(got.dtype)
        held = (want.to(got.dtype).double() == want) & ((want.abs() >= size.smallest_normal) | (want == 0))
        off = (got.double() - want).abs()
        assert bool((off == 0)[held].all()), f"{int((off != 0)[held].sum())} of {int(held.sum())} off"
        small = ~held & (want.abs() < size.smallest_normal)
        assert bool((off[small] <= size.smallest_normal * size.eps).all())

    # weights and kept inputs: a power of two for each line and 32 of its values, of either sign
    def signed(lines, n):
        e = torch.randint(-110, 111, (lines, -(-n // 32)), generator=g, device=DEV).repeat_interleave(32, 1)[:, :n]
        sign = torch.randint(0, 2, (lines, n), generator=g, device=DEV) * 2 - 1
        return sign.double() * torch.exp2(e.double())

    wide = signed(outputs, inputs)
    w = lowbit.quantise4(wide.float())
    assert torch.equal(w.values().double(), wide)
    for k, call in ((inputs, lowbit.product), (outputs, lowbit.product_grad)):
        at = torch.randint(0, k, (tokens,), generator=g, device=DEV)
        v = _numbers(tokens, dtype, g)
        a = torch.zeros((tokens, k), dtype=dtype, device=DEV)
        a[torch.arange(tokens, device=DEV), at] = v
        lines = wide.t()[at] if call is lowbit.product else wide[at]
        check(call(plain.layouts(a)[layout], w), v.double()[:, None] * lines)
    v = _numbers(outputs, dtype, g)
    at = torch.randint(0, tokens, (outputs,), generator=g, device=DEV)
    dy = torch.zeros((tokens, outputs), dtype=dtype, device=DEV)
    dy[at, torch.arange(outputs, device=DEV)] = v
    for axis in (0, 1):
        x = signed(tokens, inputs) if axis else signed(inputs, tokens).t()
        kept = lowbit.quantise8(x.float(), axis=axis)
        assert torch.equal(kept.values(torch.float32).double(), x)
        check(lowbit.weight_grad(plain.layouts(dy)[layout], kept), v.double()[:, None] * x[at])


def test_single_products_run_in_every_form() -> None:
    """The shapes above, by their plans: small tiles whole and in ranges, large ones whole and in ranges."""
    lib, small, large = _lib.load(), set(), set()
    for tokens, inputs, outputs in ONES:
        x = torch.empty((tokens, inputs), device=DEV)
        w = lowbit.Mx4._empty(outputs, inputs, DEV)
        ranges = _ranges("product", w, x)
        if ranges:
            large.add(min(ranges, 2))
        elif tokens > 16:
            small.add(lib.plx_mx_workspace(0, tokens, inputs, outputs, 0, x.data_ptr(), inputs, 1) > 0)
    assert small == {False, True} and large == {1, 2}


# ---------------------------------------------------------------------------
# Large products
# ---------------------------------------------------------------------------
def _spread(shape, g) -> torch.Tensor:
    """Values from 2^-4 to 2^4, a tenth of them zeros."""
    x = _randn(shape, g) * torch.exp2(torch.randint(-4, 4, shape, generator=g, device=DEV).float())
    return torch.where(torch.rand(shape, generator=g, device=DEV) < 0.1, 0.0, x)


@pytest.mark.parametrize("layout", ["rows", "columns", "offset_columns", "steps"])
@pytest.mark.parametrize("dtype", plain.DTYPES)
def test_infinities_and_nan_in_large_products(dtype, layout) -> None:
    tokens, inputs, outputs = 2056, 2120, 3300
    _say("large nan", dtype, layout)
    g = _gen(8)
    wf = _randn((outputs, inputs), g)
    wf[7, 40], wf[3001, 2119] = torch.nan, torch.inf  # their blocks of 32 become NaN, the last one of 8 values
    w = lowbit.quantise4(wf)
    w64 = plain.values4(w.codes, w.scales, inputs)
    assert int(torch.isnan(w64).sum()) == 40

    def places(n):
        a = _randn((tokens, n), g).to(dtype)
        a[0, 3], a[300, n - 1], a[1999, 9] = torch.inf, -torch.inf, torch.nan
        a[2000, 64:72] = torch.tensor([torch.nan, torch.inf, -torch.inf, 1, 0, -1, torch.nan, torch.inf]).to(dtype)
        return a

    def same(got, want):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        inf = torch.isinf(want)
        assert torch.equal(torch.isinf(got), inf) and torch.equal(got.double()[inf], want[inf])

    x, dy = places(inputs), places(outputs)
    a = plain.layouts(x)[layout]
    assert _ranges("product", w, a)
    same(lowbit.product(a, w), x.double() @ w64.t())
    a = plain.layouts(dy)[layout]
    assert _ranges("product_grad", w, a)
    same(lowbit.product_grad(a, w), dy.double() @ w64)
    h = _randn((tokens, inputs), g)
    h[0, 8], h[500, 2119], h[2055, 77] = torch.nan, torch.inf, -torch.inf
    for axis in (0, 1):
        kept = lowbit.quantise8(h, axis=axis)
        x8 = kept.values(torch.float32).double()
        assert _ranges("weight_grad", kept, a)
        same(lowbit.weight_grad(a, kept), dy.double().t() @ x8)


@pytest.mark.parametrize("dtype", plain.DTYPES)
def test_infinities_and_nan_in_large_products_of_two_in_4_bits(dtype) -> None:
    tokens, inputs, outputs = 2056, 2120, 6000
    g = _gen(9)
    wf, xf = _randn((outputs, inputs), g), _randn((tokens, inputs), g)
    wf[7, 40], wf[5999, 2119], xf[300, 2], xf[2055, 64] = torch.nan, torch.inf, -torch.inf, torch.nan
    w, x = lowbit.quantise4(wf), lowbit.quantise4(xf)
    assert _large4(tokens, inputs, outputs)
    want = plain.values4(x.codes, x.scales, inputs) @ plain.values4(w.codes, w.scales, inputs).t()
    got = lowbit.product(x, w, dtype=dtype)
    assert int(torch.isnan(want).sum()) == 2 * tokens + 2 * outputs - 4
    assert torch.equal(torch.isnan(got), torch.isnan(want))


def _large4(tokens, inputs, outputs) -> bool:
    """Whether a product of two in 4 bits runs as a large one: its workspace then holds the scales of whole tiles."""
    scales = (-(-tokens // 256) + -(-outputs // 256)) * -(-inputs // 256) * 2048
    need = _lib.load().plx_mx4_workspace(tokens, inputs, outputs)
    return need >= scales and (need - scales) % (4 * tokens * outputs) == 0


@pytest.mark.parametrize("layout", ["offset_columns", "steps"])
@pytest.mark.parametrize("dtype", plain.DTYPES)
def test_large_products_of_other_layouts(dtype, layout) -> None:
    tokens, inputs, outputs = 2056, 2120, 3300
    _say("large layouts", dtype, layout)
    g = _gen(10)
    w = lowbit.quantise4(_spread((outputs, inputs), g))
    w64 = plain.values4(w.codes, w.scales, inputs)
    x = plain.layouts(_spread((tokens, inputs), g).to(dtype))[layout]
    assert _ranges("product", w, x)
    plain.assert_product(lowbit.product(x, w), x.double(), w64)
    dy = plain.layouts(_spread((tokens, outputs), g).to(dtype))[layout]
    assert _ranges("product_grad", w, dy)
    plain.assert_product(lowbit.product_grad(dy, w), dy.double(), w64.t().contiguous())
    for axis in (0, 1):
        kept = lowbit.quantise8(x, axis=axis)
        assert _ranges("weight_grad", kept, dy)
        plain.assert_product(lowbit.weight_grad(dy, kept), dy.double().t().contiguous(),
                             kept.values(torch.float32).double().t().contiguous())


@pytest.mark.parametrize("shape", [(2304, 2176, 4700), (256, 36864, 1024)])
def test_large_products_on_another_stream_and_in_a_graph(shape) -> None:
    tokens, inputs, outputs = shape
    g = _gen(11)
    w = lowbit.quantise4(_randn((outputs, inputs), g))
    wide = lowbit.quantise4(_randn((6200, inputs), g))
    x, dy = _randn((tokens, inputs), g).bfloat16(), _randn((tokens, outputs), g).bfloat16()

    def step():
        kept = lowbit.quantise8(x)
        low = lowbit.product(lowbit.quantise4(x), wide, dtype=torch.bfloat16)
        return (lowbit.product(x, w), lowbit.product(x.float(), w), lowbit.product_grad(dy, w),
                lowbit.product_grad(dy.half(), w), lowbit.weight_grad(dy, kept), lowbit.weight_grad(dy.float(), kept), low)

    assert _ranges("product", w, x) and _large4(tokens, inputs, 6200)
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(3):
        x.copy_(_randn((tokens, inputs), g))
        want = [t.clone() for t in step()]  # eager work between the replays
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b), k


def test_products_of_more_tiles_than_a_launch_holds() -> None:
    """2^26 rows are a launch of 64 x 64 tiles; results go past 2^32 elements."""
    border, tokens, inputs, outputs = 1 << 26, (1 << 26) + 100, 8, 64
    g = _gen(12)
    w = lowbit.quantise4(_randn((outputs, inputs), g))
    w64 = plain.values4(w.codes, w.scales, inputs)
    x = torch.zeros((tokens, inputs), dtype=torch.bfloat16, device=DEV)
    parts = [slice(0, 70), slice(border // 2 - 50, border // 2 + 50), slice(border - 70, tokens)]
    for part in parts:
        x[part] = _randn((part.stop - part.start, inputs), g)
    for y, values in ((lowbit.product(x, w), lambda v: v.double()),
                      (lowbit.product(lowbit.quantise4(x), w, dtype=torch.bfloat16),
                       lambda v: plain.values4(*plain.quantise4(v), inputs))):
        for part in parts:
            plain.assert_product(y[part], values(x[part]), w64)
        assert not y[border // 4 : border // 4 + 1000].any() and not y[border - 1000 : border - 70].any()
        del y
