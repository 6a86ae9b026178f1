"""plastax_amd.lowbit on the GPU against the plain 64-bit forms: codes and
scales bit for bit; sums of exact products, and elementary functions, to
bounds that count their roundings."""

from __future__ import annotations

import pytest
import torch

import lowbit_plain as plain
from plastax_amd import lowbit

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
FNS = ["relu", "tanh", "sigmoid", "silu"]
LAYOUTS = ["rows", "columns", "offset", "offset_columns", "steps"]
LINES = [(1, 1), (3, 31), (5, 32), (2, 33), (7, 127), (4, 128), (3, 129), (65, 1003), (70, 2049), (130, 64), (600, 72)]
# tokens, inputs, outputs
SHAPES = [(1, 1, 1), (1, 33, 17), (2, 128, 64), (3, 129, 65), (15, 31, 128), (16, 256, 777), (17, 1003, 33),
          (63, 64, 96), (64, 512, 130), (65, 1100, 63), (130, 1, 70), (300, 130, 1100), (513, 770, 520),
          (256, 256, 256), (257, 1344, 300), (600, 576, 904), (264, 2049, 1030), (1100, 520, 512),
          (1, 4096, 1024), (33, 2048, 2049)]


# large products: whole and odd tiles, lines of whole, odd and half steps, ranges of k over workgroups
LARGE = [(2056, 2120, 2304), (1100, 2049, 4608), (264, 9600, 4104), (4104, 257, 9601), (2304, 16704, 264), (256, 36864, 1024)]


def _gen(*key: int) -> torch.Generator:
    seed = 0
    for k in key:
        seed = seed * 10007 + k
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(shape, g) -> torch.Tensor:
    return torch.randn(shape, generator=g, device=DEV)


def _spread(shape, g, low: int = -20, high: int = 20) -> torch.Tensor:
    """Values of very different sizes, some zeros."""
    e = torch.randint(low, high, shape, generator=g, device=DEV).float()
    x = _randn(shape, g) * torch.exp2(e)
    return torch.where(torch.rand(shape, generator=g, device=DEV) < 0.1, 0.0, x)


def _hard(shape, dtype, g) -> torch.Tensor:
    """Lines of ties, of equal sizes, subnormals, the type's largest, zeros of both signs, infinities and NaN."""
    r, n = shape
    x = _spread(shape, g)
    top = torch.finfo(dtype)
    kinds = [torch.randint(-24, 25, (n,), generator=g, device=DEV).float() / 4,
             torch.randint(-448, 449, (n,), generator=g, device=DEV).float() * 2.0**-7,
             _randn((n,), g) * top.tiny, (_randn((n,), g) * 0.3).clamp(-1, 1) * top.max,
             torch.where(_randn((n,), g) < 0, -0.0, 0.0), torch.full((n,), top.max, device=DEV)]
    for i, k in enumerate(kinds):
        if i < r:
            x[i] = k
    x = x.to(dtype)
    if r > 6:
        x[6, :: 45] = torch.inf
        x[6, 20::70] = torch.nan
    if r > 7:
        x[7, n // 2] = -torch.inf
    return x


def _same(a: torch.Tensor, b: torch.Tensor) -> bool:
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def _say(*what) -> None:
    print(*what, flush=True)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("shape", LINES)
def test_quantise4_gives_the_formats_codes(shape, dtype, layout) -> None:
    _say("quantise4", shape, dtype, layout)
    x = plain.layouts(_hard(shape, dtype, _gen(*shape)))[layout]
    m = lowbit.quantise4(x)
    codes, scales = plain.quantise4(x)
    assert torch.equal(m.scales, scales)
    assert torch.equal(m.codes, codes)
    want = plain.values4(codes, scales, shape[1])
    for out in plain.DTYPES:  # (float32's largest goes up to 2^128, which is an infinity there)
        assert _same(m.values(out), want.to(out))


@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("n", [1, 31, 64, 70, 257])
def test_values8_of_every_code(n, axis) -> None:
    lines, b = 256, -(-n // 32)
    codes = ((torch.arange(lines, device=DEV)[:, None] + torch.arange(32 * b, device=DEV)[None]) % 256).to(torch.uint8)
    scales = torch.randint(10, 248, (lines, b), generator=_gen(n), device=DEV).to(torch.uint8)
    m = lowbit.Mx8(codes, scales, (lines, n) if axis else (n, lines), axis)
    want = plain.values8(codes, scales, n)
    for out in plain.DTYPES:  # (the largest codes under the largest scales are infinities)
        got = m.values(out)
        assert got.shape == m.shape
        assert _same(got if axis else got.t(), want.to(out))


@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("shape", LINES)
def test_activate_and_its_gradient(shape, dtype, layout, axis) -> None:
    g = _gen(*shape, axis)
    for fn in FNS:
        _say("activate", shape, dtype, layout, axis, fn)
        h = plain.layouts(_hard(shape, dtype, g))[layout]
        y, kept = lowbit.activate(h, fn, axis=axis)
        codes, scales = plain.quantise8(h if axis else h.t())
        assert torch.equal(kept.scales, scales)
        nan = (codes & 127) == 127  # (NaN has two codes)
        alone = lowbit.quantise8(h, axis=axis)
        assert torch.equal(alone.codes, kept.codes) and torch.equal(alone.scales, kept.scales)
        assert torch.equal(torch.where(nan, 0, kept.codes), torch.where(nan, 0, codes))
        assert bool(((kept.codes & 127) == 127)[nan].all())
        # an elementary function is good to 2 steps, 1 / (1 + e) adds a step, the product half of one: 4 steps
        want = plain.act(fn, h)
        # (below the normal numbers: half the type's least step, and e^x's own, 2^-150, times h)
        least = torch.finfo(dtype).smallest_normal * plain.half_step(dtype) * 2
        tol = want.abs() * (8 * plain.U + plain.half_step(dtype)) + least + (1 + h.double().abs()) * 2.0**-148
        assert y.shape == h.shape and y.dtype == dtype
        assert _same(torch.isnan(y), torch.isnan(want))
        fine = ~torch.isnan(want)
        assert bool(((y.double() - want).abs() <= tol)[fine & torch.isfinite(want)].all())
        assert _same(y.double()[fine & ~torch.isfinite(want)], want[fine & ~torch.isfinite(want)])

        q = plain.values8(codes, scales, h.shape[axis])
        q = q if axis else q.t()
        dy = plain.layouts(_spread(shape, g, -3, 4).to(dtype))[layout]
        dh = lowbit.activate_grad(dy, kept, fn)
        # e^x 4u, 1 + t and its inverse 4u, so t r r 14u, the product with dy 1u: below 16u of the terms' sizes
        d, size = plain.act_grad(fn, q)
        want = dy.double() * d
        tol = dy.double().abs() * (size * 16 * plain.U + (1 + q.abs()) * 2.0**-148) + want.abs() * plain.half_step(dtype) + least
        assert dh.shape == dy.shape and dh.dtype == dtype
        fine = ~torch.isnan(q)
        assert bool(((dh.double() - want).abs() <= tol)[fine].all())
        if fn != "relu":
            assert bool(torch.isnan(dh)[~fine].all())


@pytest.mark.parametrize("fn", FNS)
def test_activate_grad_is_the_slope(fn) -> None:
    """Against differences of the function in 64 bits at the kept values (away from the rectifier's corner)."""
    h = _randn((64, 96), _gen(5)) * 3
    _, kept = lowbit.activate(h, fn)
    q = kept.values(torch.float32).double()
    step = 2.0**-16
    slope = (plain.act(fn, q + step) - plain.act(fn, q - step)) / (2 * step)
    got = lowbit.activate_grad(torch.ones_like(h), kept, fn).double()
    # the third derivative is below 4: step^2 / 6 * 4, and 64-bit rounding of values up to 32 over the step
    far = q.abs() > 2 * step
    assert bool(((got - slope).abs() <= step**2 + 2.0**-47 / step + 16 * plain.U * 1.3)[far].all())


def _weights(outputs, inputs, g) -> lowbit.Mx4:
    w = _spread((outputs, inputs), g, -6, 6)
    w[w.abs() < 1e-3] = 0
    return lowbit.quantise4(w)


def _w64(w: lowbit.Mx4) -> torch.Tensor:
    return plain.values4(w.codes, w.scales, w.shape[1])


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_product_and_its_gradient(shape, dtype, layout) -> None:
    tokens, inputs, outputs = shape
    _say("product", shape, dtype, layout)
    g = _gen(*shape)
    w = _weights(outputs, inputs, g)
    x = _spread((tokens, inputs), g, -4, 4).to(dtype)
    x[tokens // 2] = 0  # a sample without an active unit
    x = plain.layouts(x)[layout]
    plain.assert_product(lowbit.product(x, w), x.double(), _w64(w))
    dy = plain.layouts(_spread((tokens, outputs), g, -4, 4).to(dtype))[layout]
    dx = lowbit.product_grad(dy, w)
    plain.assert_product(dx, dy.double(), _w64(w).t())


@pytest.mark.parametrize("layout", ["rows", "columns", "offset"])
@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("shape", LARGE)
def test_large_products(shape, dtype, layout) -> None:
    tokens, inputs, outputs = shape
    _say("large", shape, dtype, layout)
    g = _gen(*shape, 5)
    w = _weights(outputs, inputs, g)
    w64 = _w64(w)
    x = plain.layouts(_spread((tokens, inputs), g, -4, 4).to(dtype))[layout]
    plain.assert_product(lowbit.product(x, w), x.double(), w64)
    dy = plain.layouts(_spread((tokens, outputs), g, -4, 4).to(dtype))[layout]
    plain.assert_product(lowbit.product_grad(dy, w), dy.double(), w64.t().contiguous())
    for axis in (0, 1):
        _, kept = lowbit.activate(x, "relu", axis=axis)
        x8 = plain.values8(kept.codes, kept.scales, (tokens, inputs)[axis])
        x8 = x8.t().contiguous() if axis else x8
        plain.assert_product(lowbit.weight_grad(dy, kept), dy.double().t().contiguous(), x8)


@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("shape", [(2056, 2120, 6000), (1100, 5000, 4608), (264, 9600, 10000), (3001, 1300, 6500),
                                   (256, 131072, 768)])
def test_large_products_of_two_in_4_bits(shape, dtype) -> None:
    tokens, inputs, outputs = shape
    _say("large4", shape, dtype)
    g = _gen(*shape, 6)
    w, x = _weights(outputs, inputs, g), lowbit.quantise4(_spread((tokens, inputs), g, -4, 4))
    got = lowbit.product(x, w, dtype=dtype)
    plain.assert_product(got, plain.values4(x.codes, x.scales, inputs), _w64(w))


@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_product_of_two_in_4_bits(shape, dtype) -> None:
    tokens, inputs, outputs = shape
    _say("product4", shape, dtype)
    g = _gen(*shape, 1)
    w = _weights(outputs, inputs, g)
    x = lowbit.quantise4(_spread((tokens, inputs), g, -4, 4))
    x64 = plain.values4(x.codes, x.scales, inputs)
    plain.assert_product(lowbit.product(x, w, dtype=dtype), x64, _w64(w))
    if dtype == torch.float32:
        assert lowbit.product(x, w).dtype == torch.float32


@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_weight_grad(shape, dtype, layout, axis) -> None:
    tokens, inputs, outputs = shape
    _say("weight_grad", shape, dtype, layout, axis)
    g = _gen(*shape, 2)
    _, kept = lowbit.activate(_spread((tokens, inputs), g, -4, 4), "relu", axis=axis)
    x = plain.values8(kept.codes, kept.scales, (tokens, inputs)[axis])
    x = x if axis else x.t()
    dy = plain.layouts(_spread((tokens, outputs), g, -4, 4).to(dtype))[layout]
    dw = lowbit.weight_grad(dy, kept)
    assert dw.dtype == torch.float32
    plain.assert_product(dw, dy.double().t(), x.t())


@pytest.mark.parametrize("shape", [(70, 300, 200), (520, 640, 770), (1, 512, 130)])
def test_gradients_are_the_products_adjoints(shape) -> None:
    """The product is linear in its input and in the weights: <g, product(d)> = <product_grad(g), d>, and
    <g, x dw^T> = <weight_grad(g), dw>, the difference of the product along d and dw."""
    tokens, inputs, outputs = shape
    g = _gen(*shape, 3)
    w = _weights(outputs, inputs, g)
    x, dy = _randn((tokens, inputs), g), _randn((tokens, outputs), g)
    y, dx = lowbit.product(x, w), lowbit.product_grad(dy, w)
    size = float((dy.double().abs() * (x.double().abs() @ _w64(w).abs().t())).sum())
    bound = (plain.sum_bound(inputs) + plain.sum_bound(outputs)) * size
    assert abs(float((dy.double() * y.double()).sum() - (dx.double() * x.double()).sum())) <= bound
    _, kept = lowbit.activate(x, "relu")
    q, dw = kept.values(torch.float32), lowbit.weight_grad(dy, kept)
    y = lowbit.product(q, w)
    size = float((dy.double().abs() * (q.double().abs() @ _w64(w).abs().t())).sum())
    bound = (plain.sum_bound(inputs) + plain.sum_bound(tokens)) * size
    assert abs(float((dy.double() * y.double()).sum() - (dw.double() * _w64(w)).sum())) <= bound


@pytest.mark.parametrize("tokens", [1, 5, 64, 300, 1024])
def test_infinities_and_nan_stay_in_their_places(tokens) -> None:
    g = _gen(tokens, 4)
    inputs, outputs = 200, 300
    wf = _randn((outputs, inputs), g)
    wf[7, 40] = torch.nan  # its block of 32 becomes NaN
    w = lowbit.quantise4(wf)
    w64 = _w64(w)
    assert bool(torch.isnan(w64[7, 32:64]).all()) and int(torch.isnan(w64).sum()) == 32
    for dtype in plain.DTYPES:
        x = _randn((tokens, inputs), g).to(dtype)
        x[0, 3] = torch.inf
        x[-1, 9] = -torch.inf if tokens > 1 else torch.inf
        if tokens > 2:
            x[2, 5] = torch.nan
            x[3, 11] = torch.finfo(dtype).max
        y = lowbit.product(x, w)
        want = x.double() @ w64.t()
        assert torch.equal(torch.isnan(y), torch.isnan(want))
        inf = torch.isinf(want)
        assert torch.equal(y.double()[inf], want[inf])
        y4 = lowbit.product(lowbit.quantise4(x), w, dtype=dtype)
        q = plain.quantise4(x)
        assert torch.equal(torch.isnan(y4), torch.isnan(plain.values4(*q, inputs) @ w64.t()))
        dy = _randn((tokens, outputs), g).to(dtype)
        dy[0, 3] = torch.inf
        dx = lowbit.product_grad(dy, w)
        assert torch.equal(torch.isnan(dx), torch.isnan(dy.double() @ w64))
        h = _randn((tokens, inputs), g)
        h[0, 8] = torch.nan
        for axis in (0, 1):
            _, kept = lowbit.activate(h, "relu", axis=axis)
            x8 = plain.values8(kept.codes, kept.scales, h.shape[axis])
            x8 = x8 if axis else x8.t()
            dw = lowbit.weight_grad(dy, kept)
            assert torch.equal(torch.isnan(dw), torch.isnan(dy.double().t() @ x8))


def test_the_whole_range_of_scales() -> None:
    """Weights from the least scale to the largest, times inputs that bring them back."""
    g = _gen(9)
    e = torch.linspace(-120, 120, 64, device=DEV).round()[:, None]
    for dtype in (torch.float32, torch.bfloat16):
        w = lowbit.quantise4(_randn((64, 96), g) * torch.exp2(e))
        x = (_randn((40, 96), g)).to(dtype)
        plain.assert_product(lowbit.product(x, w), x.double(), _w64(w))
        x4 = lowbit.quantise4(x)
        plain.assert_product(lowbit.product(x4, w, dtype=dtype), plain.values4(x4.codes, x4.scales, 96), _w64(w))


def test_nothing_to_do() -> None:
    for dtype in plain.DTYPES:
        x = torch.zeros((0, 70), dtype=dtype, device=DEV)
        w = lowbit.quantise4(torch.zeros((9, 70), device=DEV))
        assert lowbit.quantise4(x).values().shape == (0, 70)
        assert lowbit.product(x, w).shape == (0, 9)
        assert lowbit.product(lowbit.quantise4(x), w).shape == (0, 9)
        assert lowbit.product_grad(x[:, :9], w).shape == (0, 70)
        for axis in (0, 1):
            y, kept = lowbit.activate(x, "silu", axis=axis)
            assert y.shape == (0, 70) and kept.values().shape == (0, 70)
            assert lowbit.activate_grad(y, kept, "silu").shape == (0, 70)
            dw = lowbit.weight_grad(x[:, :9], kept)  # a sum over no tokens
            assert dw.shape == (9, 70) and not dw.any()
        none = lowbit.quantise4(torch.zeros((9, 0), device=DEV))
        x = torch.zeros((5, 0), dtype=dtype, device=DEV)
        assert none.values().shape == (9, 0)
        y = lowbit.product(x, none)
        assert y.shape == (5, 9) and not y.any()
        y = lowbit.product(lowbit.quantise4(x), none)
        assert y.shape == (5, 9) and not y.any()
        assert lowbit.product_grad(torch.ones((5, 9), dtype=dtype, device=DEV), none).shape == (5, 0)
        empty = lowbit.quantise4(torch.zeros((0, 70), device=DEV))
        dx = lowbit.product_grad(torch.ones((5, 0), dtype=dtype, device=DEV), empty)
        assert dx.shape == (5, 70) and not dx.any()


def test_repeated_and_spread_tensors() -> None:
    """A broadcast batch (stride 0), and the same bits from every call."""
    g = _gen(11)
    w = _weights(130, 260, g)
    row = _randn((1, 260), g)
    x = row.expand(70, 260)
    y = lowbit.product(x, w)
    assert torch.equal(y, lowbit.product(x.contiguous(), w))
    assert torch.equal(lowbit.quantise4(x).codes, lowbit.quantise4(x.contiguous()).codes)
    for axis in (0, 1):
        a, kept = lowbit.activate(x, "tanh", axis=axis)
        b, again = lowbit.activate(x.contiguous(), "tanh", axis=axis)
        assert torch.equal(a, b) and torch.equal(kept.codes, again.codes)
        dy = _randn((70, 1), g).expand(70, 260)
        assert torch.equal(lowbit.activate_grad(dy, kept, "tanh"), lowbit.activate_grad(dy.contiguous(), kept, "tanh"))
        assert torch.equal(lowbit.weight_grad(dy, kept), lowbit.weight_grad(dy.contiguous(), kept))


def _train_step(w, x, dy, axis):
    h = lowbit.product(x, w)
    y, kept = lowbit.activate(h, "silu", axis=axis)
    dh = lowbit.activate_grad(dy, kept, "silu")
    low = lowbit.product(lowbit.quantise4(y), lowbit.quantise4(h), dtype=torch.bfloat16)
    return h, y, kept.codes, dh, lowbit.product_grad(dh, w), lowbit.weight_grad(dh, kept), low


@pytest.mark.parametrize("tokens", [1, 70, 520])
def test_on_another_stream_and_in_a_graph(tokens) -> None:
    g = _gen(tokens, 12)
    w = _weights(512, 300, g)
    x, dy = _randn((tokens, 300), g).bfloat16(), _randn((tokens, 512), g).bfloat16()
    want = [t.clone() for t in _train_step(w, x, dy, 1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _train_step(w, x, dy, 1)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _train_step(w, x, dy, 1)
    for k in range(4):
        x.copy_(_randn((tokens, 300), g))
        want = [t.clone() for t in _train_step(w, x, dy, 1)]  # eager work between the replays
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b), k


def test_offsets_past_32_bits() -> None:
    """More than 2^31 values: the last lines of a long batch equal those of a short one."""
    lines, n = 70_000, 32_768
    x = torch.zeros((lines, n), dtype=torch.bfloat16, device=DEV)
    tail = (_randn((80, n), _gen(13)) * 2).bfloat16()
    x[-80:] = tail
    m = lowbit.quantise4(x)
    assert torch.equal(m.codes[-80:], lowbit.quantise4(tail).codes)
    assert torch.equal(m.values(torch.bfloat16)[-80:], lowbit.quantise4(tail).values(torch.bfloat16))
    w = lowbit.quantise4(_randn((40, n), _gen(14)))
    y = lowbit.product(x, w)
    plain.assert_product(y[-80:], tail.double(), _w64(w))
    assert not y[:1000].any()
    y, kept = lowbit.activate(x, "relu")
    assert torch.equal(y[-80:], tail.clamp_min(0))
    dh = lowbit.activate_grad(x, kept, "relu")
    assert torch.equal(dh[-80:], lowbit.activate_grad(tail, lowbit.activate(tail, "relu")[1], "relu"))
    del m, y, dh
    g = torch.zeros((lines, 40), dtype=torch.bfloat16, device=DEV)
    g[-80:] = _randn((80, 40), _gen(15))
    dw = lowbit.weight_grad(g, kept)
    q = plain.values8(kept.codes[-80:], kept.scales[-80:], n)
    size = g[-80:].double().t().abs() @ q.abs()
    want = g[-80:].double().t() @ q
    # (the other lines add zeros)
    assert bool(((dw.double() - want).abs() <= size * plain.sum_bound(lines)).all())


def test_large_products_with_offsets_past_32_bits() -> None:
    """The same through the large products: 70,000 lines of 32,768 against 260 and 256 units."""
    lines, n = 70_000, 32_768
    x = torch.zeros((lines, n), dtype=torch.bfloat16, device=DEV)
    tail = (_randn((80, n), _gen(16)) * 2).bfloat16()
    x[-80:] = tail
    w = lowbit.quantise4(_randn((260, n), _gen(17)))
    y = lowbit.product(x, w)
    plain.assert_product(y[-80:], tail.double(), _w64(w))
    assert not y[:1000].any()
    y = lowbit.product(lowbit.quantise4(x), w)
    q = plain.quantise4(tail)
    plain.assert_product(y[-80:], plain.values4(*q, n), _w64(w))
    assert not y[:1000].any()
    kept = lowbit.quantise8(x)
    g = torch.zeros((lines, 256), dtype=torch.bfloat16, device=DEV)
    g[-80:] = _randn((80, 256), _gen(18))
    dw = lowbit.weight_grad(g, kept)
    q = plain.values8(kept.codes[-80:], kept.scales[-80:], n)
    size = g[-80:].double().t().contiguous().abs() @ q.abs()
    want = g[-80:].double().t().contiguous() @ q
    assert bool(((dw.double() - want).abs() <= size * plain.sum_bound(lines)).all())
    wide = lowbit.quantise4(_randn((lines, 256), _gen(19)))
    dx = torch.zeros((300, lines), dtype=torch.bfloat16, device=DEV)
    dx[:, -80:] = _randn((300, 80), _gen(20))
    got = lowbit.product_grad(dx, wide)
    w64 = plain.values4(wide.codes[-80:], wide.scales[-80:], 256)
    want, size = dx[:, -80:].double() @ w64, dx[:, -80:].double().abs() @ w64.abs()
    assert bool(((got.double() - want).abs() <= size * plain.sum_bound(lines) + want.abs() * 2.0**-8).all())


def test_the_example_learns_and_its_answers_are_the_arenas() -> None:
    import pathlib
    import sys

    sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "examples"))
    import lowbit_mlp

    first, last, worst = lowbit_mlp.main(steps=120, samples=2)
    assert last < first / 2
    # tanh of sums of at most 256 terms through 3 levels: each sum is off by its bound times the terms' sizes (below
    # 64 for weights of this size), each tanh by 2 steps
    assert worst <= 3 * (64 * plain.sum_bound(256) + 256 * 64 * plain.U)
