"""proj_w4 and W4Weight against the formula in float64.

The kernels sum x (1 + c / 16) and x over a group and combine 16 s (first - (1 + z / 16) second), so an
output's fp32 error is at most 2^-24 per addition of the terms s |x| (16 + c) and s |x| (16 + z): up to
128 in a group, one per group, 16 for joining the parts. Then bias (an addition), activation (of slope at
most 1, itself within 2^-20) and one rounding to bf16, half a step or 2^-8 of the value.
"""

import math

import numpy as np
import pytest
import torch

from wkvm_amd import W4Weight, proj_w4

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _weight(gen, n, k, group, zero, dtype=torch.float16):
    groups = -(-k // group)
    codes = torch.randint(0, 16, (n, k), generator=gen, dtype=torch.uint8)
    scale = ((torch.rand(n, groups, generator=gen) + 0.25) / math.sqrt(k)).to(dtype)
    scale[torch.rand(n, groups, generator=gen) < 0.05] *= -1
    zeros = torch.randint(0, 16, (n, groups), generator=gen, dtype=torch.uint8) if zero else None
    return codes, scale, zeros


def _values(codes, scale, zeros, group):
    k = codes.shape[1]
    s = scale.double().repeat_interleave(group, 1)[:, :k]
    z = torch.full_like(s, 8.) if zeros is None else zeros.double().repeat_interleave(group, 1)[:, :k]
    return s * (codes.double() - z), s.abs() * (32 + codes.double() + z)


def _act(y, act):
    return torch.tanh(y) if act == "tanh" else torch.sigmoid(y) if act == "sigmoid" else y


def _check(got, x, parts, group, bias=None, act=None):
    w, mag = _values(*parts, group)
    x = x.double()
    y = x @ w.T
    err = 2.0 ** -24 * (128 + w.shape[1] // group + 17) * (x.abs() @ mag.T)
    if bias is not None:
        y = y + bias.double()
        err = err + 2.0 ** -24 * y.abs()
    if act:
        err = err + 2.0 ** -20
    y = _act(y, act)
    got = got.double().cpu()
    bound = err + 2.0 ** -8 * (y.abs() + err) + 1e-37
    worst = ((got - y).abs() / bound).max().item()
    assert worst <= 1.0, f"{worst:.2f} bounds"


def _x(gen, m, k):
    return torch.randn(m, k, generator=gen).to(BF16)


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 63, 64, 65, 130, 300, 513, 1100])
@pytest.mark.parametrize("n,k,group", [(16, 32, 32), (33, 96, 64), (100, 160, 128), (48, 1024, 32),
                                       (65, 2080, 64), (257, 512, 128), (1, 4096, 128)])
def test_products(dev, m, n, k, group):
    gen = torch.Generator().manual_seed(m + n)
    parts = _weight(gen, n, k, group, zero=n % 2 == 0)
    x = _x(gen, m, k)
    weight = W4Weight.from_codes(*(None if t is None else t.to(dev) for t in parts), group=group)
    y, = proj_w4([(x.to(dev), weight)])
    _check(y, x, parts, group)


@pytest.mark.parametrize("m", [1, 9, 40, 200])
def test_grouped_products(dev, m):
    """Several products of one launch, of different widths, lengths and groups, with bias and
    activations; outputs into views of a wider tensor; inputs with a row stride."""
    gen = torch.Generator().manual_seed(m)
    shapes = [(40, 256, 32, None, False, True), (200, 768, 128, "tanh", True, False),
              (77, 96, 64, "sigmoid", True, True), (16, 2048, 128, None, True, True)]
    products, checks, outs = [], [], []
    wide = torch.full((m, 400), 3.0, dtype=BF16, device=dev)
    for i, (n, k, group, act, bias, zero) in enumerate(shapes):
        parts = _weight(gen, n, k, group, zero, BF16 if i % 2 else torch.float16)
        x = _x(gen, m, k + 16)
        b = torch.randn(n, generator=gen).to(BF16) if bias else None
        weight = W4Weight.from_codes(*(None if t is None else t.to(dev) for t in parts),
                                     group=group)
        products.append((x.to(dev)[:, 8:8 + k], weight, None if b is None else b.to(dev), act))
        checks.append((x[:, 8:8 + k], parts, group, b, act))
        outs.append(wide[:, 40:240] if i == 1 else None)
    ys = proj_w4(products, outs)
    for y, check in zip(ys, checks):
        _check(y, *check)
    assert ys[1].data_ptr() == wide[:, 40:].data_ptr()
    assert (wide[:, :40] == 3).all() and (wide[:, 240:] == 3).all()


def test_eight_products_and_one_row_of_each_is_the_same_alone(dev):
    gen = torch.Generator().manual_seed(5)
    products = []
    for i in range(8):
        parts = _weight(gen, 64 + i, 256, 64, True)
        products.append((_x(gen, 5, 256).to(dev),
                         W4Weight.from_codes(*(t.to(dev) for t in parts), group=64)))
    together = proj_w4(products)
    for p, y in zip(products, together):
        assert torch.equal(proj_w4([p])[0], y)


@pytest.mark.parametrize("m", [3, 100, 700])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_an_infinite_or_nan_input_reaches_its_own_row(dev, m, bad):
    gen = torch.Generator().manual_seed(6)
    parts = _weight(gen, 50, 256, 64, True)
    x = _x(gen, m, 256)
    x[m // 2, 37] = bad
    weight = W4Weight.from_codes(*(t.to(dev) for t in parts), group=64)
    y = proj_w4([(x.to(dev), weight)])[0].cpu()
    want = x[m // 2].double() @ _values(*parts, 64)[0].T
    got = y[m // 2].double()
    assert (got.isnan() == want.isnan()).all()
    inf = want.isinf()
    assert (got[inf] == want[inf]).all()
    if not math.isnan(bad):
        assert inf.any()
    rest = [i for i in range(m) if i != m // 2]
    _check(y[rest], x[rest], parts, 64)


@pytest.mark.parametrize("dtype", [torch.float16, BF16])
@pytest.mark.parametrize("n,k,group", [(5, 32, 128), (16, 64, 32), (33, 416, 128), (20, 96, 64)])
def test_dequantize_gives_the_values(dev, n, k, group, dtype):
    gen = torch.Generator().manual_seed(n)
    for zero in (False, True):
        parts = _weight(gen, n, k, group, zero, dtype)
        weight = W4Weight.from_codes(*(None if t is None else t.to(dev) for t in parts),
                                     group=group)
        assert weight.shape == (n, k)
        assert torch.equal(weight.dequantize().double().cpu(), _values(*parts, group)[0])


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("n,k,group", [(7, 64, 32), (40, 288, 128), (16, 256, 64)])
def test_quantize_rounds_to_the_range(dev, n, k, group, symmetric):
    """Every value within half a step of its group (a zero point that is rounded may cut the range's
    ends by another half); zeros stay zero; groups of zeros, of one sign and of one value."""
    gen = torch.Generator().manual_seed(n)
    w = torch.randn(n, k, generator=gen).to(BF16)
    w[0, :group] = 0
    w[1, :group] = w[1, :group].abs()
    w[2, :group] = -2.5
    weight = W4Weight.quantize(w.to(dev), group=group, symmetric=symmetric)
    got = weight.dequantize().cpu()
    for g in range(-(-k // group)):
        part, back = w.float()[:, g * group:(g + 1) * group], got[:, g * group:(g + 1) * group]
        lo, hi = part.amin(1).clamp(max=0), part.amax(1).clamp(min=0)
        step = torch.maximum(-lo, hi) / 7 if symmetric else (hi - lo) / 15
        assert ((back - part).abs() <= step[:, None] * (0.5 if symmetric else 1.0) * 1.0001
                + 1e-30).all()
        assert (back[part == 0] == 0).all()
    assert (got[0, :group] == 0).all()
    # a product of the rounded weight is that of its values
    x = _x(gen, 4, k)
    y = proj_w4([(x.to(dev), weight)])[0].double().cpu()
    want = x.double() @ got.double().T
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -24 * (160 + k // group) * 48 * (
        x.double().abs().sum(1, keepdim=True) * got.double().abs().max())
    assert ((y - want).abs() <= bound).all()


def test_quantize_of_a_strided_weight(dev):
    gen = torch.Generator().manual_seed(1)
    w = torch.randn(24, 160, generator=gen).to(BF16).to(dev)
    a = W4Weight.quantize(w[:, 32:96], group=32)
    b = W4Weight.quantize(w[:, 32:96].contiguous(), group=32)
    c = W4Weight.quantize(w[:, 32:96].t().contiguous().t(), group=32)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    assert torch.equal(a.codes, c.codes) and torch.equal(a.scales, c.scales)


@pytest.mark.parametrize("m", [2, 80, 600])
def test_graph_replays_and_repeats(dev, m):
    gen = torch.Generator().manual_seed(m)
    parts = _weight(gen, 300, 1024, 128, True)
    weight = W4Weight.from_codes(*(t.to(dev) for t in parts), group=128)
    x = _x(gen, m, 1024).to(dev)
    want = proj_w4([(x, weight)])[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, = proj_w4([(x, weight)])
    for seed in range(3):
        x.copy_(_x(torch.Generator().manual_seed(seed), m, 1024))
        graph.replay()
        got = y.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, proj_w4([(x, weight)])[0])
    x.copy_(_x(torch.Generator().manual_seed(m), m, 1024))
    side = torch.cuda.Stream(dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        other = proj_w4([(x, weight)])[0]
    side.synchronize()
    assert torch.equal(other, proj_w4([(x, weight)])[0]) and want.shape == other.shape


def test_rows_of_any_count(dev):
    """No rows; and rows that share no tile with others give the same whatever the batch."""
    gen = torch.Generator().manual_seed(9)
    parts = _weight(gen, 40, 128, 64, True)
    weight = W4Weight.from_codes(*(t.to(dev) for t in parts), group=64)
    assert proj_w4([(torch.empty(0, 128, dtype=BF16, device=dev), weight)])[0].shape == (0, 40)
    x = _x(gen, 200, 128).to(dev)
    y = proj_w4([(x, weight)])[0]
    _check(y, x.cpu(), parts, 64)


def test_refusals(dev):
    gen = torch.Generator().manual_seed(2)
    codes, scale, zeros = (t.to(dev) for t in _weight(gen, 8, 64, 32, True))
    weight = W4Weight.from_codes(codes, scale, zeros, group=32)
    x = _x(gen, 3, 64).to(dev)

    def bad(match, fn):
        with pytest.raises(ValueError, match=match):
            fn()

    bad("0 .. 15", lambda: W4Weight.from_codes(codes + 16, scale, zeros, group=32))
    bad("0 .. 15", lambda: W4Weight.from_codes(codes, scale, zeros + 16, group=32))
    bad("finite", lambda: W4Weight.from_codes(codes, scale / 0, zeros, group=32))
    bad("scale must be", lambda: W4Weight.from_codes(codes, scale.float(), zeros, group=32))
    bad("scale must be", lambda: W4Weight.from_codes(codes, scale, zeros, group=64))
    bad("zero must be", lambda: W4Weight.from_codes(codes, scale, zeros[:, :1], group=32))
    bad("uint8", lambda: W4Weight.from_codes(codes.int(), scale, zeros, group=32))
    bad("group must", lambda: W4Weight.from_codes(codes, scale, zeros, group=16))
    bad("multiple of 32", lambda: W4Weight.from_codes(codes[:, :48], scale, zeros, group=32))
    bad("GPU tensor", lambda: W4Weight.from_codes(codes.cpu(), scale, zeros, group=32))
    bad("finite", lambda: W4Weight.quantize(torch.full((4, 32), math.nan, dtype=BF16, device=dev)))
    bad("bfloat16", lambda: W4Weight.quantize(torch.zeros(4, 32, device=dev)))
    bad("products per launch", lambda: proj_w4([]))
    bad("products per launch", lambda: proj_w4([(x, weight)] * 9))
    bad("W4Weight", lambda: proj_w4([(x, x)]))
    bad("bfloat16", lambda: proj_w4([(x.float(), weight)]))
    bad("x must be", lambda: proj_w4([(x[:, :32], weight)]))
    bad("same row count", lambda: proj_w4([(x, weight), (x[:2], weight)]))
    bad("act must", lambda: proj_w4([(x, weight, None, "relu")]))
    bad("bias", lambda: proj_w4([(x, weight, torch.zeros(7, dtype=BF16, device=dev))]))
    bad("out must", lambda: proj_w4([(x, weight)], [torch.empty(3, 9, dtype=BF16, device=dev)]))
    bad("GPU tensor", lambda: proj_w4([(x.cpu(), weight)]))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(2100, 2111, 160), (128, 16650, 288), (96, 16650, 288),
                                   (1700, 3100, 512), (130, 16650, 128), (70, 16650, 64)])
def test_many_tiles(dev, m, n, k, group):
    """Enough output tiles for every tile shape, k that ends inside a block of 128 and inside a group."""
    gen = torch.Generator().manual_seed(m)
    parts = _weight(gen, n, k, group, True)
    x = _x(gen, m, k)
    weight = W4Weight.from_codes(*(t.to(dev) for t in parts), group=group)
    b = torch.randn(n, generator=gen).to(BF16)
    y, = proj_w4([(x.to(dev), weight, b.to(dev), "tanh")])
    _check(y, x, parts, group, b, "tanh")


@pytest.mark.parametrize("m", [5, 40, 200])
def test_a_batch_of_infinities_or_nans(dev, m):
    gen = torch.Generator().manual_seed(m)
    parts = _weight(gen, 300, 2048, 128, True)
    weight = W4Weight.from_codes(*(t.to(dev) for t in parts), group=128)
    x = torch.full((m, 2048), math.nan, dtype=BF16)
    x[1::2] = math.inf
    y, = proj_w4([(x.to(dev), weight)])
    assert y.isnan().all()  # (infinities of both signs among an output's terms)
    x = _x(gen, m, 2048)
    x[:, 2047] = math.inf
    y, = proj_w4([(x.to(dev), weight)])
    last = _values(*parts, 128)[0][:, 2047].to(dev)
    assert (y.isnan() == (last == 0)).all()
    assert (y[:, last != 0] == math.inf * last[last != 0].sign()).all()


def test_codes_at_any_address(dev):
    gen = torch.Generator().manual_seed(4)
    parts = _weight(gen, 33, 160, 64, True)
    ref = W4Weight.from_codes(*(t.to(dev) for t in parts), group=64)
    for shift in (1, 4, 7):
        room = torch.zeros(33 * 160 + shift, dtype=torch.uint8, device=dev)
        room[shift:] = parts[0].to(dev).view(-1)
        got = W4Weight.from_codes(room[shift:].view(33, 160), *(t.to(dev) for t in parts[1:]),
                                  group=64)
        assert torch.equal(got.codes, ref.codes) and torch.equal(got.scales, ref.scales)


def test_quantize_where_the_range_is_not_finite(dev):
    """lo and hi of opposite signs and 2e38: their difference is past the largest fp32."""
    gen = torch.Generator().manual_seed(6)
    w = ((torch.rand(20, 128, generator=gen) * 2 - 1) * 2e38).to(BF16)
    w[:, 0], w[:, 1] = 2e38, -2e38
    got = W4Weight.quantize(w.to(dev), 64).dequantize().cpu().double()
    s = (w.double().view(20, 2, 64).amax(2) - w.double().view(20, 2, 64).amin(2).clamp(max=0)) / 15
    err = (got - w.double()).abs().view(20, 2, 64).amax(2)
    # the code's rounding s / 2, the zero point's s / 2 at the ends, the scale's last bits (15 steps of
    # 2^-19)
    assert (err <= s * (1 + 15 * 2.0 ** -18)).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 16500, 4128), (3, 16500, 4224), (9, 16500, 128), (4, 100, 4160),
                                   (64, 16500, 160), (500, 130, 1056), (333, 2048, 96),
                                   (16, 16500, 1056), (13, 16500, 3008), (3, 300, 4160)])
def test_kernels_of_a_few_rows(dev, m, n, k, group):
    """One row to sixteen of many columns, short and long k, and many rows of a few columns."""
    gen = torch.Generator().manual_seed(m + k)
    parts = _weight(gen, n, k, group, m % 2 == 0)
    x = _x(gen, m, k + 8)[:, :k]
    weight = W4Weight.from_codes(*(None if t is None else t.to(dev) for t in parts), group=group)
    b = torch.randn(n, generator=gen).to(BF16)
    y, = proj_w4([(x.to(dev), weight, b.to(dev), "sigmoid" if m > 8 else None)])
    _check(y, x, parts, group, b, "sigmoid" if m > 8 else None)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(230, 4700, 96), (230, 4700, 160), (200, 5000, 416),
                                   (129, 6600, 1312)])
def test_tiles_in_two_parts(dev, m, n, k, group):
    """Output tiles whose waves take blocks of k in turn: one block, two, an odd number of them."""
    gen = torch.Generator().manual_seed(m + k)
    parts = _weight(gen, n, k, group, True)
    x = _x(gen, m, k)
    weight = W4Weight.from_codes(*(t.to(dev) for t in parts), group=group)
    y, = proj_w4([(x.to(dev), weight)])
    _check(y, x, parts, group)


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("m,n", [(230, 4700), (2100, 2111), (128, 16650), (96, 16650)])
def test_an_infinite_input_of_output_tiles(dev, m, n, bad):
    gen = torch.Generator().manual_seed(6)
    parts = _weight(gen, n, 160, 64, True)
    x = _x(gen, m, 160)
    x[m // 2, 37] = bad
    weight = W4Weight.from_codes(*(t.to(dev) for t in parts), group=64)
    y = proj_w4([(x.to(dev), weight)])[0].cpu()
    want = x[m // 2].double() @ _values(*parts, 64)[0].T
    got = y[m // 2].double()
    assert (got.isnan() == want.isnan()).all()
    inf = want.isinf()
    assert (got[inf] == want[inf]).all()
    rest = [i for i in range(m) if i != m // 2]
    _check(y[rest], x[rest], parts, 64)


@pytest.mark.parametrize("m,n", [(230, 4700), (700, 6000), (70, 16650)])
def test_graph_replays_of_output_tiles(dev, m, n):
    """The sums' workspace is the graph's own: replays between eager calls of other sizes, twice the
    same weight and the same x among the products."""
    gen = torch.Generator().manual_seed(m)
    parts = _weight(gen, n, 288, 64, True)
    weight = W4Weight.from_codes(*(t.to(dev) for t in parts), group=64)
    x, other = _x(gen, m, 288).to(dev), _x(gen, 2 * m, 288).to(dev)
    proj_w4([(x, weight)])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = proj_w4([(x, weight), (x, weight, None, "tanh")])
    for step in range(4):
        x.copy_(_x(gen, m, 288))
        graph.replay()
        proj_w4([(other, weight)])
        torch.cuda.synchronize()
        want = proj_w4([(x, weight), (x, weight, None, "tanh")])
        assert all(torch.equal(a, b) for a, b in zip(ys, want)), step
        _check(ys[0], x.cpu(), parts, 64)
