"""proj_adapters on the kernel of many rows (128 or 256 x 256 tiles) against the formula in 64 bits.

Up to a few thousand rows a call takes whichever of the three tile shapes needs the least time by
its rounds over the units, so the sizes here are checked against that rule: ``_tile`` is the rule,
and every test says which shape it means to run. The tolerance is that of the other sizes (one bf16
ulp); exp and tanh add 2^-18 of a value, which is far below it.
"""

import math

import numpy as np
import pytest
import torch

from wkvm_amd import adapter_plan, proj_adapters

from .test_gpu_adapters import _assert_close, _bank, _exact, _rand

pytestmark = pytest.mark.gpu

RANKS = [16, 40, 1, 0, 100, 17, 128]
ROWS = {128: 5000, 256: 8200}  # with 1,000 columns or so


def _tile(m, widths, adapters):
    """Rows of the tile that the library takes for products of these widths (k a multiple of 64): the
    least microseconds of 128 x 64, 128 x 256 and 256 x 256 tiles by their rounds over the units."""
    units = torch.cuda.get_device_properties(0).multi_processor_count
    runs = min(m, adapters + 1)
    positions = (m + 31 * runs + 31) // 32 * 32
    best = None
    for bm, bn, us, rows in ((128, 64, 16.5, 0), (128, 256, 47.0, 128), (256, 256, 79.0, 256)):
        tiles = sum(-(-positions // bm) * -(-n // bn) for n in widths)
        time = us * -(-tiles // units)
        if best is None or time < best[0]:
            best = (time, rows)
    return best[1]


def _ids(kind, m, count, seed):
    rng = np.random.default_rng(seed)
    if kind == "none":
        return np.full(m, -1)
    if kind == "one":
        return np.full(m, 4)
    ids = rng.integers(-1, count, m)
    return np.sort(ids) if kind == "runs" else ids


@pytest.mark.parametrize("act,with_bias", [(None, False), ("tanh", True), ("sigmoid", True),
                                           ("tanh", False), (None, True)])
@pytest.mark.parametrize("k,n", [(64, 1000), (128, 1001), (192, 1024)])
@pytest.mark.parametrize("tile", [128, 256])
def test_widths_bias_and_activation(dev, tile, k, n, act, with_bias):
    gen = torch.Generator().manual_seed(k + n)
    m = ROWS[tile]
    assert _tile(m, [n], len(RANKS)) == tile
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bias = _rand((n,), gen, dev) if with_bias else None
    bank, pairs = _bank(gen, dev, RANKS, k, n)
    ids = _ids("any", m, len(RANKS), n)
    (y,) = proj_adapters([(x, w, bias, act, bank)], adapter_plan(ids, len(RANKS), dev))
    _assert_close(y, _exact(x, w, bias, act, pairs, ids))


@pytest.mark.parametrize("kind", ["none", "one", "runs"])
@pytest.mark.parametrize("tile", [128, 256])
def test_mixes(dev, tile, kind):
    gen = torch.Generator().manual_seed(5)
    m, k, n = ROWS[tile] + 17, 64, 990
    assert _tile(m, [n], len(RANKS)) == tile
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bank, pairs = _bank(gen, dev, RANKS, k, n)
    ids = _ids(kind, m, len(RANKS), 3)
    (y,) = proj_adapters([(x, w, None, None, bank)], adapter_plan(ids, len(RANKS), dev))
    _assert_close(y, _exact(x, w, None, None, pairs, ids))


@pytest.mark.parametrize("rank", [15, 33, 256])
@pytest.mark.parametrize("tile", [128, 256])
def test_ranks(dev, tile, rank):
    gen = torch.Generator().manual_seed(rank)
    m, k, n = ROWS[tile], 64, 1000
    assert _tile(m, [n], 3) == tile
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bank, pairs = _bank(gen, dev, [rank, max(1, rank // 3), rank], k, n)
    ids = _ids("any", m, 3, rank)
    (y,) = proj_adapters([(x, w, None, None, bank)], adapter_plan(ids, 3, dev))
    _assert_close(y, _exact(x, w, None, None, pairs, ids))


def test_long_k(dev):
    gen = torch.Generator().manual_seed(6)
    m, k, n = 5000, 2048, 1000
    assert _tile(m, [n], 4) == 128
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bank, pairs = _bank(gen, dev, [32, 16, 64, 8], k, n)
    ids = _ids("runs", m, 4, 8)
    (y,) = proj_adapters([(x, w, None, None, bank)], adapter_plan(ids, 4, dev))
    _assert_close(y, _exact(x, w, None, None, pairs, ids))


@pytest.mark.parametrize("tile,m", [(128, 3000), (256, 4700)])
def test_a_group_of_products(dev, tile, m):
    """Other widths, activations and banks in one call; one product has none."""
    gen = torch.Generator().manual_seed(m)
    widths, count = [1000, 40, 777], len(RANKS)
    assert _tile(m, widths, count) == tile
    ids = _ids("any", m, count, 9)
    prods, exact = [], []
    for i, (n, k, act) in enumerate(zip(widths, (128, 320, 64), ("sigmoid", None, "tanh"))):
        x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
        bias = _rand((n,), gen, dev) if i != 1 else None
        bank, pairs = (None, None) if i == 1 else _bank(gen, dev, RANKS, k, n)
        prods.append((x, w, bias, act, bank))
        exact.append(_exact(x, w, bias, act, pairs, ids))
    for y, e in zip(proj_adapters(prods, adapter_plan(ids, count, dev)), exact):
        _assert_close(y, e)


@pytest.mark.parametrize("n", [1000, 1003])
@pytest.mark.parametrize("shift", [0, 3, 8])
@pytest.mark.parametrize("tile", [128, 256])
def test_strided_inputs_and_outputs(dev, tile, n, shift):
    """Rows of x inside wider ones; rows of y that start where 16 bytes do, or between."""
    gen = torch.Generator().manual_seed(13 + shift)
    m, k = ROWS[tile], 64
    assert _tile(m, [n], 2) == tile
    x = _rand((m, 3 * k + 8), gen, dev)[:, k:2 * k]
    w = _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bank, pairs = _bank(gen, dev, [16, 8], k, n)
    ids = np.arange(m) % 3 - 1
    out = torch.zeros((m, n + 24 + (shift & 1)), dtype=torch.bfloat16, device=dev)
    view = out[:, shift:shift + n]
    proj_adapters([(x, w, None, None, bank)], adapter_plan(ids, 2, dev), outs=[view])
    _assert_close(view, _exact(x, w, None, None, pairs, ids))
    assert not out[:, :shift].any() and not out[:, shift + n:].any()


@pytest.mark.parametrize("tile", [128, 256])
def test_a_broken_adapter_stays_with_its_rows(dev, tile):
    """Infinities and NaN in one adapter, or in one row, reach no other row."""
    gen = torch.Generator().manual_seed(17)
    m, k, n = ROWS[tile], 64, 1000
    assert _tile(m, [n], 3) == tile
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bank, pairs = _bank(gen, dev, [8, 8, 8], k, n)
    ids = np.arange(m) % 4 - 1
    plan = adapter_plan(ids, 3, dev)
    (want,) = proj_adapters([(x, w, None, None, bank)], plan)
    a, b, s = pairs[1]
    bad = b.clone()
    bad[::5] = math.nan
    bad[1::5] = math.inf
    bank.load(1, a, bad, s)
    (got,) = proj_adapters([(x, w, None, None, bank)], plan)
    others = np.flatnonzero(ids != 1)
    assert torch.equal(got[others], want[others])
    assert not got[np.flatnonzero(ids == 1)][:, ::5].isfinite().any()
    bank.load(1, a, b, s)
    bad = x.clone()
    bad[5] = math.inf
    (got,) = proj_adapters([(bad, w, None, None, bank)], plan)
    rest = [i for i in range(m) if i != 5]
    assert torch.equal(got[rest], want[rest])


@pytest.mark.parametrize("tile", [128, 256])
def test_under_graph_capture(dev, tile):
    gen = torch.Generator().manual_seed(29)
    m, k, n = ROWS[tile], 128, 1000
    assert _tile(m, [n], 3) == tile
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bank, _ = _bank(gen, dev, [16, 8, 32], k, n)
    plan = adapter_plan(_ids("any", m, 3, 2), 3, dev)
    proj_adapters([(x, w, None, "sigmoid", bank)], plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (out,) = proj_adapters([(x, w, None, "sigmoid", bank)], plan)
    for _ in range(3):
        x.copy_(_rand((m, k), gen, dev))
        graph.replay()
        torch.cuda.synchronize()
        (eager,) = proj_adapters([(x, w, None, "sigmoid", bank)], plan)
        assert torch.equal(out, eager)
