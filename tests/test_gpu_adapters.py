"""proj_adapters against the formula in 64 bits.

The kernel's sums are fp32, x A^T enters the second product with all of its 24 bits, and y
is rounded once to bf16 (half an ulp). An output is therefore within one bf16 ulp of the
exact value, where an output much smaller than its terms is measured by the ulp of 1/256 of
the outputs' scale: cancellation leaves the sums' absolute error, which random sums of
k <= 4096 terms keep below a third of that ulp (2^-24 sqrt(k) of the scale against 2^-16 of it).
"""

import math

import numpy as np
import pytest
import torch

from wkvm_amd import AdapterBank, adapter_plan, ops, proj_adapters

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda", 0)


def _rand(shape, gen, dev, std=1.0):
    return (torch.randn(shape, generator=gen) * std).to(torch.bfloat16).to(dev)


def _bank(gen, dev, ranks, k, n, max_rank=None):
    """A bank of adapters (rank 0: an empty place) and its pairs."""
    bank = AdapterBank(len(ranks), k, n, max_rank or max(max(ranks), 1), dev)
    pairs = []
    for i, r in enumerate(ranks):
        if r == 0:
            pairs.append(None)
            continue
        a = _rand((r, k), gen, dev, 1 / math.sqrt(k))
        b = _rand((n, r), gen, dev, 0.5 / math.sqrt(r))
        s = 1.0 + 0.25 * i
        bank.load(i, a, b, s)
        pairs.append((a, b, s))
    return bank, pairs


def _exact(x, w, bias, act, pairs, ids):
    x = x.double().cpu()
    y = x @ w.double().cpu().T
    for a, pair in enumerate(pairs or []):
        rows = np.flatnonzero(np.asarray(ids) == a)
        if pair is None or rows.size == 0:
            continue
        A, B, s = pair
        y[rows] += s * (x[rows] @ A.double().cpu().T) @ B.double().cpu().T
    if bias is not None:
        y = y + bias.double().cpu()
    return torch.tanh(y) if act == "tanh" else torch.sigmoid(y) if act == "sigmoid" else y


def _assert_close(got, exact):
    got = got.double().cpu()
    mag = exact.abs().clamp_min(exact.pow(2).mean().sqrt().item() / 256 + 1e-30)
    ulp = torch.exp2(torch.floor(torch.log2(mag)) - 7)
    worst = ((got - exact).abs() / ulp).max().item()
    assert worst <= 1.0, f"max error {worst:.3f} bf16 ulp"


def _ids(kind, m, count, rng):
    if kind == "none":
        return np.full(m, -1)
    if kind == "one":
        return np.zeros(m, int)
    if kind == "each":
        return np.arange(m) % count
    if kind == "runs":
        return np.sort(rng.integers(-1, count, m))
    return rng.integers(-1, count, m)  # any order, some without


@pytest.mark.parametrize("kind", ["none", "one", "each", "runs", "any"])
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 129, 300, 512, 513, 1111])
def test_rows_and_mixes(dev, m, kind):
    gen = torch.Generator().manual_seed(m)
    k, n, ranks = 256, 208, [16, 8, 1, 33, 5, 0, 64, 17, 16]
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bank, pairs = _bank(gen, dev, ranks, k, n)
    ids = _ids(kind, m, len(ranks), np.random.default_rng(m))
    (y,) = proj_adapters([(x, w, None, None, bank)], adapter_plan(ids.tolist(), len(ranks), dev))
    _assert_close(y, _exact(x, w, None, None, pairs, ids))


@pytest.mark.parametrize("k,n", [(32, 1), (64, 16), (96, 17), (768, 768), (1056, 65), (2048, 2048),
                                 (2080, 529), (4096, 300)])
@pytest.mark.parametrize("m", [1, 5, 16, 40, 200, 700])
def test_widths(dev, m, k, n):
    gen = torch.Generator().manual_seed(k + n)
    ranks = [16, 40, 3]
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bias = _rand((n,), gen, dev)
    bank, pairs = _bank(gen, dev, ranks, k, n)
    ids = np.random.default_rng(k).integers(-1, 3, m)
    (y,) = proj_adapters([(x, w, bias, "tanh", bank)], adapter_plan(ids, 3, dev))
    _assert_close(y, _exact(x, w, bias, "tanh", pairs, ids))


@pytest.mark.parametrize("rank", [1, 4, 15, 16, 31, 32, 64, 100, 128, 255, 256])
@pytest.mark.parametrize("m", [3, 48, 600])
def test_ranks(dev, m, rank):
    gen = torch.Generator().manual_seed(rank)
    k, n = 512, 320
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bank, pairs = _bank(gen, dev, [rank, max(1, rank // 3), rank], k, n)
    ids = np.random.default_rng(rank).integers(-1, 3, m)
    (y,) = proj_adapters([(x, w, None, None, bank)], adapter_plan(ids, 3, dev))
    _assert_close(y, _exact(x, w, None, None, pairs, ids))


@pytest.mark.parametrize("m", [1, 9, 64, 256, 1500])
def test_a_group_of_products(dev, m):
    """Different inputs, widths, activations and banks in one call; one product has none."""
    gen = torch.Generator().manual_seed(m)
    count = 6
    ids = np.random.default_rng(m).integers(-1, count, m)
    prods, exact = [], []
    for i, (k, n, act) in enumerate([(768, 768, None), (768, 96, "tanh"), (2048, 64, "sigmoid"),
                                     (128, 1024, None)]):
        x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
        bias = _rand((n,), gen, dev) if i % 2 else None
        bank, pairs = (None, None) if i == 2 else _bank(gen, dev, [16, 8, 32, 16, 0, 4], k, n, 48)
        prods.append((x, w, bias, act, bank))
        exact.append(_exact(x, w, bias, act, pairs, ids))
    for y, e in zip(proj_adapters(prods, adapter_plan(ids, count, dev)), exact):
        _assert_close(y, e)


def test_many_rows_and_adapters(dev):
    """A prefill's row count over the 1.5B width."""
    gen = torch.Generator().manual_seed(7)
    m, k, n = 4100, 2048, 2048
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bank, pairs = _bank(gen, dev, [16, 32, 8, 16], k, n)
    ids = np.repeat([2, -1, 0, 3, 1, 0], [1000, 37, 900, 1163, 1, 999])
    (y,) = proj_adapters([(x, w, None, None, bank)], adapter_plan(ids, 4, dev))
    _assert_close(y, _exact(x, w, None, None, pairs, ids))


def test_without_adapters_it_is_the_grouped_projection(dev):
    """Rows without an adapter get proj_grouped's own bits, in batches of either kernel."""
    gen = torch.Generator().manual_seed(11)
    for m in (4, 100, 400):
        x, w = _rand((m, 2048), gen, dev), _rand((2048, 2048), gen, dev, 1 / math.sqrt(2048))
        bank, _ = _bank(gen, dev, [16, 16], 2048, 2048)
        (want,) = ops.proj_grouped([(x, w)])
        (none,) = proj_adapters([(x, w, None, None, bank)], adapter_plan([-1] * m, 2, dev))
        assert torch.equal(none, want)
        ids = [0 if i % 3 else -1 for i in range(m)]
        (some,) = proj_adapters([(x, w, None, None, bank)], adapter_plan(ids, 2, dev))
        base = [i for i in range(m) if i % 3 == 0]
        assert torch.equal(some[base], want[base])


def test_strided_inputs_and_outputs(dev):
    gen = torch.Generator().manual_seed(13)
    m, k, n = 70, 256, 130
    wide = _rand((m, 3 * k + 8), gen, dev)
    x = wide[:, k:2 * k]
    w = _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bank, pairs = _bank(gen, dev, [16, 8], k, n)
    ids = np.arange(m) % 3 - 1
    out = torch.zeros((m, n + 11), dtype=torch.bfloat16, device=dev)
    plan = adapter_plan(ids, 2, dev)
    proj_adapters([(x, w, None, None, bank)], plan, outs=[out[:, 3:3 + n]])
    _assert_close(out[:, 3:3 + n], _exact(x, w, None, None, pairs, ids))
    assert not out[:, :3].any() and not out[:, 3 + n:].any()
    odd = wide[:, 1:1 + k]  # not 16-byte aligned: copied
    (y,) = proj_adapters([(odd, w, None, None, bank)], plan)
    _assert_close(y, _exact(odd, w, None, None, pairs, ids))
    none = proj_adapters([(x[:0], w, None, None, bank)], adapter_plan([], 2, dev))
    assert none[0].shape == (0, n)


@pytest.mark.parametrize("m", [8, 48, 640])
def test_a_broken_adapter_stays_with_its_rows(dev, m):
    """Infinities and NaN in one adapter, or in one row, reach no other row."""
    gen = torch.Generator().manual_seed(17)
    k, n = 256, 96
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bank, pairs = _bank(gen, dev, [8, 8, 8], k, n)
    ids = np.arange(m) % 4 - 1
    plan = adapter_plan(ids, 3, dev)
    (want,) = proj_adapters([(x, w, None, None, bank)], plan)
    a, b, s = pairs[1]
    b = b.clone()
    b[::5] = math.nan
    b[1::5] = math.inf
    bank.load(1, a, b, s)
    (got,) = proj_adapters([(x, w, None, None, bank)], plan)
    others = np.flatnonzero(ids != 1)
    assert torch.equal(got[others], want[others])
    assert not got[np.flatnonzero(ids == 1)][:, ::5].isfinite().any()
    bank.load(1, a, pairs[1][1], s)
    bad = x.clone()
    bad[5] = math.inf
    (got,) = proj_adapters([(bad, w, None, None, bank)], plan)
    rest = [i for i in range(m) if i != 5]
    assert torch.equal(got[rest], want[rest])


def test_an_infinite_term_is_infinite_as_in_the_formula(dev):
    """h = inf in one rank: its column of B gives inf, not NaN from a rounding part or a
    padding rank."""
    k, n = 32, 16
    x = torch.zeros((1, k), dtype=torch.bfloat16, device=dev)
    x[0, 0] = math.inf
    w = torch.full((n, k), 0.0, dtype=torch.bfloat16, device=dev)
    w[:, 0] = 1.0  # (and zeros times x's zeros elsewhere)
    bank = AdapterBank(1, k, n, 16, dev)
    a = torch.zeros((1, k), dtype=torch.bfloat16, device=dev)
    a[0, 0] = 1.0
    bank.load(0, a, torch.ones((n, 1), dtype=torch.bfloat16, device=dev))
    (y,) = proj_adapters([(x, w, None, None, bank)], adapter_plan([0], 1, dev))
    assert bool((y == math.inf).all())


def test_places_are_loaded_replaced_and_cleared(dev):
    gen = torch.Generator().manual_seed(19)
    m, k, n = 20, 128, 64
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bank, pairs = _bank(gen, dev, [40, 40], k, n)
    ids = np.arange(m) % 2
    plan = adapter_plan(ids, 2, dev)
    a, b = _rand((7, k), gen, dev, 0.1), _rand((n, 7), gen, dev)  # fewer ranks than before
    bank.load(1, a, b, 0.5)
    (y,) = proj_adapters([(x, w, None, None, bank)], plan)
    _assert_close(y, _exact(x, w, None, None, [pairs[0], (a, b, 0.5)], ids))
    bank.clear(0)
    (y,) = proj_adapters([(x, w, None, None, bank)], plan)
    _assert_close(y, _exact(x, w, None, None, [None, (a, b, 0.5)], ids))


def test_calls_repeat_and_run_on_other_streams(dev):
    gen = torch.Generator().manual_seed(23)
    m, k, n = 90, 1024, 512
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bank, _ = _bank(gen, dev, [16] * 12, k, n)
    plan = adapter_plan(np.arange(m) % 13 - 1, 12, dev)
    (want,) = proj_adapters([(x, w, None, None, bank)], plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        (got,) = proj_adapters([(x, w, None, None, bank)], plan)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("m", [6, 60])
def test_under_graph_capture(dev, m):
    gen = torch.Generator().manual_seed(29)
    k, n = 2048, 256
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    bank, pairs = _bank(gen, dev, [16, 8, 32], k, n)
    ids = np.arange(m) % 4 - 1
    plan = adapter_plan(ids, 3, dev)
    proj_adapters([(x, w, None, None, bank)], plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (out,) = proj_adapters([(x, w, None, None, bank)], plan)
    for i in range(3):
        x.copy_(_rand((m, k), gen, dev))
        graph.replay()
        torch.cuda.synchronize()
        (eager,) = proj_adapters([(x, w, None, None, bank)], plan)
        assert torch.equal(out, eager)
        _assert_close(out, _exact(x, w, None, None, pairs, ids))


def test_refusals(dev):
    gen = torch.Generator().manual_seed(31)
    k, n = 64, 48
    x, w = _rand((4, k), gen, dev), _rand((n, k), gen, dev)
    bank, _ = _bank(gen, dev, [8, 8], k, n)
    plan = adapter_plan([0, 1, -1, 0], 2, dev)
    for ids in ([2], [-2], [0, 5]):
        with pytest.raises(ValueError, match="out of range"):
            adapter_plan(ids, 2, dev)
    for prods, p in [([(x[:3], w, None, None, bank)], plan),              # rows of the plan
                     ([(x, w[:, :32], None, None, bank)], plan),           # k of x and w
                     ([(x, w[:40], None, None, bank)], plan),              # n of the bank
                     ([(x, w, None, None, bank)], adapter_plan([0] * 4, 3, dev)),
                     ([(x.float(), w, None, None, bank)], plan),
                     ([(x.cpu(), w, None, None, bank)], plan),
                     ([(x, w, None, "relu", bank)], plan), ([], plan),
                     ([(x, w, None, None, bank)] * 9, plan),
                     ([(x, w, None, None, bank)], adapter_plan([0] * 4, 2, "cpu"))]:
        with pytest.raises(ValueError):
            proj_adapters(prods, p)
    a, b = _rand((8, k), gen, dev), _rand((n, 8), gen, dev)
    for args in [(2, a, b), (-1, a, b), (0, a.float(), b), (0, a, b[:, :4]), (0, a[:, :32], b),
                 (0, _rand((9, k), gen, dev), _rand((n, 9), gen, dev)), (0, a, b, math.nan)]:
        with pytest.raises(ValueError):
            bank.load(*args)
    with pytest.raises(ValueError):
        bank.clear(7)
    for args in [(0, k, n, 8), (1, 40, n, 8), (1, k, 0, 8), (1, k, n, 0), (1, k, n, 257)]:
        with pytest.raises(ValueError):
            AdapterBank(*args, dev)


def test_a_dropped_plan_stays_until_its_launches_are_done(dev):
    """A plan used on another stream than its own and dropped while that use is still to come: its
    memory is handed out again only after it."""
    gen = torch.Generator().manual_seed(37)
    m, k, n = 700, 64, 32
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev)
    bank, _ = _bank(gen, dev, [16, 8], k, n)
    ids = np.arange(m) % 3 - 1
    plan = adapter_plan(ids, 2, dev)
    (want,) = proj_adapters([(x, w, None, None, bank)], plan)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)  # some 20 ms that the launch has to wait for
        (got,) = proj_adapters([(x, w, None, None, bank)], plan)
    at, ints = plan.buf.data_ptr(), plan.buf.numel()
    del plan
    others = [torch.empty(ints, dtype=torch.int32, device=dev) for _ in range(4)]
    assert not side.query()  # (the use is still to come)
    assert all(t.data_ptr() != at for t in others)
    side.synchronize()
    assert torch.equal(got, want)


def test_adapters_that_are_only_loaded_cost_little(dev):
    """600 rows on four adapters, of 8 and of 1,000 that are loaded: the plan has room for a gap
    behind every loaded one, 19,200 positions in place of 896, whose tiles hold no row (26 and 39 us;
    with the empty tiles multiplied 26 and 255)."""
    gen = torch.Generator().manual_seed(43)
    m, k, n = 600, 2080, 2048
    x, w = _rand((m, k), gen, dev), _rand((n, k), gen, dev, 1 / math.sqrt(k))
    ids, times, outs = np.arange(m) % 4, [], []
    for loaded in (8, 1000):
        bank = AdapterBank(loaded, k, n, 8, dev)
        pairs = torch.Generator().manual_seed(47)
        for i in range(4):
            bank.load(i, _rand((8, k), pairs, dev, 1 / math.sqrt(k)), _rand((n, 8), pairs, dev))
        plan = adapter_plan(ids, loaded, dev)
        products = [(x, w, None, None, bank)]
        outs.append(proj_adapters(products, plan)[0])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(10):
                proj_adapters(products, plan)
        graph.replay()
        took = []
        for _ in range(7):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            graph.replay()
            end.record()
            end.synchronize()
            took.append(start.elapsed_time(end))
        times.append(sorted(took)[3])
    assert torch.equal(*outs)
    assert times[1] < 4 * times[0], times


@pytest.mark.parametrize("act", [None, "sigmoid"])
@pytest.mark.parametrize("m,k,n", [(1, 64, 48), (5, 256, 33), (16, 2048, 300), (40, 256, 96),
                                   (200, 2048, 130), (203, 4096, 520), (640, 256, 96),
                                   (5000, 64, 1000), (8200, 64, 1000)])
def test_an_infinite_weight_is_infinite_as_in_the_formula(dev, m, k, n, act):
    """B = +-inf in one rank of a column: h B is infinite by the sign of h, whatever h's bits are
    (powers of two, whole numbers of few bits, and all 24), and its other rank is a number. The
    rows run on every kernel: one row tile, small and large tiles, k in two parts, both tiles of
    many rows."""
    gen = torch.Generator().manual_seed(41)
    w = _rand((n, k), gen, dev, 1 / math.sqrt(k))
    x = _rand((m, k), gen, dev)
    x[:, 0] = torch.sign(x[:, 0].float()).to(torch.bfloat16)  # h of rank 0: +-1
    x[::3, 0] *= 3
    x[1::3, 0] *= 0.0078125
    bank = AdapterBank(2, k, n, 20, dev)
    a, b = _rand((18, k), gen, dev, 1 / math.sqrt(k)), _rand((n, 18), gen, dev, 0.2)
    a[0] = 0.0
    a[0, 0] = 1.0
    ranks = torch.arange(n) % 19  # the infinite one of every column, none in some
    held = torch.arange(n)[ranks < 18]
    sign = torch.where(held % 2 == 0, math.inf, -math.inf).to(torch.bfloat16).to(dev)
    b[held.to(dev), ranks[ranks < 18].to(dev)] = sign
    bank.load(1, a, b, 1.5)
    ids = np.arange(m) % 2
    ids[-1] = 1
    (y,) = proj_adapters([(x, w, None, act, bank)], adapter_plan(ids, 2, dev))
    rows = np.flatnonzero(ids == 1)
    h = 1.5 * (x.double().cpu() @ a.double().cpu().T)[rows]
    # (a sum of k terms near zero may have either sign in 32 bits)
    sure = (h.abs() > 1e-4)[:, ranks.clamp(max=17)] | (ranks == 18)
    want = _exact(x, w, None, act, [None, (a, b, 1.5)], ids)[rows]
    got = y.double().cpu()[rows]
    if act is None:
        assert int(want.isinf().sum()) == len(rows) * len(held)
        assert torch.equal(got.isinf() & sure, want.isinf() & sure)
        assert torch.equal(got[want.isinf() & sure], want[want.isinf() & sure])
    else:
        ends = (ranks < 18) & sure  # 0 or 1
        assert torch.equal(got[ends], want[ends])
    none = _exact(x, w, None, act, None, ids)
    base = np.flatnonzero(ids == 0)
    if base.size:
        _assert_close(y[base], none[base])
    plain = ranks == 18
    if plain.any():
        _assert_close(y.cpu()[rows][:, plain], want[:, plain])
