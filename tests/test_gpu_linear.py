"""linear_decode_slots / linear_prefill_varlen against the formula in float64, token by token."""

import math

import numpy as np
import pytest
import torch

from tests.linear_ref import scan, state_bound, y_bound
from wkvm_amd import RWKV7StateBank, linear_decode_slots, linear_prefill_varlen, ops
from wkvm_amd.layout import RWKV7StateLayout

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def f64(t):
    return t.detach().double().cpu().numpy()


def _decay(kind, gen, T, H):
    if kind == "fixed":
        return torch.log1p(-torch.exp2(-4 - 8 * torch.rand(H, generator=gen)))
    if kind == "none":
        return torch.zeros(T, H)
    if kind == "strong":
        return -30 * torch.rand(T, H, generator=gen)
    if kind == "forget":  # some tokens forget everything before them
        g = -0.1 * torch.rand(T, H, generator=gen)
        return torch.where(torch.rand(T, H, generator=gen) < 0.05, torch.tensor(-math.inf), g)
    if kind == "grow":  # a state that grows a little
        return 0.02 * torch.randn(T, H, generator=gen)
    rate = torch.exp(torch.rand(H, generator=gen) * 5 - 4)
    return -rate * torch.log1p(torch.exp(2 * torch.randn(T, H, generator=gen)))


def _inputs(seed, T, H, Hq, K, V, kind="token", rows=9):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(T, Hq, K, generator=gen).to(BF16)
    k = (torch.randn(T, Hq, K, generator=gen) / math.sqrt(K)).to(BF16)
    v = torch.randn(T, H, V, generator=gen).to(BF16)
    pool = torch.randn(rows, H, K, V, generator=gen)
    return pool, q, k, v, _decay(kind, gen, T, H)


def _check(pool, got_y, before, cu, ids, q, k, v, g, scale, zero_init=False):
    """Outputs, the sequences' states and every other row of the pool."""
    ref = f64(before)
    y, my, ms = scan(ref, cu, ids, f64(q), f64(k), f64(v), f64(g), scale, zero_init)
    longest = max([b - a for a, b in zip(cu, cu[1:])] + [0])
    K = q.shape[2]
    err = np.abs(f64(got_y) - y)
    bound = y_bound(y, my, longest, K, got_y.dtype == F32)
    assert np.isfinite(err).all() and (err <= bound).all(), f"y {np.max(err / bound):.2f} bounds"
    got = f64(pool)
    if len(ids):
        err = np.abs(got[ids] - ref[ids])
        bound = state_bound(ms, longest)
        assert np.isfinite(err).all() and (err <= bound).all(), \
            f"state {np.max(err / bound):.2f} bounds"
    rest = [r for r in range(len(got)) if r not in ids]
    assert (got[rest] == f64(before)[rest]).all()


SHAPES = [(4, 4, 64, 64), (6, 3, 64, 128), (4, 1, 128, 64), (2, 2, 128, 128), (3, 3, 64, 192)]


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("kind", ["fixed", "token", "strong", "forget"])
@pytest.mark.parametrize("shape", SHAPES)
def test_decode(dev, shape, kind, f32):
    H, Hq, K, V = shape
    ids = [5, 1, 8, 2, 7]
    before, q, k, v, g = _inputs(1, 5, H, Hq, K, V, kind)
    pool = before.to(dev)
    y = linear_decode_slots(pool, ids, q.to(dev), k.to(dev), v.to(dev), g.to(dev), scale=0.3,
                            out_dtype=F32 if f32 else BF16)
    _check(pool, y, before, list(range(6)), ids, q, k, v, g, 0.3)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("kind", ["fixed", "token", "none", "strong", "forget", "grow"])
@pytest.mark.parametrize("shape", SHAPES)
def test_prefill_of_ragged_sequences(dev, shape, kind, f32):
    H, Hq, K, V = shape
    lens = [0, 1, 2, 17, 64, 65, 33, 200]
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    ids = [3, 1, 8, 2, 7, 5, 4, 6]
    before, q, k, v, g = _inputs(2, cu[-1], H, Hq, K, V, kind)
    pool = before.to(dev)
    y = linear_prefill_varlen(pool, ids, cu, q.to(dev), k.to(dev), v.to(dev), g.to(dev),
                              scale=0.25, out_dtype=F32 if f32 else BF16)
    _check(pool, y, before, cu, ids, q, k, v, g, 0.25)


@pytest.mark.parametrize("length", [1, 15, 16, 31, 32, 48, 63, 64, 66, 127, 128, 129, 192])
@pytest.mark.parametrize("zero_init", [False, True])
def test_prefill_lengths(dev, length, zero_init):
    before, q, k, v, g = _inputs(length, length, 2, 2, 64, 64, rows=3)
    pool = before.to(dev)
    y = linear_prefill_varlen(pool, [2], [0, length], q.to(dev), k.to(dev), v.to(dev), g.to(dev),
                              zero_init=zero_init, out_dtype=F32)
    _check(pool, y, before, [0, length], [2], q, k, v, g, 1.0, zero_init)


@pytest.mark.parametrize("kind", ["fixed", "token", "forget"])
@pytest.mark.parametrize("lens", [[2500], [1024, 0, 700, 1, 2048, 513], [512, 512], [1537, 64],
                                  [0, 1, 4200, 0, 256, 2500, 5], [3000, 0, 2304], [1281]])
@pytest.mark.parametrize("zero_init", [False, True])
def test_prefill_in_pieces(dev, lens, kind, zero_init):
    """Long enough for the sequences to be cut (few heads), pieces that end inside and at the end of
    them, empty sequences between."""
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    ids = [6, 2, 5, 1, 8, 3, 4][:len(lens)]
    before, q, k, v, g = _inputs(4, cu[-1], 2, 1, 64, 64, kind)
    pool = before.to(dev)
    y = linear_prefill_varlen(pool, ids, cu, q.to(dev), k.to(dev), v.to(dev), g.to(dev),
                              zero_init=zero_init, scale=0.125, out_dtype=F32)
    _check(pool, y, before, cu, ids, q, k, v, g, 0.125, zero_init)


def test_prefill_in_pieces_of_wide_heads(dev):
    cu = [0, 2900, 2901]
    for f32 in (False, True):
        before, q, k, v, g = _inputs(5, cu[-1], 2, 2, 128, 128, "token")
        pool = before.to(dev)
        y = linear_prefill_varlen(pool, [4, 1], cu, q.to(dev), k.to(dev), v.to(dev), g.to(dev),
                                  out_dtype=F32 if f32 else BF16)
        _check(pool, y, before, cu, [4, 1], q, k, v, g, 1.0)


@pytest.mark.parametrize("long", [1100, 135000])
def test_more_sequences_than_a_wave(dev, long):
    """Pieces (of the long batch) find their sequence among more than 64, many of them empty."""
    rng = np.random.default_rng(3)
    lens = [int(n) if rng.random() < 0.5 else 0 for n in rng.integers(1, 40, 68)]
    lens[60] = long
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    ids = rng.permutation(np.arange(1, 81))[:68].tolist()
    before, q, k, v, g = _inputs(6, cu[-1], 1, 1, 64, 64, "token", rows=81)
    pool = before.to(dev)
    y = linear_prefill_varlen(pool, ids, cu, q.to(dev), k.to(dev), v.to(dev), g.to(dev),
                              out_dtype=F32)
    _check(pool, y, before, cu, ids, q, k, v, g, 1.0)


def test_whole_tiles_of_64_columns(dev):
    """Enough heads for the wide tile (and an odd number of them), 64 and 128 value columns."""
    for V in (64, 128):
        lens = [70, 0, 129, 64, 1]
        cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
        ids = [3, 1, 8, 2, 5]
        for f32 in (False, True):
            before, q, k, v, g = _inputs(19, cu[-1], 39, 13, 64, V, "token")
            pool = before.to(dev)
            y = linear_prefill_varlen(pool, ids, cu, q.to(dev), k.to(dev), v.to(dev), g.to(dev),
                                      scale=0.125, out_dtype=F32 if f32 else BF16)
            _check(pool, y, before, cu, ids, q, k, v, g, 0.125)


@pytest.mark.parametrize("where,bad", [
    (w, b) for w in ("v", "k", "q", "g", "state") for b in (math.inf, -math.inf, math.nan)
    if (w, b) != ("g", math.inf)])  # (a decay is at most finite)
@pytest.mark.parametrize("lens", [[150], [2500]])
def test_nothing_reaches_the_tokens_before_it(dev, where, bad, lens):
    """An infinite or NaN value reaches the outputs that the formula gives it to, and no others."""
    T = lens[0]
    before, q, k, v, g = _inputs(7, T, 2, 2, 64, 64, "token", rows=3)
    at = T - 70  # in the middle of a chunk, behind the first piece of the long one
    if where == "state":
        before[1, 0, 5, 9] = bad
    else:
        x = {"v": v, "k": k, "q": q, "g": g}[where]
        x[(at, 0) if where == "g" else (at, 0, 5)] = bad
    pool = before.to(dev)
    got = linear_prefill_varlen(pool, [1], [0, T], q.to(dev), k.to(dev), v.to(dev), g.to(dev),
                                out_dtype=F32)
    ref = f64(before)
    y, my, ms = scan(ref, [0, T], [1], f64(q), f64(k), f64(v), f64(g), 1.0)
    for got, want, mag in ((f64(got), y, my), (f64(pool)[1], ref[1], ms[0])):
        ok = np.isfinite(want)
        if where != "state":
            assert ok.any()
        bound = (y_bound(want, mag, T, 64, True) if want is y else state_bound(mag, T))[ok]
        assert (np.abs(got[ok] - want[ok]) <= bound).all()
        assert (np.isnan(got) == np.isnan(want)).all()
        inf = np.isinf(want)
        assert (got[inf] == want[inf]).all()
    if where != "state":
        assert np.isfinite(y[:at]).all()


def test_prefill_then_decode_is_one_pass(dev):
    cu, ids = [0, 90, 123], [2, 1]
    before, q, k, v, g = _inputs(8, 123, 4, 2, 64, 64)
    pool = before.to(dev)
    Q, K, V, G = (t.to(dev) for t in (q, k, v, g))
    head = [i for i in range(122) if i != 89]
    y0 = linear_prefill_varlen(pool, ids, [0, 89, 121], Q[head], K[head], V[head], G[head],
                               out_dtype=F32)
    last = [89, 122]
    y1 = linear_decode_slots(pool, ids, Q[last], K[last], V[last], G[last], out_dtype=F32)
    y = torch.empty(123, 4, 64, device=dev)
    y[head], y[last] = y0, y1
    _check(pool, y, before, cu, ids, q, k, v, g, 1.0)


def test_strided_and_misaligned_views(dev):
    """Vectors that are columns of one projection's output, and views that have to be copied."""
    before, q, k, v, g = _inputs(9, 100, 4, 2, 64, 64)
    fused = torch.cat([q.reshape(100, -1), k.reshape(100, -1), v.reshape(100, -1)], 1).to(dev)
    views = [fused[:, :128].view(100, 2, 64), fused[:, 128:256].view(100, 2, 64),
             fused[:, 256:].view(100, 4, 64)]
    assert not views[0].is_contiguous()
    wide = torch.zeros(100, 9, device=dev)
    wide[:, 3:7] = g.to(dev)
    for kind in ("columns", "transposed", "misaligned"):
        if kind == "transposed":
            xs = [t.to(dev).transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
        elif kind == "misaligned":
            xs = []
            for t in (q, k, v):
                flat = torch.empty(t.numel() + 1, dtype=BF16, device=dev)
                flat[1:] = t.reshape(-1).to(dev)
                xs.append(flat[1:].view(t.shape))
        else:
            xs = views
        pool = before.to(dev)
        y = linear_prefill_varlen(pool, [1, 4], [0, 30, 100], *xs, wide[:, 3:7])
        _check(pool, y, before, [0, 30, 100], [1, 4], q, k, v, g, 1.0)
        pool = before.to(dev)
        y = linear_decode_slots(pool, [3, 8, 1], *(x[:3] for x in xs), wide[:3, 3:7])
        _check(pool, y, before, [0, 1, 2, 3], [3, 8, 1], q[:3], k[:3], v[:3], g[:3], 1.0)


def test_refused_slots_and_rows_behind_the_last_sequence(dev):
    """Device ids out of range touch no state and give zeros; tokens of no sequence keep what ``out``
    holds."""
    before, q, k, v, g = _inputs(10, 1200, 2, 2, 64, 64)
    Q, K, V, G = (t.to(dev) for t in (q, k, v, g))
    for T, beg in ((1200, 1000), (90, 40)):
        pool = before.to(dev)
        ids = torch.tensor([9, 3], dtype=torch.int32, device=dev)
        cu = torch.tensor([0, beg, T - 10], dtype=torch.int32, device=dev)
        out = torch.full((T, 2, 64), 7.0, device=dev)
        linear_prefill_varlen(pool, ids, cu, Q[:T], K[:T], V[:T], G[:T], out=out)
        assert (out[:beg] == 0).all() and (out[T - 10:] == 7).all()
        _check(pool, out[beg:T - 10], before, [0, T - 10 - beg], [3], q[beg:T - 10],
               k[beg:T - 10], v[beg:T - 10], g[beg:T - 10], 1.0)
    pool = before.to(dev)
    out = torch.full((3, 2, 64), 7.0, device=dev)
    ids = torch.tensor([-1, 9, 4], dtype=torch.int32, device=dev)
    linear_decode_slots(pool, ids, Q[:3], K[:3], V[:3], G[:3], out=out)
    assert (out[:2] == 0).all()
    _check(pool, out[2:], before, [0, 1], [4], q[2:3], k[2:3], v[2:3], g[2:3], 1.0)


def test_offsets_that_break_their_contract_stay_in_bounds(dev):
    """Device offsets past the tokens, or falling: some tokens of the batch, never others."""
    before, q, k, v, g = _inputs(11, 700, 1, 1, 64, 64)
    Q, K, V, G = (t.to(dev) for t in (q, k, v, g))
    for offsets in ([0, 900, 650], [300, 200, 100], [-5, 2 ** 31 - 1, 700], [700, 0, 700]):
        pool = before.to(dev)
        cu = torch.tensor(offsets, dtype=torch.int32, device=dev)
        y = linear_prefill_varlen(pool, torch.tensor([1, 2], dtype=torch.int32, device=dev), cu, Q, K,
                                  V, G)
        torch.cuda.synchronize()
        rest = [0] + list(range(3, 9))
        assert (pool[rest].cpu() == before[rest]).all() and y.shape == (700, 1, 64)


def test_repeated_runs_are_bit_identical(dev):
    for T, H, K, V in ((5000, 3, 64, 64), (5000, 2, 128, 128), (900, 40, 64, 64)):
        before, q, k, v, g = _inputs(12, T, H, H, K, V)
        xs = [t.to(dev) for t in (q, k, v, g)]
        first = None
        for _ in range(5):
            pool = before.to(dev)
            y = linear_prefill_varlen(pool, [4, 2], [0, 700, T], *xs)
            if first is None:
                first = y.clone(), pool.clone()
            assert torch.equal(y, first[0]) and torch.equal(pool, first[1])


def test_a_sequence_does_not_depend_on_the_batch(dev):
    """Two requests as one batch and each alone, both uncut: the same bits."""
    before, q, k, v, g = _inputs(13, 300, 2, 2, 64, 64)
    xs = [t.to(dev) for t in (q, k, v, g)]
    both = before.to(dev)
    y = linear_prefill_varlen(both, [4, 2], [0, 130, 300], *xs)
    alone = before.to(dev)
    ya = linear_prefill_varlen(alone, [4], [0, 130], *(x[:130] for x in xs))
    yb = linear_prefill_varlen(alone, [2], [0, 170], *(x[130:].contiguous() for x in xs))
    assert torch.equal(y, torch.cat([ya, yb])) and torch.equal(both, alone)


@pytest.mark.parametrize("T", [150, 5000])
def test_graph_replays(dev, T):
    """A captured prefill and decode step, replayed with other inputs and eager work between."""
    before, q, k, v, g = _inputs(14, T, 2, 2, 64, 64)
    static = [t.to(dev) for t in (q, k, v, g)]
    pool = before.to(dev)
    ids = torch.tensor([2, 5], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, T // 3, T], dtype=torch.int32, device=dev)
    few = [t[:2].clone() for t in static]

    def step():
        y = linear_prefill_varlen(pool, ids, cu, *static)
        return y, linear_decode_slots(pool, ids, *few)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (20, 21, 22):
        b2, *xs = _inputs(seed, T, 2, 2, 64, 64)
        for dst, src in zip(static, xs):
            dst.copy_(src)
        for dst, src in zip(few, xs):
            dst.copy_(src[:2])
        pool.copy_(b2)
        graph.replay()
        got = [t.clone() for t in out] + [pool.clone()]
        torch.cuda.synchronize()
        pool.copy_(b2)
        want = [*step(), pool]
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_other_stream(dev):
    before, q, k, v, g = _inputs(15, 2000, 2, 2, 64, 64)
    xs = [t.to(dev) for t in (q, k, v, g)]
    want_pool = before.to(dev)
    want = linear_prefill_varlen(want_pool, [1], [0, 2000], *xs)
    pool = before.to(dev)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(dev)
    with torch.cuda.stream(side):
        got = [linear_prefill_varlen(pool, [1], [0, 2000], *xs)]
    side.synchronize()
    assert torch.equal(got[0], want) and torch.equal(pool, want_pool)


def test_through_the_bank(dev):
    bank = RWKV7StateBank(RWKV7StateLayout(2, 128, 2, 64, 64, BF16), 4, dev)
    before, q, k, v, g = _inputs(16, 70, 2, 2, 64, 64)
    bank.wkv[1].copy_(before[:5])
    slots = [{"wkv": 3, "shift": 3}, {"wkv": 1, "shift": 1}]
    y = bank.prefill_linear(1, slots, [0, 20, 70], q.to(dev), k.to(dev), v.to(dev), g.to(dev))
    _check(bank.wkv[1], y, before[:5], [0, 20, 70], [3, 1], q, k, v, g, 1.0)
    mid = bank.wkv[1].cpu()
    y = bank.decode_linear(1, slots, q[:2].to(dev), k[:2].to(dev), v[:2].to(dev), g[:2].to(dev),
                           out_dtype=F32)
    _check(bank.wkv[1], y, mid, [0, 1, 2], [3, 1], q[:2], k[:2], v[:2], g[:2], 1.0)
    assert (bank.wkv[0] == 0).all()


def test_nothing_to_do(dev):
    before, q, k, v, g = _inputs(17, 4, 2, 2, 64, 64)
    pool = before.to(dev)
    e = [t[:0].to(dev) for t in (q, k, v, g)]
    assert linear_decode_slots(pool, [], *e).shape == (0, 2, 64)
    assert linear_prefill_varlen(pool, [], [0], *e).shape == (0, 2, 64)
    linear_prefill_varlen(pool, [3], [0, 0], *e)
    assert torch.equal(pool.cpu(), before)
    linear_prefill_varlen(pool, [3], [0, 0], *e, zero_init=True)
    before[3] = 0
    assert torch.equal(pool.cpu(), before)


def test_refusals(dev):
    before, q, k, v, g = _inputs(18, 6, 4, 2, 64, 64)
    pool, Q, K, V, G = (t.to(dev) for t in (before, q, k, v, g))

    def bad(match, *, pool=pool, ids=(1, 2), cu=(0, 3, 6), q=Q, k=K, v=V, g=G, **kw):
        with pytest.raises(ValueError, match=match):
            linear_prefill_varlen(pool, list(ids), list(cu), q, k, v, g, **kw)

    bad("float32", pool=pool.half())
    bad("K must be", pool=torch.zeros(9, 4, 32, 64, device=dev))
    bad("V must be", pool=torch.zeros(9, 4, 64, 96, device=dev))
    bad("contiguous", pool=torch.zeros(9, 4, 64, 128, device=dev)[..., :64])
    bad("duplicate", ids=(1, 1))
    bad("out of range", ids=(1, 9))
    bad("cu_seqlens", cu=(0, 3, 5))
    bad("cu_seqlens", cu=(0, 6))
    bad("non-decreasing", ids=(1, 2, 3), cu=(0, 5, 3, 6))
    bad("bfloat16", q=Q.float())
    bad("GPU tensor", q=q)
    bad("k has|q has", k=K.repeat(1, 2, 1))
    bad("v has", v=V[:, :2])
    bad("multiple", q=Q.repeat(1, 2, 1)[:, :3], k=K.repeat(1, 2, 1)[:, :3])
    bad("q must be", q=Q[:5])
    bad("float32", g=G.double())
    bad("log_decay must be", g=G[:, :2])
    bad("y dtype", out_dtype=torch.float16)
    bad("contiguous", out=torch.empty(6, 4, 128, device=dev)[..., :64])
    with pytest.raises(ValueError, match="row_order"):
        linear_decode_slots(pool, [1, 2, 3, 4, 5, 6], Q, K, V, G, row_order=torch.arange(6))
    with pytest.raises(ValueError, match="q must be"):
        linear_decode_slots(pool, [1, 2], Q, K, V, G)
    assert torch.equal(pool.cpu(), before)


@pytest.mark.parametrize("Hq,K,V", [(4, 64, 64), (2, 128, 128)])
def test_the_order_of_the_sequences_changes_nothing(dev, Hq, K, V):
    """Offsets on the host (longest first), on the device (as they come) and in a given order; a number
    outside of the sequences runs none."""
    lens = [40, 0, 300, 1, 129, 64, 7]
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    ids = [3, 1, 8, 2, 7, 5, 4]
    before, q, k, v, g = _inputs(31, cu[-1], 4, Hq, K, V)
    args = [t.to(dev) for t in (q, k, v, g)]
    device_cu = torch.tensor(cu, dtype=torch.int32, device=dev)
    pools, ys = [], []
    for offsets, order in ((cu, None), (device_cu, None), (device_cu, [6, 5, 4, 3, 2, 1, 0]),
                           (cu, [2, 0, 1, 3, 6, 5, 4])):
        pools.append(before.to(dev))
        order = None if order is None else torch.tensor(order, dtype=torch.int32, device=dev)
        ys.append(linear_prefill_varlen(pools[-1], ids, offsets, *args, seq_order=order))
    _check(pools[0], ys[0], before, cu, ids, q, k, v, g, 1.0)
    for pool, y in zip(pools, ys):
        assert torch.equal(pool, pools[0]) and torch.equal(y, ys[0])
    pool = before.to(dev)
    order = torch.tensor([7, -1, 0, 1 << 30, -5, 9, 8], dtype=torch.int32, device=dev)
    linear_prefill_varlen(pool, ids, device_cu, *args, seq_order=order)
    assert torch.equal(pool[3], pools[0][3])
    rest = [r for r in range(9) if r != 3]
    assert torch.equal(pool[rest], before.to(dev)[rest])
    for wrong in (order[:6], order.long(), order.cpu(), torch.zeros(14, dtype=torch.int32,
                                                                    device=dev)[::2]):
        with pytest.raises(ValueError, match="seq_order"):
            linear_prefill_varlen(pool, ids, cu, *args, seq_order=wrong)


@pytest.mark.parametrize("nseq", [2, 9, 62, 63, 64])
def test_offsets_on_the_device_of_many_workgroups(dev, nseq):
    """More workgroups than units and long sequences on average, so that their lengths decide which
    starts first: equal, increasing and with empty ones among them, against host offsets."""
    H, Hq, K, V = 48, 16, 128, 256 if nseq < 9 else 64
    gen = torch.Generator().manual_seed(nseq)
    for kind in ("equal", "up", "mixed"):
        lens = [260] * nseq if kind == "equal" else [200 + 4 * i for i in range(nseq)]
        if kind == "mixed":
            lens = torch.randint(0, 640, (nseq,), generator=gen).tolist()
            lens[0] = 0
        cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
        T, ids = cu[-1], list(range(1, nseq + 1))
        q, k = (torch.randn(T, Hq, K, generator=gen).to(BF16).to(dev) / 8 for _ in range(2))
        v = torch.randn(T, H, V, generator=gen).to(BF16).to(dev)
        g = -0.1 * torch.rand(T, H, generator=gen).to(dev)
        pools = [torch.full((nseq + 2, H, K, V), 0.25, device=dev) for _ in range(2)]
        offsets = torch.tensor(cu, dtype=torch.int32, device=dev)
        ys = [linear_prefill_varlen(p, ids, c, q, k, v, g) for p, c in zip(pools, (cu, offsets))]
        assert torch.equal(ys[0], ys[1]) and torch.equal(pools[0], pools[1])
        longest = max(range(nseq), key=lambda s: lens[s])
        a, b = cu[longest], cu[longest + 1]
        alone = torch.full((2, H, K, V), 0.25, device=dev)
        y = linear_prefill_varlen(alone, [1], [0, b - a], q[a:b], k[a:b], v[a:b], g[a:b])
        assert torch.equal(y, ys[1][a:b]) and torch.equal(alone[1], pools[1][longest + 1])
        assert (pools[1][[0, nseq + 1]] == 0.25).all()
