"""linear_prefill_varlen where sequences are cut into pieces: every test here asks the library whether
its case is cut, so that none of them runs whole by a changed rule."""

import math

import numpy as np
import pytest
import torch

from tests.test_gpu_linear import BF16, F32, _check, _inputs
from wkvm_amd import _lib, linear_prefill_varlen

pytestmark = pytest.mark.gpu


def is_cut(nseq, tokens, H, Hq, K, V):
    io = _lib.LinearIO(H=H, Hq=Hq, K=K, V=V)
    return _lib.load().wkv7_linear_prefill_workspace_bytes(nseq, tokens, io) > 0


def _run(dev, seed, lens, ids, H, Hq, K, V, kind, zero_init, f32=True, rows=9):
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    assert is_cut(len(lens), cu[-1], H, Hq, K, V)
    before, q, k, v, g = _inputs(seed, cu[-1], H, Hq, K, V, kind, rows=rows)
    pool = before.to(dev)
    y = linear_prefill_varlen(pool, ids, cu, q.to(dev), k.to(dev), v.to(dev), g.to(dev),
                              zero_init=zero_init, scale=0.125, out_dtype=F32 if f32 else BF16)
    _check(pool, y, before, cu, ids, q, k, v, g, 0.125, zero_init)


@pytest.mark.parametrize("lens", [[0, 4096], [2305, 0], [1, 0, 8000], [0, 0, 5000], [5000, 0, 0],
                                  [0, 0, 0, 6000], [3000, 0, 2304], [0, 1, 6200, 0, 256, 2500, 5]])
@pytest.mark.parametrize("zero_init", [False, True])
def test_empty_sequences_among_cut_ones(dev, lens, zero_init):
    """Their slots are zeroed or left as they are, wherever they lie among the pieces of the others."""
    _run(dev, 41, lens, [6, 2, 5, 1, 8, 3, 4][:len(lens)], 2, 1, 64, 64, "token", zero_init)


@pytest.mark.parametrize("zero_init", [False, True])
def test_empty_sequences_among_cut_ones_of_wide_heads(dev, zero_init):
    for f32 in (False, True):
        _run(dev, 42, [0, 4096, 0], [4, 1, 7], 2, 2, 128, 128, "token", zero_init, f32)


@pytest.mark.parametrize("kind", ["fixed", "token", "none", "strong", "forget", "grow"])
@pytest.mark.parametrize("lens", [[1024, 0, 700, 1, 4048, 1813], [2560, 2560], [2537, 64], [4097]])
def test_pieces_that_end_inside_and_at_the_end(dev, lens, kind):
    _run(dev, 43, lens, [6, 2, 5, 1, 8, 3][:len(lens)], 2, 1, 64, 64, kind, False)


def test_pieces_find_their_sequence_among_more_than_a_wave(dev):
    """70 sequences, some of them empty, the first and the last among these."""
    rng = np.random.default_rng(3)
    lens = [int(n) if rng.random() < 0.5 else 0 for n in rng.integers(1, 4000, 70)]
    lens[0] = lens[69] = 0
    lens[66] = 168000 - sum(lens) + lens[66]
    ids = rng.permutation(np.arange(1, 81))[:70].tolist()
    _run(dev, 44, lens, ids, 1, 1, 64, 64, "token", True, rows=81)


def test_refused_slots_of_a_cut_batch(dev):
    """Ids out of range touch no state and give zeros; tokens of no sequence keep what ``out`` holds."""
    T, beg, end = 4000, 1900, 3990
    assert is_cut(2, T, 2, 2, 64, 64)
    before, q, k, v, g = _inputs(45, T, 2, 2, 64, 64)
    pool = before.to(dev)
    ids = torch.tensor([9, 3], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, beg, end], dtype=torch.int32, device=dev)
    out = torch.full((T, 2, 64), 7.0, device=dev)
    linear_prefill_varlen(pool, ids, cu, *(t.to(dev) for t in (q, k, v, g)), out=out)
    assert (out[:beg] == 0).all() and (out[end:] == 7).all()
    _check(pool, out[beg:end], before, [0, end - beg], [3], q[beg:end], k[beg:end], v[beg:end],
           g[beg:end], 1.0)


def test_broken_offsets_of_a_cut_batch_stay_in_bounds(dev):
    """Device offsets past the tokens, or falling: some tokens of the batch, never other rows."""
    T = 4000
    assert is_cut(2, T, 1, 1, 64, 64)
    before, q, k, v, g = _inputs(46, T, 1, 1, 64, 64)
    xs = [t.to(dev) for t in (q, k, v, g)]
    for offsets in ([0, 5000, 3000], [3000, 2000, 1000], [-5, 2 ** 31 - 1, T], [T, 0, T]):
        pool = before.to(dev)
        cu = torch.tensor(offsets, dtype=torch.int32, device=dev)
        linear_prefill_varlen(pool, torch.tensor([1, 2], dtype=torch.int32, device=dev), cu, *xs)
        torch.cuda.synchronize()
        rest = [0] + list(range(3, 9))
        assert (pool[rest].cpu() == before[rest]).all()


@pytest.mark.parametrize("where,bad", [
    (w, b) for w in ("v", "k", "q", "g", "state") for b in (math.inf, -math.inf, math.nan)
    if (w, b) != ("g", math.inf)])  # (a decay is at most finite)
@pytest.mark.parametrize("T", [150, 2900])
def test_infinities_of_128_keys(dev, where, bad, T):
    """An infinite or NaN value reaches the outputs that the formula gives it to, and no others."""
    from tests.linear_ref import scan, state_bound, y_bound
    from tests.test_gpu_linear import f64

    assert is_cut(1, T, 2, 2, 128, 128) == (T > 2000)
    before, q, k, v, g = _inputs(47, T, 2, 2, 128, 128, "token", rows=3)
    at = T - 70
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
    for got, want, bound in ((f64(got), y, y_bound(y, my, T, 128, True)),
                             (f64(pool)[1], ref[1], state_bound(ms[0], T))):
        ok = np.isfinite(want)
        assert (np.abs(got[ok] - want[ok]) <= bound[ok]).all()
        assert (np.isnan(got) == np.isnan(want)).all()
        inf = np.isinf(want)
        assert (got[inf] == want[inf]).all()


@pytest.mark.parametrize("kind", ["fixed", "token", "strong", "forget", "grow"])
@pytest.mark.parametrize("lens,H,Hq,K,V", [([700, 64, 1, 33], 3, 3, 64, 128), ([4097], 2, 1, 64, 64),
                                           ([150, 300], 4, 2, 128, 64), ([400] * 8, 40, 40, 64, 64)])
def test_a_bf16_output_is_the_fp32_one_rounded(dev, lens, H, Hq, K, V, kind):
    """Whatever the outputs' type, they are computed in fp32 (and the same states are left)."""
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    before, *xs = _inputs(48, cu[-1], H, Hq, K, V, kind)
    xs = [t.to(dev) for t in xs]
    got = []
    for dtype in (F32, BF16):
        pool = before.to(dev)
        got.append((linear_prefill_varlen(pool, list(range(1, len(lens) + 1)), cu, *xs, scale=0.2,
                                          out_dtype=dtype), pool))
    assert torch.equal(got[0][0].to(BF16), got[1][0]) and torch.equal(got[0][1], got[1][1])
