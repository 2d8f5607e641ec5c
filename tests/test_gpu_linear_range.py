"""linear_prefill_varlen where parts of its sums pass fp32 and the formula does not: token by token in
float64 (tests/linear_ref.py), the tests' bounds as elsewhere."""

import math

import numpy as np
import pytest
import torch

from tests.linear_ref import scan, state_bound, y_bound
from tests.test_gpu_linear import BF16, F32, _check, _inputs, f64
from tests.test_gpu_linear_pieces import is_cut
from wkvm_amd import linear_prefill_varlen

pytestmark = pytest.mark.gpu


def _run(dev, cu, ids, before, q, k, v, g, zero_init=False, f32=True):
    pool = before.to(dev)
    y = linear_prefill_varlen(pool, ids, cu, q.to(dev), k.to(dev), v.to(dev), g.to(dev),
                              zero_init=zero_init, out_dtype=F32 if f32 else BF16)
    return pool, y


# -- pieces: the decay of a whole piece -----------------------------------------------------------

@pytest.mark.parametrize("g0", [-0.5, -9.0, -30.0, -80.0])
@pytest.mark.parametrize("T", [300, 2900])
def test_an_infinite_state_stays_so_under_any_decay(dev, T, g0):
    """However far a piece decays it, as long as no token's factor is 0; it is NaN behind one that
    forgets."""
    assert is_cut(1, T, 2, 2, 64, 64) == (T > 2000)
    before, q, k, v, _ = _inputs(61, T, 2, 2, 64, 64, rows=3)
    before[1, 0, 5, 9], before[1, 1, 7, 3] = math.inf, -math.inf
    g = torch.full((T, 2), g0)
    g[T - 90, 1] = -math.inf  # (the second head forgets in a later piece)
    pool, y = _run(dev, [0, T], [1], before, q, k, v, g)
    ref = f64(before)
    want, my, ms = scan(ref, [0, T], [1], f64(q), f64(k), f64(v), f64(g), 1.0)
    assert ref[1, 0, 5, 9] == math.inf and np.isnan(ref[1, 1, 7, 3])
    for got, w, bound in ((f64(y), want, y_bound(want, my, T, 64, True)),
                          (f64(pool)[1], ref[1], state_bound(ms[0], T))):
        ok = np.isfinite(w)
        assert (np.isnan(got) == np.isnan(w)).all() and (got[np.isinf(w)] == w[np.isinf(w)]).all()
        assert (np.abs(got[ok] - w[ok]) <= bound[ok]).all()


@pytest.mark.parametrize("zero_init", [False, True])
def test_a_piece_that_grows_past_fp32(dev, zero_init):
    """A piece's factor e^128 over a state of 1e-30 (or of zeros), then back: no entry passes fp32. (A
    chunk's exponent, 46 in powers of two, is rounded to fp32: 16 roundings' worth in each of the 8
    chunks here, of the 472 that the bound holds for 46.)"""
    T = 2900
    assert is_cut(1, T, 2, 2, 64, 64)
    before, q, k, v, _ = _inputs(62, T, 2, 2, 64, 64, rows=3)
    before *= 1e-30
    before[1, 0, :, 5] = 0
    k[:512] = 0
    g = torch.full((T, 2), -0.05)
    g[:256], g[256:512] = 0.5, -0.5
    pool, y = _run(dev, [0, T], [1], before, q, k, v, g, zero_init)
    _check(pool, y, before, [0, T], [1], q, k, v, g, 1.0, zero_init)


# -- chunks: growth across the middle ---------------------------------------------------------------

@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("K", [64, 128])
def test_growth_and_decay_across_the_middle_of_a_chunk(dev, K, f32):
    """e^(G_t - G_31) falls below fp32, e^(G_t - G_s) of the tokens s before does not. (The values behind
    are zeros, so that only these tokens and the state count.)"""
    T = 150
    before, q, k, v, _ = _inputs(63, T, 2, 2, K, 64, rows=3)
    g = torch.full((T, 2), -0.01)
    g[27:32], g[34:39] = 12.0, -20.0
    v[27:] = 0
    pool, y = _run(dev, [0, T], [1], before, q, k, v, g, f32=f32)
    _check(pool, y, before, [0, T], [1], q, k, v, g, 1.0)


# -- products before their decay ---------------------------------------------------------------------

@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("T", [100, 2900])
def test_growth_past_fp32_of_small_values(dev, T, f32):
    """Six tokens grow by e^90 in all, which passes fp32; what they grow does not."""
    before, q, k, v, _ = _inputs(66, T, 2, 2, 64, 64, rows=3)
    g = torch.full((T, 2), -0.01)
    g[T - 73:T - 70], g[T - 70:T - 67], g[T - 60:T - 57] = -30.0, 30.0, -40.0
    v[T - 76:T - 66] *= 1e-6
    pool, y = _run(dev, [0, T], [1], before, q, k, v, g, f32=f32)
    _check(pool, y, before, [0, T], [1], q, k, v, g, 1.0)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("first", [-50.0, -math.inf])
@pytest.mark.parametrize("T", [1, 40, 150, 2900])
def test_a_large_state_that_a_token_decays(dev, T, first, f32):
    """Queries times the state pass fp32 before its decay, and not under it."""
    before, q, k, v, g = _inputs(64, T, 2, 2, 64, 64, rows=3)
    q = q.abs() + 0.5
    before[1] = before[1].abs() * 3e37
    g[0] = first
    pool, y = _run(dev, [0, T], [1], before, q, k, v, g, f32=f32)
    _check(pool, y, before, [0, T], [1], q, k, v, g, 1.0)


@pytest.mark.parametrize("zero_init", [False, True])
@pytest.mark.parametrize("T", [90, 2900])
def test_large_queries_and_keys_of_small_values(dev, T, zero_init):
    """A score passes fp32; the state, which holds the keys times the values, does not."""
    before, q, k, v, g = _inputs(65, T, 2, 2, 64, 64, rows=3)
    at = T - 70
    q[at:at + 3] *= 1e20
    k[at:at + 3] *= 1e20
    v[at:at + 3] *= 1e-30
    pool, y = _run(dev, [0, T], [1], before, q, k, v, g, zero_init)
    _check(pool, y, before, [0, T], [1], q, k, v, g, 1.0, zero_init)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("H,Hq,K,V,T", [(2, 2, 128, 128, 200), (4, 2, 128, 64, 130), (3, 1, 64, 192, 77),
                                        (2, 1, 128, 64, 2900), (40, 40, 64, 64, 100)])
def test_a_sequence_that_is_run_again_leaves_the_others(dev, H, Hq, K, V, T, f32):
    """One of three sequences has large queries and keys of small values: it is as the formula says, the
    others as they are beside a usual one."""
    before, q, k, v, g = _inputs(67, 3 * T, H, Hq, K, V)
    g = g.clamp(max=-0.3)  # (a bound holds 8 additions for each 64 tokens of one by one: some 30 count)
    cu, ids = [0, T, 2 * T, 3 * T], [4, 1, 7]
    assert is_cut(3, 3 * T, H, Hq, K, V) == (T > 2000)
    usual_pool, usual = _run(dev, cu, ids, before, q, k, v, g, f32=f32)
    at = 2 * T - 40
    q[at] *= 1e20
    k[at] *= 1e20
    v[at] *= 1e-30
    pool, y = _run(dev, cu, ids, before, q, k, v, g, f32=f32)
    _check(pool, y, before, cu, ids, q, k, v, g, 1.0)
    rest = list(range(T)) + list(range(2 * T, 3 * T))
    assert torch.equal(y[rest], usual[rest]) and torch.equal(pool[[4, 7]], usual_pool[[4, 7]])


def test_outputs_over_the_inputs_are_refused(dev):
    before, q, k, v, g = _inputs(68, 70, 2, 2, 64, 64, rows=3)
    q, k, v, g = (t.to(dev) for t in (q, k, v, g))
    pool, both = before.to(dev), torch.zeros(140, 2, 64, dtype=BF16, device=dev)
    both[:70] = v
    for out in (q, k, v):
        with pytest.raises(ValueError, match="overlap"):
            linear_prefill_varlen(pool, [1], [0, 70], q, k, v, g, out=out)
    with pytest.raises(ValueError, match="overlap"):
        linear_prefill_varlen(pool, [1], [0, 70], q, k, both[:70], g, out=both[69:139])
    assert torch.equal(pool.cpu(), before)
    want = linear_prefill_varlen(pool.clone(), [1], [0, 70], q, k, v, g)
    linear_prefill_varlen(pool, [1], [0, 70], q, k, both[:70], g, out=both[70:])
    assert torch.equal(both[70:], want) and torch.equal(both[:70], v)
