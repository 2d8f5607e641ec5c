"""linear_prefill_varlen where sequences are cut into pieces: every test here asks the library whether
its case is cut, so that none of them runs whole by a changed rule."""

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


def test_pieces_find_their_sequence_among_more_than_a_wave(dev):
    """70 sequences, some of them empty, the first and the last among these."""
    rng = np.random.default_rng(3)
    lens = [int(n) if rng.random() < 0.5 else 0 for n in rng.integers(1, 4000, 70)]
    lens[0] = lens[69] = 0
    lens[66] = 168000 - sum(lens) + lens[66]
    ids = rng.permutation(np.arange(1, 81))[:70].tolist()
    _run(dev, 44, lens, ids, 1, 1, 64, 64, "token", True, rows=81)
