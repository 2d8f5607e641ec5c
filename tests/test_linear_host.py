"""Argument checks of the linear-attention entry points: host code, no GPU."""

import ctypes

import pytest
import torch

from wkvm_amd import _lib, linear_decode_slots, linear_prefill_varlen
from tests.linear_ref import scan

import numpy as np


def _io(**kw):
    p = ctypes.c_void_p(4096)
    io = _lib.LinearIO(p, p, p, p, p, 256, 256, 256, 4, 4, 4, 64, 64, 0, 1.0)
    for name, value in kw.items():
        setattr(io, name, value)
    return io


@pytest.mark.parametrize("change,code", [
    (dict(H=0), "ARG"), (dict(Hq=0), "ARG"), (dict(Hq=3), "ARG"), (dict(y_dtype=7), "ARG"),
    (dict(q=None), "ARG"), (dict(log_decay=None), "ARG"), (dict(y=None), "ARG"),
    (dict(K=32), "SHAPE"), (dict(K=96), "SHAPE"), (dict(V=0), "SHAPE"), (dict(V=96), "SHAPE"),
    (dict(V=2048), "SHAPE"), (dict(ldq=248), "SHAPE"), (dict(ldk=260), "SHAPE"),
    (dict(ldv=128), "SHAPE"), (dict(ld_decay=3), "SHAPE"), (dict(q=4098), "SHAPE"),
    (dict(v=4104), "SHAPE"), (dict(y=4100), "SHAPE"), (dict(log_decay=4098), "SHAPE")])
def test_abi_refusals(change, code):
    lib, dummy = _lib.load(), ctypes.c_void_p(4096)
    want = getattr(_lib, "WKV7_ERR_" + code)
    io = _io(**change)
    assert lib.wkv7_linear_decode(dummy, 5, dummy, None, 2, io, None) == want
    assert lib.wkv7_linear_prefill(dummy, 5, dummy, dummy, None, 1, 2, io, 0, None, 0, None) == want


def test_abi_refusals_of_the_call():
    lib, p, io = _lib.load(), ctypes.c_void_p(4096), _io()
    A, S = _lib.WKV7_ERR_ARG, _lib.WKV7_ERR_SHAPE
    assert lib.wkv7_linear_decode(None, 5, p, None, 2, io, None) == A
    assert lib.wkv7_linear_decode(ctypes.c_void_p(4104), 5, p, None, 2, io, None) == S
    assert lib.wkv7_linear_decode(p, 0, p, None, 2, io, None) == A
    assert lib.wkv7_linear_decode(p, 5, None, None, 2, io, None) == A
    assert lib.wkv7_linear_decode(p, 5, p, None, -1, io, None) == A
    assert lib.wkv7_linear_decode(p, 5, p, None, 2, None, None) == A
    assert lib.wkv7_linear_decode(p, 5, None, None, 0, io, None) == _lib.WKV7_OK
    assert lib.wkv7_linear_prefill(p, 5, p, p, None, -1, 2, io, 0, None, 0, None) == A
    assert lib.wkv7_linear_prefill(p, 5, None, p, None, 1, 2, io, 0, None, 0, None) == A
    assert lib.wkv7_linear_prefill(p, 5, p, None, None, 1, 2, io, 0, None, 0, None) == A
    assert lib.wkv7_linear_prefill(p, 5, p, p, None, 1, 1 << 31, io, 0, None, 0, None) == A
    assert lib.wkv7_linear_prefill(p, 5, p, p, None, 1, -1, io, 0, None, 0, None) == A
    assert lib.wkv7_linear_prefill(p, 5, None, None, None, 0, 0, io, 0, None, 0, None) == _lib.WKV7_OK
    assert lib.wkv7_linear_prefill_workspace_bytes(0, 100, io) == 0
    assert lib.wkv7_linear_prefill_workspace_bytes(1, 100, None) == 0


def test_there_is_no_cpu_path():
    pool = torch.zeros(3, 2, 64, 64)
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU tensor"):
        linear_decode_slots(pool, [1], x, x, x, torch.zeros(2))
    with pytest.raises(ValueError, match="GPU tensor"):
        linear_prefill_varlen(pool, [1], [0, 1], x, x, x, torch.zeros(2))


def test_the_reference_is_the_sum_over_tokens():
    """y_t = scale sum_{s <= t} e^(g_{s+1} + .. + g_t) (q_t . k_s) v_s, plus the initial state's part."""
    rng = np.random.default_rng(0)
    T, H, K, V = 9, 2, 4, 3
    q, k, v = rng.normal(size=(T, 1, K)), rng.normal(size=(T, 1, K)), rng.normal(size=(T, H, V))
    g = -rng.random((T, H))
    state = rng.normal(size=(2, H, K, V))
    s0 = state[1].copy()
    y, _, _ = scan(state, [0, T], [1], q, k, v, g, 0.5)
    G = np.cumsum(g, 0)
    for h in range(H):
        for t in range(T):
            want = np.exp(G[t, h]) * q[t, 0] @ s0[h]
            for s in range(t + 1):
                want = want + np.exp(G[t, h] - G[s, h]) * (q[t, 0] @ k[s, 0]) * v[s, h]
            np.testing.assert_allclose(y[t, h], 0.5 * want, rtol=1e-12)


def test_overlaps():
    from wkvm_amd.linear import overlaps

    buf = torch.zeros(12, 8)
    assert overlaps(buf, buf) and overlaps(buf[:6], buf[5:]) and overlaps(buf[:, :2], buf[:, 4:])
    assert not overlaps(buf[:6], buf[6:]) and not overlaps(buf[:0], buf)
    assert not overlaps(buf[:1, :4], buf[:1, 4:]) and not overlaps(buf, torch.zeros(12, 8))
    assert overlaps(buf[3].expand(5, 8), buf[3:4]) and not overlaps(buf[3].expand(5, 8), buf[4:])
