"""Linear attention with head decays from its definition, token by token in float64, with the
magnitudes that the tests' bounds are relative to."""

from __future__ import annotations

import numpy as np


def scan(state, cu, ids, q, k, v, g, scale, zero_init=False):
    """``state [rows, H, K, V]`` float64 (changed in place), host arrays q, k ``[T, Hq, K]``, v ``[T, H,
    V]``, g ``[T, H]`` or ``[H]``. Returns ``(y, my, ms)``: outputs, the outputs' and the final states'
    sums of absolute terms (``ms`` shaped like the sequences' states)."""
    T, H, V = v.shape
    Hq = q.shape[1]
    whose = np.arange(H) // (H // Hq)
    if g.ndim == 1:
        g = np.broadcast_to(g, (T, H))
    y, my = np.zeros((T, H, V)), np.zeros((T, H, V))
    ms = np.zeros((len(ids),) + state.shape[1:])
    with np.errstate(invalid="ignore", over="ignore"):
        for s, row in enumerate(ids):
            h = np.zeros(state.shape[1:]) if zero_init else state[row].copy()
            m = np.abs(h)
            for t in range(cu[s], cu[s + 1]):
                d = np.exp(g[t])[:, None, None]
                qt, kt = q[t][whose], k[t][whose]
                kv = kt[:, :, None] * v[t][:, None, :]
                h = d * h + kv
                m = d * m + np.abs(kv)
                y[t] = scale * np.einsum("hk,hkv->hv", qt, h)
                my[t] = abs(scale) * np.einsum("hk,hkv->hv", np.abs(qt), m)
            state[row] = h
            ms[s] = m
    return y, my, ms


def state_bound(ms, tokens):
    """Of the final states of sequences of up to ``tokens`` tokens, relative to their absolute terms.
    In a chunk: at most 38 fp32 additions (6 products of 32 terms), the decayed key's rounding, an
    exponential (2^-22) of a difference that is itself off by 2^-24 of it (of weight 2^-d at a
    distance d, so 2^-24 at most): under 48 roundings, taken twice. Each later chunk multiplies by
    an exponential (4 roundings), rounds the product and adds: 8."""
    return 2.0 ** -24 * (96 + 8 * (tokens // 64 + 1)) * ms + 1e-37


def y_bound(y, my, tokens, K, f32):
    """Of the outputs: K products per score and per state column, at most 128 further additions, the
    state's own bound; for bf16 its rounding and the two-part split of scores and state (2^-18)."""
    fp32 = 2.0 ** -24 * (K + 128 + 96 + 8 * (tokens // 64 + 1)) * my + 1e-37
    return fp32 if f32 else fp32 + 2.0 ** -8 * np.abs(y) + 2.0 ** -18 * my
