"""Sampling of a decode batch's next tokens on the GPU.

The reference samples per request on the host, from logits copied back
(``sample_token``, wkvm/runner/sampling.py:40), and takes a batched argmax for
greedy decoding (wkvm/engine.py:163). Here every row of a batch is sampled in
one call (two launches) by its own temperature, top-k, top-p and min-p, from random numbers
that the caller brings, so a request's tokens do not depend on the batch
around it.
"""

from __future__ import annotations

import math

import numpy as np
import torch

from . import _lib, ops

SAMPLE_GROUP = _lib.WKV7_SAMPLE_GROUP


def sample_noise_size(vocab: int) -> int:
    """Random numbers that one row of ``vocab`` logits takes: one per token of a
    group of 256 and one per group."""
    return SAMPLE_GROUP + (int(vocab) + SAMPLE_GROUP - 1) // SAMPLE_GROUP


# name -> (dtype of the per-row tensor, lowest and highest value)
_SETTINGS = {"temperature": (torch.float32, 0.0, math.inf), "top_k": (torch.int32, 0, 2**31 - 1),
             "top_p": (torch.float32, 0.0, 1.0), "min_p": (torch.float32, 0.0, 1.0)}


def _setting(name: str, value, rows: int, device: torch.device):
    """``(per-row tensor or None, value of every row)``. Numbers and host
    sequences are checked; a device tensor is taken as it is (the kernel holds
    its values to the ranges)."""
    dtype, lo, hi = _SETTINGS[name]
    if isinstance(value, torch.Tensor) and value.is_cuda:
        if (value.dtype != dtype or value.shape != (rows,) or value.device != device
                or not value.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous {dtype} tensor of {rows} values on "
                             f"{device}")
        return value, 0
    if isinstance(value, (torch.Tensor, np.ndarray)):
        if value.ndim > 1:
            raise ValueError(f"{name} must be a number or {rows} values, got {tuple(value.shape)}")
        value = value.tolist()
    many = value if isinstance(value, ops._IDS) else [value]
    for v in many:
        if not lo <= v <= hi or (dtype is torch.int32 and v != int(v)):  # (NaN fails too)
            raise ValueError(f"{name} must be in [{lo}, {hi}], got {v}")
    if many is not value:
        return None, int(value) if dtype is torch.int32 else float(value)
    if len(many) != rows:
        raise ValueError(f"{len(many)} values of {name} for {rows} rows")
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{name} given as host values under graph capture: pass a device tensor")
    return torch.tensor(many, dtype=dtype, pin_memory=True).to(device, non_blocking=True), 0


def sample_tokens(logits: torch.Tensor, noise: torch.Tensor, *, temperature=1.0, top_k=0,
                  top_p=1.0, min_p=0.0, logprobs: bool = True,
                  ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The next token of every row of ``logits [B, V]`` (bf16 or fp32, rows may be
    strided) and its log-probability ``x - logsumexp(row)``.

    The settings are numbers (all rows), host sequences or device tensors of B
    values (fp32; ``top_k`` int32). After the temperature, ``top_k`` keeps the
    largest logits (0: all), ``top_p`` of those the shortest prefix that reaches
    that share of their probability (1: all), ``min_p`` of those the tokens with
    at least that share of the largest probability (0: all); equal logits are
    ordered by index. Temperature 0 is greedy. NaN logits count as -inf and
    +inf as the largest finite number; a row with nothing above -inf gets token -1.

    ``noise [B, sample_noise_size(V)]`` fp32 holds independent exponential variates
    (``torch.empty(..).exponential_(generator=g)``): one per group of 256 tokens decides
    the group, one per token of it the token.

    Returns ``(tokens [B] int32, logprobs [B] fp32, or None)``.
    """
    ops._require_cuda(logits, "logits")
    ops._require_cuda(noise, "noise")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be [B, V], got {tuple(logits.shape)}")
    code = ops._y_code(logits.dtype)
    B, V = logits.shape
    dev = logits.device
    if V > _lib.WKV7_SAMPLE_MAX_VOCAB:
        raise ValueError(f"at most {_lib.WKV7_SAMPLE_MAX_VOCAB} tokens per row, got {V}")
    if noise.dtype != torch.float32 or noise.dim() != 2 or noise.shape[0] != B or \
            noise.shape[1] < sample_noise_size(V) or noise.device != dev:
        raise ValueError(f"noise must be float32 [{B}, {sample_noise_size(V)}] on {dev}, got "
                         f"{noise.dtype} {tuple(noise.shape)} on {noise.device}")
    if logits.stride(1) != 1 or B > 1 and logits.stride(0) < V:
        logits = logits.contiguous()
    if noise.stride(1) != 1 or B > 1 and noise.stride(0) < noise.shape[1]:
        noise = noise.contiguous()
    got = {n: _setting(n, v, B, dev) for n, v in (("temperature", temperature), ("top_k", top_k),
                                                   ("top_p", top_p), ("min_p", min_p))}
    tokens = torch.empty(B, dtype=torch.int32, device=dev)
    logp = torch.empty(B, dtype=torch.float32, device=dev) if logprobs else None
    if B == 0:
        return tokens, logp
    params = _lib.SampleParams(*(ops._ptr(t) for t, _ in got.values()),
                               *(v for _, v in got.values()))
    lib = _lib.load()
    ws = torch.empty(lib.wkv7_sample_workspace_bytes(B, V), dtype=torch.uint8, device=dev)
    rc = lib.wkv7_sample_tokens(
        logits.data_ptr(), code, B, V, logits.stride(0) if B > 1 else V, noise.data_ptr(),
        noise.stride(0) if B > 1 else noise.shape[1], params, tokens.data_ptr(), ops._ptr(logp),
        ws.data_ptr(), ws.numel(), ops._stream_ptr(dev))
    _lib.check(rc, "wkv7_sample_tokens")
    return tokens, logp
