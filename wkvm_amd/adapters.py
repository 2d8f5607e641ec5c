"""Low-rank adapters of many requests at once, beside the projections they share.

A batch whose requests run on different fine-tunings of one base model shares
every weight but the low-rank pairs (A, B): row m of a product with adapter a is
``act(x w^T + bias + scale_a (x A_a^T) B_a^T)``. ``AdapterBank`` holds the pairs of one
weight in the kernels' layout, ``adapter_plan`` the batch's adapter ids, and
``proj_adapters`` runs up to 8 products of a batch (a decode step's rows or
the tokens of packed prompts) in two launches whatever the mix.

The reference has no counterpart (its projections are plain nn.Linear calls of
the external model, wkvm/runner/runner.py:80-88).
"""

from __future__ import annotations

import ctypes
import math
from typing import Sequence

import numpy as np
import torch

from . import _lib, ops

_SLAB = _lib.WKV7_ADAPTER_SLAB
_SET_ARRAYS = [_lib.AdapterSet * n for n in range(_lib.WKV7_PROJ_MAX_GROUPS + 1)]


class AdapterBank:
    """The adapters of one ``[n, k]`` weight: ``num_adapters`` places of up to ``max_rank``
    ranks. ``a`` ``[N, R, k]`` and ``b`` ``[N, R/16, n, 16]`` bf16 hold the pairs with zeros
    past each one's rank (R is ``max_rank`` rounded up to 16), ``scale`` fp32 and ``rank``
    int32 ``[N]`` the rest. An empty place has rank 0 and adds nothing."""

    def __init__(self, num_adapters: int, k: int, n: int, max_rank: int,
                 device: torch.device | str = "cuda") -> None:
        if num_adapters < 1:
            raise ValueError("num_adapters must be >= 1")
        if not 1 <= max_rank <= _lib.WKV7_ADAPTER_MAX_RANK:
            raise ValueError(f"max_rank must be in [1, {_lib.WKV7_ADAPTER_MAX_RANK}], "
                             f"got {max_rank}")
        if k < 32 or k % 32:
            raise ValueError(f"k must be a positive multiple of 32, got {k}")
        if n < 1:
            raise ValueError("n must be >= 1")
        self.num_adapters, self.k, self.n = int(num_adapters), int(k), int(n)
        self.max_rank = int(max_rank)
        self.device = torch.device(device)
        self.slabs = (self.max_rank + _SLAB - 1) // _SLAB
        bf16, dev = torch.bfloat16, self.device
        self.a = torch.zeros((num_adapters, self.slabs * _SLAB, k), dtype=bf16, device=dev)
        self.b = torch.zeros((num_adapters, self.slabs, n, _SLAB), dtype=bf16, device=dev)
        self.scale = torch.zeros(num_adapters, dtype=torch.float32, device=dev)
        self.rank = torch.zeros(num_adapters, dtype=torch.int32, device=dev)
        self.set = _lib.AdapterSet(self.a.data_ptr(), self.b.data_ptr(), self.scale.data_ptr(),
                                   self.rank.data_ptr(), self.num_adapters, self.slabs)

    def _check_place(self, index: int) -> int:
        if not 0 <= index < self.num_adapters:
            raise ValueError(f"adapter {index} out of range [0, {self.num_adapters})")
        return int(index)

    def load(self, index: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0) -> None:
        """Put the pair ``a [r, k]``, ``b [n, r]`` (bf16) with its factor (alpha / r) into a
        place, on the current stream."""
        index = self._check_place(index)
        for t, name in ((a, "a"), (b, "b")):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16 or t.dim() != 2:
                raise ValueError(f"{name} must be a 2-D bfloat16 tensor")
        r = int(a.shape[0])
        if not 1 <= r <= self.max_rank:
            raise ValueError(f"rank must be in [1, {self.max_rank}], got {r}")
        if tuple(a.shape) != (r, self.k) or tuple(b.shape) != (self.n, r):
            raise ValueError(f"a must be [{r}, {self.k}] and b [{self.n}, {r}], got "
                             f"{tuple(a.shape)} and {tuple(b.shape)}")
        if not math.isfinite(ctypes.c_float(scale).value):  # (as the kernels hold it)
            raise ValueError(f"scale must be finite in 32 bits, got {scale}")
        for t, name in ((a, "a"), (b, "b")):
            ops._require_cuda(t, name)
            if t.device != self.a.device:
                raise ValueError(f"{name} on {t.device}, the bank on {self.a.device}")
        if a.stride(1) != 1 or r > 1 and a.stride(0) < self.k:
            a = a.contiguous()
        if b.stride(1) != 1 or self.n > 1 and b.stride(0) < r:
            b = b.contiguous()
        rc = _lib.load().wkv7_adapter_load(self.set, index, self.n, self.k, a.data_ptr(),
                                           max(a.stride(0), self.k), b.data_ptr(),
                                           max(b.stride(0), r), r, float(scale),
                                           ops._stream_ptr(self.a.device))
        _lib.check(rc, "wkv7_adapter_load")

    def clear(self, index: int) -> None:
        """Empty a place: rows that name it get the shared product alone."""
        self.rank[self._check_place(index)] = 0


class AdapterPlan:
    """A batch's adapter ids on the device: its rows in the order of their adapters."""

    def __init__(self, rows: int, num_adapters: int, buf: torch.Tensor) -> None:
        self.rows, self.num_adapters, self.buf = rows, num_adapters, buf
        self._made_on = ops._stream_ptr(buf.device) if buf.is_cuda else None

    def use(self) -> int:
        """The plan's address for a launch on the current stream, on which its memory is then in
        use also after the plan is dropped. (A graph capture leaves keeping it to the caller.)"""
        if ops._stream_ptr(self.buf.device) != self._made_on and \
                not torch.cuda.is_current_stream_capturing():
            self.buf.record_stream(torch.cuda.current_stream(self.buf.device))
        return self.buf.data_ptr()


def plan_ints(ids, num_adapters: int) -> np.ndarray:
    """The plan of ``ids`` (host integers, -1: no adapter) in host memory."""
    if isinstance(ids, torch.Tensor):
        ids = ids.tolist() if ids.is_cuda else ids.numpy()
    wide = np.asarray(ids, dtype=np.int64).reshape(-1)
    bad = wide[(wide < -1) | (wide >= num_adapters)]
    if bad.size:
        raise ValueError(f"adapter id {bad[0]} out of range [-1, {num_adapters})")
    flat = np.ascontiguousarray(wide, dtype=np.int32)
    lib = _lib.load()
    out = np.empty(lib.wkv7_adapter_plan_ints(flat.size, num_adapters), dtype=np.int32)
    rc = lib.wkv7_adapter_plan(flat.ctypes.data, flat.size, num_adapters, out.ctypes.data, out.size)
    _lib.check(rc, "wkv7_adapter_plan")
    return out


def adapter_plan(ids, num_adapters: int, device: torch.device | str = "cuda") -> AdapterPlan:
    """Device plan of a batch whose row m runs on adapter ``ids[m]`` (host integers; -1: the
    base model alone). It is complete when returned, serves every product of the batch
    and stays right for as long as the rows keep their adapters. Refused under graph
    capture, before the stream is touched: a replay would not see other ids."""
    device = torch.device(device)
    if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("adapter_plan under graph capture: its ids are host values")
    host = plan_ints(ids, num_adapters)
    rows = int(np.asarray(ids).size) if not isinstance(ids, torch.Tensor) else ids.numel()
    return AdapterPlan(rows, int(num_adapters), torch.from_numpy(host).to(device))


def proj_adapters(products: Sequence[tuple], plan: AdapterPlan,
                  outs: Sequence[torch.Tensor | None] | None = None) -> list[torch.Tensor]:
    """``ops.proj_grouped`` with the rows' adapters beside the shared weights
    (``wkv7_proj_adapters``): ``products`` holds up to 8 tuples ``(x, w, bias, act, bank)``, all but
    the first two optional; ``bank`` is the ``AdapterBank`` of ``w`` or None. Every ``x`` has the
    plan's row count, at most 2^28. Returns the ``[M, n]`` bf16 outputs."""
    groups, ys, keep, M = ops.proj_groups(products, outs)
    if M != plan.rows:
        raise ValueError(f"products of {M} rows for a plan of {plan.rows}")
    n = len(products)
    dev = ys[0].device
    if plan.buf.device != dev:
        raise ValueError(f"plan on {plan.buf.device}, products on {dev}")
    sets = _SET_ARRAYS[n]()
    for i, prod in enumerate(products):
        bank = prod[4] if len(prod) > 4 else None
        if bank is None:
            continue
        group = groups[i]
        if bank.k != group.k or bank.n != group.n:
            raise ValueError(f"adapters of a [{bank.n}, {bank.k}] weight beside a "
                             f"[{group.n}, {group.k}] one")
        if bank.num_adapters < plan.num_adapters:
            raise ValueError(f"a bank of {bank.num_adapters} adapters for a plan of "
                             f"{plan.num_adapters}")
        if bank.a.device != dev:
            raise ValueError(f"adapters on {bank.a.device}, products on {dev}")
        sets[i] = bank.set
    if M:
        lib = _lib.load()
        ws_bytes = int(lib.wkv7_proj_adapters_workspace_bytes(M, groups, sets, n,
                                                              plan.num_adapters))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
        rc = lib.wkv7_proj_adapters(M, groups, sets, n, plan.use(), plan.num_adapters,
                                    ops._ptr(ws), ws_bytes, ops._stream_ptr(dev))
        _lib.check(rc, "wkv7_proj_adapters")
    return ys
