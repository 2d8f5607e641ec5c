"""Projections with 4-bit weights: codes with a scale and a zero point for each group of inputs.

``W4Weight`` holds one ``[n, k]`` weight in the kernels' layout, made from a checkpoint's codes, scales
and zero points (``from_codes``) or by rounding a bf16 weight (``quantize``); ``proj_w4`` runs up to 8
products ``act(x W^T + bias)`` of a batch in one call, as ``ops.proj_grouped`` does with bf16 weights.
They take a quarter of the memory, and products of few rows, which are bound by the weights' bytes, less
time; from some hundred rows on they take as long as with bf16 weights, those of prompts longer (three of
4096 x 4096: 16 rows 11 us; 256 rows 41, bf16 in the library 41 to 56; 4,096 rows 411, bf16 303).

The reference has no counterpart (its projections are plain nn.Linear calls of the external model,
wkvm/runner/runner.py:80-88).
"""

from __future__ import annotations

import ctypes
import struct
from typing import Sequence

import torch

from . import _lib, ops
from .linear import on_device

GROUPS = (32, 64, 128)
_GROUP_ARRAYS = [_lib.W4Group * n for n in range(_lib.WKV7_PROJ_MAX_GROUPS + 1)]
_GROUP_PACK = struct.Struct("@QQQiiiiQQqqii")  # the fields of W4Group
assert _GROUP_PACK.size == ctypes.sizeof(_lib.W4Group)


class W4Weight:
    """One ``[n, k]`` weight as 4-bit codes: ``W[n, k] = s (c - z)`` with a scale s and a zero point z in
    0 .. 15 for each row and ``group`` (32, 64 or 128) consecutive inputs, the last group possibly
    shorter. ``codes`` and ``scales`` are device buffers in the kernels' layout, zeros until they
    are filled."""

    def __init__(self, n: int, k: int, group: int = 128,
                 device: torch.device | str = "cuda") -> None:
        self._hold(n, k, group, device)
        self._codes.zero_()
        self._scales.zero_()

    def _hold(self, n: int, k: int, group: int, device) -> W4Weight:
        """Checks the sizes and allocates the buffers."""
        if n < 1:
            raise ValueError("n must be >= 1")
        if k < 32 or k % 32:
            raise ValueError(f"k must be a positive multiple of 32, got {k}")
        if group not in GROUPS:
            raise ValueError(f"group must be one of {GROUPS}, got {group}")
        self.n, self.k, self.group = int(n), int(k), int(group)
        self.groups = (self.k + self.group - 1) // self.group
        lib = _lib.load()
        self._codes = torch.empty(lib.wkv7_w4_code_bytes(n, k) // 4, dtype=torch.int32,
                                  device=device)
        self._scales = torch.empty(lib.wkv7_w4_scale_bytes(n, k, group) // 4, dtype=torch.int32,
                                   device=device)
        self.device = self._codes.device
        self.fields = (self._codes.data_ptr(), self._scales.data_ptr(), self.n, self.k, self.group, 0)
        self.desc = _lib.W4Desc(*self.fields)
        return self

    # (the launches hold the buffers' addresses: they are written into, not replaced)
    @property
    def codes(self) -> torch.Tensor:
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        return self._scales

    @property
    def shape(self) -> tuple[int, int]:
        return self.n, self.k

    def nbytes(self) -> int:
        return 4 * (self.codes.numel() + self.scales.numel())

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None = None,
                   group: int = 128) -> W4Weight:
        """From codes ``[n, k]`` (uint8, 0 .. 15), scales ``[n, ceil(k / group)]`` (bf16 or fp16, finite)
        and zero points (uint8, 0 .. 15, of the scales' shape; None: 8). Checks the values, so it waits
        for the device."""
        ops._require_cuda(codes, "codes")
        if codes.dtype != torch.uint8 or codes.dim() != 2:
            raise ValueError("codes must be a 2-D uint8 tensor")
        n, k = codes.shape
        weight = cls.__new__(cls)._hold(n, k, group, codes.device)
        want = (n, weight.groups)
        ops._require_cuda(scale, "scale")
        if scale.dtype not in (torch.bfloat16, torch.float16) or tuple(scale.shape) != want:
            raise ValueError(f"scale must be a bf16 or fp16 {want} tensor, got {scale.dtype} "
                             f"{tuple(scale.shape)}")
        if zero is not None:
            ops._require_cuda(zero, "zero")
            if zero.dtype != torch.uint8 or tuple(zero.shape) != want:
                raise ValueError(f"zero must be a uint8 {want} tensor, got {zero.dtype} "
                                 f"{tuple(zero.shape)}")
        for t, name in ((scale, "scale"), (zero, "zero")):
            if t is not None and t.device != codes.device:
                raise ValueError(f"{name} on {t.device}, codes on {codes.device}")
        wrong = torch.stack([codes.amax() > 15, codes.new_zeros((), dtype=torch.bool) if zero is None
                             else zero.amax() > 15, ~torch.isfinite(scale).all()]).tolist()
        if wrong[0] or wrong[1]:
            raise ValueError("codes and zero points must be in 0 .. 15")
        if wrong[2]:
            raise ValueError("scales must be finite")
        codes, scale = codes.contiguous(), scale.contiguous()
        zero = None if zero is None else zero.contiguous()
        kind = _lib.WKV7_SCALE_BF16 if scale.dtype == torch.bfloat16 else _lib.WKV7_SCALE_F16
        with on_device(weight.device):
            rc = _lib.load().wkv7_w4_pack(weight.desc, codes.data_ptr(), scale.data_ptr(), kind,
                                          ops._ptr(zero), ops._stream_ptr(weight.device))
        _lib.check(rc, "wkv7_w4_pack")
        return weight

    @classmethod
    def quantize(cls, w: torch.Tensor, group: int = 128, symmetric: bool = False) -> W4Weight:
        """By rounding a finite bf16 weight ``[n, k]`` group by group to its range, zero among it
        (``symmetric``: to plus and minus its largest magnitude). Checks the values, so it waits for
        the device."""
        ops._require_cuda(w, "w")
        if w.dtype != torch.bfloat16 or w.dim() != 2:
            raise ValueError("w must be a 2-D bfloat16 tensor")
        n, k = w.shape
        weight = cls.__new__(cls)._hold(n, k, group, w.device)
        if not bool(torch.isfinite(w).all()):
            raise ValueError("the weight must be finite")
        if w.stride(1) != 1 or n > 1 and w.stride(0) < k:
            w = w.contiguous()
        with on_device(weight.device):
            rc = _lib.load().wkv7_w4_quantize(weight.desc, w.data_ptr(), max(w.stride(0), k),
                                              int(bool(symmetric)),
                                              ops._stream_ptr(weight.device))
        _lib.check(rc, "wkv7_w4_quantize")
        return weight

    def dequantize(self) -> torch.Tensor:
        """The values ``[n, k]`` in fp32."""
        ops._require_cuda(self.codes, "the weight")
        w = torch.empty((self.n, self.k), dtype=torch.float32, device=self.device)
        with on_device(self.device):
            rc = _lib.load().wkv7_w4_unpack(self.desc, w.data_ptr(), ops._stream_ptr(self.device))
        _lib.check(rc, "wkv7_w4_unpack")
        return w


def proj_w4(products: Sequence[tuple], outs: Sequence[torch.Tensor | None] | None = None,
            ) -> list[torch.Tensor]:
    """Independent projections ``act(x @ W.T + bias)`` with 4-bit weights in one call
    (``wkv7_proj_w4``): ``products`` holds up to 8 tuples ``(x, weight)``, ``(x, weight, bias)`` or
    ``(x, weight, bias, act)`` with ``weight`` a ``W4Weight`` and the rest as for ``ops.proj_grouped``:
    bf16 ``x [M, k]``, every one of the same M (any number of rows), ``bias [n]`` or None, ``act``
    None, ``"tanh"`` or ``"sigmoid"``. Returns the ``[M, n]`` bf16 outputs (written into ``outs[i]``
    where given). A group's ``x (16 + c)`` and ``x (16 + z)`` are summed in fp32 and subtracted, so errors
    are 2^-24 of the size of these terms, also where a code is near its zero point."""
    n_products = len(products)
    if not 1 <= n_products <= _lib.WKV7_PROJ_MAX_GROUPS:
        raise ValueError(f"1..{_lib.WKV7_PROJ_MAX_GROUPS} products per launch, got {n_products}")
    packed = bytearray(_GROUP_PACK.size * n_products)
    ys, keep = [], []
    M = dev = last = None
    bf16 = torch.bfloat16
    for i, prod in enumerate(products):
        x, w = prod[0], prod[1]
        bias = prod[2] if len(prod) > 2 else None
        act = prod[3] if len(prod) > 3 else None
        if act not in ops.ACTIVATIONS:
            raise ValueError(f"act must be one of {list(ops.ACTIVATIONS)}, got {act!r}")
        if not isinstance(w, W4Weight):
            raise ValueError(f"the weight must be a W4Weight, got {type(w).__name__}")
        if x is not last:  # (products often share one)
            if not (isinstance(x, torch.Tensor) and x.is_cuda):
                ops._require_cuda(x, "x")
            if x.dtype is not bf16 or x.dim() != 2:
                raise ValueError("x must be a 2-D bfloat16 tensor")
            last = x
            m, k = x.shape
            if M is None:
                M, dev = m, x.device
            if m != M:
                raise ValueError("every product needs the same row count")
            if x.device != dev:
                raise ValueError("projection tensors must share a device")
            ldx, step = x.stride()
            if m <= 1 and step == 1:
                ldx = k
            ptr = x.data_ptr()
            if step != 1 or ldx < k or ldx % 8 or ptr % 16:
                x = x.clone(memory_format=torch.contiguous_format)
                ldx, ptr = k, x.data_ptr()
            keep.append(x)
        if k != w.k:
            raise ValueError(f"x must be [{M}, {w.k}], got {tuple(last.shape)}")
        n = w.n
        if bias is None:
            bias_ptr = 0
        else:
            if not (bias.dtype is bf16 and bias.shape == (n,) and bias.is_contiguous()
                    and bias.is_cuda):
                bias = ops._bf16_2d(bias.reshape(-1), "bias", (n,))
            if bias.device != dev:
                raise ValueError("projection tensors must share a device")
            bias_ptr = bias.data_ptr()
            keep.append(bias)
        y = outs[i] if outs is not None and i < len(outs) else None
        if y is None:
            y = last.new_empty((M, n))
            ldy = n
        else:
            ops._require_cuda(y, "out")
            if y.dtype != bf16 or tuple(y.shape) != (M, n) or n > 1 and y.stride(1) != 1:
                raise ValueError(f"out must be a bf16 [{M}, {n}] tensor with unit column stride")
            if y.device != dev:
                raise ValueError("projection tensors must share a device")
            ldy = n if M <= 1 else y.stride(0)
        if w.device != dev:
            raise ValueError("projection tensors must share a device")
        _GROUP_PACK.pack_into(packed, _GROUP_PACK.size * i, ptr, *w.fields,
                              bias_ptr, y.data_ptr(), ldx, ldy, ops.ACTIVATIONS[act], 0)
        ys.append(y)
    if M:
        lib = _lib.load()
        groups = _GROUP_ARRAYS[n_products].from_buffer(packed)
        with on_device(dev):
            ws_bytes = (int(lib.wkv7_proj_w4_workspace_bytes(M, groups, n_products))
                        if M > _lib.WKV7_W4_NO_WORKSPACE_ROWS else 0)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
            rc = lib.wkv7_proj_w4(M, groups, n_products, ops._ptr(ws), ws_bytes,
                                  ops._stream_ptr(dev))
        _lib.check(rc, "wkv7_proj_w4")
    return ys
