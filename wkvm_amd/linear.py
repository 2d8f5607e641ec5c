"""Linear attention with a decay for each head, over the slot pool.

Layers whose state has the slots of a WKV7 layer and a plainer update: per token and head

    S <- exp(g) S + k v^T        y = scale q^T S

with ``S [K, V]`` fp32 in its slot's row and a log-decay ``g`` that is fixed for a head or comes from
the token. ``linear_decode_slots`` advances one token per slot, ``linear_prefill_varlen`` ragged prompts
in chunks on the matrix cores; both take slot ids, offsets and outputs as ``wkv7_decode_slots`` and
``wkv7_prefill_varlen`` do, and refuse what those refuse.

The reference has no counterpart (its recurrent layers are RWKV-7's, wkvm/models/rwkv7.py:38-113).
"""

from __future__ import annotations

import contextlib
import ctypes
import struct

import torch

from . import _lib, ops

KEY_SIZES = (64, 128)
_IO_PACK = struct.Struct("@QQQQQqqqqiiiiif")  # the fields of LinearIO
assert _IO_PACK.size == ctypes.sizeof(_lib.LinearIO)
_MAX_LD = 1 << 24  # elements from one token to the next that the kernels address


_HERE = contextlib.nullcontext()


def on_device(device: torch.device):
    """A context in which ``device`` is the current one (launches go to the current device)."""
    if device.index is None or device.index == torch.cuda.current_device():
        return _HERE
    return torch.cuda.device(device)


def _check_state(state: torch.Tensor) -> tuple[int, int, int, int]:
    ops._require_cuda(state, "state")
    if state.dtype != torch.float32:
        raise ValueError(f"state must be float32, got {state.dtype}")
    if state.dim() != 4:
        raise ValueError(f"state must be [rows, H, K, V], got {tuple(state.shape)}")
    rows, H, K, V = state.shape
    if rows < 1 or H < 1:
        raise ValueError(f"state must have rows and heads, got {tuple(state.shape)}")
    if K not in KEY_SIZES:
        raise ValueError(f"K must be one of {KEY_SIZES}, got {K}")
    if V < 64 or V % 64 or V > _lib.WKV7_LINEAR_MAX_V:
        raise ValueError(f"V must be a multiple of 64 up to {_lib.WKV7_LINEAR_MAX_V}, got {V}")
    if not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError("state must be contiguous and 16-byte aligned")
    return rows, H, K, V


def _vectors(x: torch.Tensor, name: str, tokens: int, size: int, device: torch.device):
    """``[tokens, heads, size]`` bf16 with whole tokens in one piece (copied where they are not), its
    heads and the elements from one token to the next."""
    if not (isinstance(x, torch.Tensor) and x.is_cuda):
        ops._require_cuda(x, name)
    if x.dtype is not torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16, got {x.dtype}")
    shape = x.shape
    if len(shape) != 3 or shape[0] != tokens or shape[2] != size:
        raise ValueError(f"{name} must be [{tokens}, heads, {size}], got {tuple(shape)}")
    if x.device != device:
        raise ValueError(f"{name} on {x.device}, state on {device}")
    heads = shape[1]
    own = heads * size
    ld, sh, se = x.stride()
    if tokens <= 1:
        ld = own
    if (se != 1 or heads > 1 and sh != size or ld < own or ld % 8 or ld > _MAX_LD
            or x.data_ptr() % 16):
        x = x.clone(memory_format=torch.contiguous_format)
        ld = own
    return x, heads, ld


def _span(x: torch.Tensor) -> tuple[int, int]:
    """Addresses from the first element of ``x`` to behind its last."""
    last = sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
    return x.data_ptr(), x.data_ptr() + (last + 1) * x.element_size()


def overlaps(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory from a's first to its last element meets b's."""
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def _io(q, k, v, log_decay, dims, dev, tokens, scale, out, out_dtype):
    """The checked vectors as a ``LinearIO``, the output and the tensors that the launch reads;
    ``dims`` are the state's."""
    rows, H, K, V = dims
    q, Hq, ldq = _vectors(q, "q", tokens, K, dev)
    k, Hk, ldk = _vectors(k, "k", tokens, K, dev)
    v, Hv, ldv = _vectors(v, "v", tokens, V, dev)
    if Hk != Hq:
        raise ValueError(f"q has {Hq} heads, k {Hk}")
    if Hv != H:
        raise ValueError(f"v has {Hv} heads, the state {H}")
    if Hq < 1 or H % Hq:
        raise ValueError(f"the state's {H} heads must be a multiple of the {Hq} of q and k")
    ops._require_cuda(log_decay, "log_decay")
    if log_decay.dtype is not torch.float32:
        raise ValueError(f"log_decay must be float32, got {log_decay.dtype}")
    if log_decay.shape not in ((H,), (tokens, H)):
        raise ValueError(f"log_decay must be [{H}] or [{tokens}, {H}], got "
                         f"{tuple(log_decay.shape)}")
    if log_decay.device != dev:
        raise ValueError(f"log_decay on {log_decay.device}, state on {dev}")
    fixed = log_decay.dim() == 1
    if not log_decay.is_contiguous() and (
            H > 1 and log_decay.stride(-1) != 1
            or not fixed and tokens > 1 and log_decay.stride(0) < H):
        log_decay = log_decay.clone(memory_format=torch.contiguous_format)
    ldd = 0 if fixed else H if tokens <= 1 else log_decay.stride(0)
    dtype = out.dtype if out is not None else out_dtype
    code = ops._y_code(dtype)
    if out is None:
        y = torch.empty((tokens, H, V), dtype=dtype, device=dev)
    else:
        y = ops._out(out, (tokens, H, V), dtype, dev, "out")
        if y.device != dev or y.data_ptr() % 16:
            raise ValueError("out must be 16-byte aligned and on the state's device")
    io = _lib.LinearIO.from_buffer(bytearray(_IO_PACK.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), y.data_ptr(), ldq, ldk, ldv,
        ldd, H, Hq, K, V, code, scale)))
    return io, y, (q, k, v, log_decay)


def linear_decode_slots(state: torch.Tensor, slot_ids, q, k, v, log_decay, *, scale: float = 1.0,
                        out: torch.Tensor | None = None,
                        out_dtype: torch.dtype = torch.bfloat16,
                        row_order: torch.Tensor | None = None) -> torch.Tensor:
    """One token per slot, in place on ``state`` (``[rows, H, K, V]`` fp32, K 64 or 128, V a multiple of
    64).

    ``q``, ``k`` bf16 ``[B, Hq, K]`` (H a multiple of Hq: head h reads head ``h // (H / Hq)``), ``v``
    bf16 ``[B, H, V]``, rows of any stride; ``log_decay`` fp32 ``[H]`` or ``[B, H]``. Returns
    ``y [B, H, V]`` in ``out_dtype`` (bf16 or fp32; computed in fp32, rounded once). ``slot_ids`` and
    ``row_order`` as for ``wkv7_decode_slots``."""
    dims = _check_state(state)
    rows, dev = dims[0], state.device
    ids, order = ops.decode_plan(slot_ids, rows, dev, wait=False)
    B = int(ids.shape[0])
    if row_order is not None:
        order = ops.packed_ints(row_order, B, dev, "row_order")
    io, y, keep = _io(q, k, v, log_decay, dims, dev, B, scale, out, out_dtype)
    if B:
        with on_device(dev):
            rc = _lib.load().wkv7_linear_decode(state.data_ptr(), rows, ids.data_ptr(),
                                                ops._ptr(order), B, io, ops._stream_ptr(dev))
        _lib.check(rc, "wkv7_linear_decode")
    return y


def linear_prefill_varlen(state: torch.Tensor, slot_ids, cu_seqlens, q, k, v, log_decay, *,
                          zero_init: bool = False, scale: float = 1.0,
                          out: torch.Tensor | None = None,
                          out_dtype: torch.dtype = torch.bfloat16,
                          seq_order: torch.Tensor | None = None) -> torch.Tensor:
    """Ragged prompts: sequence ``s`` runs tokens ``cu_seqlens[s]:cu_seqlens[s+1]`` from the state of
    slot ``slot_ids[s]`` (from zero with ``zero_init``) and leaves its final state there; an empty
    sequence leaves it as it is (zeroes it with ``zero_init``).

    ``q``, ``k``, ``v``, ``log_decay`` and the result as for ``linear_decode_slots``, over the T packed
    tokens (``out`` may not overlap them). ``cu_seqlens`` is a host sequence or a device int32 tensor, ``seq_order`` as for
    ``wkv7_prefill_varlen``. A token's output does not depend on later tokens, whatever they hold. Few
    sequences are cut into pieces that run side by side, through a workspace from torch's
    allocator."""
    dims = _check_state(state)
    rows, dev = dims[0], state.device
    ids = ops.device_ids(slot_ids, rows, dev, "slot_ids", distinct=True, wait=False)
    nseq = int(ids.shape[0])
    ops._require_cuda(v, "v")
    T = int(v.shape[0]) if v.dim() == 3 else -1
    io, y, keep = _io(q, k, v, log_decay, dims, dev, T, scale, out, out_dtype)
    if out is not None and any(overlaps(out, x) for x in (*keep, state)):
        raise ValueError("out must not overlap the inputs, which may be read again")
    if isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.is_cuda:
        cu = ops.packed_ints(cu_seqlens, nseq + 1, dev, "cu_seqlens")
    else:
        lst = ops._host_cu(cu_seqlens, T)
        if len(lst) != nseq + 1:
            raise ValueError(f"cu_seqlens has {len(lst)} entries for {nseq} sequences")
        cu = ops._device_plan(lst, dev)
        if seq_order is None:
            seq_order = cu[nseq + 1:]
    if seq_order is not None:
        ops.packed_ints(seq_order, nseq, dev, "seq_order")
    if nseq:
        lib = _lib.load()
        with on_device(dev):
            ws_bytes = int(lib.wkv7_linear_prefill_workspace_bytes(nseq, T, io))
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
            rc = lib.wkv7_linear_prefill(state.data_ptr(), rows, ids.data_ptr(), cu.data_ptr(),
                                         ops._ptr(seq_order), nseq, T, io, int(bool(zero_init)),
                                         ops._ptr(ws), ws_bytes, ops._stream_ptr(dev))
        _lib.check(rc, "wkv7_linear_prefill")
    return y
