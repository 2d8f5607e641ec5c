"""The adapter plan and the argument checks of the adapter and sampling entry points: all of it
host code, no GPU."""

import ctypes
import math

import numpy as np
import pytest
import torch

from wkvm_amd import (AdapterBank, AdapterPlan, _lib, adapter_plan, ops, proj_adapters,
                      sample_noise_size, sample_tokens)
from wkvm_amd.adapters import plan_ints
from wkvm_amd.layout import RWKV7StateLayout
from wkvm_amd.timemix import RWKV7TimeMix, TimeMixDecodeGraph

SLAB, PACKED, ALIGN = _lib.WKV7_ADAPTER_SLAB, 512, 32
TILE = 20  # ints of a tile: first position, rows, adapter, 0, its rows


def _parts(plan, m, count):
    """(order, adapter, end of its run) of every position, and the tiles that hold rows."""
    runs = min(m, count + 1)
    all_ = m if m <= PACKED else (m + (ALIGN - 1) * runs + ALIGN - 1) // ALIGN * ALIGN
    step = (all_ + 3) // 4 * 4
    order, ids, end = (plan[i * step:i * step + all_] for i in range(3))
    tiles = plan[3 * step:].reshape(-1, TILE)
    return order, ids, end, tiles[tiles[:, 1] > 0]


@pytest.mark.parametrize("m,count,kind", [
    (0, 3, "any"), (1, 1, "any"), (5, 3, "any"), (64, 64, "own"), (300, 7, "any"), (512, 4, "any"),
    (513, 4, "any"), (600, 200, "any"), (3000, 5, "runs"), (3000, 1, "none"), (2048, 3, "one")])
def test_plan(m, count, kind):
    rng = np.random.default_rng(m)
    ids = {"any": lambda: rng.integers(-1, count, m), "own": lambda: rng.permutation(m),
           "runs": lambda: np.sort(rng.integers(-1, count, m)), "none": lambda: np.full(m, -1),
           "one": lambda: np.zeros(m, int)}[kind]()
    order, adapter, end, tiles = _parts(plan_ints(ids, count), m, count)
    held = order >= 0
    assert sorted(order[held].tolist()) == list(range(m))  # every row once
    assert (adapter[held] == ids[order[held]]).all()
    assert (adapter[~held] == -1).all()
    # one run per adapter, in the rows' own order, none of them split; rows without one last
    used = [a for a in sorted(set(ids.tolist())) if a >= 0]
    for a in used:
        at = np.flatnonzero(adapter == a)
        assert (np.diff(at) == 1).all() and (end[at] == at[-1] + 1).all()
        assert (np.diff(order[at]) > 0).all()
        if m > PACKED:
            assert at[0] % ALIGN == 0
    none = np.flatnonzero(held & (adapter < 0))
    if none.size and used:
        assert none[0] > np.flatnonzero(adapter >= 0)[-1]
        if m > PACKED:
            assert none[0] % ALIGN == 0
    # the tiles cover every position that has an adapter once
    seen = []
    for first, rows, a, _, *row in tiles.tolist():
        assert 1 <= rows <= SLAB and (adapter[first:first + rows] == a).all()
        assert row[:rows] == order[first:first + rows].tolist()
        seen += range(first, first + rows)
    assert sorted(seen) == np.flatnonzero(adapter >= 0).tolist()


def test_plan_refusals():
    for ids in ([3], [-2], [0, 1, 2, 2**31], [-2**31]):
        with pytest.raises(ValueError, match="out of range"):
            plan_ints(ids, 3)
    lib = _lib.load()
    ids = np.zeros(4, np.int32)
    out = np.zeros(lib.wkv7_adapter_plan_ints(4, 2), np.int32)
    p, o = ids.ctypes.data, out.ctypes.data
    assert lib.wkv7_adapter_plan(p, 4, 2, o, out.size) == _lib.WKV7_OK
    assert lib.wkv7_adapter_plan(p, 4, 2, o, out.size - 1) == _lib.WKV7_ERR_WORKSPACE
    assert lib.wkv7_adapter_plan(p, -1, 2, o, out.size) == _lib.WKV7_ERR_ARG
    assert lib.wkv7_adapter_plan(p, 4, -1, o, out.size) == _lib.WKV7_ERR_ARG
    assert lib.wkv7_adapter_plan(None, 4, 2, o, out.size) == _lib.WKV7_ERR_ARG
    assert lib.wkv7_adapter_plan(p, 4, 0, o, out.size) == _lib.WKV7_ERR_ARG  # (id 0 of none)
    assert lib.wkv7_adapter_plan_ints(-1, 2) == 0


def test_proj_adapters_rejects_bad_arguments_before_any_launch():
    lib = _lib.load()

    def groups(**kw):
        base = dict(x=4096, w=8192, bias=None, y=12288, ldx=64, ldw=64, ldy=32, n=32, k=64, act=0,
                    reserved=0)
        base.update(kw)
        arr = (_lib.ProjGroup * 1)()
        arr[0] = _lib.ProjGroup(**base)
        return arr

    def sets(**kw):
        base = dict(a=4096, b=8192, scale=64, rank=128, count=4, slabs=1)
        base.update(kw)
        arr = (_lib.AdapterSet * 1)()
        arr[0] = _lib.AdapterSet(**base)
        return arr

    def call(m=4, g=None, s=None, n=1, plan=4096, count=4, ws=None, ws_bytes=0):
        return lib.wkv7_proj_adapters(m, g or groups(), s or sets(), n, plan, count, ws, ws_bytes,
                                      None)

    assert call(m=0) == _lib.WKV7_OK
    assert call(m=0, plan=None) == _lib.WKV7_OK
    for kw in (dict(m=-1), dict(n=0), dict(n=9), dict(plan=None), dict(count=-1), dict(count=5),
               dict(m=(1 << 28) + 1), dict(g=groups(k=48)), dict(s=sets(b=None)),
               dict(s=sets(scale=None)), dict(s=sets(rank=None)), dict(s=sets(slabs=0)),
               dict(s=sets(slabs=17))):
        assert call(**kw) == _lib.WKV7_ERR_ARG, kw
    for kw in (dict(g=groups(ldx=32)), dict(s=sets(a=4100)), dict(s=sets(b=8194)), dict(plan=4100)):
        assert call(**kw) == _lib.WKV7_ERR_SHAPE, kw
    assert lib.wkv7_proj_adapters_workspace_bytes(0, groups(), sets(), 1, 4) == 0
    assert lib.wkv7_proj_adapters_workspace_bytes(4, groups(k=48), sets(), 1, 4) == 0
    assert lib.wkv7_proj_adapters_workspace_bytes(4, groups(), sets(), 1, 5) == 0


def test_sample_rejects_bad_arguments_before_any_launch():
    lib = _lib.load()
    d = 4096

    def call(logits=d, dtype=1, rows=2, vocab=1000, stride=1000, noise=d, noise_stride=260,
             params=True, tokens=d, ws=d, ws_bytes=None):
        p = _lib.SampleParams() if params else None
        if ws_bytes is None:
            ws_bytes = lib.wkv7_sample_workspace_bytes(max(rows, 1), min(max(vocab, 1), 1 << 21))
        return lib.wkv7_sample_tokens(logits, dtype, rows, vocab, stride, noise, noise_stride, p,
                                      tokens, None, ws, ws_bytes, None)

    assert call(rows=0) == _lib.WKV7_OK
    for kw in (dict(rows=-1), dict(vocab=0), dict(params=False), dict(dtype=2), dict(logits=None),
               dict(noise=None), dict(tokens=None)):
        assert call(**kw) == _lib.WKV7_ERR_ARG, kw
    for kw in (dict(stride=999), dict(noise_stride=259), dict(logits=4098), dict(noise=4097),
               dict(vocab=(1 << 21) + 1, stride=1 << 22, noise_stride=1 << 20)):
        assert call(**kw) == _lib.WKV7_ERR_SHAPE, kw
    for kw in (dict(ws=None), dict(ws=4104), dict(ws_bytes=64)):
        assert call(**kw) == _lib.WKV7_ERR_WORKSPACE, kw
    assert lib.wkv7_sample_workspace_bytes(0, 10) == 0
    assert lib.wkv7_sample_workspace_bytes(4, (1 << 21) + 1) == 0


def test_no_cpu_path():
    logits = torch.zeros((2, 300))
    noise = torch.ones((2, sample_noise_size(300)))
    with pytest.raises(ValueError, match="GPU"):
        sample_tokens(logits, noise)
    x = torch.zeros((2, 32), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        proj_adapters([(x, x)], adapter_plan([-1, -1], 1, "cpu"))


def test_bank_refusals():
    bank = AdapterBank(2, 32, 16, 20, "cpu")
    assert bank.slabs == 2 and bank.a.shape == (2, 32, 32) and bank.b.shape == (2, 2, 16, 16)
    a, b = torch.zeros((4, 32), dtype=torch.bfloat16), torch.zeros((16, 4), dtype=torch.bfloat16)
    for args in [(2, a, b), (-1, a, b), (0, a.float(), b), (0, a, b.float()), (0, a, b[:, :3]),
                 (0, a[:, :16], b), (0, a, b, math.inf), (0, a[:0], b[:, :0]), (0, a[0], b)]:
        with pytest.raises(ValueError):
            bank.load(*args)
    with pytest.raises(ValueError):
        bank.clear(2)


def test_noise_size():
    assert [sample_noise_size(v) for v in (1, 256, 257, 65536)] == [257, 257, 258, 512]


def test_a_projection_keeps_its_bank():
    """A decode graph captures the banks' addresses, so a second bank must not take one's place."""
    block = RWKV7TimeMix.random(RWKV7StateLayout(1, 64, 1, 64, 64, torch.bfloat16), 0, "cpu")
    held = dict(block.add_adapters(2, 8, names=("r", "o")))
    for names in (("r",), ("k", "o"), ("k", "g1")):
        with pytest.raises(ValueError, match="already holds|r, k, v and o"):
            block.add_adapters(4, 8, names=names)
        assert block.adapters == held  # (and none of the names got one)
    more = block.add_adapters(3, 4, names=iter(("k", "v")))
    assert all(more[name] is bank for name, bank in held.items())
    assert more["k"].num_adapters == more["v"].num_adapters == 3


def test_plans_of_more_positions_than_32_bits_are_refused():
    """Many rows over very many adapters: every adapter's run may leave a gap, and the plan's
    positions are 32-bit numbers. (Refused before anything is read or written.)"""
    lib = _lib.load()
    most = 1 << 28
    for count in (1000, 60_000_000):  # 2^28 + 31 * 60,000,001 is below 2^31
        assert lib.wkv7_adapter_plan_ints(most, count) > 3 * most
    groups, sets = (_lib.ProjGroup * 1)(), (_lib.AdapterSet * 1)()
    groups[0] = _lib.ProjGroup(x=4096, w=8192, bias=None, y=12288, ldx=64, ldw=64, ldy=32, n=32,
                               k=64, act=0, reserved=0)
    for m, count in [(most, most), (most, 2**31 - 1), (most, 61_000_000), (1 << 27, 1 << 27)]:
        assert lib.wkv7_adapter_plan_ints(m, count) == 0
        assert lib.wkv7_adapter_plan(4096, m, count, 4096, 0) == _lib.WKV7_ERR_ARG
        sets[0] = _lib.AdapterSet(a=4096, b=8192, scale=64, rank=128, count=count, slabs=1)
        assert lib.wkv7_proj_adapters_workspace_bytes(m, groups, sets, 1, count) == 0
        assert lib.wkv7_proj_adapters(m, groups, sets, 1, 4096, count, None, 0,
                                      None) == _lib.WKV7_ERR_ARG


def test_a_scale_that_32_bits_make_infinite_is_refused():
    bank = AdapterBank(1, 32, 16, 4, "cpu")
    a, b = torch.zeros((4, 32), dtype=torch.bfloat16), torch.zeros((16, 4), dtype=torch.bfloat16)
    for scale in (1e39, -1e300, math.inf, -math.inf, math.nan):
        with pytest.raises(ValueError, match="scale must be finite"):
            bank.load(0, a, b, scale)
    with pytest.raises(ValueError, match="GPU"):  # (a bank on the host has nothing to load into)
        bank.load(0, a, b, -3e38)


def test_host_ids_under_graph_capture_are_refused_by_name(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="adapter_plan under graph capture"):
        adapter_plan([0, -1], 1, "cuda")
    graph = TimeMixDecodeGraph.__new__(TimeMixDecodeGraph)  # (a graph itself needs the GPU)
    graph.batch_size, graph.num_adapters, graph._order = 2, 1, ops.ReplayOrder()
    graph.adapter_plan = AdapterPlan(2, 1, torch.zeros(64, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="set_adapters under graph capture"):
        graph.set_adapters([0, -1])
    with pytest.raises(RuntimeError, match="set_slots under graph capture"):
        ops.ReplayOrder().refresh(torch.zeros(2, dtype=torch.int32), [1, 2])
