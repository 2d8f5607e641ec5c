"""Adapters through the time-mix block, its decode graph and the example's decode loop."""

import gc
import math
import os
import sys
import weakref

import numpy as np
import pytest
import torch

from wkvm_amd import RWKV7StateBank, RWKV7StateLayout
from wkvm_amd.timemix import RWKV7TimeMix, TimeMixDecodeGraph, TokenBatch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "examples"))

pytestmark = pytest.mark.gpu

LAYOUT = RWKV7StateLayout(2, 768, 12, 64, 64, torch.bfloat16)


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda", 0)


def _blocks(dev, adapters=3, rank=16, std=0.1):
    gen = torch.Generator(device=dev).manual_seed(5)
    blocks = [RWKV7TimeMix.random(LAYOUT, i, dev, seed=1) for i in range(2)]
    pairs = []
    for block in blocks:
        held = {}
        for name, bank in block.add_adapters(adapters, rank).items():
            held[name] = []
            for i in range(adapters):
                a = (torch.randn((rank, bank.k), generator=gen, device=dev)
                     / math.sqrt(bank.k)).to(torch.bfloat16)
                b = (torch.randn((bank.n, rank), generator=gen, device=dev)
                     * std / math.sqrt(rank)).to(torch.bfloat16)
                bank.load(i, a, b, 2.0)
                held[name].append((a, b, 2.0))
        pairs.append(held)
    return blocks, pairs


def _run(dev, blocks, ids, lengths=None, adapter_ids=None, adapters=3):
    """Both blocks over a batch from given states: their outputs and the new states."""
    gen = torch.Generator(device=dev).manual_seed(9)
    bank = RWKV7StateBank(LAYOUT, 40, dev)
    bank.wkv.normal_(generator=gen)
    bank.wkv *= 0.1
    cu = None if lengths is None else np.concatenate([[0], np.cumsum(lengths)]).tolist()
    batch = TokenBatch.plan(bank, ids, cu, adapter_ids, adapters)
    out, v_first = [], None
    for block in blocks:
        x = torch.randn((batch.tokens, 768), generator=gen, device=dev).to(torch.bfloat16)
        o, v_first = block.forward(bank, x, batch, v_first)
        out.append(o)
    return out, bank.wkv


@pytest.mark.parametrize("ids,lengths", [([3, 9, 1, 20], None), (list(range(1, 34)), None),
                                         ([5, 2], [7, 40])])
def test_no_adapter_is_the_plain_block(dev, ids, lengths):
    blocks, _ = _blocks(dev)
    plain, plain_state = _run(dev, blocks, ids, lengths)
    none, none_state = _run(dev, blocks, ids, lengths, [-1] * len(ids))
    for a, b in zip(plain, none):
        assert torch.equal(a, b)
    assert torch.equal(plain_state, none_state)


@pytest.mark.parametrize("ids,lengths,adapter_ids", [
    ([3, 9, 1, 20, 7], None, [0, 2, -1, 1, 0]), ([5, 2, 8], [70, 1, 33], [1, -1, 2]),
    ([5, 2, 8], [600, 3, 500], [1, 2, -1])])
def test_an_adapter_is_a_merged_weight(dev, ids, lengths, adapter_ids):
    """Every sequence against blocks whose r, k, v and o hold W + s B A, rounded to bf16. That
    rounding (2^-9 of a weight) and the block's own bf16 stages leave about 1 % of the
    output's scale; the adapters themselves change it by more than 5 %."""
    blocks, pairs = _blocks(dev)
    got, _ = _run(dev, blocks, ids, lengths, adapter_ids)
    plain, _ = _run(dev, blocks, ids, lengths)
    lens = lengths or [1] * len(ids)
    starts = np.concatenate([[0], np.cumsum(lens)])
    for a in sorted(set(adapter_ids) - {-1}):
        merged = []
        for block, held in zip(blocks, pairs):
            w = dict(block.w)
            for name, places in held.items():
                A, B, s = places[a]
                w[name] = (w[name].float() + s * B.float() @ A.float()).to(torch.bfloat16)
            merged.append(RWKV7TimeMix(LAYOUT, block.layer_idx, w))
        want, _ = _run(dev, merged, ids, lengths)
        for s in (i for i, x in enumerate(adapter_ids) if x == a):
            rows = slice(int(starts[s]), int(starts[s + 1]))
            for g, e, p in zip(got, want, plain):
                scale = e[rows].float().norm()
                assert (g[rows].float() - e[rows].float()).norm() <= 0.02 * scale
                assert (p[rows].float() - e[rows].float()).norm() >= 0.05 * scale


def test_decode_graph_with_adapters(dev):
    """Replays with changing adapters against the eager blocks, state by state."""
    blocks, _ = _blocks(dev)
    B, ids = 6, [4, 1, 9, 30, 2, 17]
    bank = RWKV7StateBank(LAYOUT, 40, dev)
    graph = TimeMixDecodeGraph(bank, blocks, B, num_adapters=3)
    graph.set_slots(ids)
    ref = RWKV7StateBank(LAYOUT, 40, dev)
    gen = torch.Generator(device=dev).manual_seed(3)
    for adapter_ids in ([-1] * 6, [0, 1, 2, -1, 0, 2], [2] * 6, [0, 1, 2, -1, 0, 2]):
        graph.set_adapters(adapter_ids)
        graph.x.normal_(generator=gen)
        out = graph.replay()
        torch.cuda.synchronize()
        batch = TokenBatch.plan(ref, ids, None, adapter_ids, 3)
        v_first = None
        for i, block in enumerate(blocks):
            o, v_first = block.forward(ref, graph.x[i].clone(), batch, v_first)
            assert torch.equal(o, out[i])
        assert torch.equal(bank.wkv, ref.wkv) and torch.equal(bank.shift, ref.shift)
    with pytest.raises(ValueError, match="adapter ids"):
        graph.set_adapters([0] * 5)
    with pytest.raises(ValueError, match="out of range"):
        graph.set_adapters([3] * 6)
    with pytest.raises(ValueError, match="num_adapters"):
        TimeMixDecodeGraph(bank, blocks, 2).set_adapters([0, 0])


def test_refusals(dev):
    blocks, _ = _blocks(dev)
    bank = RWKV7StateBank(LAYOUT, 4, dev)
    with pytest.raises(ValueError, match="adapter ids"):
        TokenBatch.plan(bank, [1, 2], None, [0], 3)
    with pytest.raises(ValueError, match="out of range"):
        TokenBatch.plan(bank, [1, 2], None, [0, 3], 3)
    with pytest.raises(ValueError, match="r, k, v and o"):
        blocks[0].add_adapters(2, 8, names=("g1",))


def test_the_example_decodes(dev):
    """Greedy rows of the example do not depend on the batch around them or on other rows'
    adapters, and sampled tokens come from the vocabulary with their log-probabilities."""
    import adapter_decode as ex

    model = ex.AdapterModel("0.1B", 2, 1009, 8, 3, 16, dev, seed=2)
    settings = {"temperature": [0.0, 0.0, 0.8, 1.0], "top_k": [0, 0, 20, 0],
                "top_p": [1.0, 1.0, 0.9, 0.95], "min_p": [0.0, 0.0, 0.0, 0.1]}
    tokens, logp, _ = ex.decode(model, [1, 2, 3, 4], [0, -1, 2, 1], settings, 6)
    assert tokens.shape == logp.shape == (6, 4)
    assert bool(((tokens >= 0) & (tokens < 1009)).all()) and bool((logp <= 0).all())
    model.bank.wkv.zero_()
    model.bank.shift.zero_()
    other = {k: [v[1], v[0]] for k, v in settings.items()}
    again, _, _ = ex.decode(model, [7, 5], [-1, 0], other, 6)
    assert torch.equal(again[:, 0], tokens[:, 1]) and torch.equal(again[:, 1], tokens[:, 0])


def test_a_decode_graph_holds_its_banks(dev):
    """Blocks that give their banks up after the capture: the graph replays the ones it captured."""
    blocks, _ = _blocks(dev)
    ids, adapter_ids = [4, 1, 9], [0, 2, -1]
    state, want_state = (RWKV7StateBank(LAYOUT, 40, dev) for _ in range(2))
    graph, want = (TimeMixDecodeGraph(b, blocks, 3, num_adapters=3) for b in (state, want_state))
    gen = torch.Generator(device=dev).manual_seed(3)
    for g in (graph, want):
        g.set_slots(ids)
        g.set_adapters(adapter_ids)
    want.x.normal_(generator=gen)
    graph.x.copy_(want.x)
    expected = [o.clone() for o in want.replay()]
    held = {id(b) for block in blocks for b in block.adapters.values()}
    assert {id(b) for b in graph.adapter_banks} == held and len(held) == 8
    refs = [weakref.ref(b.a) for block in blocks for b in block.adapters.values()]
    for block in blocks:
        block.adapters.clear()
        for bank in block.add_adapters(3, 16).values():
            bank.a.fill_(math.nan)
    del want, g
    assert all(r() is not None for r in refs)
    for o, e in zip(graph.replay(), expected):
        assert torch.equal(o, e)
    del graph, o, e
    gc.collect()
    assert all(r() is None for r in refs)
