"""4-bit weights and linear attention as a layer uses them: in the time-mix block and its decode graph,
and one after the other over the slots of a bank."""

import gc

import numpy as np
import pytest
import torch

from tests import util as U
from tests.linear_ref import scan, state_bound, y_bound
from wkvm_amd import RWKV7StateBank, RWKV7StateLayout, W4Weight, proj_w4
from wkvm_amd.timemix import RWKV7TimeMix, TimeMixDecodeGraph, TokenBatch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
LAYOUT = RWKV7StateLayout(2, 256, 4, 64, 64, BF16)


def _grid(shape, group, gen, dev):
    """Weights that 4-bit codes hold: multiples of 2^-5 from -8 to 7 of them, both in each group."""
    codes = torch.randint(0, 16, shape, generator=gen, device=dev)
    codes[:, ::group], codes[:, 1::group] = 0, 15
    return ((codes - 8) / 32).to(BF16)


def _blocks(dev, group):
    gen = torch.Generator(device=dev).manual_seed(group)
    plain, quant = [], []
    for i in range(2):
        w = dict(RWKV7TimeMix.random(LAYOUT, i, dev, seed=4).w)
        for name in ("r", "k", "v", "o"):
            w[name] = _grid((256, 256), group, gen, dev)
        plain.append(RWKV7TimeMix(LAYOUT, i, w))
        quant.append(RWKV7TimeMix(LAYOUT, i, w))
        quant[-1].quantize(group)
        assert set(quant[-1].w4) == {"r", "k", "v", "o"} and "r" in w and "r" not in quant[-1].w
    return plain, quant


def _bank(dev, slots=90):
    bank = RWKV7StateBank(LAYOUT, slots, dev)
    gen = torch.Generator(device=dev).manual_seed(9)
    bank.wkv.normal_(0.0, 0.1, generator=gen)
    bank.shift.copy_(torch.randn(bank.shift.shape, generator=gen, device=dev))
    return bank


def _run(bank, blocks, x, ids, lengths, adapter_ids=None, adapters=0, streams=None):
    cu = None if lengths is None else np.concatenate([[0], np.cumsum(lengths)]).tolist()
    batch = TokenBatch.plan(bank, ids, cu, adapter_ids, adapters)
    out, v_first = [], None
    for block in blocks:
        o, v_first = block.forward(bank, x[:batch.tokens], batch, v_first, streams=streams)
        out.append(o)
    return out


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("ids,lengths", [([7], None), (list(range(1, 81)), None),
                                         ([5, 2, 8], [70, 1, 33]), ([5, 2, 8], [600, 3, 500])])
def test_block_is_the_one_with_the_values_of_its_codes(dev, ids, lengths, group):
    """The products differ in the order of their sums, so in a rounding of their bf16 outputs here and
    there, as the block's own two ways of computing them do."""
    plain, quant = _blocks(dev, group)
    for name in ("r", "o"):
        err = (quant[0].w4[name].dequantize() - plain[0].w[name].float()).abs().max().item()
        assert err <= 2.0 ** -2 * 2.0 ** -18  # (a scale's last bits hold its zero point)
    x = torch.randn((1200, 256), generator=torch.Generator(device=dev).manual_seed(2),
                    device=dev).to(BF16)
    banks = _bank(dev), _bank(dev)
    ref = _run(banks[0], plain, x, ids, lengths)
    got = _run(banks[1], quant, x, ids, lengths)
    assert torch.equal(banks[0].shift, banks[1].shift)
    assert U.normwise_max(U.f64(banks[1].wkv), U.f64(banks[0].wkv)) <= 1e-2
    for a, b in zip(got, ref):
        assert U.rel_l2(U.f64(a), U.f64(b)) <= 1e-2


def test_block_on_side_streams_and_with_some_adapters(dev):
    _, quant = _blocks(dev, 64)
    x = torch.randn((700, 256), generator=torch.Generator(device=dev).manual_seed(3),
                    device=dev).to(BF16)
    banks = [_bank(dev) for _ in range(2)]
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    a = _run(banks[0], quant, x, [3, 4], [600, 100])
    b = _run(banks[1], quant, x, [3, 4], [600, 100], streams=streams)
    torch.cuda.synchronize()
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    assert torch.equal(banks[0].wkv, banks[1].wkv)

    # v and o as codes, r and k with adapters: none in the batch, then some
    w = RWKV7TimeMix.random(LAYOUT, 0, dev, seed=4).w
    mixed = RWKV7TimeMix(LAYOUT, 0, w)
    mixed.quantize(64, ("v", "o"))
    gen = torch.Generator(device=dev).manual_seed(6)
    merged = dict(w)
    for name, bank in mixed.add_adapters(2, 16, ("r", "k")).items():
        pair = [torch.randn(shape, generator=gen, device=dev).to(BF16) / 16
                for shape in ((16, 256), (256, 16))]
        bank.load(1, *pair, 1.0)
        merged[name] = (w[name].float() + pair[1].float() @ pair[0].float()).to(BF16)
    one = RWKV7TimeMix(LAYOUT, 0, merged)
    one.quantize(64, ("v", "o"))
    banks = [_bank(dev) for _ in range(2)]
    got, = _run(banks[0], [mixed], x, [3, 4], [600, 50], [1, 1], 2)
    ref, = _run(banks[1], [one], x, [3, 4], [600, 50])
    assert U.rel_l2(U.f64(got), U.f64(ref)) <= 2e-2  # (the merged weights round once more)
    with pytest.raises(ValueError, match="takes no adapters"):
        mixed.add_adapters(2, 16, ("v",))
    with pytest.raises(ValueError, match="holds adapters"):
        mixed.quantize(64, ("k",))
    with pytest.raises(ValueError, match="already holds a 4-bit"):
        mixed.quantize(64, ("o",))


@pytest.mark.parametrize("B", [6, 80])
def test_decode_graph_with_codes(dev, B, monkeypatch):
    """Replays against the eager blocks, the library's products beside them on side streams for the
    larger batch; a graph of the plain blocks keeps its weights when these become codes."""
    if B == 80:
        monkeypatch.setattr(RWKV7TimeMix, "PROJ_MAX_ROWS", 64)
    plain, quant = _blocks(dev, 128)
    eager, graphed, banks = _bank(dev), _bank(dev), (_bank(dev), _bank(dev))
    graph = TimeMixDecodeGraph(graphed, quant, B)
    other = TimeMixDecodeGraph(banks[0], plain, B)
    kept = [RWKV7TimeMix(LAYOUT, i, b.w) for i, b in enumerate(plain)]
    kept = [RWKV7TimeMix(LAYOUT, i, {n: t.clone() for n, t in b.w.items()})
            for i, b in enumerate(kept)]
    for b in plain:
        b.w = dict(b.w)
        b.quantize(32)
    gc.collect()
    spoil = [torch.full((256, 256), 3.0, dtype=BF16, device=dev) for _ in range(64)]
    gen = torch.Generator().manual_seed(B)
    for step in range(4):
        slots = (torch.randperm(90, generator=gen)[:B] + 1).tolist()
        x = torch.randn((2, B, 256), generator=gen).to(BF16).to(dev)
        for g, bank, blocks in ((graph, eager, quant), (other, banks[1], kept)):
            batch = TokenBatch.plan(bank, slots)
            v_first, ref = None, []
            for i, block in enumerate(blocks):
                o, v_first = block.forward(bank, x[i], batch, v_first)
                ref.append(o)
            g.set_slots(slots)
            g.x.copy_(x)
            out = g.replay()
            torch.cuda.synchronize()
            assert torch.equal(torch.stack(out), torch.stack(ref)), f"step {step}"
            assert torch.equal(g.bank.wkv, bank.wkv)
    del spoil


# -- a linear-attention layer whose projections are 4-bit codes ---------------------------------

class Layer:
    """x -> q, k, v, an output gate and the tokens' decays -> linear attention -> gate -> o."""

    H, HQ, D = 4, 2, 256

    def __init__(self, dev, group):
        gen = torch.Generator(device=dev).manual_seed(group)
        self.parts = {}
        for name, n in (("q", 128), ("k", 128), ("v", 256), ("g", 256), ("o", 256)):
            codes = torch.randint(0, 16, (n, 256), generator=gen, device=dev, dtype=torch.uint8)
            scale = ((torch.rand(n, 256 // group, generator=gen, device=dev) + .5) / 64).to(BF16)
            self.parts[name] = W4Weight.from_codes(codes, scale, group=group)
        self.rate = torch.rand(self.H, generator=gen, device=dev) * 0.1

    def project(self, x):
        p = self.parts
        q, k, v, g = proj_w4([(x, p["q"]), (x, p["k"]), (x, p["v"]), (x, p["g"], None, "sigmoid")])
        T = len(x)
        return (q.view(T, self.HQ, 64), k.view(T, self.HQ, 64), v.view(T, self.H, 64), g,
                -self.rate * (1 + x[:, :self.H].float().abs()))

    def out(self, y, g):
        return proj_w4([(y.reshape(g.shape) * g, self.parts["o"])])[0]

    def prefill(self, bank, x, ids, cu):
        q, k, v, g, d = self.project(x)
        return self.out(bank.prefill_linear(1, ids, cu, q, k, v, d, scale=0.125), g)

    def decode(self, bank, x, ids, order=None):
        q, k, v, g, d = self.project(x)
        return self.out(bank.decode_linear(1, ids, q, k, v, d, scale=0.125, row_order=order), g)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_layer_over_a_bank(dev, group):
    """Ragged prompts, then captured decode steps: each stage against its formula in float64 on what
    the stage before it gave, and the replays against the eager steps."""
    layer, banks = Layer(dev, group), [_bank(dev, 12) for _ in range(2)]
    gen = torch.Generator(device=dev).manual_seed(1)
    cu, ids = [0, 1, 71, 71, 400], [4, 9, 2, 7]
    slots = [{"wkv": i} for i in ids]
    x = torch.randn((400, 256), generator=gen, device=dev).to(BF16)
    before = banks[0].wkv.clone()
    got = layer.prefill(banks[0], x, slots, cu)
    layer.prefill(banks[1], x, slots, cu)
    assert torch.equal(banks[0].wkv, banks[1].wkv)

    q, k, v, g, d = layer.project(x)
    ref = U.f64(before[1])
    y, my, ms = scan(ref, cu, ids, *(U.f64(t) for t in (q, k, v, d)), 0.125)
    # each product: 2^-24 of its terms' size (32 + code + zero point per value) for every sum and join
    for name, act, t, inp in (("q", 0, q, x), ("v", 0, v, x), ("g", 1, g, x)):
        w = U.f64(layer.parts[name].dequantize())
        p, xin = U.f64(inp) @ w.T, np.abs(U.f64(inp))
        scale = np.abs(w).max()  # s times 7 at least somewhere; 55 s bounds s (32 + c + z)
        err = 2.0 ** -24 * (128 + 8 + 17) * xin.sum(1, keepdims=True) * 8 * scale
        err, p = (err + 2.0 ** -20, 1 / (1 + np.exp(-p))) if act else (err, p)
        assert (np.abs(U.f64(t).reshape(p.shape) - p) <= err + 2.0 ** -8 * (np.abs(p) + err)).all()
    again = _bank(dev, 12)
    yk = again.prefill_linear(1, slots, cu, q, k, v, d, scale=0.125)
    assert (np.abs(U.f64(yk) - y) <= y_bound(y, my, 329, 64, False)).all()
    assert (np.abs(U.f64(again.wkv[1])[ids] - ref[ids]) <= state_bound(ms, 329)).all()
    assert torch.equal(layer.out(yk, g), got)
    assert torch.equal(banks[0].wkv[0], before[0])
    rest = [r for r in range(13) if r not in ids]
    assert torch.equal(banks[0].wkv[:, rest], before[:, rest])

    rows = torch.tensor(ids, dtype=torch.int32, device=dev)
    order = torch.tensor([2, 0, 3, 1], dtype=torch.int32, device=dev)
    xs = torch.zeros((4, 256), dtype=BF16, device=dev)
    side = torch.cuda.Stream(dev)
    with torch.cuda.stream(side):
        layer.decode(banks[0], xs, rows, order)
    side.synchronize()
    banks[0].wkv.copy_(banks[1].wkv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.decode(banks[0], xs, rows, order)
    for _ in range(5):
        step = torch.randn((4, 256), generator=gen, device=dev).to(BF16)
        want = layer.decode(banks[1], step, slots)
        xs.copy_(step)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(banks[0].wkv, banks[1].wkv)
        torch.randn(1 << 16, device=dev).sum().item()


def test_prompt_at_once_and_token_by_token(dev):
    """The decode steps' states and outputs are the prefill's to the bounds of both: products of few
    and of many rows round their outputs alike but for ties."""
    layer, banks = Layer(dev, 128), [_bank(dev, 12) for _ in range(2)]
    x = torch.randn((130, 256), generator=torch.Generator(device=dev).manual_seed(8),
                    device=dev).to(BF16)
    a = layer.prefill(banks[0], x, [{"wkv": 5}], [0, 130])
    b = torch.cat([layer.decode(banks[1], x[t:t + 1], [{"wkv": 5}]) for t in range(130)])
    assert U.rel_l2(U.f64(a), U.f64(b)) <= 1e-2
    assert U.normwise_max(U.f64(banks[0].wkv[1, 5]), U.f64(banks[1].wkv[1, 5])) <= 1e-2
