"""Decoding for many requests on one base model, each with an adapter and sampling settings of
its own: token -> embedding -> time-mix blocks -> head -> next token, all rows together.

    python examples/adapter_decode.py [--shape 0.1B] [--layers 4] [--requests 16] [--steps 32]

Weights are random (there are no checkpoints here), so the text means nothing; what the example
shows is the calls of a decode step and what they cost.
"""

from __future__ import annotations

import argparse
import math
import os
import sys
import time

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from wkvm_amd import (AdapterBank, RWKV7StateBank, RWKV7StateLayout, proj_adapters,  # noqa: E402
                      sample_noise_size, sample_tokens)
from wkvm_amd.timemix import RWKV7TimeMix, TokenBatch  # noqa: E402


class AdapterModel:
    """An embedding, ``layers`` time-mix blocks with adapters of their projections, and a head
    with adapters."""

    def __init__(self, shape: str, layers: int, vocab: int, slots: int, adapters: int, rank: int,
                 device, seed: int = 0) -> None:
        full = RWKV7StateLayout.for_shape(shape)
        layout = RWKV7StateLayout(layers, full.hidden_size, full.num_heads, full.head_dim,
                                  full.head_v_dim, full.dtype)
        D = layout.hidden_size
        self.gen = torch.Generator(device=device).manual_seed(seed)

        def normal(shape, std):
            return (torch.randn(shape, generator=self.gen, device=device) * std).to(torch.bfloat16)

        self.bank = RWKV7StateBank(layout, slots, device)
        self.blocks = [RWKV7TimeMix.random(layout, i, device, seed=seed) for i in range(layers)]
        self.embedding = normal((vocab, D), 1.0)
        self.head = normal((vocab, D), 1 / math.sqrt(D))
        self.head_adapters = AdapterBank(adapters, D, vocab, rank, device)
        self.adapters, self.vocab = adapters, vocab
        banks = [self.head_adapters]
        for block in self.blocks:
            banks += block.add_adapters(adapters, rank).values()
        for bank in banks:
            for i in range(adapters):  # ranks differ from adapter to adapter
                r = max(1, rank // (1 + i % 2))
                bank.load(i, normal((r, bank.k), 1 / math.sqrt(bank.k)),
                          normal((bank.n, r), 0.2 / math.sqrt(r)), scale=2.0)

    def step(self, tokens: torch.Tensor, batch: TokenBatch) -> torch.Tensor:
        """Logits ``[B, V]`` of the next tokens; the requests' states advance."""
        x = F.embedding(tokens, self.embedding)
        v_first = None
        for block in self.blocks:
            o, v_first = block.forward(self.bank, F.layer_norm(x, x.shape[1:]), batch, v_first)
            x = x + o
        x = F.layer_norm(x, x.shape[1:])
        return proj_adapters([(x, self.head, None, None, self.head_adapters)], batch.adapters)[0]


def decode(model: AdapterModel, slots, adapter_ids, settings, steps: int, first_tokens=None):
    """``steps`` tokens of every request: ``(tokens [steps, B], log-probabilities [steps, B],
    seconds per step)``. ``settings``: sample_tokens' keyword arguments, one value per request."""
    dev = model.bank.device
    batch = TokenBatch.plan(model.bank, slots, adapter_ids=adapter_ids,
                            num_adapters=model.adapters)
    B = len(slots)
    kinds = {"top_k": torch.int32}
    rows = {k: torch.tensor(v, dtype=kinds.get(k, torch.float32), device=dev)
            for k, v in settings.items()}
    noise = torch.empty((B, sample_noise_size(model.vocab)), device=dev)
    tokens = torch.zeros(B, dtype=torch.int32, device=dev) if first_tokens is None else first_tokens
    out, logp = [], []
    torch.cuda.synchronize(dev)
    start = time.perf_counter()
    for _ in range(steps):
        logits = model.step(tokens, batch)
        tokens, lp = sample_tokens(logits, noise.exponential_(generator=model.gen), **rows)
        out.append(tokens)
        logp.append(lp)
    torch.cuda.synchronize(dev)
    return torch.stack(out), torch.stack(logp), (time.perf_counter() - start) / steps


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--shape", default="0.1B")
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--adapters", type=int, default=6)
    ap.add_argument("--rank", type=int, default=16)
    ap.add_argument("--vocab", type=int, default=65536)
    ap.add_argument("--steps", type=int, default=32)
    args = ap.parse_args()
    B = args.requests
    model = AdapterModel(args.shape, args.layers, args.vocab, B, args.adapters, args.rank,
                         torch.device("cuda", 0))
    adapter_ids = [i % (args.adapters + 1) - 1 for i in range(B)]  # some on the base model
    settings = {"temperature": [0.0 if i % 5 == 4 else 0.7 + 0.1 * (i % 4) for i in range(B)],
                "top_k": [0 if i % 3 else 40 for i in range(B)],
                "top_p": [1.0 if i % 2 else 0.95 for i in range(B)],
                "min_p": [0.05 if i % 4 == 1 else 0.0 for i in range(B)]}
    slots = list(range(1, B + 1))
    decode(model, slots, adapter_ids, settings, 2)
    tokens, logp, seconds = decode(model, slots, adapter_ids, settings, args.steps)
    for i in range(min(B, 4)):
        print(f"request {i}: adapter {adapter_ids[i]}, tokens {tokens[:8, i].tolist()}, "
              f"log-probability {logp[:, i].sum().item():.2f}")
    print(f"{seconds * 1e6:.0f} us per step of {B} requests, {args.layers} blocks")


if __name__ == "__main__":
    main()
