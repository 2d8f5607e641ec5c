"""What a request brings of its own to a batched decode step, as operators: timing cases.

* ``adapters``  ``proj_adapters``: projections shared by every row of a batch, with a low-rank
                adapter of the row's own request beside them
* ``sample``    ``sample_tokens``: each row's next token by its own temperature, top-k, top-p and
                min-p, from given random numbers, with its log-probability

``listed()`` holds the cases, ``draw(rng)`` makes more of the same ranges. ``run`` computes a case in
its plain form (elementary torch operations in 32 bits) or, where ``own`` is set, through the
framework's entry points. ``exact`` computes it from the definition in 64 bits.

Hidden sizes are those of RWKV-7 0.1B, 1.5B and 7B; batches and prompts are those of the
repository's benchmark and of a serving engine around them.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
GROUP = 256  # tokens of one group of the sampling race
LARGEST_SAMPLE = 512 * 131077
LARGEST_ADAPTERS = 3 * 32768 * 2048 * 2048  # rows x (k n + rank (k + n)) over all products


def listed():
    return [
        # One live request of the small model, with its adapter: a launch's latency is all.
        {"name": "adapters_one", "kind": "adapters", "rows": 1, "seqs": 1, "k": 768, "n": 768,
         "products": 3, "adapters": 4, "rank": 8, "none": 0.0, "act": False},
        # A handful of requests that share two adapters.
        {"name": "adapters_8", "kind": "adapters", "rows": 8, "seqs": 8, "k": 2048, "n": 2048,
         "products": 3, "adapters": 2, "rank": 16, "none": 0.2, "act": False},
        # Every request of a batch with an adapter of its own.
        {"name": "adapters_64_own", "kind": "adapters", "rows": 64, "seqs": 64, "k": 2048,
         "n": 2048, "products": 3, "adapters": 64, "rank": 16, "none": 0.0, "act": False},
        # The headline decode batch over a few dozen adapters of up to 32 ranks, popular ones
        # first, a quarter of the requests on the base model.
        {"name": "adapters_256", "kind": "adapters", "rows": 256, "seqs": 256, "k": 2048,
         "n": 2048, "products": 3, "adapters": 32, "rank": 32, "none": 0.25, "act": False},
        # One wide product of the 7B shape with bias and activation, odd row count, high ranks.
        {"name": "adapters_7b", "kind": "adapters", "rows": 203, "seqs": 203, "k": 4096,
         "n": 4096, "products": 1, "adapters": 24, "rank": 64, "none": 0.1, "act": True},
        # A few prompts in one prefill, ragged.
        {"name": "adapters_prompts", "kind": "adapters", "rows": 3001, "seqs": 7, "k": 2048,
         "n": 2048, "products": 3, "adapters": 5, "rank": 16, "none": 0.1, "act": False},
        # The benchmark's prefill: eight long prompts' worth of tokens.
        {"name": "adapters_prefill", "kind": "adapters", "rows": 32768, "seqs": 11, "k": 2048,
         "n": 2048, "products": 3, "adapters": 8, "rank": 32, "none": 0.1, "act": False},
        # One chat request's next token.
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 65536, "bf16": False,
         "mode": "all"},
        # A few requests over an odd vocabulary, each with its own settings, logits in bf16.
        {"name": "sample_odd", "kind": "sample", "rows": 9, "vocab": 32003, "bf16": True,
         "mode": "mixed"},
        # The headline decode batch, every request with its own settings.
        {"name": "sample_256", "kind": "sample", "rows": 256, "vocab": 65536, "bf16": False,
         "mode": "mixed"},
        # The same batch with temperature alone: nothing is cut off.
        {"name": "sample_256_plain", "kind": "sample", "rows": 256, "vocab": 65536, "bf16": False,
         "mode": "plain"},
        # A large batch over a large vocabulary, nucleus sampling.
        {"name": "sample_wide", "kind": "sample", "rows": 512, "vocab": 131077, "bf16": True,
         "mode": "nucleus"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        vocab = _log(rng, 1000, 200003)
        return {"kind": "sample", "rows": _log(rng, 1, min(1024, LARGEST_SAMPLE // vocab)),
                "vocab": vocab, "bf16": rng.random() < 0.5,
                "mode": rng.choice(["mixed", "mixed", "all", "plain", "nucleus", "top_k"])}
    k = rng.choice([768, 2048, 2048, 4096, 32 * _log(rng, 4, 128)])
    n = rng.choice([k, k, _log(rng, 64, 4096)])
    products = rng.choice([1, 2, 3])
    rank = rng.choice([4, 8, 16, 16, 32, 64, _log(rng, 1, 128)])
    rows = _log(rng, 1, min(32768, LARGEST_ADAPTERS // (products * (k * n + rank * (k + n)))))
    decode = rows <= 512 and rng.random() < 0.8
    return {"kind": "adapters", "rows": rows, "seqs": rows if decode else min(rows, _log(rng, 1, 32)),
            "k": k, "n": n, "products": products, "adapters": _log(rng, 1, 64), "rank": rank,
            "none": rng.choice([0.0, 0.1, 0.5]), "act": rng.random() < 0.3}


# -- inputs ---------------------------------------------------------------------------------------

def _requests(case):
    """Adapter of every row (-1: the base model), from the case alone: sequences of random
    lengths (one row each where there are as many as rows), popular adapters more often."""
    rng = random.Random("%(rows)d rows of %(seqs)d requests over %(adapters)d adapters" % case)
    rows, seqs, many = case["rows"], case["seqs"], case["adapters"]
    cuts = sorted(rng.sample(range(1, rows), seqs - 1)) if seqs < rows else list(range(1, rows))
    order = list(range(many))
    rng.shuffle(order)
    ids = np.empty(rows, dtype=np.int64)
    for i, (lo, hi) in enumerate(zip([0] + cuts, cuts + [rows])):
        if rng.random() < case["none"]:
            a = -1
        elif many >= seqs:
            a = order[i]  # each request its own
        else:
            a = order[min(int(many * rng.random() ** 2), many - 1)]
        ids[lo:hi] = a
    return ids


def _ranks(case):
    """Every adapter's rank: the case's largest, some of them half of it."""
    rng = random.Random("%(adapters)d adapters of rank %(rank)d" % case)
    return [case["rank"] if i == 0 or rng.random() < 0.7 else max(1, case["rank"] // 2)
            for i in range(case["adapters"])]


def _adapter_inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def n(shape, std):
        return (torch.randn(shape, generator=gen, device=DEV) * std).to(torch.bfloat16)

    k, cols = case["k"], case["n"]
    ids, ranks = _requests(case), _ranks(case)
    used = sorted(set(ids[ids >= 0].tolist()))
    state = {"products": [], "rows": {a: torch.from_numpy(np.flatnonzero(ids == a)).to(DEV)
                                      for a in used}}
    for _ in range(case["products"]):
        state["products"].append({
            "x": n((case["rows"], k), 1.0), "w": n((cols, k), 1 / math.sqrt(k)),
            "bias": n((cols,), 0.5) if case["act"] else None,
            "act": "sigmoid" if case["act"] else None,
            "a": [n((r, k), 1 / math.sqrt(k)) for r in ranks],
            "b": [n((cols, r), 0.2 / math.sqrt(r)) for r in ranks],
            "scale": [2.0 if i % 3 else 1.5 for i in range(len(ranks))],
        })
    return state


def _load_adapters(case, state):
    """The banks that hold the adapters and the plan of the batch's adapter ids."""
    from wkvm_amd import AdapterBank, adapter_plan

    dev = torch.device(DEV)
    state["plan"] = adapter_plan(_requests(case).tolist(), case["adapters"], dev)
    for p in state["products"]:
        p["bank"] = AdapterBank(case["adapters"], case["k"], case["n"], case["rank"], dev)
        for i, (a, b, s) in enumerate(zip(p["a"], p["b"], p["scale"])):
            p["bank"].load(i, a, b, s)


def _settings(case):
    """Temperature, top-k, top-p and min-p of every row (off: 0, 1 and 0)."""
    rng = random.Random("%(rows)d rows of %(vocab)d tokens, %(mode)s" % case)
    out = []
    for _ in range(case["rows"]):
        temp = rng.choice([0.6, 0.8, 1.0, 1.0, 1.3])
        k, p, m = rng.choice([20, 40, 50, 200]), rng.choice([0.8, 0.9, 0.95, 0.98]), \
            rng.choice([0.02, 0.05, 0.1])
        kind = case["mode"]
        if kind == "mixed":
            kind = rng.choice(["plain", "top_k", "nucleus", "min_p", "all", "all", "greedy"])
        out.append((0.0 if kind == "greedy" else temp,
                    k if kind in ("top_k", "all") else 0,
                    p if kind in ("nucleus", "all") else 1.0,
                    m if kind in ("min_p", "all") else 0.0))
    return out


def _sample_inputs(case, seed):
    """Logits as a language model gives them: probabilities that fall as a power of the rank,
    steeper for the surer rows, a little noise, and banned tokens at -inf."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    rank = torch.rand((rows, vocab), generator=gen, device=DEV).clamp_(min=1e-7).mul_(vocab)
    steep = 1.0 + 0.8 * torch.rand((rows, 1), generator=gen, device=DEV)
    logits = rank.log_().mul_(-steep)
    logits += 0.3 * torch.randn((rows, vocab), generator=gen, device=DEV)
    logits += 12.0 + torch.randn((rows, 1), generator=gen, device=DEV)
    banned = torch.randint(0, vocab, (rows, 16), generator=gen, device=DEV)
    logits.scatter_(1, banned, -math.inf)
    numbers = GROUP + (vocab + GROUP - 1) // GROUP
    noise = torch.empty((rows, numbers), device=DEV).exponential_(generator=gen)
    temp, k, p, m = zip(*_settings(case))
    return {"logits": logits.to(torch.bfloat16 if case["bf16"] else torch.float32),
            "noise": noise,
            "temperature": torch.tensor(temp, dtype=torch.float32, device=DEV),
            "top_k": torch.tensor(k, dtype=torch.int32, device=DEV),
            "top_p": torch.tensor(p, dtype=torch.float32, device=DEV),
            "min_p": torch.tensor(m, dtype=torch.float32, device=DEV)}


def prepare(case, seed):
    if case["kind"] == "sample":
        return _sample_inputs(case, seed)
    state = _adapter_inputs(case, seed)
    if own:
        _load_adapters(case, state)
    return state


# -- one pass -------------------------------------------------------------------------------------

def _plain_adapters(state):
    out = []
    for p in state["products"]:
        x = p["x"].float()
        y = x @ p["w"].float().t()
        for a, rows in state["rows"].items():
            h = (x[rows] @ p["a"][a].float().t()) * p["scale"][a]
            y[rows] += h @ p["b"][a].float().t()
        if p["bias"] is not None:
            y += p["bias"].float()
        if p["act"] == "sigmoid":
            y = 1.0 / (1.0 + torch.exp(-y))
        out.append(y.to(torch.bfloat16))
    return out


def _sample(logits, noise, temperature, top_k, top_p, min_p):
    """The definition, in the inputs' own precision: tokens and log-probabilities."""
    rows, vocab = logits.shape
    x = torch.where(torch.isnan(logits), -math.inf, logits)
    top = x.amax(1, keepdim=True)
    d = torch.where(x == top, 0.0, x - top)
    total = torch.exp(d).sum(1)
    greedy = temperature <= 0
    z = d / torch.where(greedy, 1.0, temperature)[:, None]
    # in order of the logits, ties by index
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    zs = torch.gather(z, 1, order)
    ws = torch.exp(zs)
    place = torch.arange(vocab, device=x.device)[None, :]
    many = torch.where(top_k > 0, top_k, vocab)[:, None]
    ws = torch.where(place < many, ws, 0.0)
    before = torch.cumsum(ws, 1) - ws
    keep = (place < many) & (before < (top_p * ws.sum(1))[:, None]) | (top_p >= 1)[:, None] & (place < many)
    keep |= place == 0
    keep &= zs >= torch.log(min_p)[:, None]
    w = torch.zeros_like(x).scatter_(1, order, torch.where(keep, ws, 0.0))
    groups = (vocab + GROUP - 1) // GROUP
    padded = torch.zeros((rows, groups * GROUP), dtype=x.dtype, device=x.device)
    padded[:, :vocab] = w
    padded = padded.view(rows, groups, GROUP)
    g = torch.argmin(noise[:, GROUP:GROUP + groups] / padded.sum(2), 1)
    chosen = padded[torch.arange(rows, device=x.device), g]
    token = g * GROUP + torch.argmin(noise[:, :GROUP] / chosen, 1)
    token = torch.where(greedy, torch.argmax(x, 1), token)
    logp = torch.gather(d, 1, token[:, None])[:, 0] - torch.log(total)
    return token, logp


def _plain_sample(state):
    token, logp = _sample(state["logits"].float(), state["noise"], state["temperature"],
                          state["top_k"], state["top_p"], state["min_p"])
    return token.int(), logp


def run(state):
    if "products" in state:
        if not own:
            return _plain_adapters(state)
        from wkvm_amd import proj_adapters

        return proj_adapters([(p["x"], p["w"], p["bias"], p["act"], p["bank"])
                              for p in state["products"]], state["plan"])
    if not own:
        return _plain_sample(state)
    from wkvm_amd import sample_tokens

    return sample_tokens(state["logits"], state["noise"], temperature=state["temperature"],
                         top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])


# -- from the definitions, in 64 bits ----------------------------------------------------------------

def _exact_adapters(case, seed):
    state = _adapter_inputs(case, seed)
    ids, ranks = _requests(case), _ranks(case)
    out = []
    for p in state["products"]:
        x, w = p["x"].double(), p["w"].double()
        # every adapter's A beside W: one product gives the base result and all rows' A x
        stacked = torch.cat([w] + [a.double() for a in p["a"]])
        both = x.matmul(stacked.t())
        y, h = both[:, :case["n"]], both[:, case["n"]:]
        # a row keeps the columns of its own adapter, scaled
        owner = np.repeat(np.arange(len(ranks)), ranks)
        mine = torch.from_numpy((ids[:, None] == owner[None, :]).astype(np.float64)).to(DEV)
        scale = torch.from_numpy(np.repeat(np.asarray(p["scale"]), ranks)).to(DEV)
        y = y + (h * mine * scale).matmul(torch.cat([b.double() for b in p["b"]], 1).t())
        if p["bias"] is not None:
            y = y + p["bias"].double()
        out.append(torch.sigmoid(y) if p["act"] == "sigmoid" else y)
    return out


def _exact_row(x, noise, temp, top_k, top_p, min_p):
    """One row by walking its logits from the largest down."""
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    lse = torch.logsumexp(x, 0)
    values, index = torch.sort(x, descending=True, stable=True)
    if temp <= 0:
        return index[0], values[0] - lse
    if top_k > 0:
        values, index = values[:top_k], index[:top_k]
    weights = ((values - values[0]) / temp).exp()
    if top_p < 1:
        reached = torch.searchsorted(weights.cumsum(0), top_p * weights.sum())
        weights = torch.where(torch.arange(len(weights), device=x.device) <= reached, weights, 0.0)
    weights = torch.where(weights >= min_p, weights, 0.0)
    mass = torch.zeros(len(noise) - GROUP, dtype=x.dtype, device=x.device)
    mass.index_add_(0, index // GROUP, weights)
    first = torch.argmax(mass / noise[GROUP:])
    score = torch.where(index // GROUP == first, weights / noise[index % GROUP], -1.0)
    # of equal scores the lowest index
    won = torch.where(score == score.max(), index, x.shape[0]).min()
    return won, x[won] - lse


def _exact_sample(case, seed):
    state = _sample_inputs(case, seed)
    rows = _settings(case)
    x, noise = state["logits"].double(), state["noise"].double()
    # the settings as they are held in 32 bits
    got = [_exact_row(x[i], noise[i], float(np.float32(t)), k, float(np.float32(p)),
                      float(np.float32(m))) for i, (t, k, p, m) in enumerate(rows)]
    return torch.stack([t for t, _ in got]).int(), torch.stack([l for _, l in got])


def exact(case, seed):
    return _exact_adapters(case, seed) if case["kind"] == "adapters" else _exact_sample(case, seed)


# -- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    if case["kind"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        numbers = GROUP + (vocab + GROUP - 1) // GROUP
        return {"bytes": rows * (vocab * (2 if case["bf16"] else 4) + 4 * numbers + 16 + 8),
                "flops": 8 * rows * vocab}
    rows, k, n = case["rows"], case["k"], case["n"]
    ids, ranks = _requests(case), _ranks(case)
    used = set(ids[ids >= 0].tolist())
    low = sum(int((ids == a).sum()) * ranks[a] for a in used)
    return {"bytes": case["products"] * 2 * (rows * (k + n) + n * k
                                             + sum(ranks[a] for a in used) * (k + n)),
            "flops": case["products"] * 2 * (rows * n * k + low * (k + n))}
