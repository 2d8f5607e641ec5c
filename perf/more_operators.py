"""Linear attention with a decay for each head, and products with 4-bit weights: timing cases.

* ``linear``  ``linear_decode_slots`` / ``linear_prefill_varlen``: the state of every request in its
              slot, ``S <- exp(g) S + k v^T``, ``y = scale q^T S``, one token per slot or ragged
              prompts
* ``w4``      ``proj_w4``: projections whose weights are 4-bit codes with a scale (and a zero point)
              for each group of inputs

``listed()`` holds the cases, ``draw(rng)`` makes more of the same ranges. ``run`` computes a case in
its plain form (elementary torch operations in 32 bits) or, where ``own`` is set, through the
framework's entry points. ``exact`` computes it from the definition in 64 bits.

Hidden sizes, heads and slots are those of RWKV-7 0.1B, 1.5B and 7B; batches and prompts are those of
the repository's benchmark and of a serving engine around them. Heads of 128 channels and queries and
keys shared by several heads are what other models with such a state have.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
CHUNK = 64          # tokens of a chunk of the plain form
LONGEST = 16384     # tokens of one prompt
LARGEST_TOKENS = 8 * 4096 * 32 * 64 * 64      # tokens x heads x K x V
LARGEST_DECODE = 3 * 256 * 32 * 64 * 64       # layers x rows x heads x K x V
LARGEST_W4 = 3 * 3001 * 2048 * 2048           # products x rows x n x k
LARGEST_WEIGHT = 65536 * 2048


def listed():
    return [
        # A few live requests of the small model, decay fixed for each head: latency is all.
        {"name": "linear_decode_4", "kind": "decode", "rows": 4, "slots": 16, "layers": 1,
         "heads": 12, "shared": 1, "K": 64, "V": 64, "token_decay": False, "f32": False},
        # Heads of 128 channels, queries and keys shared by four heads, odd batch, fp32 outputs.
        {"name": "linear_decode_61", "kind": "decode", "rows": 61, "slots": 64, "layers": 2,
         "heads": 16, "shared": 4, "K": 128, "V": 128, "token_decay": True, "f32": True},
        # The headline decode batch over three layers, decays from the token.
        {"name": "linear_decode_256", "kind": "decode", "rows": 256, "slots": 512, "layers": 3,
         "heads": 32, "shared": 1, "K": 64, "V": 64, "token_decay": True, "f32": False},
        # One slice of a prompt, as the reference prefills a request.
        {"name": "linear_slice", "kind": "prefill", "tokens": 512, "seqs": 1, "heads": 32,
         "shared": 1, "K": 64, "V": 64, "token_decay": True, "fresh": False, "f32": False},
        # One long prompt: few heads to share the work, so its length has to.
        {"name": "linear_long", "kind": "prefill", "tokens": 16384, "seqs": 1, "heads": 12,
         "shared": 1, "K": 64, "V": 64, "token_decay": False, "fresh": True, "f32": False},
        # Ragged prompts (one empty, one of a single token), heads of 128 channels.
        {"name": "linear_ragged", "kind": "prefill", "tokens": 9001, "seqs": 19, "heads": 16,
         "shared": 4, "K": 128, "V": 128, "token_decay": True, "fresh": False, "f32": True},
        # The benchmark's prefill: eight prompts of 4,096 tokens.
        {"name": "linear_batch", "kind": "prefill", "tokens": 32768, "seqs": 8, "heads": 32,
         "shared": 1, "K": 64, "V": 64, "token_decay": True, "fresh": True, "f32": False},
        # One request of the small model: three projections of one row.
        {"name": "w4_one", "kind": "w4", "rows": 1, "k": 768, "n": 768, "products": 3,
         "group": 32, "zero": True, "act": False},
        # One request's logits: the vocabulary's product is the largest weight there is.
        {"name": "w4_vocab", "kind": "w4", "rows": 1, "k": 2048, "n": 65536, "products": 1,
         "group": 128, "zero": False, "act": False},
        # A handful of requests, odd width, bias and activation.
        {"name": "w4_9", "kind": "w4", "rows": 9, "k": 2048, "n": 2047, "products": 3,
         "group": 64, "zero": True, "act": True},
        # A decode batch of the 7B shape.
        {"name": "w4_256", "kind": "w4", "rows": 256, "k": 4096, "n": 4096, "products": 3,
         "group": 128, "zero": True, "act": False},
        # A few prompts in one prefill, ragged.
        {"name": "w4_prompts", "kind": "w4", "rows": 3001, "k": 2048, "n": 2048, "products": 3,
         "group": 128, "zero": False, "act": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decode", "prefill", "w4", "w4"])
    if kind == "w4":
        k = rng.choice([768, 2048, 4096, 32 * _log(rng, 1, 128)])
        n = rng.choice([k, k, _log(rng, 1, 4096), _log(rng, 4096, LARGEST_WEIGHT // 4096)])
        products = 1 if n > 4096 else rng.choice([1, 2, 3])
        rows = _log(rng, 1, max(1, min(8192, LARGEST_W4 // (products * k * n))))
        return {"kind": "w4", "rows": rows, "k": k, "n": n, "products": products,
                "group": rng.choice([32, 64, 128]), "zero": rng.random() < 0.5,
                "act": rng.random() < 0.3}
    dims = rng.choice([(64, 64), (64, 64), (128, 128), (64, 128), (128, 64)])
    shared = rng.choice([1, 1, 2, 4])
    heads = shared * max(1, _log(rng, 4, 48) // shared)
    both = {"heads": heads, "shared": shared, "K": dims[0], "V": dims[1],
            "token_decay": rng.random() < 0.6, "f32": rng.random() < 0.4}
    size = heads * dims[0] * dims[1]
    if kind == "decode":
        layers = rng.choice([1, 1, 2, 3])
        rows = _log(rng, 1, max(1, min(512, LARGEST_DECODE // (layers * size))))
        return {"kind": "decode", "rows": rows, "slots": rows + rng.randint(0, rows),
                "layers": layers, **both}
    tokens = _log(rng, 1, min(32768, LARGEST_TOKENS // size))
    few = max(1, -(-tokens // LONGEST))
    seqs = max(few, min(_log(rng, 1, 64), tokens))
    return {"kind": "prefill", "tokens": tokens, "seqs": seqs, "fresh": rng.random() < 0.5, **both}


# -- inputs ---------------------------------------------------------------------------------------

def _lengths(case):
    """Tokens of every sequence, from the case alone: equal where they divide the tokens and there
    are at most eight, else random cuts (so that empty sequences occur), none past ``LONGEST``."""
    tokens, seqs = case["tokens"], case["seqs"]
    if seqs <= 8 and tokens % seqs == 0:
        return [tokens // seqs] * seqs
    rng = random.Random("%(tokens)d tokens in %(seqs)d prompts" % case)
    while True:
        cuts = sorted(rng.randint(0, tokens) for _ in range(seqs - 1))
        if seqs >= 8 and tokens > 1:  # (an empty one and one of a single token)
            cuts[0] = cuts[1] = 0
            cuts[2] = 1
            cuts.sort()
        out = [b - a for a, b in zip([0] + cuts, cuts + [tokens])]
        if max(out) <= LONGEST:
            return out


def _slots(case, rows, slots):
    rng = random.Random("%d of %d slots" % (rows, slots))
    return rng.sample(range(1, slots + 1), rows)


def _tensors(case, gen, tokens):
    """Queries, keys, values and log-decays of one layer, as projections give them."""
    heads, qk = case["heads"], case["heads"] // case["shared"]

    def n(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    q, k = n(tokens, qk, case["K"]), n(tokens, qk, case["K"])
    k /= math.sqrt(case["K"])
    v = n(tokens, heads, case["V"])
    if case["token_decay"]:  # -rate softplus(x): a few tokens forget nearly everything
        rate = torch.exp(torch.rand(heads, generator=gen, device=DEV) * 5 - 4)
        g = -rate * torch.log1p(torch.exp(2 * n(tokens, heads)))
    else:  # each head its own span, 16 to some thousand tokens
        g = torch.log1p(-torch.exp2(-4 - 8 * torch.rand(heads, generator=gen, device=DEV)))
    return {"q": q.to(torch.bfloat16), "k": k.to(torch.bfloat16), "v": v.to(torch.bfloat16),
            "g": g}


def _linear_inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    decode = case["kind"] == "decode"
    rows = case["rows"] if decode else case["seqs"]
    slots = case["slots"] if decode else rows + 3
    tokens = rows if decode else case["tokens"]
    layers = case["layers"] if decode else 1
    pool = torch.randn((layers, slots + 1, case["heads"], case["K"], case["V"]), generator=gen,
                       device=DEV)
    ids = _slots(case, rows, slots)
    state = {"pool": pool, "ids": ids, "rows": torch.tensor(ids, device=DEV),
             "layers": [_tensors(case, gen, tokens) for _ in range(layers)],
             "scale": 1 / math.sqrt(case["K"]), "shared": case["shared"],
             "dtype": torch.float32 if case["f32"] else torch.bfloat16}
    if not decode:
        lengths = _lengths(case)
        cu = [0]
        for length in lengths:
            cu.append(cu[-1] + length)
        longest = -(-max(lengths) // CHUNK) * CHUNK
        at = torch.arange(longest, device=DEV)[None, :]
        first = torch.tensor(cu[:-1], device=DEV)[:, None]
        real = at < torch.tensor(lengths, device=DEV)[:, None]
        state.update(cu=cu, real=real, token=torch.where(real, first + at, 0),
                     fresh=case["fresh"])
    return state


def _w4_inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    k, n, group = case["k"], case["n"], case["group"]
    groups = -(-k // group)
    products = []
    for _ in range(case["products"]):
        # codes as rounding a weight's group to its range leaves them: middle ones more often
        codes = torch.randn((n, k), generator=gen, device=DEV).mul_(3).add_(7.5)
        codes = codes.clamp_(0, 15).round_().to(torch.uint8)
        scale = (torch.rand((n, groups), generator=gen, device=DEV) + 0.5) / (4.0 * math.sqrt(k))
        zero = torch.randint(5, 11, (n, groups), generator=gen, device=DEV).to(torch.uint8)
        products.append({
            "x": torch.randn((case["rows"], k), generator=gen, device=DEV).to(torch.bfloat16),
            "codes": codes, "scale": scale.to(torch.float16),
            "zero": zero if case["zero"] else None,
            "bias": ((torch.randn(n, generator=gen, device=DEV) * 0.5).to(torch.bfloat16)
                     if case["act"] else None),
            "act": "sigmoid" if case["act"] else None})
    return {"products": products, "group": group}


def prepare(case, seed):
    if case["kind"] == "w4":
        state = _w4_inputs(case, seed)
        if own:
            from wkvm_amd import W4Weight

            for p in state["products"]:
                p["weight"] = W4Weight.from_codes(p["codes"], p["scale"], p["zero"],
                                                  group=state["group"])
        return state
    state = _linear_inputs(case, seed)
    if own:
        from wkvm_amd import ops

        rows = state["pool"].shape[1]
        if case["kind"] == "decode":
            state["plan"] = ops.decode_plan(state["ids"], rows, torch.device(DEV))
        else:
            state["plan"] = (state["rows"].int(),
                             torch.tensor(state["cu"], dtype=torch.int32, device=DEV))
    return state


# -- one pass -------------------------------------------------------------------------------------

def _per_head(x, shared):
    return x.float().repeat_interleave(shared, dim=1) if shared > 1 else x.float()


def _plain_decode(state):
    out = []
    for pool, t in zip(state["pool"], state["layers"]):
        q, k = _per_head(t["q"], state["shared"]), _per_head(t["k"], state["shared"])
        h = pool[state["rows"]] * torch.exp(t["g"])[..., None, None]
        h = h + k[..., :, None] * t["v"].float()[..., None, :]
        pool[state["rows"]] = h
        out.append(((q * state["scale"])[..., :, None] * h).sum(2).to(state["dtype"]))
    return out


def _plain_prefill(state):
    """Chunk by chunk, every sequence padded to the longest: within a chunk the scores under their
    decays, before it the state."""
    (t,), pool, real = state["layers"], state["pool"][0], state["real"]
    q, k = _per_head(t["q"], state["shared"]), _per_head(t["k"], state["shared"])
    v = t["v"].float()
    tokens, heads, V = v.shape
    K = q.shape[2]
    g = t["g"] if t["g"].dim() == 2 else t["g"].expand(tokens, heads)
    y = torch.zeros((tokens + 1, heads, V), device=v.device)
    h = pool[state["rows"]]
    if state["fresh"]:
        h = torch.zeros_like(h)
    seqs, longest = real.shape
    mask = real[:, None, :]
    causal = torch.ones((CHUNK, CHUNK), dtype=torch.bool, device=v.device).tril()
    for c in range(0, longest, CHUNK):
        at = state["token"][:, c:c + CHUNK].reshape(-1)
        live = mask[..., c:c + CHUNK]

        def take(x, width):
            x = x[at].reshape(seqs, CHUNK, heads, width).transpose(1, 2)
            return torch.where(live[..., None], x, 0.0).contiguous()

        qc, kc, vc = take(q, K), take(k, K), take(v, V)
        total = take(g[..., None], 1)[..., 0].double().cumsum(-1)
        between = total[..., :, None] - total[..., None, :]
        decay = torch.where(causal, torch.exp(between.float()), 0.0)
        scores = torch.matmul(qc, kc.transpose(-1, -2).contiguous()) * decay
        o = torch.matmul(scores, vc) + torch.matmul(qc, h) * torch.exp(total.float())[..., None]
        left = torch.exp((total[..., -1:] - total).float())
        kd = (kc * left[..., None]).transpose(-1, -2).contiguous()
        h = h * torch.exp(total[..., -1].float())[..., None, None] + torch.matmul(kd, vc)
        where = torch.where(real[:, c:c + CHUNK].reshape(-1), at, tokens)
        y[where] = o.transpose(1, 2).reshape(-1, heads, V)
    pool[state["rows"]] = h
    return (y[:tokens] * state["scale"]).to(state["dtype"])


def _plain_w4(state):
    out = []
    for p in state["products"]:
        n, k = p["codes"].shape
        zero = 8.0 if p["zero"] is None else p["zero"].float().repeat_interleave(
            state["group"], dim=1)[:, :k]
        scale = p["scale"].float().repeat_interleave(state["group"], dim=1)[:, :k]
        y = p["x"].float() @ ((p["codes"].float() - zero) * scale).t()
        if p["bias"] is not None:
            y = y + p["bias"].float()
        if p["act"] == "sigmoid":
            y = 1.0 / (1.0 + torch.exp(-y))
        out.append(y.to(torch.bfloat16))
    return out


def run(state):
    if "products" in state:
        if not own:
            return _plain_w4(state)
        from wkvm_amd import proj_w4

        return proj_w4([(p["x"], p["weight"], p["bias"], p["act"]) for p in state["products"]])
    pool = state["pool"]
    if "cu" not in state:
        if not own:
            y = _plain_decode(state)
        else:
            from wkvm_amd import linear_decode_slots

            ids, order = state["plan"]
            y = [linear_decode_slots(layer, ids, t["q"], t["k"], t["v"], t["g"],
                                     scale=state["scale"], out_dtype=state["dtype"],
                                     row_order=order)
                 for layer, t in zip(pool, state["layers"])]
        return *y, pool
    if not own:
        return _plain_prefill(state), pool
    from wkvm_amd import linear_prefill_varlen

    (t,), (ids, cu) = state["layers"], state["plan"]
    return linear_prefill_varlen(pool[0], ids, cu, t["q"], t["k"], t["v"], t["g"],
                                 zero_init=state["fresh"], scale=state["scale"],
                                 out_dtype=state["dtype"]), pool


# -- from the definitions, in 64 bits ----------------------------------------------------------------

def _step(h, q, k, v, g):
    """One token of ``[n, heads]`` states in 64 bits: the new state and its output."""
    h = h * g.exp()[..., None, None]
    h.addcmul_(k[..., None], v[..., None, :])
    return h, torch.matmul(q[..., None, :], h)[..., 0, :]


def _exact_linear(case, seed):
    state = _linear_inputs(case, seed)
    heads, shared = case["heads"], case["shared"]
    whose = torch.arange(heads, device=DEV) // shared  # a head's queries and keys
    pool = state["pool"].double()
    ys = []
    for pool_layer, t in zip(pool, state["layers"]):
        q, k = t["q"].double()[:, whose], t["k"].double()[:, whose]
        v, g = t["v"].double(), t["g"].double()
        if g.dim() == 1:
            g = g[None, :].expand(len(v), heads)
        if case["kind"] == "decode":
            h, y = _step(pool_layer[state["ids"]], q, k, v, g)
            pool_layer[state["ids"]] = h
            ys.append(y * state["scale"])
            continue
        # token by token, the sequences side by side, longest first so that the live ones lead
        cu = state["cu"]
        lengths = [b - a for a, b in zip(cu, cu[1:])]
        order = sorted(range(len(lengths)), key=lambda s: -lengths[s])
        first = torch.tensor([cu[s] for s in order], device=DEV)
        rows = [state["ids"][s] for s in order]
        h = pool_layer[rows]
        if case["fresh"]:
            h.zero_()
        y = torch.zeros_like(v)
        live = len(order)
        for i in range(max(lengths)):
            while lengths[order[live - 1]] <= i:
                live -= 1
            at = first[:live] + i
            h[:live], y[at] = _step(h[:live], q[at], k[at], v[at], g[at])
        pool_layer[rows] = h
        ys.append(y * state["scale"])
    return *ys, pool


def _exact_w4(case, seed):
    state = _w4_inputs(case, seed)
    out = []
    for p in state["products"]:
        n, k = p["codes"].shape
        w = p["codes"].double()
        for i in range(p["scale"].shape[1]):  # group by group, in place
            part = w[:, i * case["group"]:(i + 1) * case["group"]]
            part -= 8 if p["zero"] is None else p["zero"][:, i:i + 1].double()
            part *= p["scale"][:, i:i + 1].double()
        y = torch.nn.functional.linear(p["x"].double(), w)
        if p["bias"] is not None:
            y = y + p["bias"].double()
        out.append(torch.sigmoid(y) if p["act"] == "sigmoid" else y)
    return out


def exact(case, seed):
    return _exact_w4(case, seed) if case["kind"] == "w4" else _exact_linear(case, seed)


# -- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    if case["kind"] == "w4":
        rows, k, n = case["rows"], case["k"], case["n"]
        groups = -(-k // case["group"])
        weight = n * k // 2 + n * groups * 2 + (n * groups // 2 if case["zero"] else 0)
        return {"bytes": case["products"] * (weight + 2 * rows * (k + n)),
                "flops": case["products"] * 2 * rows * n * k}
    heads, K, V = case["heads"], case["K"], case["V"]
    qk = heads // case["shared"]
    decode = case["kind"] == "decode"
    layers = case["layers"] if decode else 1
    seqs = case["rows"] if decode else case["seqs"]
    tokens = case["rows"] if decode else case["tokens"]
    state = seqs * heads * K * V * 4
    reads = 1 if decode or not case["fresh"] else 0
    token = 2 * (2 * qk * K + heads * V) + heads * V * (4 if case["f32"] else 2)
    decay = 4 * heads * (tokens if case["token_decay"] else 1)
    # a token's share of the state's update and of reading it: two multiply-adds per entry
    return {"bytes": layers * (state * (1 + reads) + tokens * token + decay),
            "flops": layers * tokens * heads * K * V * 4}
