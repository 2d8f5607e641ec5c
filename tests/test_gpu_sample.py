"""sample_tokens against the definition in 64 bits.

The kernel's weights are exp2((x - M) c) in fp32: relative error at most
|z| 2^-23 + 2^-22 for z = (x - M) / T, so below 1.5e-5 for |z| <= 100 (smaller weights
never decide a row here). Group sums add at most 256 roundings of 2^-24 (or the
2^-42 steps of the fixed-point sums), 1.6e-5. An arrival time is therefore within
TOL = 1e-4 of the exact one, and a prefix sum within 1e-4 of the exact one. A row
whose two earliest arrivals lie within TOL, or whose outcome depends on
top_p (1 -+ TOL), has more than one right answer; every other row has one.
"""

import math

import numpy as np
import pytest
import torch

from wkvm_amd import sample_noise_size, sample_tokens

pytestmark = pytest.mark.gpu

TOL = 1e-4
G = 256


def _clean(x):
    x = np.where(np.isnan(x), -np.inf, x)
    return np.minimum(x, float(np.finfo(np.float32).max))


def _race(arrivals):
    """Indices of the arrivals that may be the first one."""
    return np.flatnonzero(arrivals <= arrivals.min() * (1 + TOL))


def _outcomes(x, e, temp, top_k, top_p, min_p):
    """Every token that a row may give, one almost always."""
    x = _clean(x)
    if x.max() == -np.inf:
        return {-1}
    if not temp > 0:
        return {int(np.argmax(x))}
    order = np.argsort(-x, kind="stable")
    z = (x[order] - x[order[0]]) / temp
    if 0 < top_k < len(x):
        order, z = order[:top_k], z[:top_k]
    w = np.exp(z)
    out = set()
    for slack in ((1 - TOL, 1 + TOL) if top_p < 1 else (1,)):
        keep = np.ones(len(w), bool)
        if top_p < 1:
            keep[1:] = np.cumsum(w)[:-1] < top_p * slack * w.sum()
        if min_p > 0:
            keep &= w >= min(min_p, 1.0) * (1 - 1e-6)
        ids, ws = order[keep], w[keep]
        mass = np.bincount(ids // G, ws)
        with np.errstate(divide="ignore"):
            groups = _race(e[G:G + len(mass)] / mass)
            for g in groups:
                mine = ids // G == g
                for i in _race(e[ids[mine] % G] / ws[mine]):
                    out.add(int(ids[mine][i]))
    return out


def _check(logits, noise, temp, top_k, top_p, min_p, got, ambiguous=0.05):
    tokens, logp = (t.cpu().numpy() for t in got)
    x = logits.double().cpu().numpy()
    e = noise.double().cpu().numpy()
    rows = len(x)

    def per_row(v):
        v = v.cpu().numpy() if isinstance(v, torch.Tensor) else v
        return np.broadcast_to(np.asarray(v, dtype=np.float64), rows)
    temp, top_p, min_p = (per_row(np.float32(v) if np.isscalar(v) else v)
                          for v in (temp, top_p, min_p))
    top_k = per_row(top_k).astype(int)
    several = 0
    for r in range(rows):
        may = _outcomes(x[r], e[r], temp[r], top_k[r], top_p[r], min_p[r])
        assert int(tokens[r]) in may, (r, int(tokens[r]), may, temp[r], top_k[r], top_p[r], min_p[r])
        several += len(may) > 1
        c = _clean(x[r])
        if tokens[r] < 0:
            assert logp[r] == -np.inf
            continue
        d = c - c.max()
        want = d[tokens[r]] - math.log(np.exp(d).sum())
        # fp32: the difference x - M (2^-24 of it) and log of a sum of relative error
        # 1.5e-5 at most, most of it in terms that hardly count
        assert abs(logp[r] - want) <= 2e-5 + 2e-7 * abs(want), (r, logp[r], want)
    assert several <= max(1, ambiguous * rows), several


def _inputs(rows, vocab, dtype, seed, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn((rows, vocab), generator=gen) * spread).to(dtype).cuda()
    noise = torch.empty((rows, sample_noise_size(vocab))).exponential_(generator=gen).cuda()
    return logits, noise


def _settings(rows, seed):
    """Every combination of filters, in turn."""
    rng = np.random.default_rng(seed)
    on = np.arange(rows)
    temp = torch.tensor(rng.choice([0.3, 0.7, 1.0, 1.5], rows), dtype=torch.float32)
    temp[on % 11 == 10] = 0.0
    k = torch.tensor(np.where(on & 1, rng.choice([1, 2, 17, 50, 300], rows), 0), dtype=torch.int32)
    p = torch.tensor(np.where(on & 2, rng.choice([0.1, 0.5, 0.9, 0.99], rows), 1.0),
                     dtype=torch.float32)
    m = torch.tensor(np.where(on & 4, rng.choice([0.01, 0.1, 0.5], rows), 0.0),
                     dtype=torch.float32)
    return temp, k, p, m


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 255, 256, 257, 1000, 4095, 4097, 8191, 16385, 32003,
                                   65536, 65537, 131072, 131077, 200003])
def test_mixed_settings(vocab, dtype):
    rows = 24
    logits, noise = _inputs(rows, vocab, dtype, vocab)
    temp, k, p, m = _settings(rows, vocab)
    got = sample_tokens(logits, noise, temperature=temp.cuda(), top_k=k.cuda(), top_p=p.cuda(),
                        min_p=m.cuda())
    # (a small vocabulary in bf16 has few weights: none of them makes more rows ambiguous)
    _check(logits, noise, temp, k, p, m, got)


@pytest.mark.parametrize("vocab", [800003, 1048579, 1 << 21])
def test_large_vocabularies(vocab):
    """More groups than the candidates' group weights have room for."""
    rows = 8
    logits, noise = _inputs(rows, vocab, torch.bfloat16, 7)
    temp, k, p, m = _settings(rows, 9)
    got = sample_tokens(logits, noise, temperature=temp.cuda(), top_k=k.cuda(), top_p=p.cuda(),
                        min_p=m.cuda())
    _check(logits, noise, temp, k, p, m, got, ambiguous=0.5)


@pytest.mark.parametrize("top_k,top_p,min_p", [(0, 1.0, 0.0), (40, 1.0, 0.0), (0, 0.95, 0.0),
                                               (0, 1.0, 0.05), (50, 0.9, 0.02), (5000, 1.0, 0.0),
                                               (20000, 0.99, 0.0), (0, 0.0, 0.0), (1, 1.0, 0.0),
                                               (40000, 0.5, 1.0), (39999, 0.999, 0.0)])
@pytest.mark.parametrize("spread", [0.0, 0.02, 1.0, 8.0, 300.0])
def test_filters_over_flat_and_steep_rows(top_k, top_p, min_p, spread):
    logits, noise = _inputs(5, 40000, torch.float32, 5, spread)
    got = sample_tokens(logits, noise, temperature=0.9, top_k=top_k, top_p=top_p, min_p=min_p)
    _check(logits, noise, 0.9, top_k, top_p, min_p, got)


@pytest.mark.parametrize("top_k", [1, 3, 100, 2500, 9000])
@pytest.mark.parametrize("top_p", [1.0, 0.6, 0.05])
def test_ties_go_to_the_lowest_index(top_k, top_p):
    """A few distinct values only: nearly every cut falls among equal logits."""
    gen = torch.Generator().manual_seed(top_k)
    logits = torch.randint(0, 3, (6, 20000), generator=gen).float()
    logits[1:4] *= -0.0  # rows of zeros of either sign
    logits[2, ::2] = 0.0
    noise = torch.empty((6, sample_noise_size(20000))).exponential_(generator=gen)
    logits, noise = logits.cuda(), noise.cuda()
    got = sample_tokens(logits, noise, temperature=1.0, top_k=top_k, top_p=top_p)
    _check(logits, noise, 1.0, top_k, top_p, 0.0, got, ambiguous=1.0 if top_p < 1 else 0.05)


@pytest.mark.parametrize("settings", [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.9, 0.05), (0.0, 0, 1.0, 0.0),
                                      (1.0, 5, 1.0, 0.0), (1.0, 0, 0.9, 0.0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_rows_and_special_values(settings, dtype):
    temp, k, p, m = settings
    vocab = 5003
    logits, noise = _inputs(10, vocab, torch.float32, 3)
    low = torch.finfo(dtype).min
    logits[0] = -math.inf                      # a mask that leaves nothing
    logits[1] = math.nan
    logits[2] = low                            # the lowest value everywhere: all equal
    logits[3] = -math.inf
    logits[3, 4999] = -7.0                     # a single token left
    logits[4, ::3] = math.nan
    logits[4, 1::3] = -math.inf
    logits[5, 17] = logits[5, 4100] = math.inf  # two tokens at +inf
    logits[6] = low
    logits[6, 100:130] = 2.0
    logits[7] = -math.inf
    logits[7, :3] = low                        # three tokens at the lowest value beside -inf
    logits[8] *= 1e-30                         # differences far below one
    logits = logits.to(dtype)
    got = sample_tokens(logits, noise, temperature=temp, top_k=k, top_p=p, min_p=m)
    _check(logits, noise, temp, k, p, m, got, ambiguous=0.4)
    assert got[0][:2].tolist() == [-1, -1]
    assert got[0][3].item() == 4999 and got[0][5].item() in (17, 4100)
    assert 100 <= got[0][6].item() < 130 and 0 <= got[0][7].item() < 3


@pytest.mark.parametrize("shift", [0.0, -3e4, 1e6])
@pytest.mark.parametrize("top_p,min_p", [(0.6, 0.0), (0.9, 0.0), (0.98, 0.0), (0.999, 0.0),
                                         (0.98, 0.3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_top_p_far_down_flat_rows(dtype, top_p, min_p, shift):
    """Tens of thousands of tokens kept, many of them equal (in bf16, and far from zero), with
    NaN and -inf among them; one row's mass lies in a few groups, one row is all equal but -inf."""
    vocab = 50021
    logits, noise = _inputs(8, vocab, torch.float32, 23, 0.7)
    logits[1] *= 3.0
    logits[2] *= 0.01
    logits[3, ::2] = math.nan
    logits[4, 5::7] = -math.inf
    logits[5, 2000:] -= 9.0
    logits[6] = 0.0
    logits[6, ::5] = -math.inf
    logits = (logits + shift).to(dtype)
    for temp in (0.7, 1.3):
        got = sample_tokens(logits, noise, temperature=temp, top_p=top_p, min_p=min_p)
        _check(logits, noise, temp, 0, top_p, min_p, got, ambiguous=0.25)


@pytest.mark.parametrize("temperature", [1e-30, 1e-6, 1e6, 1e30, math.inf])
def test_extreme_temperatures(temperature):
    logits, noise = _inputs(4, 3000, torch.float32, 9)
    got = sample_tokens(logits, noise, temperature=temperature)
    if temperature < 1:
        assert got[0].tolist() == logits.argmax(1).tolist()
    else:  # every token weighs 1 to 1e-4
        _check(logits, noise, 1e9, 0, 1.0, 0.0, got, ambiguous=1.0)


def test_strided_rows_and_one_row():
    wide, noise = _inputs(7, 3001, torch.float32, 11)
    many = torch.empty((7, noise.shape[1] + 5), device="cuda").exponential_()
    many[:, :noise.shape[1]] = noise
    view = wide[:, 1:2500]  # rows 3001 apart, starting at an odd element
    a = sample_tokens(view, many, top_k=30, top_p=0.9)
    b = sample_tokens(view.contiguous(), noise, top_k=30, top_p=0.9)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c = sample_tokens(view[3:4], many[3:4], top_k=30, top_p=0.9, logprobs=False)
    assert c[1] is None and c[0].item() == b[0][3].item()
    t = sample_tokens(view.t().contiguous().t(), many, top_k=30, top_p=0.9)  # columns apart
    assert torch.equal(t[0], b[0])
    none = sample_tokens(wide[:0], noise[:0])
    assert none[0].shape == (0,) and none[1].shape == (0,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_do_not_depend_on_the_batch_and_calls_repeat(dtype):
    logits, noise = _inputs(40, 70001, dtype, 13)
    temp, k, p, m = (t.cuda() for t in _settings(40, 2))
    a = sample_tokens(logits, noise, temperature=temp, top_k=k, top_p=p, min_p=m)
    for _ in range(3):
        b = sample_tokens(logits, noise, temperature=temp, top_k=k, top_p=p, min_p=m)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for r in (0, 7, 23, 39):
        one = sample_tokens(logits[r:r + 1], noise[r:r + 1], temperature=temp[r].item(),
                            top_k=int(k[r]), top_p=p[r].item(), min_p=m[r].item())
        assert one[0].item() == a[0][r].item() and one[1].item() == a[1][r].item()


def test_host_sequences_equal_device_tensors():
    logits, noise = _inputs(12, 1234, torch.float32, 17)
    temp, k, p, m = _settings(12, 4)
    a = sample_tokens(logits, noise, temperature=temp.tolist(), top_k=k.tolist(), top_p=p, min_p=m)
    b = sample_tokens(logits, noise, temperature=temp.cuda(), top_k=k.cuda(), top_p=p.cuda(),
                      min_p=m.cuda())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_device_settings_out_of_range_stay_in_the_vocabulary():
    """Values that the host cannot check: NaN turns a filter off, a negative or NaN
    temperature is greedy, min_p is held to 1; bad noise still gives a token."""
    logits, noise = _inputs(6, 999, torch.float32, 19)
    nan, f32 = math.nan, torch.float32
    temp = torch.tensor([1.0, -1.0, nan, 1.0, 1.0, 1.0], dtype=f32)
    k = torch.tensor([0, 0, 0, -5, 5000, 0], dtype=torch.int32)
    p = torch.tensor([nan, 1.0, 1.0, -3.0, 7.0, 1.0], dtype=f32)
    m = torch.tensor([nan, 0.0, 0.0, 0.0, -1.0, 9.0], dtype=f32)
    got = sample_tokens(logits, noise, temperature=temp.cuda(), top_k=k.cuda(), top_p=p.cuda(),
                        min_p=m.cuda())
    top = logits.argmax(1)
    assert got[0][1].item() == top[1].item() and got[0][2].item() == top[2].item()
    assert got[0][3].item() == top[3].item() and got[0][5].item() == top[5].item()
    plain = sample_tokens(logits, noise)
    assert got[0][0].item() == plain[0][0].item() and got[0][4].item() == plain[0][4].item()
    for bad in (0.0, -1.0, nan, math.inf):
        t = sample_tokens(logits, torch.full_like(noise, bad), top_k=50, top_p=0.9)[0]
        assert bool(((t >= 0) & (t < 999)).all())


def test_frequencies_follow_the_probabilities():
    """40,000 draws from one row: each token's count within 5 standard deviations of its
    probability, with and without a nucleus."""
    vocab, draws = 600, 40000
    gen = torch.Generator().manual_seed(23)
    row = torch.randn(vocab, generator=gen) * 2
    logits = row.cuda().expand(draws, vocab).contiguous()
    dev_gen = torch.Generator("cuda").manual_seed(29)
    noise = torch.empty((draws, sample_noise_size(vocab)), device="cuda").exponential_(
        generator=dev_gen)
    for top_p in (1.0, 0.8):
        tokens = sample_tokens(logits, noise, temperature=0.8, top_p=top_p)[0].cpu().numpy()
        w = np.exp(row.double().numpy() / 0.8)
        order = np.argsort(-w, kind="stable")
        if top_p < 1:
            cum = np.cumsum(w[order])
            w[order[1:][cum[:-1] >= top_p * cum[-1]]] = 0
        prob = w / w.sum()
        count = np.bincount(tokens, minlength=vocab)
        assert count[prob == 0].sum() == 0
        dev = np.abs(count - draws * prob) / np.sqrt(np.maximum(draws * prob * (1 - prob), 1.0))
        assert dev.max() < 5, dev.max()


def test_under_graph_capture():
    logits, noise = _inputs(8, 5000, torch.float32, 31)
    temp, k, p, m = (t.cuda() for t in _settings(8, 6))
    eager = sample_tokens(logits, noise, temperature=temp, top_k=k, top_p=p, min_p=m)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample_tokens(logits, noise, temperature=temp, top_k=k, top_p=p, min_p=m)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])
        logits.copy_(_inputs(8, 5000, torch.float32, 40 + i)[0])
        eager = sample_tokens(logits, noise, temperature=temp, top_k=k, top_p=p, min_p=m)
        torch.cuda.synchronize()


def test_on_another_stream():
    logits, noise = _inputs(16, 30011, torch.float32, 37)
    want = sample_tokens(logits, noise, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sample_tokens(logits, noise, top_p=[0.9] * 16)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals():
    logits, noise = _inputs(4, 1000, torch.float32, 41)
    for kw, match in [({"temperature": -1.0}, "temperature"), ({"temperature": math.nan}, "temperature"),
                      ({"top_k": -1}, "top_k"), ({"top_k": 1.5}, "top_k"), ({"top_p": 1.1}, "top_p"),
                      ({"top_p": [0.5] * 3}, "3 values"), ({"min_p": -0.1}, "min_p"),
                      ({"min_p": torch.zeros(4, device="cuda").double()}, "min_p"),
                      ({"top_k": torch.zeros(4, device="cuda")}, "top_k"),
                      ({"temperature": torch.ones(5, device="cuda")}, "temperature"),
                      ({"temperature": torch.ones(8, device="cuda")[::2]}, "temperature")]:
        with pytest.raises(ValueError, match=match):
            sample_tokens(logits, noise, **kw)
    for bad_logits, bad_noise in [(logits.half(), noise), (logits[0], noise), (logits.cpu(), noise),
                                  (logits, noise[:3]), (logits, noise[:, :-1]),
                                  (logits, noise.double()), (logits, noise.cpu()),
                                  (logits[:, :0], noise)]:
        with pytest.raises(ValueError):
            sample_tokens(bad_logits, bad_noise)
    with pytest.raises(ValueError, match="tokens per row"):
        sample_tokens(torch.zeros((1, (1 << 21) + 1), device="cuda"), noise[:1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,down", [(1 << 21, 22.25), (1 << 21, 23.5), (200003, 21.0)])
def test_a_flat_tail_far_below_one_sure_token(dtype, vocab, down):
    """One token at 0 and all others at -down (weights of 2^-30 to 2^-34), of which top-p keeps the
    first half. Whole groups 2 % of the tail before and after that cut are drawn or not. The tail
    weighs 1.3e-4 to 4.6e-4 of the row. The row's weight and top-p's share of it hold 24 bits, which
    moves the cut by at most 2 x 2^-24 / 1.3e-4 = 0.1 % of the tail, and a weight of 2^-34 held to
    2^-42 moves it by 0.4 %."""
    x = torch.full((3, vocab), -down, dtype=dtype)
    at = 777
    x[:, at] = 0.0
    tail = math.exp(-float(-x[0, 0])) * (vocab - 1)
    share = (1 + 0.5 * tail) / (1 + tail)
    top_p = float(np.float32(share))
    kept = (top_p * (1 + tail) - 1) / tail  # of the tail, by the share as it is held
    assert abs(kept - 0.5) < 0.01
    groups = (vocab + G - 1) // G
    inside, outside = int((kept - 0.02) * groups), int((kept + 0.02) * groups)
    noise = torch.empty((3, sample_noise_size(vocab))).exponential_(
        generator=torch.Generator().manual_seed(3)).clamp_(min=1e-3)
    noise[:, G + at // G] = 1e30           # the sure token's group comes last
    noise[0, G + inside] = 1e-12           # kept, and first
    noise[1, G + outside] = 1e-12          # would be first, but is cut off
    noise[1, G + inside] = 1e-9
    noise[2, G + groups - 1] = 1e-12
    noise[2, G + inside - 1] = 1e-9
    noise[:, :G] = torch.linspace(1, 2, G)  # token 0 of a group comes first
    tokens = sample_tokens(x.cuda(), noise.cuda(), top_p=top_p)[0].cpu().tolist()
    assert tokens == [inside * G, inside * G, (inside - 1) * G]


def test_host_arrays_and_ranges_are_sequences():
    logits, noise = _inputs(12, 1234, torch.float32, 17)
    temp, k, p, m = _settings(12, 4)
    want = sample_tokens(logits, noise, temperature=temp.cuda(), top_k=k.cuda(), top_p=p.cuda(),
                         min_p=m.cuda())
    got = sample_tokens(logits, noise, temperature=temp.numpy(), top_k=k.numpy(),
                        top_p=p.double().numpy(), min_p=tuple(m.tolist()))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    ranks = torch.arange(1, 13, dtype=torch.int32)
    a = sample_tokens(logits, noise, top_k=range(1, 13), temperature=np.float32(0.5))
    b = sample_tokens(logits, noise, top_k=ranks.cuda(), temperature=np.asarray(0.5))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for bad in (np.ones((12, 1)), torch.ones((12, 1)), np.ones(11)):
        with pytest.raises(ValueError, match="values"):
            sample_tokens(logits, noise, temperature=bad)
