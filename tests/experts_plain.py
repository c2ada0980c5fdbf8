"""Plain forms in 64 bits of the int8 linear and mixture-of-experts operators, on the CPU."""
import math

import numpy as np
import torch

TINY = 2.0 ** -100
LARGEST = float(np.finfo(np.float32).max)
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def codes(g, shape, lo=-128, hi=127):
    return torch.randint(lo, hi + 1, shape, generator=g, dtype=torch.int8)


def route(x, bias, k, scoring, renormalise, groups=1, top_groups=1, best=1, scale=1.0, live=None):
    """ids, weights, offsets, rows, places: one token after the other."""
    x = x.double().numpy()
    T, E = x.shape
    b = np.zeros(E) if bias is None else bias.double().numpy()
    live = T if live is None else max(0, min(T, live))
    ids, weights = np.full((T, k), -1), np.zeros((T, k))
    for t in range(live):
        there = (x[t] > -math.inf) & (b > -math.inf)
        v = np.minimum(x[t], LARGEST)
        s = np.zeros(E)
        if there.any():
            with np.errstate(over="ignore"):
                if scoring == "sigmoid":
                    s[there] = 1 / (1 + np.exp(-v[there]))
                else:
                    p = np.exp(v[there] - v[there].max())
                    s[there] = p / p.sum()
        value = s + np.minimum(b, LARGEST)
        order = v if bias is None else value
        left = [e for e in range(E) if there[e]]
        if groups > 1:
            size = E // groups
            of = []
            for g in range(groups):
                mine = sorted((float((order if best == 1 else value)[e]) for e in left if e // size == g), reverse=True)[:best]
                if mine:
                    of.append((-sum(mine), g))
            stay = {g for _, g in sorted(of)[:top_groups]}
            left = [e for e in left if e // size in stay]
        chosen = sorted(left, key=lambda e: (-order[e], e))[:k]
        ids[t, :len(chosen)] = chosen
        w = s[chosen]
        if renormalise:
            w = w / w.sum() if w.sum() > 0 else 0 * w
        weights[t, :len(chosen)] = w * scale
    return (torch.from_numpy(ids).int(), torch.from_numpy(weights)) + tables(torch.from_numpy(ids), E)


def tables(ids, E):
    flat = ids.flatten().tolist()
    rows = [i for e in range(E) for i in np.flatnonzero(np.array(flat) == e).tolist()]
    offsets = np.concatenate([[0], np.cumsum([flat.count(e) for e in range(E)])])
    places = np.full(len(flat), -1)
    places[rows] = np.arange(len(rows))
    return tuple(torch.tensor(np.array(v), dtype=torch.int32) for v in (offsets, rows + [-1] * (len(flat) - len(rows)), places))


def quantize(x):
    """(codes, scales): fp32 scales, codes of the quotient in 64 bits rounded to fp32 first, as the formula says."""
    finite = x.float().isfinite().all(dim=1)
    amax = torch.where(finite, x.float().abs().amax(dim=1), torch.ones(x.shape[0])).clamp(min=TINY)
    q = (x.double() * 127.0 / amax.double()[:, None]).float().round()
    q = torch.where(finite[:, None], q, torch.zeros_like(q))
    return q.to(torch.int8), torch.where(finite, amax / 127.0, torch.full_like(amax, math.nan))


def scaled(a, b, sa, sb, bias, gated, out):
    """(C in 64 bits, how far an output of type `out` may be from it).

    Of D = float(acc) * sa * sb + bias: three roundings of the product and one of the sum, 2^-24 each. Of silu(g) = g / (1 + exp(-g)),
    whose derivative is under 1.1: g's error, and of the value the sum's and the quotient's rounding and the exponential's error; the
    last is 2 * 2^-24 in fp32 (a whole step), and with the fast forms behind 16-bit outputs |g| * 2^-24 (g * log2 e is rounded) and
    2 * 2^-24 each for the power of two and the reciprocal. Rounded up to 8 (+ |g|). Under 2^-120 the fast reciprocal gives 0."""
    u = 2.0 ** -24
    p = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()[None, :]
    d = p if bias is None else p + bias.double()[None, :]
    e = 3.01 * u * p.abs() + (0 if bias is None else u * (d.abs() + 4 * u * p.abs()))
    if gated:
        N = d.shape[1] // 2
        g, v, eg, ev = d[:, :N], d[:, N:], e[:, :N], e[:, N:]
        s = g * torch.sigmoid(g)
        es = 1.1 * eg + s.abs() * (8 + (0 if out == torch.float32 else g.abs())) * u + 2.0 ** -112
        d = s * v
        e = es * v.abs() + s.abs() * ev + es * ev + u * d.abs()
    return d, e + HALF_STEP[out] * (d.abs() + e) + 2.0 ** -149 + (2.0 ** -25 if out == torch.float16 else 0)


def combine(y, places, weights, add, out):
    """(sums in 64 bits, how far an output may be): k + 1 roundings of sums of the terms' sizes, and the output's own."""
    T, k = places.shape
    o = torch.zeros(T, y.shape[1], dtype=torch.float64) if add is None else add.double()
    mag = o.abs()
    for j in range(k):
        there = (places[:, j] >= 0) & (places[:, j] < y.shape[0])
        term = torch.where(there[:, None], y[places[:, j].clamp(0, max(0, y.shape[0] - 1)).long()].double() * weights[:, j].double()[:, None], torch.zeros(()).double())
        o, mag = o + term, mag + term.abs()
    e = (k + 1) * 2.0 ** -24 * mag
    return o, e + HALF_STEP[out] * (o.abs() + e) + 2.0 ** -149 + (2.0 ** -25 if out == torch.float16 else 0)


def near(got, want, bound, what=""):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4], want[bad][:4])
