"""Plain forms in 64 bits of the 8-bit serving operators, on the CPU, and the inputs their tests share."""
import numpy as np
import torch

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
TINY = 2.0 ** -100
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def to_code(x32, dtype):
    """fp32 values to codes, ties to even (the arithmetic before it is fp32 too: codes are compared bit for bit)."""
    return torch.round(x32).to(torch.int8) if dtype == torch.int8 else x32.to(torch.float8_e4m3fn)


def quantize(x):
    """(codes, scales [M, groups]): fp32 scales, codes of the quotient in 64 bits rounded to fp32 first, as the formula says."""
    M, K = x.shape
    groups = -(-K // 128)
    pad = torch.zeros((M, groups * 128))
    pad[:, :K] = x.float()
    pad = pad.view(M, groups, 128)
    amax = torch.where(pad.isnan(), torch.zeros_like(pad), pad).abs().amax(dim=2)
    amax = torch.clamp(amax, min=TINY)
    q = (pad.double() * 448.0 / amax.double()[:, :, None]).float().view(M, groups * 128)[:, :K].to(torch.float8_e4m3fn)
    return q, amax / 448.0


def gemm(a, b, sa, sb):
    """(C, sum of the absolute products, what the 8-bit matrix instruction may cut) in 64 bits; sa [M, groups], sb [ceil(N / 128),
    groups].

    The instruction adds products in eights (k = 8i ... 8i + 7) on a grid of 2^-13 times a power of two that is at most the
    largest product of the eight, and drops what lies under the grid: +2^16, -2^16 and 1.875^2 * 2^e side by side give 1.875^2 *
    2^e cut to multiples of 8, for every e. So each of the seven others loses less than 2^-13 of the largest product, which is at
    most the product of the eights' largest magnitudes."""
    K, N = a.shape[1], b.shape[0]
    wide = lambda s, n: s.double().repeat_interleave(128, dim=1)[:, :n]
    x = a.double() * wide(sa, K)
    y = b.double() * wide(sb, K).repeat_interleave(128, dim=0)[:N]
    eights = lambda v: torch.nn.functional.pad(v.abs(), (0, -K % 8)).view(v.shape[0], -1, 8).amax(dim=2)
    return x @ y.t(), x.abs() @ y.abs().t(), 7 * 2.0 ** -13 * (eights(x) @ eights(y).t())


def store(cache, scale, x, slots):
    """In place: cache [blocks, heads, size, D], scale [blocks, heads], x [T, heads, D]."""
    size, q = cache.shape[2], QMAX[cache.dtype]
    t, T = 0, len(slots)
    inside = lambda s: 0 <= s < cache.shape[0] * size
    while t < T:
        if not inside(slots[t]):
            t += 1
            continue
        block, end = slots[t] // size, t
        while end < T and inside(slots[end]) and slots[end] // size == block:
            end += 1
        begin = slots[t] % size
        new = x[t:end].float()
        for h in range(cache.shape[1]):
            v = new[:, h]
            amax = torch.clamp(v.abs().max(), min=TINY)
            s = torch.tensor(float("nan")) if v.isnan().any() else amax / q
            quotient = (v.double() * q / amax.double()).float()
            if begin > 0:
                old = scale[block, h].clone()
                if not old.isnan() and not old >= s:
                    codes = cache[block, h, :begin].float() * (old / s)
                    cache[block, h, :begin] = to_code(torch.nan_to_num(codes, nan=0.0), cache.dtype)
                else:
                    s = old
                    quotient = (v.double() / s.double()).float()
            scale[block, h] = s
            codes = to_code(torch.nan_to_num(quotient, nan=0.0), cache.dtype)
            for i in range(t, end):
                cache[block, h, slots[i] % size] = codes[i - t]
        t = end


def attention(q, table, cu, kv_lens, k, v, ks, vs, scale, causal):
    """(output, the bound's ingredients) in 64 bits. Returns o [T, heads, D], weighted magnitudes sum_j p_j |v_j|, and per row the
    largest scale * sum |q| |k|."""
    T, heads, D = q.shape
    H, size = k.shape[1], k.shape[2]
    G = heads // H
    o = torch.zeros(T, heads, D, dtype=torch.float64)
    mag = torch.zeros_like(o)
    big = torch.zeros(T, heads, dtype=torch.float64)
    for b in range(len(kv_lens)):
        n, L = cu[b + 1] - cu[b], min(kv_lens[b], table.shape[1] * size)
        for h in range(H):
            keys = torch.zeros(max(L, 0), D, dtype=torch.float64)
            vals = torch.zeros_like(keys)
            there = torch.zeros(max(L, 0), dtype=torch.bool)
            for j in range(0, L, size):
                blk, m = int(table[b, j // size]), min(size, L - j)
                if 0 <= blk < k.shape[0]:
                    keys[j:j + m] = k[blk, h, :m].double() * ks[blk, h].double()
                    vals[j:j + m] = v[blk, h, :m].double() * vs[blk, h].double()
                    there[j:j + m] = True
            for i in range(n):
                seen = there.clone()
                if causal:
                    seen[max(0, L - n + i + 1):] = False
                if not seen.any():
                    continue
                for hq in range(h * G, h * G + G):
                    x = q[cu[b] + i, hq].double()
                    s = (keys[seen] @ x) * scale
                    p = torch.softmax(s, dim=0)
                    o[cu[b] + i, hq] = p @ vals[seen]
                    mag[cu[b] + i, hq] = p @ vals[seen].abs()
                    big[cu[b] + i, hq] = (keys[seen].abs() @ x.abs()).max() * abs(scale)
    return o, mag, big


def attention_bound(o, mag, big, dtype, D, kv):
    """Per element: half a step of the output; of every summand half an fp16 step, twice the error of its score (an fp32 sum of
    D products, a multiply and a subtraction: D + 4 roundings of 2^-23 of the sum of magnitudes, in the exponent) and the
    roundings of the sums over the cached tokens (each 2^-23). The score sums enter numerator and denominator alike."""
    return HALF_STEP[dtype] * o.abs() + mag * (2.0 ** -11 + 2 * (D + 4) * 2.0 ** -23 * big[:, :, None] + 2 * (kv + 16) * 2.0 ** -23) + 1e-30


def small_products(scale, dtype, kv):
    """What fp16's subnormal numbers cost, for scores far apart, where attention_bound's relative terms alone do not hold: a
    probability (at most 1 beside the row's largest) times a value scale relative to the largest value scale is off by at most half
    of fp16's smallest step, 2^-25; the sum of up to kv of them, times codes of at most QMAX and that scale, is divided by a sum of
    probabilities of at least 1."""
    return kv * 2.0 ** -25 * QMAX[dtype] * float(scale.abs().max())


def random_cache(g, blocks, heads, size, D, dtype, layout="bhsd"):
    shape = (blocks, heads, size, D) if layout == "bhsd" else (blocks, size, heads, D)
    def codes():
        x = torch.randn(shape, generator=g)
        c = (x * 32).round().clamp(-127, 127).to(torch.int8) if dtype == torch.int8 else (x * 112).clamp(-448, 448).to(dtype)
        return c if layout == "bhsd" else c.permute(0, 2, 1, 3)
    unit = 1 / 32 if dtype == torch.int8 else 1 / 112
    scales = lambda: (0.3 + 1.4 * torch.rand(blocks, heads, generator=g)) * unit
    return codes(), codes(), scales(), scales()


def same_codes(a, b):
    """Codes bit for bit, all NaN alike."""
    if a.dtype == torch.int8:
        return torch.equal(a, b)
    x, y = a.float(), b.float()
    return bool(((x == y) | (x.isnan() & y.isnan())).all())
