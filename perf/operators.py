"""The 8-bit serving operators this library is timed on, over the range of sizes and types they are used with.

    quant      DeviceBlockQuantizeF8: activations to e4m3 with one scale per row and group of 128 columns
    gemm       DeviceGemmBlockScaleF8: the product of two such operands (weights: one scale per 128 x 128 block)
    tables     DeviceKvCacheTables: block tables and slot maps of a step from the request lengths
    store      DeviceKvCacheStore8: new keys and values into a cache of 8-bit blocks, one scale per block and head
    attention  DevicePagedAttention8: attention of the new tokens over that cache

`own` chooses between the operators and their plain form in elementary torch operations (32-bit arithmetic, rounded once).
"""
import math

import numpy as np
import torch

own = False

E4M3_MAX, INT8_MAX, TINY, GROUP = 448.0, 127.0, 2.0 ** -100, 128
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _quant(name, dtype, M, K):
    return {"name": name, "kind": "quant", "dtype": dtype, "M": M, "K": K}


def _gemm(name, out, M, N, K):
    return {"name": name, "kind": "gemm", "out": out, "M": M, "N": N, "K": K}


def _tables(name, B, ctx, new, block):
    return {"name": name, "kind": "tables", "B": B, "ctx": ctx, "new": new, "block": block}


def _store(name, dtype, B, ctx, new, kv_heads, D, block):
    return {"name": name, "kind": "store", "dtype": dtype, "B": B, "ctx": ctx, "new": new, "kv_heads": kv_heads, "D": D, "block": block}


def _attention(name, dtype, cache, B, ctx, new, heads, kv_heads, D, block, causal=True):
    return {"name": name, "kind": "attention", "dtype": dtype, "cache": cache, "B": B, "ctx": ctx, "new": new, "heads": heads,
            "kv_heads": kv_heads, "D": D, "block": block, "causal": causal}


def listed():
    return [
        # one token's activations on their way into a linear layer: latency
        _quant("quant_bf16_m1_k4096", "bf16", 1, 4096),
        # a long prompt's activations in front of the layer with the long reduction
        _quant("quant_bf16_m8192_k11008", "bf16", 8192, 11008),
        # one token through a linear layer: the weights are read once
        _gemm("gemm_m1_n11008_k4096", "bf16", 1, 11008, 4096),
        # a long prompt through the same layer
        _gemm("gemm_m4096_n11008_k4096", "bf16", 4096, 11008, 4096),
        # sizes that are no multiple of a tile, the last group of K short
        _gemm("gemm_m2001_n1003_k1040", "f16", 2001, 1003, 1040),
        # a decoding step's tables for 64 sequences
        _tables("tables_b64_decode", 64, 4096, 1, 16),
        # the prompts of a full batch arrive at once
        _tables("tables_b1024_new256", 1024, 64, 256, 16),
        # a decoding step's keys and values
        _store("store_b64_decode", "bf16", 64, 4096, 1, 8, 128, 16),
        # a long prompt's keys and values
        _store("store_b4_new4096", "bf16", 4, 100, 4096, 8, 128, 16),
        # one sequence, one new token, a short context: the smallest call
        _attention("attention_b1_ctx1000", "bf16", "e4m3", 1, 1000, 1, 32, 8, 128, 16),
        # a decoding step over long contexts of different lengths
        _attention("attention_b64_ctx8192", "bf16", "e4m3", 64, 8192, 1, 32, 8, 128, 16),
        # prompts (or pieces of them) behind cached tokens
        _attention("attention_b4_ctx4096_new1024", "f16", "int8", 4, 4096, 1024, 32, 8, 128, 32),
    ]


# ------------------------------------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi, step=1):
    """A whole multiple of `step` in [lo, hi], uniform in its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step * step, max(-(-lo // step) * step, int(round(v / step)) * step))


def _draw_one(rng):
    kind = rng.choice(["quant", "gemm", "gemm", "tables", "store", "attention", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "quant":
        return _quant("", rng.choice(["bf16", "bf16", "f16", "f32"]), _log(rng, 1, 16384), rng.choice([_log(rng, 128, 16384, 128), _log(rng, 100, 12288)]))
    if kind == "gemm":
        M = rng.choice([_log(rng, 1, 64), _log(rng, 65, 512), _log(rng, 512, 8192)])
        return _gemm("", rng.choice(["bf16", "bf16", "f16", "f32"]), M, rng.choice([_log(rng, 512, 12288, 128), _log(rng, 500, 12288)]),
                     rng.choice([_log(rng, 512, 12288, 128), _log(rng, 512, 12288, 16)]))
    block = rng.choice([16, 16, 32, 64])
    if kind == "tables":
        new = rng.choice([1, 1, _log(rng, 2, 1024)])
        return _tables("", _log(rng, 1, 2048), _log(rng, 1, 16384), new, block)
    kv_heads, D = rng.choice([1, 2, 4, 8, 8, 16]), rng.choice([64, 128, 128, 80])
    if kind == "store":
        return _store("", dtype, _log(rng, 1, 256), _log(rng, 1, 4096), rng.choice([1, 1, _log(rng, 2, 4096)]), kv_heads, D, block)
    return _attention("", dtype, rng.choice(["e4m3", "e4m3", "int8"]), _log(rng, 1, 128), _log(rng, 1, 16384),
                      rng.choice([1, 1, 1, 2, _log(rng, 3, 1024)]), kv_heads * rng.choice([1, 4, 4, 7, 8]), kv_heads, D, block,
                      rng.random() < 0.8)


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = {k: max(_cost(c) for c in listed() if c["kind"] == k) for k in ("quant", "gemm", "tables", "store", "attention")}
    while True:
        c = _draw_one(rng)
        if _cost(c) > most[c["kind"]]:
            continue
        if c["kind"] == "attention" and c["B"] * c["heads"] * c["new"] * (c["ctx"] + c["new"]) > 4 * 32 * 1024 * 5120:
            continue  # (the plain form's scores)
        if c["kind"] in ("attention", "store") and c["B"] * c["kv_heads"] * c["D"] * (c["ctx"] + c["new"]) > 1 << 29:
            continue
        del c["name"]
        return c


# ------------------------------------------------------------------------------------------------ sizes
def _lengths(case):
    """(tokens in the cache, new tokens) of every sequence. Requests of one batch differ: the lengths are spread over the
    upper half of what the case names."""
    b = np.arange(case["B"])
    share = 1.0 - 0.5 * np.mod(b * 0.6180339887, 1.0)
    ctx = np.maximum(1, (case["ctx"] * share).astype(np.int64))
    new = np.maximum(1, (case["new"] * share).astype(np.int64))
    return ctx, new


def work(case):
    if case["kind"] == "quant":
        M, K = case["M"], case["K"]
        es = 4 if case["dtype"] == "f32" else 2
        return {"bytes": float(M * K * (es + 1) + 4 * M * -(-K // GROUP)), "flops": 3.0 * M * K}
    if case["kind"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        kb = -(-K // GROUP)
        es = 4 if case["out"] == "f32" else 2
        return {"bytes": float(M * K + N * K + M * N * es + 4 * kb * (M + -(-N // GROUP))), "flops": 2.0 * M * N * K}
    ctx, new = _lengths(case)
    bs = case["block"]
    if case["kind"] == "tables":
        need = int((-(-(ctx + new) // bs) + -ctx // bs).sum())  # (blocks after less blocks before)
        return {"bytes": float(4 * (4 * case["B"] + 2 * need + int(new.sum()))), "flops": float(int(new.sum()))}
    H, D = case["kv_heads"], case["D"]
    if case["kind"] == "store":
        return {"bytes": float(int(new.sum()) * (2 * H * D * 3 + 4)), "flops": 6.0 * int(new.sum()) * H * D}
    seen = new * ctx + (new * (new + 1) // 2 if case["causal"] else new * new)
    bytes_ = 2 * int((ctx + new).sum()) * H * D + 2 * 2 * int(new.sum()) * case["heads"] * D
    return {"bytes": float(bytes_), "flops": 4.0 * int(seen.sum()) * case["heads"] * D}


# ------------------------------------------------------------------------------------------------ what a program holds
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype=torch.float32, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def _uniform(g, shape, lo, hi):
    return torch.rand(shape, generator=g, device="cuda", dtype=torch.float32).mul_(hi - lo).add_(lo)


def _cache(case, g, seed):
    """A cache whose blocks are spread over its whole memory, the block table of the sequences, their lengths, and the slots of
    the new tokens."""
    ctx, new = _lengths(case)
    bs, H, D, B = case["block"], case["kv_heads"], case["D"], case["B"]
    each = -(-(ctx + new) // bs)
    blocks, width = int(each.sum()) + 3, int(each.max())
    rng = np.random.default_rng(seed)
    order = rng.permutation(blocks)[: int(each.sum())].astype(np.int32)
    first = np.concatenate([[0], np.cumsum(each)])
    table = np.full((B, width), -1, np.int32)
    for b in range(B):
        table[b, : each[b]] = order[first[b]:first[b + 1]]
    cu = np.concatenate([[0], np.cumsum(new)])
    seq = np.repeat(np.arange(B), new)
    pos = np.arange(int(cu[-1])) - cu[seq] + ctx[seq]
    slots = table[seq, pos // bs].astype(np.int64) * bs + pos % bs
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a.astype(np.int32))).cuda()
    int8 = case.get("cache") == "int8"
    codes = lambda: (_normal(g, (blocks, H, bs, D), scale=32.0).round_().clamp_(-127, 127).to(torch.int8) if int8
                     else _normal(g, (blocks, H, bs, D), scale=112.0).clamp_(-448, 448).to(torch.float8_e4m3fn))
    unit = 1.0 / 32.0 if int8 else 1.0 / 112.0
    scales = lambda: _uniform(g, (blocks, H), 0.6 * unit, 1.4 * unit)
    return {"k_cache": codes(), "v_cache": codes(), "k_scale": scales(), "v_scale": scales(), "table": dev(table), "cu": dev(cu),
            "kv_lens": dev(ctx + new), "ctx_lens": dev(ctx), "new_lens": dev(new), "slots": dev(slots), "tokens": int(cu[-1]),
            "longest_new": int(new.max()), "longest": int((ctx + new).max())}


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind == "quant":
        M, K = case["M"], case["K"]
        # (activations: normal, with columns that stand out)
        x = _normal(g, (M, K)).mul_(torch.exp(_normal(g, (1, K)))).to(DTYPES[case["dtype"]])
        s = {"x": x, "q": torch.empty((M, K), device="cuda", dtype=torch.float8_e4m3fn),
             "scale": torch.empty((-(-K // GROUP), M), device="cuda")}
    elif kind == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        kb = -(-K // GROUP)
        code = lambda shape: _normal(g, shape, scale=112.0).clamp_(-448, 448).to(torch.float8_e4m3fn)
        s = {"a": code((M, K)), "b": code((N, K)), "scale_a": _uniform(g, (kb, M), 0.5 / 112, 1.5 / 112),
             "scale_b": _uniform(g, (-(-N // GROUP), kb), 0.5 / 112, 1.5 / 112).mul_(K ** -0.5),
             "c": torch.empty((M, N), device="cuda", dtype=DTYPES[case["out"]])}
    elif kind == "tables":
        s = _tables_state(case, seed)
    else:
        s = _cache(case, g, seed)
        T, H, D, dt = s["tokens"], case["kv_heads"], case["D"], DTYPES[case["dtype"]]
        if kind == "store":
            # keys and values as a fused projection leaves them: columns of one matrix; tokens of different magnitude
            kv = _normal(g, (T, 2 * H * D)).mul_(torch.exp(_normal(g, (T, 1), scale=0.5))).to(dt)
            s["k"], s["v"] = kv[:, : H * D].view(T, H, D), kv[:, H * D:].view(T, H, D)
        else:
            qkv = _normal(g, (T, (case["heads"] + 2 * H) * D)).to(dt)
            s["q"] = qkv[:, : case["heads"] * D].view(T, case["heads"], D)
            s["o"] = torch.empty((T, case["heads"], D), device="cuda", dtype=dt)
    s["case"] = case
    if own:
        s["call"] = _handle(case, s)
    return s


def _tables_state(case, seed):
    ctx, new = _lengths(case)
    bs, B = case["block"], case["B"]
    before, after = -(-ctx // bs), -(-(ctx + new) // bs)
    rng = np.random.default_rng(seed)
    order = rng.permutation(int(after.sum()) + 64).astype(np.int32)
    width = int(after.max()) + 1
    table = np.full((B, width), -1, np.int32)
    at = 0
    for b in range(B):
        table[b, : before[b]] = order[at:at + before[b]]
        at += before[b]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a.astype(np.int32))).cuda()
    T = int(new.sum()) + 5  # (a step's buffers are made for more tokens than it has)
    return {"ctx_lens": dev(ctx), "new_lens": dev(new), "free": dev(order[at:]), "table": dev(table),
            "cu": torch.empty(B + 1, device="cuda", dtype=torch.int32), "kv_lens": torch.empty(B, device="cuda", dtype=torch.int32),
            "slots": torch.empty(T, device="cuda", dtype=torch.int32), "used": torch.empty(1, device="cuda", dtype=torch.int32)}


def _handle(case, s):
    """The operator's invoker with its argument, workspace and stream, which a program keeps."""
    import composable_kernel_amd as ck
    kind = case["kind"]
    if kind == "quant":
        M, K = case["M"], case["K"]
        op = ck.DeviceBlockQuantizeF8(case["dtype"])
        arg = op.MakeArgumentPointer(s["x"], s["q"], s["scale"], M, K, K, K, 1, M)
    elif kind == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        op = ck.DeviceGemmBlockScaleF8(case["out"])
        arg = op.MakeArgumentPointer(s["a"], s["b"], s["c"], s["scale_a"], s["scale_b"], M, N, K, K, K, N, (1, M), (-(-K // GROUP), 1))
    elif kind == "tables":
        op = ck.DeviceKvCacheTables()
        arg = op.MakeArgumentPointer(s["ctx_lens"], s["new_lens"], s["free"], s["table"], s["cu"], s["kv_lens"], s["slots"], s["used"],
                                     case["B"], s["free"].numel(), s["table"].shape[1], s["table"].shape[1], s["slots"].numel(), case["block"])
    else:
        cache = ck.KvCache8(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
        if kind == "store":
            op = ck.DeviceKvCacheStore8(case["dtype"])
            arg = op.MakeArgumentPointer(s["k"], s["v"], s["slots"], cache, s["tokens"], s["k"].stride()[:2], s["v"].stride()[:2])
        else:
            op = ck.DevicePagedAttention8(case["dtype"], Causal=case["causal"])
            arg = op.MakeArgumentPointer(s["q"], s["o"], s["table"], s["cu"], s["kv_lens"], cache, case["B"], s["tokens"], case["heads"],
                                         s["longest"], s["table"].shape[1], s["table"].shape[1], s["q"].stride()[:2],
                                         s["o"].stride()[:2], ck.Scale(case["D"] ** -0.5))
    if not op.IsSupportedArgument(arg):
        raise ValueError(op.GetTypeString() + ": " + ck.capi.last_error())
    need = op.GetWorkSpaceSize(arg)
    if need:
        op.SetWorkSpacePointer(arg, torch.empty(need, device="cuda", dtype=torch.uint8))
    return op.MakeInvokerPointer(), arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream)


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        invoker, argument, config = s["call"]
        invoker.Run(argument, config)
    else:
        {"quant": _plain_quant, "gemm": _plain_gemm, "tables": _plain_tables, "store": _plain_store, "attention": _plain_attention}[kind](s)
    names = {"quant": ("q", "scale"), "gemm": ("c",), "tables": ("table", "cu", "kv_lens", "slots", "used"),
             "store": ("k_cache", "v_cache", "k_scale", "v_scale"), "attention": ("o",)}[kind]
    return {n: s[n] for n in names}


def _plain_quant(s):
    M, K = s["x"].shape
    kb = -(-K // GROUP)
    x = torch.zeros((M, kb * GROUP), device="cuda")
    x[:, :K] = s["x"]
    x = x.view(M, kb, GROUP)
    scale = x.abs().amax(dim=2).clamp_(min=TINY) / E4M3_MAX
    s["q"].copy_((x * (1.0 / scale)[:, :, None]).view(M, kb * GROUP)[:, :K])
    s["scale"].copy_(scale.t())


def _plain_gemm(s):
    M, K = s["a"].shape
    N = s["b"].shape[0]
    a = s["a"].float() * s["scale_a"].t().repeat_interleave(GROUP, dim=1)[:, :K]
    b = s["b"].float() * s["scale_b"].repeat_interleave(GROUP, dim=0)[:N].repeat_interleave(GROUP, dim=1)[:, :K]
    s["c"].copy_(torch.matmul(a, b.t().contiguous()))


def _plain_tables(s):
    bs, table, ctx, new = s["case"]["block"], s["table"], s["ctx_lens"], s["new_lens"]
    B, width = table.shape
    kv = ctx + new
    before, after = (ctx + bs - 1) // bs, (kv + bs - 1) // bs
    need = after - before
    base = torch.cumsum(need, 0) - need
    col = torch.arange(width, device="cuda")[None, :]
    fresh = (col >= before[:, None]) & (col < after[:, None])
    take = (base[:, None] + col - before[:, None]).clamp_(0, s["free"].numel() - 1)
    table.copy_(torch.where(fresh, s["free"][take], table))
    s["cu"][0] = 0
    s["cu"][1:] = torch.cumsum(new, 0)
    s["kv_lens"].copy_(kv)
    s["used"].copy_(need.sum(dim=0, keepdim=True))
    t = torch.arange(s["slots"].numel(), device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["cu"][1:], t, right=True).clamp_(max=B - 1)
    pos = (ctx[seq] + t - s["cu"][seq]).clamp_(min=0)
    block = table[seq, (pos // bs).clamp_(max=width - 1)]
    s["slots"].copy_(torch.where(t < s["cu"][B], block * bs + pos % bs, -1))


def _plain_store(s):
    bs, slots = s["case"]["block"], s["slots"].long()
    block, at = slots // bs, slots % bs
    leads = torch.ones_like(block, dtype=torch.bool)
    leads[1:] = block[1:] != block[:-1]
    run = torch.cumsum(leads, 0) - 1                       # the token's run
    lead = torch.nonzero(leads).flatten()
    blk, o = block[lead], at[lead]                         # a run's block, and where in it the run begins
    part = torch.nonzero(o > 0).flatten()                  # runs that go on in a block begun earlier
    older = torch.arange(bs, device="cuda")[None, None, :, None] < o[part][:, None, None, None]
    for x, cache, scales in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        x = x.float()
        amax = torch.zeros((lead.numel(), x.shape[1]), device="cuda").index_reduce_(0, run, x.abs().amax(dim=2), "amax")
        fresh = amax.clamp_(min=TINY) / E4M3_MAX
        was = scales[blk]
        now = torch.where(o[:, None] > 0, torch.maximum(was, fresh), fresh)
        shrink = (was / now)[part]
        codes = cache[blk[part]]
        cache[blk[part]] = torch.where(older, (codes.float() * shrink[:, :, None, None]).to(cache.dtype).float(), codes.float()).to(cache.dtype)
        scales[blk] = now
        cache[block, :, at] = (x * (1.0 / now)[run][:, :, None]).to(cache.dtype)


def _plain_attention(s):
    c, q, table, cu, kv = s["case"], s["q"], s["table"], s["cu"].long(), s["kv_lens"].long()
    T, heads, D = q.shape
    B, H, bs, new = c["B"], c["kv_heads"], c["block"], s["longest_new"]
    G, L = heads // H, table.shape[1] * bs
    blocks = table.clamp(min=0).long()

    def gather(cache, scale):
        x = cache[blocks].float() * scale[blocks][:, :, :, None, None]          # [B, blocks, H, bs, D]
        return x.permute(0, 2, 1, 3, 4).reshape(B, H, L, D)
    k, v = gather(s["k_cache"], s["k_scale"]), gather(s["v_cache"], s["v_scale"])
    i = torch.arange(new, device="cuda")[None, :]
    count = cu[1:] - cu[:-1]
    live = i < count[:, None]                                                   # [B, new]
    rows = (cu[:-1, None] + i).clamp_(max=T - 1)
    x = q[rows].float().view(B, new, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, new * G, D)
    scores = torch.matmul(x, k.transpose(2, 3).contiguous()).mul_(D ** -0.5).view(B, H, new, G, L)
    last = (kv - count)[:, None] + i if c["causal"] else (kv - 1)[:, None].expand(B, new)
    seen = torch.arange(L, device="cuda")[None, None, :] <= last[:, :, None]    # [B, new, L]
    scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    scores.sub_(scores.amax(dim=4, keepdim=True).clamp_(min=-1e30)).exp_()
    total = scores.sum(dim=4, keepdim=True)
    scores.div_(torch.where(total > 0, total, torch.ones_like(total)))
    out = torch.matmul(scores.view(B, H, new * G, L), v).view(B, H, new, G, D).permute(0, 2, 1, 3, 4).reshape(B, new, heads, D)
    # (a token's row is found from its sequence and its place in it)
    t = torch.arange(T, device="cuda")
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    s["o"].copy_(out[seq, t - cu[seq]])


# ------------------------------------------------------------------------------------------------ in 64 bits
def _to_e4m3(x):
    """Doubles rounded to the nearest e4m3 value, ties to the even one."""
    size = x.abs()
    power = torch.floor(torch.log2(torch.where(size > 0, size, torch.ones_like(size)))).clamp_(min=-6.0)
    step = torch.exp2(power - 3.0)
    return torch.round(x / step).mul_(step)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"quant": _exact_quant, "gemm": _exact_gemm, "tables": _exact_tables, "store": _exact_store, "attention": _exact_attention}[case["kind"]](s)


def _exact_quant(s):
    M, K = s["x"].shape
    scales, codes = [], []
    for k in range(0, K, GROUP):
        x = s["x"][:, k:k + GROUP].double()
        scales.append(x.abs().max(dim=1).values.clamp(min=TINY) / E4M3_MAX)
        codes.append(_to_e4m3(x / scales[-1][:, None]).float())
    return {"q": torch.cat(codes, dim=1), "scale": torch.stack(scales)}


def _exact_gemm(s):
    (M, K), N = s["a"].shape, s["b"].shape[0]
    c = torch.zeros((M, N), device="cuda", dtype=torch.float64)
    for j, k in enumerate(range(0, K, GROUP)):
        per_row = s["scale_b"][:, j].double()[torch.arange(N, device="cuda") // GROUP]
        a = s["a"][:, k:k + GROUP].double() * s["scale_a"][j].double()[:, None]
        c += a @ (s["b"][:, k:k + GROUP].double() * per_row[:, None]).t().contiguous()
    return {"c": c}


def _exact_tables(s):
    return None  # (whole numbers)


def _exact_store(s):
    bs, slots = s["case"]["block"], s["slots"].cpu().numpy()
    out = {}
    starts = np.flatnonzero(np.concatenate([[True], slots[1:] // bs != slots[:-1] // bs]))
    if len(starts) > 6000:
        return None
    ends = np.concatenate([starts[1:], [len(slots)]])
    for name in ("k", "v"):
        cache, scales, x = s[name + "_cache"].double(), s[name + "_scale"].double(), s[name].double()
        for lo, hi in zip(starts.tolist(), ends.tolist()):
            b, o = divmod(int(slots[lo]), bs)
            now = x[lo:hi].abs().amax(dim=(0, 2)).clamp(min=TINY) / E4M3_MAX
            if o:
                now = torch.maximum(now, scales[b])
                cache[b, :, :o] = _to_e4m3(cache[b, :, :o] * (scales[b] / now)[:, None, None])
            scales[b] = now
            cache[b, :, o:o + hi - lo] = _to_e4m3(x[lo:hi].transpose(0, 1) / now[:, None, None])
        out[name + "_cache"], out[name + "_scale"] = cache.float(), scales
    return out


def _exact_attention(s):
    c = s["case"]
    cu, kv, table = s["cu"].tolist(), s["kv_lens"].tolist(), s["table"]
    H, G = c["kv_heads"], c["heads"] // c["kv_heads"]
    o = torch.zeros(s["o"].shape, device="cuda", dtype=torch.float64)
    for b in range(c["B"]):
        L, n = kv[b], cu[b + 1] - cu[b]
        blocks = table[b, : -(-L // c["block"])].long()
        for h in range(H):
            k = (s["k_cache"][blocks, h].double() * s["k_scale"][blocks, h].double()[:, None, None]).flatten(0, 1)[:L]
            v = (s["v_cache"][blocks, h].double() * s["v_scale"][blocks, h].double()[:, None, None]).flatten(0, 1)[:L]
            for j in range(h * G, h * G + G):
                p = s["q"][cu[b]:cu[b + 1], j].double() @ k.t().contiguous() / math.sqrt(c["D"])
                if c["causal"]:
                    p.masked_fill_(torch.arange(L, device="cuda")[None, :] > torch.arange(L - n, L, device="cuda")[:, None], -math.inf)
                o[cu[b]:cu[b + 1], j] = torch.softmax(p, dim=1) @ v
    return {"o": o}
