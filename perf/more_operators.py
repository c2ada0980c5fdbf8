"""The operators of mixture-of-experts layers in 8-bit integers, over the range of sizes and types they are used with.

    route      DeviceRouteExperts: each token's experts and their weights from its logits, and the experts' rows in order
    quant      DeviceTokenQuantizeI8: activations to int8 with one scale per token
    gemm       DeviceGemmTokenScaleI8: int8 product with a scale for each token and channel (gated: silu(gate) * up)
    experts    DeviceExpertsGemmI8: that product for each expert's rows, gathered from their tokens
    combine    DeviceExpertsCombine: the weighted sum of a token's rows

`own` chooses between the operators and their plain form in elementary torch operations (32-bit arithmetic, rounded once; the
router's scores, whose order decides, in 64).
"""
import math

import numpy as np
import torch

own = False

INT8_MAX, TINY, LARGEST = 127.0, 2.0 ** -100, float(np.finfo(np.float32).max)
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def _route(name, dtype, T, E, k, scoring="softmax", bias=False, groups=1, top_groups=1, best=1, padded=False, masked=False):
    return {"name": name, "kind": "route", "dtype": dtype, "T": T, "E": E, "k": k, "scoring": scoring, "bias": bias, "groups": groups,
            "top_groups": top_groups, "best": best, "padded": padded, "masked": masked}


def _quant(name, dtype, M, K):
    return {"name": name, "kind": "quant", "dtype": dtype, "M": M, "K": K}


def _gemm(name, out, M, N, K, gated=False, bias=False):
    return {"name": name, "kind": "gemm", "out": out, "M": M, "N": N, "K": K, "gated": gated, "bias": bias}


def _experts(name, out, T, E, k, N, K, gated, gather):
    return {"name": name, "kind": "experts", "out": out, "T": T, "E": E, "k": k, "N": N, "K": K, "gated": gated, "gather": gather}


def _combine(name, dtype, T, k, N, add=False):
    return {"name": name, "kind": "combine", "dtype": dtype, "T": T, "k": k, "N": N, "add": add}


def listed():
    return [
        # one token finds its experts: latency
        _route("route_t1_e64_k8", "f32", 1, 64, 8),
        # a batch of long prompts, many experts in groups, biases that balance their load
        _route("route_t16384_e256_k8_groups", "f32", 16384, 256, 8, "sigmoid", True, 8, 4, 2),
        # a decoding step's activations on their way into a layer
        _quant("quant_bf16_m16_k4096", "bf16", 16, 4096),
        # a long prompt's activations in front of the layer with the long reduction
        _quant("quant_bf16_m8192_k11008", "bf16", 8192, 11008),
        # one token through a linear layer: the weights are read once
        _gemm("gemm_m1_n11008_k4096", "bf16", 1, 11008, 4096),
        # a long prompt through the same layer
        _gemm("gemm_m4096_n11008_k4096", "bf16", 4096, 11008, 4096),
        # gate and up projection in one, with biases, sizes that are no multiple of a tile
        _gemm("gemm_gated_m777_n2744_k2064", "f16", 777, 2744, 2064, True, True),
        # one token through its experts' gate and up projections
        _experts("experts_up_t1_e64_k8", "bf16", 1, 64, 8, 1408, 4096, True, True),
        # a decoding step's rows through the experts' down projections: few rows each
        _experts("experts_down_t64_e64_k8", "bf16", 64, 64, 8, 4096, 1408, False, False),
        # a prompt through the gate and up projections
        _experts("experts_up_t4096_e64_k8", "bf16", 4096, 64, 8, 1408, 4096, True, True),
        # a decoding step's rows back to their tokens
        _combine("combine_t16_k8_n4096", "bf16", 16, 8, 4096),
        # a prompt's rows back to their tokens, onto what the shared layer gave
        _combine("combine_t8192_k8_n4096", "bf16", 8192, 8, 4096, True),
    ]


# ------------------------------------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi, step=1):
    """A whole multiple of `step` in [lo, hi], uniform in its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step * step, max(-(-lo // step) * step, int(round(v / step)) * step))


def _draw_one(rng):
    kind = rng.choice(["route", "route", "quant", "gemm", "gemm", "gemm", "experts", "experts", "experts", "experts", "combine"])
    out = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "route":
        E = rng.choice([8, 16, 60, 64, 128, 160, 256, _log(rng, 2, 256)])
        groups = rng.choice([1, 1, 4, 8])
        if E % groups or E < 16:
            groups = 1
        k = min(E, rng.choice([1, 2, 2, 4, 6, 8, 8]))
        scoring = rng.choice(["softmax", "sigmoid"])
        return _route("", rng.choice(["f32", "f32", "bf16", "f16"]), _log(rng, 1, 16384), E, k, scoring, rng.random() < 0.5, groups,
                      rng.randint(1, groups), rng.choice([1, 2]), rng.random() < 0.3, rng.random() < 0.3)
    if kind == "quant":
        return _quant("", out, _log(rng, 1, 16384), rng.choice([_log(rng, 128, 16384, 128), _log(rng, 100, 12288)]))
    if kind == "gemm":
        M = rng.choice([_log(rng, 1, 64), _log(rng, 65, 512), _log(rng, 512, 8192)])
        return _gemm("", out, M, rng.choice([_log(rng, 256, 12288, 128), _log(rng, 250, 12288)]),
                     rng.choice([_log(rng, 512, 12288, 128), _log(rng, 512, 12288, 16)]), rng.random() < 0.4, rng.random() < 0.3)
    if kind == "experts":
        E = rng.choice([4, 8, 16, 60, 64, 128])
        return _experts("", out, rng.choice([_log(rng, 1, 64), _log(rng, 64, 8192)]), E, min(E, rng.choice([1, 2, 4, 6, 8])),
                        rng.choice([_log(rng, 256, 4096, 64), _log(rng, 250, 4096)]), rng.choice([_log(rng, 256, 4096, 128), _log(rng, 256, 4096, 16)]),
                        rng.random() < 0.5, rng.random() < 0.5)
    return _combine("", out, _log(rng, 1, 16384), rng.choice([1, 2, 4, 6, 8]), rng.choice([_log(rng, 512, 8192, 128), _log(rng, 500, 8192)]),
                    rng.random() < 0.5)


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = {k: max(_cost(c) for c in listed() if c["kind"] == k) for k in ("route", "quant", "gemm", "experts", "combine")}
    while True:
        c = _draw_one(rng)
        if _cost(c) > most[c["kind"]] or (c["kind"] == "experts" and c["E"] * c["N"] * (1 + c["gated"]) * c["K"] > 64 * 2816 * 4096):
            continue
        del c["name"]
        return c


# ------------------------------------------------------------------------------------------------ sizes
def work(case):
    kind = case["kind"]
    if kind == "route":
        T, E, k = case["T"], case["E"], case["k"]
        return {"bytes": float(T * E * SIZE[case["dtype"]] + 16 * T * k + 4 * E), "flops": float(T * E * (8 + k))}
    if kind == "quant":
        M, K = case["M"], case["K"]
        return {"bytes": float(M * K * (SIZE[case["dtype"]] + 1) + 4 * M), "flops": 3.0 * M * K}
    if kind == "combine":
        T, k, N = case["T"], case["k"], case["N"]
        return {"bytes": float(T * N * SIZE[case["dtype"]] * (k + 1 + case["add"]) + 8 * T * k), "flops": 2.0 * T * k * N}
    N, K, rows = case["N"], case["K"], case["M"] if kind == "gemm" else case["T"] * case["k"]
    wide = N * (1 + case["gated"])
    if kind == "gemm":
        matrices, rows_a = 1.0, rows
    else:
        # experts that a call meets; a gathered token is read once
        matrices = case["E"] * (1 - (1 - case["k"] / case["E"]) ** case["T"])
        rows_a = case["T"] if case["gather"] else rows
    return {"bytes": float(rows_a * (K + 4) + matrices * wide * (K + 4) + rows * N * SIZE[case["out"]]), "flops": 2.0 * rows * wide * K}


# ------------------------------------------------------------------------------------------------ what a program holds
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype=torch.float32, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def _uniform(g, shape, lo, hi):
    return torch.rand(shape, generator=g, device="cuda", dtype=torch.float32).mul_(hi - lo).add_(lo)


def _codes(g, shape):
    return _normal(g, shape, scale=36.0).round_().clamp_(-127, 127).to(torch.int8)


def _int(n, *more):
    return torch.empty((n, *more), device="cuda", dtype=torch.int32)


def _choice(case, g):
    """Each token's experts, some of them more in demand than others: ids [T, k] and weights."""
    T, E, k = case["T"], case["E"], case["k"]
    scores = _normal(g, (T, E)) + _normal(g, (1, E), scale=0.5)
    best, ids = torch.sort(scores, dim=1, descending=True, stable=True)
    return ids[:, :k].contiguous(), torch.softmax(best[:, :k], dim=1).contiguous()


def _tables(ids, E):
    """offsets [E + 1], rows and places [T * k] (int32) of ids [T, k]; ids of -1 are in none."""
    key = torch.where(ids < 0, E, ids).flatten().long()
    order = torch.sort(key, stable=True).indices
    offsets = torch.searchsorted(key[order].contiguous(), torch.arange(E + 1, device="cuda"))
    rank = torch.arange(key.numel(), device="cuda")
    there = rank < offsets[E]
    rows = torch.where(there, order, -1)
    places = torch.empty_like(order)
    places[order] = torch.where(there, rank, -1)
    return offsets.int(), rows.int(), places.int()


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind == "route":
        T, E, k = case["T"], case["E"], case["k"]
        s = {"x": (_normal(g, (T, E), scale=1.5) + _normal(g, (1, E), scale=0.5)).to(DTYPES[case["dtype"]]), "bias": None, "live": None,
             "ids": _int(T, k), "weights": torch.empty((T, k), device="cuda"), "offsets": _int(E + 1), "rows": _int(T * k), "places": _int(T * k)}
        if case["masked"]:  # experts that are switched off for some tokens
            s["x"].masked_fill_(_uniform(g, (T, E), 0, 1) < 0.1, -math.inf)
        if case["bias"]:
            s["bias"] = _normal(g, (E,), scale=0.1)
        if case["padded"]:  # (a captured step's buffers are made for more tokens than it has)
            s["live"] = torch.tensor([T - T // 5], device="cuda", dtype=torch.int32)
    elif kind == "quant":
        M, K = case["M"], case["K"]
        # (activations: normal, with columns that stand out)
        x = _normal(g, (M, K)).mul_(torch.exp(_normal(g, (1, K)))).to(DTYPES[case["dtype"]])
        s = {"x": x, "q": torch.empty((M, K), device="cuda", dtype=torch.int8), "scale": torch.empty(M, device="cuda")}
    elif kind == "combine":
        T, k, N, dt = case["T"], case["k"], case["N"], DTYPES[case["dtype"]]
        ids, weights = _choice({"T": T, "E": 64, "k": k}, g)
        s = {"y": _normal(g, (T * k, N), dt), "places": _tables(ids, 64)[2], "weights": weights,
             "add": _normal(g, (T, N), dt) if case["add"] else None, "out": torch.empty((T, N), device="cuda", dtype=dt)}
    else:
        N, K = case["N"], case["K"]
        wide = N * (1 + case["gated"])
        E = case["E"] if kind == "experts" else 1
        rows = case["M"] if kind == "gemm" else case["T"] * case["k"]
        rows_a = case["T"] if kind == "experts" and case["gather"] else rows
        s = {"a": _codes(g, (rows_a, K)), "scale_a": _uniform(g, (rows_a,), 0.5 / 36, 1.5 / 36), "b": _codes(g, (E, wide, K)),
             "scale_b": _uniform(g, (E, wide), 0.5 / 36, 1.5 / 36).mul_(K ** -0.5), "c": torch.empty((rows, N), device="cuda", dtype=DTYPES[case["out"]])}
        if kind == "gemm":
            s["b"], s["scale_b"] = s["b"][0], s["scale_b"][0]
            s["bias"] = _normal(g, (wide,)) if case["bias"] else None
        else:
            ids, _ = _choice(case, g)
            s["offsets"], s["rows"], _ = _tables(ids, E)
            s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
    s["case"] = case
    if own:
        s["call"] = _handle(case, s)
    return s


def _handle(case, s):
    """The operator's invoker with its argument, workspace and stream, which a program keeps."""
    import composable_kernel_amd as ck
    kind = case["kind"]
    if kind == "route":
        T, E, k = case["T"], case["E"], case["k"]
        op = ck.DeviceRouteExperts(case["dtype"], Scoring=case["scoring"], Renormalise=True)
        arg = op.MakeArgumentPointer(s["x"], s["bias"], s["live"], s["ids"], s["weights"], s["offsets"], s["rows"], s["places"], T, E, k, E,
                                     case["groups"], case["top_groups"], case["best"], ck.Scale(1.0))
    elif kind == "quant":
        M, K = case["M"], case["K"]
        op = ck.DeviceTokenQuantizeI8(case["dtype"])
        arg = op.MakeArgumentPointer(s["x"], s["q"], s["scale"], M, K, K, K)
    elif kind == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        op = ck.DeviceGemmTokenScaleI8(case["out"], Gated=case["gated"])
        arg = op.MakeArgumentPointer(s["a"], s["b"], s["c"], s["scale_a"], s["scale_b"], s["bias"], M, N, K, K, K, N)
    elif kind == "experts":
        N, K = case["N"], case["K"]
        op = ck.DeviceExpertsGemmI8(case["out"], Gated=case["gated"])
        arg = op.MakeArgumentPointer(s["a"], s["b"], s["c"], s["scale_a"], s["scale_b"], None, s["offsets"], s["rows"] if case["gather"] else None,
                                     s["c"].shape[0], s["a"].shape[0], case["E"], N, K, K, K, N, s["b"].stride(0), case["k"] if case["gather"] else 1)
    else:
        T, k, N = case["T"], case["k"], case["N"]
        op = ck.DeviceExpertsCombine(case["dtype"])
        arg = op.MakeArgumentPointer(s["y"], s["places"], s["weights"], s["add"], s["out"], T, k, T * k, N, N, N, N)
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
        {"route": _plain_route, "quant": _plain_quant, "gemm": _plain_gemm, "experts": _plain_experts, "combine": _plain_combine}[kind](s)
    names = {"route": ("ids", "weights", "offsets", "rows", "places"), "quant": ("q", "scale"), "gemm": ("c",), "experts": ("c",),
             "combine": ("out",)}[kind]
    return {n: s[n] for n in names}


def _plain_route(s):
    c = s["case"]
    T, E, k, G = c["T"], c["E"], c["k"], c["groups"]
    x = s["x"].double()
    there = x > -math.inf                                    # (NaN is not)
    if s["bias"] is not None:
        there = there & (s["bias"] > -math.inf)
    x = x.clamp(max=LARGEST).masked_fill(~there, -math.inf)
    if c["scoring"] == "softmax":
        p = torch.exp(x - x.amax(dim=1, keepdim=True).clamp(min=-LARGEST))
        total = p.sum(dim=1, keepdim=True)
        p = p / torch.where(total > 0, total, torch.ones_like(total))
    else:
        p = 1 / (1 + torch.exp(-x))
    value = p if s["bias"] is None else p + s["bias"].double().clamp(max=LARGEST)
    value = value.masked_fill(~there, -math.inf)
    order = x if s["bias"] is None else value
    if G > 1:
        best = torch.sort((order if c["best"] == 1 else value).view(T, G, E // G), dim=2, descending=True, stable=True).values
        of_group = best[:, :, 0]
        if c["best"] == 2 and E // G > 1:
            of_group = of_group + torch.where(best[:, :, 1] > -math.inf, best[:, :, 1], torch.zeros_like(of_group))
        place = torch.sort(of_group, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        stays = torch.zeros((T, G), device="cuda", dtype=torch.bool).scatter_(1, place, True)
        order = order.masked_fill(~stays.repeat_interleave(E // G, dim=1), -math.inf)
    best, ids = torch.sort(order, dim=1, descending=True, stable=True)
    best, ids = best[:, :k], ids[:, :k]
    has = best > -math.inf
    if s["live"] is not None:
        has = has & (torch.arange(T, device="cuda") < s["live"])[:, None]
    w = torch.where(has, torch.gather(p, 1, ids), torch.zeros_like(best))
    total = w.sum(dim=1, keepdim=True)
    s["weights"].copy_(w / torch.where(total > 0, total, torch.ones_like(total)))
    ids = torch.where(has, ids, -1)
    s["ids"].copy_(ids)
    offsets, rows, places = _tables(ids, E)
    s["offsets"].copy_(offsets)
    s["rows"].copy_(rows)
    s["places"].copy_(places)


def _plain_quant(s):
    x = s["x"]
    amax = x.abs().amax(dim=1).float().clamp_(min=TINY)
    if x.dtype == torch.float32:  # (the quotient as if rounded once)
        t = (x.double() * INT8_MAX / amax.double()[:, None]).float()
    else:                         # (16-bit values times 127 are exact)
        t = x.float() * INT8_MAX / amax[:, None]
    s["q"].copy_(t.round_())
    s["scale"].copy_(amax / INT8_MAX)


def _silu(x):
    return x / (1 + torch.exp(-x))


def _plain_gemm(s):
    c = torch.matmul(s["a"].float(), s["b"].float().t().contiguous())
    c = c * s["scale_a"][:, None] * s["scale_b"][None, :]
    if s["bias"] is not None:
        c = c + s["bias"][None, :]
    N = s["c"].shape[1]
    s["c"].copy_(_silu(c[:, :N]) * c[:, N:] if s["case"]["gated"] else c)


def _plain_experts(s):
    case, offsets = s["case"], s["offsets"].long()
    P, E, N = s["c"].shape[0], case["E"], case["N"]
    row = torch.arange(P, device="cuda")
    expert = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
    at = s["rows"].long() // case["k"] if case["gather"] else row
    a, scale_a = s["a"][at].float(), s["scale_a"][at]
    if P < E:  # each row with its expert's matrix
        c = torch.bmm(a[:, None, :], s["b"][expert].float().transpose(1, 2).contiguous())[:, 0]
    else:      # each expert with all of its rows, as many as the fullest has
        place = row - offsets[expert]
        wide = torch.zeros((E, s["most"], case["K"]), device="cuda")
        wide[expert, place] = a
        c = torch.bmm(wide, s["b"].float().transpose(1, 2).contiguous())[expert, place]
    c = c * scale_a[:, None] * s["scale_b"][expert]
    s["c"].copy_(_silu(c[:, :N]) * c[:, N:] if case["gated"] else c)


def _plain_combine(s):
    T, N = s["out"].shape
    y = s["y"].float()[s["places"].long()].view(T, -1, N)
    out = (y * s["weights"][:, :, None]).sum(dim=1)
    s["out"].copy_(out if s["add"] is None else out + s["add"].float())


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"route": _exact_route, "quant": _exact_quant, "gemm": _exact_gemm, "experts": _exact_experts, "combine": _exact_combine}[case["kind"]](s)


def _exact_route(s):
    c = s["case"]
    T, E, k, G = c["T"], c["E"], c["k"], c["groups"]
    x = s["x"].double().cpu().numpy()
    bias = np.zeros(E) if s["bias"] is None else s["bias"].double().cpu().numpy()
    live = T if s["live"] is None else int(s["live"])
    off = np.isneginf(x) | np.isneginf(bias)
    with np.errstate(over="ignore"):
        score = 1 / (1 + np.exp(-x)) if c["scoring"] == "sigmoid" else np.exp(x - x.max(axis=1, keepdims=True))
    if c["scoring"] == "softmax":
        score /= score.sum(axis=1, keepdims=True)
    value = np.where(off, -np.inf, score + bias)
    if G > 1:
        per = value.reshape(T, G, E // G)
        two = np.sort(per, axis=2)[:, :, -c["best"]:]
        two = np.where(np.isneginf(two), 0.0, two).sum(axis=2)
        two[np.isneginf(per).all(axis=2)] = -np.inf
        rank = np.argsort(np.argsort(-two, axis=1, kind="stable"), axis=1, kind="stable")
        value[np.repeat(rank >= c["top_groups"], E // G, axis=1)] = -np.inf
    w = np.zeros((T, k))
    row = np.arange(T)
    for j in range(k):
        e = value.argmax(axis=1)
        has = ~np.isneginf(value[row, e]) & (row < live)
        w[has, j] = score[row, e][has]
        value[row, e] = -np.inf
    total = w.sum(axis=1, keepdims=True)
    return {"ids": None, "weights": torch.from_numpy(w / np.where(total > 0, total, 1)), "offsets": None, "rows": None, "places": None}


def _exact_quant(s):
    return {"q": None, "scale": s["x"].double().abs().max(dim=1).values.clamp(min=TINY) / INT8_MAX}


def _gated(c, N):
    gate, up = c[..., :N], c[..., N:]
    return gate * up * torch.sigmoid(gate)


def _exact_gemm(s):
    M, N = s["c"].shape
    c = torch.empty((M, N), device="cuda", dtype=torch.float64)
    b = (s["b"].double() * s["scale_b"].double()[:, None]).t().contiguous()
    for m in range(0, M, 1024):
        part = (s["a"][m:m + 1024].double() * s["scale_a"][m:m + 1024].double()[:, None]) @ b
        if s["bias"] is not None:
            part += s["bias"].double()
        c[m:m + 1024] = _gated(part, N) if s["case"]["gated"] else part
    return {"c": c}


def _exact_experts(s):
    case, offsets = s["case"], s["offsets"].tolist()
    c = torch.empty(s["c"].shape, device="cuda", dtype=torch.float64)
    for e in range(case["E"]):
        lo, hi = offsets[e], offsets[e + 1]
        if lo == hi:
            continue
        at = torch.div(s["rows"][lo:hi].long(), case["k"], rounding_mode="floor") if case["gather"] else slice(lo, hi)
        part = (s["a"][at].double() * s["scale_a"][at].double()[:, None]) @ (s["b"][e].double() * s["scale_b"][e].double()[:, None]).t().contiguous()
        c[lo:hi] = _gated(part, case["N"]) if case["gated"] else part
    return {"c": c}


def _exact_combine(s):
    T, N = s["out"].shape
    out = torch.zeros((T, N), device="cuda", dtype=torch.float64) if s["add"] is None else s["add"].double()
    places = s["places"].long().view(T, -1)
    for j in range(places.shape[1]):
        out += s["y"][places[:, j]].double() * s["weights"][:, j].double()[:, None]
    return {"out": out}
