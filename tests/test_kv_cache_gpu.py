"""Tables and store of the 8-bit cache against plain forms on the CPU: whole numbers, codes and scales bit for bit."""
import numpy as np
import pytest
import torch

import composable_kernel_amd as ck
import serving_plain as sp

pytestmark = pytest.mark.gpu


def stream():
    return ck.StreamConfig(torch.cuda.current_stream().cuda_stream)


def plain_tables(ctx, new, free, table, slots_n, bs):
    table, cu, used = table.copy(), [0], 0
    slots = np.full(slots_n, -1, np.int64)
    at = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(int(c), 0), max(int(n), 0)
        had, need = -(-c // bs), -(-(c + n) // bs)
        blocks = {}
        for col in range(had, need):
            f = used + col - had
            if f < len(free):
                blocks[col] = free[f]
                if col < table.shape[1]:
                    table[b, col] = free[f]
        used += need - had
        for i in range(n):
            col = (c + i) // bs
            blk = -1
            if col < table.shape[1]:
                blk = table[b, col] if col < had else blocks.get(col, -1)
            if at < slots_n and blk >= 0:
                slots[at] = blk * bs + (c + i) % bs
            at += 1
        cu.append(at)
    return table, cu, [max(int(c), 0) + max(int(n), 0) for c, n in zip(ctx, new)], slots, used


def run_tables(ctx, new, free, table, slots_n, bs, max_blocks=None):
    dev = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")
    B = len(ctx)
    d = [dev(ctx), dev(new), dev(free), dev(table)]
    cu, kv, used = (torch.full((n,), -77, dtype=torch.int32, device="cuda") for n in (B + 1, B, 1))
    slots = torch.full((slots_n + 3,), -77, dtype=torch.int32, device="cuda")
    op = ck.DeviceKvCacheTables()
    width = table.shape[1]
    arg = op.MakeArgumentPointer(*d, cu, kv, slots, used, B, len(free), width if max_blocks is None else max_blocks, width, slots_n, bs)
    op.MakeInvokerPointer().Run(arg, stream())
    torch.cuda.synchronize()
    assert bool((slots[slots_n:] == -77).all()), "wrote behind the slots"
    return d[3].cpu().numpy(), cu.tolist(), kv.tolist(), slots[:slots_n].cpu().numpy(), int(used)


@pytest.mark.parametrize("B,ctx_hi,new_hi,bs", [(1, 0, 1, 16), (1, 100, 1, 16), (7, 40, 5, 16), (64, 300, 1, 32), (300, 90, 40, 16),
                                                (1000, 20, 3, 64), (3, 10, 5000, 128), (257, 200, 0, 16), (8192, 30, 2, 16)])
def test_tables(B, ctx_hi, new_hi, bs):
    rng = np.random.default_rng(B + bs)
    ctx, new = rng.integers(0, ctx_hi + 1, B), rng.integers(0, new_hi + 1, B)
    had, need = -(-ctx // bs), -(-(ctx + new) // bs)
    order = rng.permutation(int(need.sum()) + 9).astype(np.int32)
    table = np.full((B, int(need.max()) + 2), -5, np.int32)
    at = 0
    for b in range(B):
        table[b, :had[b]] = order[at:at + had[b]]
        at += had[b]
    free, T = order[at:], int(new.sum()) + 11
    want = plain_tables(ctx, new, free, table, T, bs)
    got = run_tables(ctx, new, free, table, T, bs)
    assert np.array_equal(got[0], want[0]) and got[1] == want[1] and got[2] == want[2] and got[4] == want[4]
    assert np.array_equal(got[3], want[3])


@pytest.mark.parametrize("case", ["free list short", "no free block", "table narrow", "slots short", "no sequence", "negative lengths"])
def test_tables_that_do_not_fit(case):
    bs, ctx, new = 16, np.array([5, 20, 0, 33]), np.array([30, 1, 50, 16])
    table = np.full((4, 6), -1, np.int32)
    table[0, 0], table[1, :2], table[3, :3] = 3, (9, 1), (0, 2, 7)
    free, T = np.arange(20, 32, dtype=np.int32), int(new.sum())
    if case == "free list short":
        free = free[:3]
    elif case == "no free block":
        free = free[:0]
    elif case == "table narrow":
        table = table[:, :3]
    elif case == "slots short":
        T = 40
    elif case == "no sequence":
        ctx, new, table, T = ctx[:0], new[:0], table[:0], 5
    else:
        ctx, new, T = np.array([5, -3, 0, 33]), np.array([30, 1, -50, 16]), 47
        table[1, :2] = -1
    want, got = plain_tables(ctx, new, free, table, T, bs), run_tables(ctx, new, free, table, T, bs)
    assert np.array_equal(got[0], want[0]) and got[1] == want[1] and got[2] == want[2] and got[4] == want[4]
    assert np.array_equal(got[3], want[3])


def run_store(k, v, slots, cache, xt):
    kc, vc, ks, vs = (x.clone().cuda() for x in cache)     # (clone keeps the strides of a dense layout)
    kv = torch.cat([k.flatten(1), v.flatten(1)], dim=1).cuda()
    T, H, D = k.shape
    kd, vd = kv[:, :H * D].view(T, H, D), kv[:, H * D:].view(T, H, D)
    op = ck.DeviceKvCacheStore8(xt)
    arg = op.MakeArgumentPointer(kd, vd, torch.tensor(slots, dtype=torch.int32, device="cuda"), ck.KvCache8(kc, vc, ks, vs), T,
                                 kd.stride()[:2], vd.stride()[:2])
    assert op.IsSupportedArgument(arg), ck.capi.last_error()
    op.MakeInvokerPointer().Run(arg, stream())
    torch.cuda.synchronize()
    return [x.cpu() for x in (kc, vc, ks, vs)]


def check_store(k, v, slots, cache, xt):
    want = [x.clone() for x in cache]
    sp.store(want[0], want[2], k, slots)
    sp.store(want[1], want[3], v, slots)
    got = run_store(k, v, slots, cache, xt)
    for name, g, w in zip(("k", "v"), got[:2], want[:2]):
        assert sp.same_codes(g, w), name
    for name, g, w in zip(("k", "v"), got[2:], want[2:]):
        assert torch.equal(g.nan_to_num(nan=-1.0), w.nan_to_num(nan=-1.0)), name
    return want


DT = {"bf16": torch.bfloat16, "f16": torch.float16}


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("xt", ["bf16", "f16"])
@pytest.mark.parametrize("H,D,size,layout", [(2, 64, 16, "bhsd"), (1, 128, 16, "bshd"), (3, 80, 32, "bhsd"), (2, 16, 64, "bshd"),
                                             (2, 112, 128, "bhsd"), (5, 48, 16, "bhsd")])
def test_store(code, xt, H, D, size, layout):
    g = sp.gen(H * 100 + D + size)
    cache = sp.random_cache(g, 24, H, size, D, code, layout)
    order = torch.randperm(24, generator=g).tolist()
    slots, at = [], 0
    for ctx, new in ((0, 1), (3, 1), (size - 1, 1), (size - 2, 5), (7, 2 * size + 3), (0, size), (0, 3 * size + 1), (size, 2)):
        blocks = order[at:at + -(-(ctx + new) // size)]
        at += len(blocks)
        slots += [blocks[(ctx + i) // size] * size + (ctx + i) % size for i in range(new)]
    T = len(slots)
    # magnitudes on both sides of what the blocks hold already, so that some scales grow and some stay
    grow = torch.exp2(torch.randint(-3, 3, (T, H, 1), generator=g).float())
    k, v = (sp.normal(g, (T, H, D)) * grow).to(DT[xt]), (sp.normal(g, (T, H, D)) * grow).to(DT[xt])
    check_store(k, v, slots, cache, xt)


@pytest.mark.parametrize("tokens", [300, 700, 2600, 5200])
def test_store_of_many_tokens(tokens):
    """One token, four and sixteen a wave, runs that begin anywhere, skipped tokens between and inside them."""
    g = sp.gen(8)
    blocks = tokens // 8
    cache = sp.random_cache(g, blocks, 2, 16, 64, torch.float8_e4m3fn)
    order = torch.randperm(blocks, generator=g).tolist()
    slots, at = [], 0
    while len(slots) < tokens:
        first, n = int(torch.randint(0, 16, (1,), generator=g)), int(torch.randint(1, 60, (1,), generator=g))
        mine = order[at:at + -(-(first + n) // 16)]
        at += len(mine)
        slots += [mine[(first + i) // 16] * 16 + (first + i) % 16 for i in range(n)] + [-1] * int(torch.randint(0, 3, (1,), generator=g))
    k, v = sp.normal(g, (len(slots), 2, 64), torch.bfloat16, 2.0), sp.normal(g, (len(slots), 2, 64), torch.bfloat16, 0.2)
    check_store(k, v, slots, cache, "bf16")


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
def test_store_skips_slots_outside_the_cache_and_keeps_the_rest(code):
    g = sp.gen(4)
    cache = sp.random_cache(g, 3, 2, 16, 32, code)
    k, v = sp.normal(g, (6, 2, 32), torch.bfloat16), sp.normal(g, (6, 2, 32), torch.bfloat16)
    want = check_store(k, v, [-1, 48, 5, 6, 1 << 30, -(1 << 31)], cache, "bf16")
    for i in (1, 2):
        assert sp.same_codes(want[0][i], cache[0][i])


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
def test_store_of_nan_infinity_and_zero(code):
    g = sp.gen(6)
    cache = sp.random_cache(g, 6, 1, 16, 64, code)
    k = sp.normal(g, (8, 1, 64), torch.bfloat16)
    v = k.clone()
    k[0, 0, 3], k[1, 0, 9], k[4], v[5, 0, 63] = float("nan"), float("inf"), 0.0, -float("inf")
    # blocks 0: NaN in the middle of a filled one; 1: infinity at its start; 2: two tokens; 3: zeros alone; 4, 5
    want = check_store(k, v, [5, 16, 32, 33, 48, 64, 80, 81], cache, "bf16")
    assert bool(want[2][0, 0].isnan()) and bool(want[2][1, 0].isinf()) and float(want[2][3, 0]) > 0
    # begun anew, a block is sound again; continued, it is not
    again = [x.clone() for x in want]
    x = sp.normal(g, (2, 1, 64), torch.bfloat16)
    after = check_store(x, x, [0, 17], again, "bf16")
    assert bool(after[2][0, 0].isfinite()) and not bool(after[2][1, 0].isfinite())


def test_a_cache_past_32_bit_offsets():
    """Blocks behind 4 GiB: a cache of few heads with rows far apart."""
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GiB of device memory")
    size, D, stride = 16, 64, 1 << 20
    blocks = 5000
    flat = torch.zeros(blocks * stride, dtype=torch.int8, device="cuda")
    kc = flat.as_strided((blocks, 1, size, D), (stride, size * D, D, 1))
    vc = flat.as_strided((blocks, 1, size, D), (stride, size * D, D, 1), stride // 2)
    ks, vs = torch.ones(blocks, 1, device="cuda"), torch.ones(blocks, 1, device="cuda")
    cache = ck.KvCache8(kc, vc, ks, vs)
    g = sp.gen(2)
    k, v = sp.normal(g, (2, 1, D), torch.bfloat16).cuda(), sp.normal(g, (2, 1, D), torch.bfloat16).cuda()
    slots = torch.tensor([4999 * size, 4999 * size + 1], dtype=torch.int32, device="cuda")
    op = ck.DeviceKvCacheStore8("bf16")
    op.MakeInvokerPointer().Run(op.MakeArgumentPointer(k, v, slots, cache, 2, k.stride()[:2], v.stride()[:2]), stream())
    q, o = k.repeat(1, 2, 1).contiguous(), torch.zeros(2, 2, D, dtype=torch.bfloat16, device="cuda")
    at = ck.DevicePagedAttention8("bf16")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    table, cu, kv = i32([[4999]]), i32([0, 2]), i32([2])
    at.MakeInvokerPointer().Run(at.MakeArgumentPointer(q, o, table, cu, kv, cache, 1, 2, 2, 2, 1, 1, q.stride()[:2], o.stride()[:2],
                                                       ck.Scale(0.125)), stream())
    torch.cuda.synchronize()
    want = [torch.zeros(1, 1, size, D, dtype=torch.int8), torch.ones(1, 1)], [torch.zeros(1, 1, size, D, dtype=torch.int8), torch.ones(1, 1)]
    sp.store(*want[0], k.cpu(), [0, 1])
    sp.store(*want[1], v.cpu(), [0, 1])
    assert torch.equal(kc[4999].cpu(), want[0][0][0]) and torch.equal(vc[4999].cpu(), want[1][0][0])
    assert int(flat.count_nonzero()) == int(want[0][0].count_nonzero() + want[1][0].count_nonzero())
    ref, mag, big = sp.attention(q.cpu(), torch.zeros(1, 1), [0, 2], [2], want[0][0], want[1][0], want[0][1], want[1][1], 0.125, True)
    assert bool(((o.cpu().double() - ref).abs() <= sp.attention_bound(ref, mag, big, torch.bfloat16, D, 2)).all())


def test_tables_block_numbers_without_a_slot():
    """Numbers past 2^31 / block_size, in the table or the free list, would wrap to another block's slots."""
    top = 2 ** 31 // 16
    table = np.array([[top + 3, 5, -1], [top - 1, 2 ** 31 - 1, -1]])
    got = run_tables([16, 31], [18, 3], [top, 9, top - 2], table, 21, 16)
    want = [-1] * 16 + [9 * 16, 9 * 16 + 1] + [-1, (top - 2) * 16, (top - 2) * 16 + 1]
    assert got[1] == [0, 18, 21] and got[4] == 3 and got[3].tolist() == want


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
def test_a_started_block_with_a_negative_scale(code):
    """Blocks that hold (-codes, -scales) instead of (codes, scales) stand for the same values, and go on doing so: where the scale
    stays, the new codes are the negative ones, where it grows, codes and scale are the same in both."""
    g = sp.gen(21)
    cache = sp.random_cache(g, 8, 2, 16, 64, code)
    turned = [(-x.float()).to(code) for x in cache[:2]] + [-x for x in cache[2:]]
    slots = [b * 16 + i for b, (o, n) in enumerate(((0, 4), (1, 3), (7, 1), (15, 1), (3, 13), (9, 2), (4, 1), (0, 16))) for i in range(o, o + n)]
    # blocks 1, 3, 5: tokens small enough for the scale to stay; 2, 4, 6: large ones
    size = torch.tensor([4.0 if (s // 16) % 2 == 0 else 0.05 for s in slots])[:, None, None]
    k, v = ((sp.normal(g, (len(slots), 2, 64)) * size).to(torch.bfloat16) for _ in range(2))
    want, got = run_store(k, v, slots, cache, "bf16"), run_store(k, v, slots, turned, "bf16")
    value = lambda c, s, i: c[i].float() * s[i][:, None, None]
    for i in range(2):
        assert torch.equal(want[2 + i][1::2][:3], cache[2 + i][1::2][:3])
        for b in range(8):
            end = max(s for s in slots if s // 16 == b) % 16 + 1    # (what lies behind the run is unwritten)
            assert torch.equal(value(got[i], got[2 + i], b)[:, :end], value(want[i], want[2 + i], b)[:, :end]), (i, b)
