"""DevicePagedAttention8 against attention in 64 bits (bound: serving_plain.attention_bound)."""
import math

import pytest
import torch

import composable_kernel_amd as ck
import serving_plain as sp

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


class Problem:
    def __init__(self, news, kvs, heads, H, D, size, code=torch.float8_e4m3fn, xt="bf16", layout="bhsd", seed=0, causal=True, scale=None,
                 spare=0):
        g = sp.gen(seed + heads + D + size + sum(kvs))
        self.news, self.kvs, self.heads, self.D, self.size, self.xt, self.causal = news, kvs, heads, D, size, xt, causal
        self.scale = D ** -0.5 if scale is None else scale
        self.cu = [0]
        for n in news:
            self.cu.append(self.cu[-1] + n)
        each = [-(-kv // size) for kv in kvs]
        blocks = sum(each) + 3
        self.cache = list(sp.random_cache(g, blocks, H, size, D, code, layout))
        order, at = torch.randperm(blocks, generator=g).tolist(), 0
        self.table = torch.full((len(news), max(each + [1]) + 1), -1, dtype=torch.int32)
        for b, n in enumerate(each):
            self.table[b, :n] = torch.tensor(order[at:at + n])
            at += n
        self.T = self.cu[-1] + spare
        self.q = sp.normal(g, (self.T, heads, D), DT[xt])

    def run(self, max_kv=None, tokens=None, o=None, sync=True):
        kc, vc, ks, vs = (x.cuda() for x in self.cache)
        self.dev = [kc, vc, ks, vs, self.table.cuda(), torch.tensor(self.cu, dtype=torch.int32, device="cuda"),
                    torch.tensor(self.kvs, dtype=torch.int32, device="cuda")]
        # queries as columns of a fused projection, outputs with a gap behind every token
        qkv = torch.zeros(self.T, (self.heads + 3) * self.D, dtype=DT[self.xt], device="cuda")
        q = qkv[:, :self.heads * self.D].view(self.T, self.heads, self.D)
        q.copy_(self.q)
        out = torch.full((self.T, self.heads * self.D + 8), 5.0, dtype=DT[self.xt], device="cuda")
        o = out[:, :self.heads * self.D].view(self.T, self.heads, self.D)
        op = ck.DevicePagedAttention8(self.xt, Causal=self.causal)
        arg = op.MakeArgumentPointer(q, o, self.dev[4], self.dev[5], self.dev[6], ck.KvCache8(kc, vc, ks, vs), len(self.news), self.T,
                                     self.heads, max(self.kvs + [0]) if max_kv is None else max_kv, self.table.shape[1],
                                     self.table.shape[1], q.stride()[:2], o.stride()[:2], ck.Scale(self.scale))
        assert op.IsSupportedArgument(arg), ck.capi.last_error()
        need = op.GetWorkSpaceSize(arg)
        if need:
            op.SetWorkSpacePointer(arg, torch.full((need,), 0x7F, device="cuda", dtype=torch.uint8))
        op.MakeInvokerPointer().Run(arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert bool((out[:, self.heads * self.D:] == 5).all()) and bool((out[self.cu[-1]:] == 5).all()), "wrote outside the rows"
        return o.cpu()[:self.cu[-1]]

    def check(self, **kw):
        got = self.run(**kw).double()
        kc, vc, ks, vs = self.cache
        want, mag, big = sp.attention(self.q[:self.cu[-1]], self.table, self.cu, self.kvs, kc, vc, ks, vs, self.scale, self.causal)
        bound = sp.attention_bound(want, mag, big, DT[self.xt], self.D, max(self.kvs + [0]))
        bad = ~((got - want).abs() <= bound)
        assert not bool(bad.any()), (float((got - want).abs().max()), bad.nonzero()[:4].tolist(), int(bad.sum()))
        return got


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("xt", ["bf16", "f16"])
@pytest.mark.parametrize("heads,H,D,size", [(4, 1, 64, 16), (8, 2, 128, 16), (7, 1, 80, 32), (3, 3, 16, 64), (32, 2, 112, 128), (20, 1, 96, 16)])
def test_single_tokens(code, xt, heads, H, D, size):
    Problem([1, 1, 1, 1, 1], [1, 15, 33, 64, 300], heads, H, D, size, code, xt).check()


@pytest.mark.parametrize("kv", [1, 2, 16, 31, 32, 33, 127, 128, 129, 255, 257, 511, 1000, 2049, 5000])
def test_lengths(kv):
    Problem([1], [kv], 8, 2, 64, 16).check()


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,H,D,size", [(4, 1, 64, 16), (8, 2, 128, 32), (6, 6, 48, 16), (14, 2, 80, 64), (48, 2, 64, 16)])
def test_prompts(code, causal, heads, H, D, size):
    Problem([5, 1, 17, 40], [5, 9, 50, 100], heads, H, D, size, code, "bf16", causal=causal).check()
    Problem([33, 70], [33, 200], heads, H, D, size, code, "f16", causal=causal).check()


@pytest.mark.parametrize("news,kvs", [([130], [130]), ([200, 3], [333, 3]), ([64, 128, 256], [64, 129, 300]), ([1, 257], [400, 257])])
@pytest.mark.parametrize("heads,H,D", [(4, 1, 128), (2, 2, 64), (7, 1, 64)])
def test_longer_prompts(news, kvs, heads, H, D):
    Problem(news, kvs, heads, H, D, 16).check()
    Problem(news, kvs, heads, H, D, 32, torch.int8, "f16", causal=False).check()


def test_rows_that_see_nothing_are_zero():
    # a sequence without cached tokens, one with fewer than it has queries (its first rows see none), one without queries
    p = Problem([2, 5, 0, 1], [0, 3, 40, 20], 8, 2, 64, 16)
    got = p.check()
    assert bool((got[:4] == 0).all()) and bool((got[4:] != 0).any())
    p = Problem([2, 70, 0, 1], [0, 3, 40, 20], 8, 2, 64, 16)
    got = p.check()
    assert bool((got[:69] == 0).all())
    p = Problem([2, 5, 0, 1], [0, 3, 40, 20], 8, 2, 64, 16, causal=False)
    assert bool((p.check()[:2] == 0).all())


def test_no_sequence_and_no_token():
    assert Problem([], [], 4, 1, 64, 16, spare=3).run().shape[0] == 0
    assert Problem([0, 0], [5, 0], 4, 1, 64, 16, spare=2).run().shape[0] == 0


def test_rows_behind_the_last_sequence_stay():
    Problem([1, 3, 1], [40, 50, 600], 8, 2, 64, 16, spare=7).check()
    Problem([90, 40], [90, 600], 8, 2, 64, 16, spare=200).check()


@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
def test_cache_layouts(layout):
    Problem([1, 4], [77, 300], 8, 2, 64, 32, layout=layout).check()
    Problem([100], [300], 8, 2, 128, 32, torch.int8, layout=layout).check()


@pytest.mark.parametrize("news", [[1, 1, 1], [1, 2, 3], [80, 1, 30]])
def test_stale_codes_scales_and_table_entries_do_not_matter(news):
    """Behind the last token of a block: NaN codes; blocks that no sequence has: NaN codes and scales; table columns behind the
    last block: numbers of those blocks, and numbers outside the cache."""
    p = Problem(news, [17, 100, 47], 8, 2, 64, 16)
    want = p.run()
    kc, vc, ks, vs = p.cache
    nan = torch.tensor(float("nan")).to(torch.float8_e4m3fn)
    used = set()
    for b, kv in enumerate(p.kvs):
        for c in range(-(-kv // 16)):
            used.add(int(p.table[b, c]))
        for x in (kc, vc):
            if kv % 16:
                x[int(p.table[b, kv // 16]), :, kv % 16:] = nan
    free = [i for i in range(kc.shape[0]) if i not in used]
    for i in free:
        kc[i], vc[i], ks[i], vs[i] = nan, nan, float("nan"), float("inf")
    for b, kv in enumerate(p.kvs):
        p.table[b, -(-kv // 16):] = free[b % len(free)]
    p.table[0, -1], p.table[1, -1] = 1 << 30, -(1 << 31)
    assert torch.equal(p.run(), want)


@pytest.mark.parametrize("bad", [-1, 1 << 30, -(1 << 31)])
@pytest.mark.parametrize("news", [[1, 1], [60, 2]])
def test_blocks_outside_the_cache_count_as_not_there(news, bad):
    p = Problem(news, [90, 64], 8, 2, 64, 16)
    p.table[0, 1], p.table[1, 3], p.table[1, 0] = bad, bad, bad
    p.check()
    p = Problem(news, [90, 64], 8, 2, 64, 16)
    p.table[:] = bad
    assert bool((p.check() == 0).all())


def test_lengths_past_the_table_end_with_it():
    p = Problem([1, 2], [60, 40], 4, 1, 64, 16)
    p.kvs = [10000, 10000]
    p.table[p.table < 0] = 0
    p.check(max_kv=64)


@pytest.mark.parametrize("max_kv", [0, 1, 300, 5000, 100000])
def test_the_bound_on_the_lengths_does_not_change_results(max_kv):
    Problem([1, 1], [1500, 300], 8, 2, 64, 16).check(max_kv=max_kv)


def test_a_poisoned_block_reaches_only_rows_that_see_it():
    p = Problem([1, 40, 1], [64, 64, 64], 8, 2, 64, 16)
    first = int(p.table[1, 3])                     # tokens 48 ... 63 of the sequence with 40 queries (24 ... 63)
    p.cache[3][first] = float("nan")
    p.cache[1][first] = 0.0
    got = p.run()
    assert bool(got[0].isfinite().all()) and bool(got[41].isfinite().all())
    assert bool(got[1:25].isfinite().all()) and bool(got[25:41].isnan().all())
    p = Problem([1, 40, 1], [64, 64, 64], 8, 2, 64, 16)
    p.cache[2][int(p.table[1, 3])] = float("nan")
    got = p.run()
    assert bool(got[1:25].isfinite().all()) and bool(got[25:41].isnan().all()) and bool(got[41].isfinite().all())


def test_large_scores_and_uneven_scales():
    p = Problem([1, 50], [500, 200], 8, 2, 64, 16, scale=3.0)
    p.check()
    p = Problem([1, 50], [500, 200], 8, 2, 64, 16, torch.int8)
    p.cache[3] *= torch.exp2(torch.randint(-6, 7, p.cache[3].shape, generator=sp.gen(1)).float())
    p.cache[2] *= torch.exp2(torch.randint(-3, 2, p.cache[2].shape, generator=sp.gen(2)).float())
    p.check()
    Problem([3, 70], [90, 70], 8, 2, 64, 16, scale=-0.2).check()


def test_the_same_call_twice_gives_the_same_bits():
    p = Problem([1, 1, 130], [3000, 2000, 700], 8, 2, 128, 16)
    assert torch.equal(p.run(), p.run())


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("news,kvs", [([64], [3000]), ([33, 40], [2100, 700]), ([100], [4097])])
def test_prompts_over_long_caches(news, kvs, code):
    """Few tiles, many cached tokens: the shares of the cached tokens are joined, some of them empty."""
    Problem(news, kvs, 4, 1, 64, 16, code).check()
    Problem(news, kvs, 2, 2, 128, 64, code, "f16", causal=False).check()


@pytest.mark.parametrize("max_kv", [0, 1023, 1024, 1500, 100000])
@pytest.mark.parametrize("causal", [True, False])
def test_shares_of_prompts(max_kv, causal):
    """Shares of two steps and more, most of them empty for the short sequences; the bound only steers how many there are."""
    Problem([60, 40, 70], [1500, 30, 70], 4, 1, 80, 16, causal=causal).check(max_kv=max_kv)
    Problem([200], [1100], 8, 2, 128, 32, torch.int8, "f16", causal=causal).check(max_kv=max_kv)


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("D,size", [(64, 16), (128, 64)])
def test_one_share_of_a_long_cache(code, D, size):
    """Over 8192 tokens a share: the block numbers and scales of a wave's 32 turns are fetched anew."""
    Problem([1, 2, 1], [8193, 20000, 8192], 4, 1, D, size, code).check(max_kv=0)


def _rows_largest_scale(p):
    """[rows]: the largest value scale among the blocks that a row sees."""
    top = torch.zeros(p.cu[-1], dtype=torch.float64)
    for b, (n, kv) in enumerate(zip(p.news, p.kvs)):
        for i in range(n):
            see = kv - n + i + 1 if p.causal else kv
            blocks = [int(x) for x in p.table[b, :-(-max(see, 0) // p.size)]]
            top[p.cu[b] + i] = max([float(p.cache[3][x].abs().max()) for x in blocks] + [0.0])
    return top


def _check_to_each_rows_own_scale(p, **kw):
    """attention_bound, and what probabilities under fp16's normal numbers cost (serving_plain.small_products), row by row."""
    got = p.run(**kw).double()
    kc, vc, ks, vs = p.cache
    want, mag, big = sp.attention(p.q, p.table, p.cu, p.kvs, kc, vc, ks, vs, p.scale, p.causal)
    small = max(p.kvs) * 2.0 ** -25 * sp.QMAX[vc.dtype] * _rows_largest_scale(p)
    bound = sp.attention_bound(want, mag, big, DT[p.xt], p.D, max(p.kvs)) + small[:, None, None]
    bad = ~((got - want).abs() <= bound)
    assert not bool(bad.any()), (float(((got - want).abs() / bound).nan_to_num(nan=1e9).max()), bad.nonzero()[:4].tolist(), int(bad.sum()))


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("up", [10, 30])
@pytest.mark.parametrize("news,kvs,heads,H,D", [([5], [50], 8, 2, 64), ([7, 9], [50, 70], 6, 3, 128), ([40], [64], 8, 2, 64),
                                                ([100, 33], [200, 40], 8, 2, 128), ([70, 60], [1500, 70], 4, 1, 80)])
def test_a_value_scale_reaches_only_rows_that_see_its_block(news, kvs, heads, H, D, up, code):
    """Value scales that grow 2^up-fold from block to block over the new tokens: a row that sees the first of them keeps its own
    precision, whatever the scales of the blocks behind it are."""
    p = Problem(news, kvs, heads, H, D, 16, code)
    for b, (n, kv) in enumerate(zip(news, kvs)):
        first = (kv - n) // 16
        for c in range(first + 1, -(-kv // 16)):
            p.cache[3][int(p.table[b, c])] *= 2.0 ** min(up * (c - first), 90)
    _check_to_each_rows_own_scale(p)


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("news,kvs,heads,H,D", [([5], [50], 8, 2, 64), ([10, 9], [311, 70], 8, 2, 128), ([40], [64], 8, 2, 64),
                                                ([100, 33], [250, 40], 8, 2, 128), ([70, 60], [1524, 70], 4, 1, 80)])
def test_blocks_that_a_row_does_not_see_change_none_of_its_bits(news, kvs, heads, H, D, code):
    """Large key and value scales in the last block of every sequence, which only the last rows see."""
    p = Problem(news, kvs, heads, H, D, 16, code)
    want, blind = p.run(), []
    for b, (n, kv) in enumerate(zip(news, kvs)):
        last = (kv - 1) // 16
        for x in p.cache[2:]:
            x[int(p.table[b, last])] *= 2.0 ** 6
        blind += [p.cu[b] + i for i in range(n) if kv - n + i < last * 16]
    got = p.run()
    assert len(blind) >= 3 and torch.equal(got[blind], want[blind]) and not torch.equal(got, want)


def test_no_probability_is_lost_beside_a_value_scale_far_below_the_others():
    """One token whose value is 1, and 80000 behind it whose values are zero (their blocks' scales are what the store makes of zeros),
    with scores 26.5 powers of two under the first one's: the output is 1 / (1 + sum of their probabilities). Off by half a step of
    fp16 under 1 (2^-12), by 2^-24 for each of the 5000 additions of eight probabilities to a sum near 1 (a lane has every other
    eight), and 2^-18 for the exponents (26.5 and 109 rounded to fp32, twice)."""
    size, D, heads, kv, below = 16, 64, 4, 80000, 26.5
    p = Problem([30], [kv], heads, 1, D, size, torch.int8, "f16", causal=False, scale=1.0)
    kc, vc, ks, vs = p.cache
    p.q.zero_()
    p.q[:, :, 0] = 1.0
    for x in (kc, vc):
        x.zero_()
    ks.fill_(below * math.log(2.0) / 127)
    vs.fill_(2.0 ** -100 / 127)
    first = int(p.table[0, 0])
    kc[first, 0, 0, 0], vc[first, 0, 0], vs[first] = 127, 127, 1 / 127
    got = p.run(max_kv=0).double()   # (one share)
    want = 1 / (1 + (kv - 1) * 2.0 ** -below)
    assert bool(((got - want).abs() <= 2.0 ** -12 + 5000 * 2.0 ** -24 + 2.0 ** -18).all()), (float(got.min()), float(got.max()), want)



@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("news,kvs", [([1, 3], [300, 77]), ([60, 40], [90, 1100])])
def test_tiny_key_scales_under_large_queries(news, kvs, code):
    """Keys 2^-100 and queries 2^100 times as large, exact in bf16 and fp32: the same scores, and the same bits."""
    p = Problem(news, kvs, 8, 2, 64, 16, code)
    want = p.check()
    p.cache[2] *= 2.0 ** -100
    p.q *= 2.0 ** 100
    assert torch.equal(p.run().double(), want)


@pytest.mark.parametrize("news,kvs", [([1, 3], [300, 77]), ([60, 40], [90, 1100])])
def test_key_scales_of_zero(news, kvs):
    """All scores zero, masked ones apart, whatever the codes: the mean of the values that a row sees."""
    p = Problem(news, kvs, 8, 2, 64, 16)
    p.cache[2].zero_()
    p.q *= 2.0 ** 100
    p.check()
    p.cache[2].fill_(0.1)
    p.q *= 2.0 ** -100
    p.scale = 0.0
    p.check()


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("news,kvs,D", [([1, 3], [300, 77], 64), ([1], [5000], 128), ([60, 40], [90, 1100], 64), ([120, 7], [333, 30], 128)])
@pytest.mark.parametrize("which", ["keys", "values", "both", "all values", "all keys"])
def test_scales_of_either_sign(which, news, kvs, D, code):
    p = Problem(news, kvs, 8, 2, D, 16, code)
    g = sp.gen(12)
    signs = lambda x: torch.randint(0, 2, x.shape, generator=g) * 2.0 - 1
    if which in ("keys", "both"):
        p.cache[2] *= signs(p.cache[2])
    if which in ("values", "both"):
        p.cache[3] *= signs(p.cache[3])
    if which.startswith("all"):
        p.cache[2 if which == "all keys" else 3].neg_()
    p.check()
    if which == "both":
        p.scale = -p.scale
        p.check()


@pytest.mark.parametrize("news,kvs,heads,H,D,rows", [([2, 5], [40, 300], 8, 2, 64, 4), ([1, 4, 3], [9, 20, 33], 4, 1, 128, 3),
                                                     ([60, 70], [90, 400], 8, 2, 64, 83), ([150], [1500], 4, 1, 128, 101), ([40, 40], [40, 64], 8, 8, 64, 80)])
@pytest.mark.parametrize("causal", [True, False])
def test_fewer_rows_than_the_sequences_have(news, kvs, heads, H, D, rows, causal):
    """num_tokens ends inside a sequence: its rows up to there keep their places in it, the others are neither read nor written."""
    p = Problem(news, kvs, heads, H, D, 16, causal=causal)
    cache, (kc, vc, ks, vs) = [x.cuda() for x in p.cache], p.cache
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    table, cu, kv = p.table.cuda(), i32(p.cu), i32(kvs)
    q, o = p.q.cuda(), torch.full((p.T, heads, D), 5.0, dtype=torch.bfloat16, device="cuda")
    q[rows:] = float("nan")
    op = ck.DevicePagedAttention8("bf16", Causal=causal)
    arg = op.MakeArgumentPointer(q, o, table, cu, kv, ck.KvCache8(*cache), len(news), rows, heads, max(kvs), table.shape[1], table.shape[1],
                                 q.stride()[:2], o.stride()[:2], ck.Scale(p.scale))
    need = op.GetWorkSpaceSize(arg)
    if need:
        op.SetWorkSpacePointer(arg, torch.full((need,), 0x7F, device="cuda", dtype=torch.uint8))
    op.MakeInvokerPointer().Run(arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert bool((o[rows:] == 5).all())
    want, mag, big = sp.attention(p.q, p.table, p.cu, kvs, kc, vc, ks, vs, p.scale, causal)
    bound = sp.attention_bound(want, mag, big, torch.bfloat16, D, max(kvs))
    assert bool(((o.cpu().double() - want).abs() <= bound)[:rows].all())


@pytest.mark.parametrize("heads,H,D,size", [(8, 2, 64, 16), (4, 4, 128, 32)])
@pytest.mark.parametrize("most", [1, 3, 90])
def test_many_sequences(most, heads, H, D, size):
    """Past 64, 128 and 192 sequences, some without queries, some without cached tokens, rows in front of the first sequence."""
    g = sp.gen(most + heads)
    B = 200 if most < 90 else 130
    news = torch.randint(0, most + 1, (B,), generator=g).tolist()
    kvs = [n + int(torch.randint(0, 60, (1,), generator=g)) if b % 7 else 0 for b, n in enumerate(news)]
    p = Problem(news, kvs, heads, H, D, size, spare=5)
    p.check()
