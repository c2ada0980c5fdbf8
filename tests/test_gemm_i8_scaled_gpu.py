"""DeviceGemmTokenScaleI8 and DeviceExpertsGemmI8 against their formulas in 64 bits."""
import itertools

import pytest
import torch

import composable_kernel_amd as ck
import experts_plain as ep

pytestmark = pytest.mark.gpu


def stream():
    return ck.StreamConfig(torch.cuda.current_stream().cuda_stream)


def strided(x, pad, offset):
    """x on the GPU, rows `pad` elements further apart, `offset` elements into its memory (what lies between is 3)."""
    M, K = x.shape
    d = torch.full((M * (K + pad) + offset + 16,), 3, dtype=x.dtype, device="cuda")[offset:offset + M * (K + pad)].view(M, K + pad)
    d[:, :K] = x.cuda()
    return d


def dense(M, N, K, kind, gated=False, biased=False, pads=(0, 0, 0), offset=0, workspace=True, seed=0):
    g = ep.gen(seed + M * 7 + N * 3 + K)
    wide = N * (1 + gated)
    a, b = ep.codes(g, (M, K)), ep.codes(g, (wide, K))
    sa = (0.5 + torch.rand(M, generator=g)) / 60
    sb = (0.5 + torch.rand(wide, generator=g)) / 60 / max(1, K) ** 0.5
    bias = ep.normal(g, (wide,)) if biased else None
    ad, bd = strided(a, pads[0], offset), strided(b, pads[1], offset)
    c = torch.full((M, N + pads[2]), 55.0, dtype=ep.DT[kind], device="cuda")
    op = ck.DeviceGemmTokenScaleI8(kind, Gated=gated)
    arg = op.MakeArgumentPointer(ad, bd, c, sa.cuda(), sb.cuda(), None if bias is None else bias.cuda(), M, N, K, K + pads[0], K + pads[1], N + pads[2])
    assert op.IsSupportedArgument(arg), ck.capi.last_error()
    need = op.GetWorkSpaceSize(arg)
    if need and workspace:
        op.SetWorkSpacePointer(arg, torch.full((need,), 0x7D, dtype=torch.uint8, device="cuda"))
    op.MakeInvokerPointer().Run(arg, stream())
    torch.cuda.synchronize()
    c = c.cpu()
    assert bool((c[:, N:] == 55).all()), "wrote behind the row"
    want, bound = ep.scaled(a, b, sa, sb, bias, gated, ep.DT[kind])
    ep.near(c[:, :N], want, bound, (M, N, K, kind, gated))
    return c


SIZES = [(1, 1, 1), (1, 64, 16), (3, 70, 128), (16, 256, 512), (17, 100, 256), (33, 129, 272), (64, 128, 4096), (65, 257, 144), (128, 128, 128),
         (130, 200, 400), (200, 520, 1024), (257, 300, 1040), (300, 1000, 2064), (1, 1000, 11008), (5, 333, 131071), (520, 769, 640)]


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("gated,biased", [(False, False), (True, True), (False, True), (True, False)])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_sizes(kind, gated, biased, M, N, K):
    dense(M, N, K, kind, gated, biased)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,N,K", [(7, 90, 100), (130, 140, 333), (40, 33, 1), (1, 7, 15), (260, 270, 130)])
@pytest.mark.parametrize("pads,offset", [((0, 0, 0), 0), ((1, 3, 5), 0), ((16, 32, 8), 0), ((0, 0, 0), 1), ((12, 12, 1), 4)])
def test_strides_and_addresses(gated, M, N, K, pads, offset):
    dense(M, N, K, "bf16", gated, True, pads, offset)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,N,K", [(20, 96, 256), (300, 320, 512), (600, 600, 256)])
@pytest.mark.parametrize("pads", [(16, 32, 8), (0, 0, 3)])
def test_strides_of_whole_vectors(gated, M, N, K, pads):
    for kind in ("bf16", "f32"):
        dense(M, N, K, kind, gated, True, pads, 16)


def test_sums_are_exact_at_the_largest_reduction():
    K = 131071
    a = torch.full((2, K), -128, dtype=torch.int8)
    b = torch.full((3, K), -128, dtype=torch.int8)
    b[1], b[2, 1:] = 127, 0
    one = torch.ones(3)
    c = torch.zeros(2, 3, device="cuda")
    op = ck.DeviceGemmTokenScaleI8("f32")
    arg = op.MakeArgumentPointer(a.cuda(), b.cuda(), c, one[:2].cuda(), one.cuda(), None, 2, 3, K, K, K, 3)
    op.MakeInvokerPointer().Run(arg, stream())
    torch.cuda.synchronize()
    want = torch.tensor([128 * 128 * K, -128 * 127 * K, 128 * 128], dtype=torch.int64).float()
    assert torch.equal(c.cpu(), want.expand(2, 3))


def test_nothing_to_reduce_gives_the_bias():
    for gated in (False, True):
        dense(5, 40, 0, "f32", gated, True)
        dense(5, 40, 0, "bf16", gated, False)


def test_scales_that_are_not_finite():
    """A token that could not be quantised (scale NaN) is NaN in its own row and nowhere else."""
    M, N, K = 40, 64, 128
    a, b = ep.codes(ep.gen(1), (M, K)), ep.codes(ep.gen(2), (N, K))
    sa, sb = torch.ones(M), torch.ones(N)
    sa[7] = float("nan")
    c = torch.zeros(M, N, device="cuda", dtype=torch.float16)
    op = ck.DeviceGemmTokenScaleI8("f16")
    op.MakeInvokerPointer().Run(op.MakeArgumentPointer(a.cuda(), b.cuda(), c, sa.cuda(), sb.cuda(), None, M, N, K, K, K, N), stream())
    torch.cuda.synchronize()
    c = c.cpu()
    assert bool(c[7].isnan().all()) and not bool(c[:7].isnan().any()) and not bool(c[8:].isnan().any())
    want = (a.double() @ b.double().t())
    over = want.abs() >= 65520
    over[7] = False
    assert bool(over.any()) and bool(c[over].isinf().all())  # past fp16: infinities


# ------------------------------------------------------------------------------------------------ experts
def experts(counts, N, K, kind, gated=False, gather=None, biased=False, spare=3, pads=(0, 0, 0), offset=0, batch_pad=0, bad_rows=(), seed=0):
    """counts: rows of each expert. gather: rows of A that pairs of `gather` rows each come from, in any order."""
    g = ep.gen(seed + sum(counts) * 11 + N + K)
    E, P = len(counts), sum(counts)
    wide, size = N * (1 + gated), P + spare
    per = gather or 1
    rows_a = max(1, -(-P // per)) if gather else size
    a, b = ep.codes(g, (rows_a, K)), ep.codes(g, (E * wide, K))
    sa = (0.5 + torch.rand(rows_a, generator=g)) / 60
    sb = (0.5 + torch.rand(E, wide, generator=g)) / 60 / max(1, K) ** 0.5
    bias = ep.normal(g, (E, wide)) if biased else None
    offsets = torch.tensor([0] + list(itertools.accumulate(counts)), dtype=torch.int32)
    rows = None
    if gather:
        rows = torch.cat([torch.randperm(rows_a * per, generator=g)[:P], torch.full((spare,), -1)]).int()
        for i in bad_rows:
            rows[i] = [-1, rows_a * per, 2 ** 31 - 1][i % 3]
    ad = strided(a, pads[0], offset)
    bd = torch.full((E, wide * (K + pads[1]) + batch_pad), 5, dtype=torch.int8, device="cuda")
    bd[:, :wide * (K + pads[1])].view(E, wide, K + pads[1])[:, :, :K] = b.view(E, wide, K).cuda()
    c = torch.full((size, N + pads[2]), 55.0, dtype=ep.DT[kind], device="cuda")
    op = ck.DeviceExpertsGemmI8(kind, Gated=gated)
    arg = op.MakeArgumentPointer(ad, bd, c, sa.cuda(), sb.cuda(), None if bias is None else bias.cuda(), offsets.cuda(), None if rows is None else rows.cuda(),
                                 size, rows_a, E, N, K, K + pads[0], K + pads[1], N + pads[2], bd.stride(0), per)
    assert op.IsSupportedArgument(arg), ck.capi.last_error()
    op.MakeInvokerPointer().Run(arg, stream())
    torch.cuda.synchronize()
    c = c.cpu()
    assert bool((c[:, N:] == 55).all()) and bool((c[P:] == 55).all()), "wrote outside the experts' rows"
    for e in range(E):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        at = torch.arange(lo, hi) if rows is None else torch.div(rows[lo:hi].long(), per, rounding_mode="floor")
        there = (at >= 0) & (at < rows_a)
        x = torch.where(there[:, None], a[at.clamp(0, rows_a - 1)].int(), 0)
        s = torch.where(there, sa[at.clamp(0, rows_a - 1)], torch.zeros(()))
        want, bound = ep.scaled(x, b.view(E, wide, K)[e], s, sb[e], None if bias is None else bias[e], gated, ep.DT[kind])
        ep.near(c[lo:hi, :N], want, bound, (e, counts[e]))


COUNTS = [[1], [0, 1, 0], [3, 0, 5, 2], [1] * 8, [17, 0, 0, 16, 15, 1], [40, 64, 65, 0, 7], [130, 1, 0, 128, 127], [300, 5, 260], [0, 0, 0, 0], [2] * 70]


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("gated,gather", [(True, 2), (False, None), (True, None), (False, 4)])
@pytest.mark.parametrize("N,K", [(64, 128), (100, 272), (300, 512)])
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "_".join(map(str, c[:6])))
def test_experts(kind, gated, gather, N, K, counts):
    experts(counts, N, K, kind, gated, gather)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("N,K,pads,offset,batch_pad", [(70, 100, (0, 0, 0), 0, 0), (64, 256, (16, 16, 8), 0, 32), (64, 256, (1, 0, 0), 0, 0),
                                                       (64, 256, (0, 5, 3), 0, 0), (64, 256, (0, 0, 0), 1, 0), (64, 256, (0, 0, 0), 0, 7)])
def test_experts_strides_and_biases(gated, N, K, pads, offset, batch_pad):
    for counts in ([5, 0, 9], [70, 140, 1]):
        experts(counts, N, K, "f16", gated, 3, True, 2, pads, offset, batch_pad)


def test_rows_outside_a_count_as_zeros():
    experts([5, 7, 200], 96, 256, "f32", False, 2, True, bad_rows=(0, 4, 5, 11, 100))
    experts([5, 7, 200], 96, 256, "bf16", True, 2, True, bad_rows=(0, 4, 5, 11, 100))


def test_nothing_to_reduce_and_many_experts():
    experts([3, 0, 4], 40, 0, "f32", False, 2, True)
    experts([i % 3 for i in range(1024)], 32, 64, "bf16", False, 2)
    experts([0] * 1000 + [9] + [0] * 23, 32, 64, "bf16", True, 2)


@pytest.mark.parametrize("offsets", [[0, 9, 4, 12], [5, 5, 1000, 1000], [-7, 3, 3, 6], [12, 12, 12, 12]])
def test_offsets_are_cut_to_the_rows(offsets):
    """Offsets that no router gives: whatever they say, only rows that exist are written."""
    P, N, K = 12, 64, 128
    a, b = ep.codes(ep.gen(1), (P, K)), ep.codes(ep.gen(2), (3, N, K))
    c = torch.full((P + 8, N), 55.0, device="cuda")
    op = ck.DeviceExpertsGemmI8("f32")
    arg = op.MakeArgumentPointer(a.cuda(), b.cuda(), c, torch.ones(P).cuda(), torch.ones(3, N).cuda(), None, torch.tensor(offsets, dtype=torch.int32).cuda(), None,
                                 P, P, 3, N, K, K, K, N, N * K)
    op.MakeInvokerPointer().Run(arg, stream())
    torch.cuda.synchronize()
    assert bool((c[P:].cpu() == 55).all())
