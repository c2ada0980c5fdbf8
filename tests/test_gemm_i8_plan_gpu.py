"""Every kernel of DeviceGemmTokenScaleI8 and DeviceExpertsGemmI8 by the plan that leads to it: small products whose sizes, or whose little
workspace, make the rule take it, against the formula in 64 bits."""
import pytest
import torch

import composable_kernel_amd as ck
import experts_plain as ep
from composable_kernel_amd import capi
from test_gemm_i8_scaled_gpu import dense, strided, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,N,K,tile,runs", [(16, 100, 272, 16, 1), (13, 40, 9216, 16, 1), (40, 200, 1040, 16, 1), (62, 2000, 1040, 32, 1), (200, 130, 16384, 64, 2), (150, 4096, 256, 128, 1), (300, 4096, 1024, 64, 1),
                                             (1000, 4100, 512, 128, 1), (2050, 4100, 512, 256, 1), (30, 64, 100, 16, 0), (60, 64, 100, 128, 0), (1, 500, 4099, 16, 0), (130, 300, 4099, 128, 0)])
def test_plan(kind, gated, M, N, K, tile, runs):
    N = N // 2 if gated and M > 100 else N
    need = capi.lib().ckx_gemm_i8_tokenscale_workspace_bytes(M, N, K, int(gated))
    p = capi.gemm_i8_plan(M, N, K, gated=gated, workspace_bytes=need)
    assert p[0] == tile and (p[2] >= runs if runs > 1 else p[2] == runs), p
    dense(M, N, K, kind, gated, True)


def test_a_workspace_too_small_for_the_runs_is_left_alone():
    M, N, K = 130, 128, 16384
    need = capi.lib().ckx_gemm_i8_tokenscale_workspace_bytes(M, N, K, 0)
    most = capi.gemm_i8_plan(M, N, K, workspace_bytes=need)[2]
    fewer = capi.gemm_i8_plan(M, N, K, workspace_bytes=need - 4)[2]
    assert most > fewer >= 1
    with_it, without = dense(M, N, K, "f32"), dense(M, N, K, "f32", workspace=False)
    assert torch.equal(with_it, without)             # (sums of whole numbers)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("gathered", [False, True])
@pytest.mark.parametrize("rows,E,N,K,tile", [(20, 16, 100, 2048, 16), (200, 4, 130, 272, 16), (2400, 3, 200, 400, 64), (200, 4, 130, 100, 0),
                                             (400, 8, 2100, 1040, 64), (708, 8, 2100, 272, 128), (6000, 8, 2100, 272, 256)])
def test_plan_of_experts(gated, gathered, rows, E, N, K, tile):
    g = ep.gen(rows + N)
    R, wide = 50, N * (1 + gated)
    counts = torch.multinomial(torch.tensor([1.0] + [0.2] * (E - 1)), rows, replacement=True, generator=g).bincount(minlength=E)
    of_experts(g, counts, rows, E, N, K, R, wide, gated, gathered, tile)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("gathered", [False, True])
@pytest.mark.parametrize("counts", [[0, 1, 255, 256, 257, 0, 5200, 31], [6000, 0, 0, 0, 0, 0, 0, 0], [0, 0, 0, 0, 0, 0, 0, 6000], [128, 129, 127, 512, 513, 511, 4000, 80]])
def test_experts_of_every_size_on_the_largest_tiles(gated, gathered, counts):
    of_experts(ep.gen(sum(counts[:5])), torch.tensor(counts), 6000, 8, 2100, 272, 50, 2100 * (1 + gated), gated, gathered, 256)


def test_rows_outside_a_and_outside_c_on_the_largest_tiles():
    """Row numbers that A does not have count as rows of zeros; offsets past C's rows are cut."""
    rows, E, N, K, R = 6000, 8, 2100, 272, 40
    g = ep.gen(9)
    a, sa, b, sb = ep.codes(g, (R, K)), torch.rand(R, generator=g), ep.codes(g, (E, N, K)), torch.rand(E, N, generator=g) / 100
    pick = torch.randint(-R, 3 * R, (rows,), generator=g, dtype=torch.int32)
    pick[7] = -2 ** 31
    offsets = torch.tensor([-5, 700, 700, 2000, 1900, 2500, 3000, 5000, 9000], dtype=torch.int32)
    desc = capi.ExpertsDesc(rows, R, E, N, K, K, K, N, 1, 0, capi.TYPE_F32, 0, N * K)
    assert capi.experts_gemm_i8_plan(desc, True)[0] == 256
    c = torch.full((rows + 3, N), 55.0, device="cuda")
    op = ck.DeviceExpertsGemmI8("f32")
    arg = op.MakeArgumentPointer(a.cuda(), b.cuda(), c, sa.cuda(), sb.cuda(), None, offsets.cuda(), pick.cuda(), rows, R, E, N, K, K, K, N, N * K)
    op.MakeInvokerPointer().Run(arg, stream())
    torch.cuda.synchronize()
    c = c.cpu()
    assert bool((c[rows:] == 55).all())
    for e, (i, j) in enumerate([(0, 700), (700, 700), (700, 2000), (2000, 1900), (2000, 2500), (2500, 3000), (3000, 5000), (5000, 6000)]):
        if e in (2, 4) or i >= j:                    # (rows that two experts claim are either's)
            continue
        from_ = pick[i:j].long()
        there = (from_ >= 0) & (from_ < R)
        at = from_.clamp(0, R - 1)
        want, bound = ep.scaled(a[at] * there[:, None], b[e], sa[at] * there, sb[e], None, False, torch.float32)
        ep.near(c[i:j], want, bound, e)


def of_experts(g, counts, rows, E, N, K, R, wide, gated, gathered, tile):
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]).int()
    b, sb, bias = ep.codes(g, (E, wide, K)), (0.5 + torch.rand(E, wide, generator=g)) / 60 / K ** 0.5, ep.normal(g, (E, wide))
    pick = torch.randint(0, R * 2, (rows,), generator=g, dtype=torch.int32)
    a, sa = ep.codes(g, (R if gathered else rows, K)), (0.5 + torch.rand(R if gathered else rows, generator=g)) / 60
    c = torch.full((rows + 3, N), 55.0, dtype=torch.bfloat16, device="cuda")
    desc = capi.ExpertsDesc(rows, a.shape[0], E, N, K, K, K, N, 2 if gathered else 1, int(gated), capi.TYPE_BF16, 0, wide * K)
    p = capi.experts_gemm_i8_plan(desc, gathered)
    assert p[2] == 0 if tile == 0 else p[0] == tile and p[2] == 1, p
    op = ck.DeviceExpertsGemmI8("bf16", gated)
    arg = op.MakeArgumentPointer(strided(a, 0, 0), b.cuda(), c, sa.cuda(), sb.cuda(), bias.cuda(), offsets.cuda(), pick.cuda() if gathered else None, rows,
                                 a.shape[0], E, N, K, K, K, N, wide * K, 2 if gathered else 1)
    op.MakeInvokerPointer().Run(arg, stream())
    torch.cuda.synchronize()
    assert bool((c[rows:] == 55).all())
    for e in range(E):
        i, j = int(offsets[e]), int(offsets[e + 1])
        from_ = (pick[i:j] // 2).long() if gathered else torch.arange(i, j)
        ep.near(c[i:j].cpu(), *ep.scaled(a[from_], b[e], sa[from_], sb[e], bias[e], gated, torch.bfloat16), e)


@pytest.mark.parametrize("M,far", [(80, 1 << 26), (1100, 1 << 22)])
def test_rows_far_apart_and_a_far_matrix(M, far):
    """Offsets past 32 bits: rows of A 64 MB apart (the kernel for any call) or 4 MB (in order: a tile's rows lie within 2 GiB), an expert's B
    2 GiB behind the last."""
    N, K = 64, 128
    desc = capi.ExpertsDesc(M, M, 2, N, K, far, K, N, 1, 0, capi.TYPE_F32, 0, (1 << 31) + 4096)
    assert [capi.experts_gemm_i8_plan(desc, gathered)[2] for gathered in (True, False)] == [0, int(M > 80)]
    g = ep.gen(4)
    a, sa, sb = ep.codes(g, (M, K)), torch.rand(M, generator=g) / 60, torch.rand(2, N, generator=g) / 600
    big = torch.empty((M - 1) * far + K, dtype=torch.int8, device="cuda")
    ad = big.as_strided((M, K), (far, 1))
    ad.copy_(a)
    b = ep.codes(g, (2, N, K))
    bd = torch.empty((1 << 31) + 4096 + N * K, dtype=torch.int8, device="cuda").as_strided((2, N, K), ((1 << 31) + 4096, K, 1))
    bd.copy_(b)
    pick = torch.randperm(M, generator=g).int()
    offsets = torch.tensor([0, 30, M], dtype=torch.int32)
    for rows in (pick, None):
        c = torch.zeros(M, N, dtype=torch.float32, device="cuda")
        op = ck.DeviceExpertsGemmI8("f32")
        arg = op.MakeArgumentPointer(ad, bd, c, sa.cuda(), sb.cuda(), None, offsets.cuda(), None if rows is None else rows.cuda(), M, M, 2, N, K, far, K, N,
                                     (1 << 31) + 4096)
        assert op.IsSupportedArgument(arg), capi.last_error()
        op.MakeInvokerPointer().Run(arg, stream())
        torch.cuda.synchronize()
        for e, (i, j) in enumerate(((0, 30), (30, M))):
            from_ = torch.arange(i, j) if rows is None else pick[i:j].long()
            ep.near(c[i:j].cpu(), *ep.scaled(a[from_], b[e], sa[from_], sb[e], None, False, torch.float32), e)
