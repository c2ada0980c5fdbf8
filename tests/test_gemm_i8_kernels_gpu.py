"""Every kernel of DeviceGemmTokenScaleI8 and DeviceExpertsGemmI8 by its name, against the formula in 64 bits: sizes at which its tiles, its
stages and its runs of K end raggedly, and experts' rows around the borders of its tiles."""
import pytest
import torch

import composable_kernel_amd as ck
import experts_plain as ep
from composable_kernel_amd import capi
from test_gemm_i8_scaled_gpu import COUNTS, dense, experts, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,N,K,gated,kernel,runs", [
    (1, 1000, 8240, True, "direct16x16 eight waves", 1), (16, 333, 8720, False, "direct16x16 eight waves", 1),
    (49, 3647, 16, False, "direct32x32", 1), (17, 3782, 816, True, "direct32x32", 1),
    (137, 8, 160, False, "tile64x128", 1), (130, 9, 160, True, "tile64x128", 1), (17, 9, 9712, False, "tile64x128", 16), (18, 8, 10496, True, "tile64x128", 14),
    (777, 2744, 2064, False, "tile128x128", 1), (1604, 1153, 1616, False, "tile128x128", 1), (325, 2723, 1568, True, "tile128x128", 1),
    (68, 5733, 14512, False, "tile128x128", 5), (70, 2744, 13248, True, "tile128x128", 5),
    (131, 8, 16, False, "tile128x128 two a CU", 1), (133, 9, 16, True, "tile128x128 two a CU", 1),
    (132, 8, 3984, False, "tile128x128 two a CU", 16), (133, 8, 3776, True, "tile128x128 two a CU", 15),
    (2312, 5658, 48, False, "tile256x256", 1), (1349, 4436, 16, True, "tile256x256", 1),
    (16, 100, 4100, True, "any16x16", 0), (200, 130, 333, True, "any128x128", 0)])
def test_dense(kind, M, N, K, gated, kernel, runs):
    need = capi.lib().ckx_gemm_i8_tokenscale_workspace_bytes(M, N, K, int(gated))
    assert capi.gemm_i8_kernel(M, N, K, gated=gated, workspace_bytes=need) == kernel
    assert capi.gemm_i8_plan(M, N, K, gated=gated, workspace_bytes=need)[2] == runs
    dense(M, N, K, kind, gated, True)


# sizes at which some number of rows leads to the kernel
SIZES = {"tile64x128": [(1030, 400), (300, 272)], "tile64x128 two a CU": [(2100, 1040), (300, 272)], "tile128x128 two a CU": [(1030, 400), (300, 272)],
         "tile256x256": [(2100, 272), (1030, 400), (2100, 1040)]}


def sizes_for(kernel, counts, kind, gated, gather):
    """N, K, and rows of C behind the experts' (the plan knows their number alone) with which the kernel is the one that is taken."""
    E, P, per = len(counts), sum(counts), gather or 1
    for N, K in SIZES[kernel]:
        for rows in (3, 20, 50, 100, 200, 400, 700, 1000, 1500, 2000, 3000, 4000, 6000, 10000, 20000, 40000):
            rows_a = max(1, -(-P // per)) if gather else P + rows
            c_type = {"bf16": capi.TYPE_BF16, "f16": capi.TYPE_F16, "f32": capi.TYPE_F32}[kind]
            desc = capi.ExpertsDesc(P + rows, rows_a, E, N, K, K, K, N, per, int(gated), c_type, 0, N * (1 + gated) * K)
            if capi.experts_gemm_i8_kernel(desc, gather is not None) == kernel:
                return N, K, rows
    raise AssertionError((kernel, counts))


FEW = [c + [0] * (8 - len(c)) for c in COUNTS if len(c) <= 8]
MANY = [[0] * 70 + [300, 0, 5, 64, 63, 0, 256, 257] + [0] * 22, [1] * 64 + [130] + [2] * 64 + [0, 500], [2] * 70]


@pytest.mark.parametrize("kind,gated,gather", [("bf16", True, 2), ("bf16", False, None), ("f32", True, None), ("f32", False, 4), ("f16", True, 3)])
@pytest.mark.parametrize("counts", FEW, ids=lambda c: "_".join(map(str, c[:6])))
@pytest.mark.parametrize("kernel", sorted(SIZES))
def test_experts(kernel, counts, kind, gated, gather):
    N, K, spare = sizes_for(kernel, counts, kind, gated, gather)
    experts(counts, N, K, kind, gated, gather, counts[0] == 300, spare)


@pytest.mark.parametrize("kind,gated,gather", [("bf16", True, 2), ("f32", False, None), ("f16", False, 4)])
@pytest.mark.parametrize("counts", MANY, ids=lambda c: f"{len(c)}")
@pytest.mark.parametrize("kernel", sorted(set(SIZES) - {"tile64x128"}))
def test_more_experts_than_lanes(kernel, counts, kind, gated, gather):
    N, K, spare = sizes_for(kernel, counts, kind, gated, gather)
    experts(counts, N, K, kind, gated, gather, True, spare)


@pytest.mark.parametrize("kernel", sorted(SIZES))
@pytest.mark.parametrize("gated", [False, True])
def test_rows_outside_a(kernel, gated):
    counts = [5, 7, 200, 0, 0, 130, 0, 1]
    N, K, spare = sizes_for(kernel, counts, "f32", gated, 2)
    experts(counts, N, K, "f32", gated, 2, True, spare, bad_rows=(0, 4, 5, 11, 100, 212, 342))


@pytest.mark.parametrize("E,P,N,K,kernel,offsets", [
    (3, 12, 64, 128, "direct16x16", [5, 5, 1000, 1000]), (3, 12, 64, 128, "direct16x16", [-7, 3, 3, 6]), (3, 12, 64, 128, "direct16x16", [12, 12, 12, 12]),
    (3, 700, 1030, 400, "tile64x128", [-100, 65, 65, 2 ** 31 - 1]), (3, 700, 1030, 400, "tile64x128", [70, 70, 300, 301]),
    (8, 720, 2100, 1040, "tile64x128 two a CU", [-2 ** 31, -1, 0, 1, 66, 66, 500, 699, 900]),
    (3, 3000, 1030, 400, "tile128x128 two a CU", [129, 1000, 1000, 5000]), (3, 3000, 1030, 400, "tile128x128 two a CU", [-3, -2, -1, 0]),
    (3, 7000, 2100, 272, "tile256x256", [257, 600, 1113, 9000]), (3, 7000, 2100, 272, "tile256x256", [7000, 7000, 7001, 8000])])
def test_offsets_past_the_rows(E, P, N, K, kernel, offsets):
    """Offsets that ascend but leave C: cut, and what they leave is each expert's; rows of none stay as they are."""
    g = ep.gen(P + offsets[1])
    a, b, sa, sb = ep.codes(g, (P, K)), ep.codes(g, (E, N, K)), torch.rand(P, generator=g), torch.rand(E, N, generator=g) / 100
    desc = capi.ExpertsDesc(P, P, E, N, K, K, K, N, 1, 0, capi.TYPE_F32, 0, N * K)
    assert capi.experts_gemm_i8_kernel(desc, False) == kernel
    c = torch.full((P + 8, N), 55.0, device="cuda")
    op = ck.DeviceExpertsGemmI8("f32")
    arg = op.MakeArgumentPointer(a.cuda(), b.cuda(), c, sa.cuda(), sb.cuda(), None, torch.tensor(offsets, dtype=torch.int32).cuda(), None, P, P, E, N, K, K, K, N,
                                 N * K)
    op.MakeInvokerPointer().Run(arg, stream())
    torch.cuda.synchronize()
    c, cut = c.cpu(), [max(0, min(P, o)) for o in offsets]
    for e, (i, j) in enumerate(zip(cut, cut[1:])):
        ep.near(c[i:j], *ep.scaled(a[i:j], b[e], sa[i:j], sb[e], None, False, torch.float32), e)
    assert bool((c[:cut[0]] == 55).all()) and bool((c[cut[-1]:] == 55).all())


@pytest.mark.parametrize("M,N,K,gated", [(130, 128, 16384, False), (70, 2744, 13248, True), (133, 8, 3776, True)])
def test_less_workspace_takes_fewer_runs(M, N, K, gated):
    wide = N * (1 + gated)
    need = capi.lib().ckx_gemm_i8_tokenscale_workspace_bytes(M, N, K, int(gated))
    g = ep.gen(N)
    a, b, sa, sb = ep.codes(g, (M, K)), ep.codes(g, (wide, K)), torch.rand(M, generator=g), torch.rand(wide, generator=g) / K
    want, bound = ep.scaled(a, b, sa, sb, None, gated, torch.float32)
    runs = []
    for there in (need, need - 4, need // 2, 4 * M * wide * 2, 4 * M * wide * 2 - 4, 16, 0):
        runs.append(capi.gemm_i8_plan(M, N, K, gated=gated, workspace_bytes=there, c_type=capi.TYPE_F32)[2])
        ws = torch.full((need + 256,), 0x7D, dtype=torch.uint8, device="cuda")
        c = torch.full((M, N), 55.0, device="cuda")
        op = ck.DeviceGemmTokenScaleI8("f32", Gated=gated)
        arg = op.MakeArgumentPointer(a.cuda(), b.cuda(), c, sa.cuda(), sb.cuda(), None, M, N, K, K, K, N)
        op.SetWorkSpacePointer(arg, ws, there)
        op.MakeInvokerPointer().Run(arg, stream())
        torch.cuda.synchronize()
        ep.near(c.cpu(), want, bound, there)
        assert bool((ws[there:] == 0x7D).all()), there
    assert runs[0] > runs[1] and runs[-1] == 1 and sorted(runs, reverse=True) == runs
