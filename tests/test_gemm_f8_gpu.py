"""DeviceGemmBlockScaleF8 against the product in 64 bits. Bound per element: half a step of C's type, and for the fp32 sums
(128 products and one multiply-add a group, the product of the two scales) 2^-23 of the sum of magnitudes for each of the
128 + groups + 4 roundings on the way of a summand; with 16-bit outputs also what the 8-bit matrix instruction cuts
(serving_plain.gemm)."""
import pytest
import torch

import composable_kernel_amd as ck
import serving_plain as sp

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def operands(M, N, K, seed):
    g = sp.gen(seed)
    groups = -(-K // 128)
    code = lambda shape: sp.normal(g, shape, scale=100.0).clamp(-448, 448).to(torch.float8_e4m3fn)
    return (code((M, K)), code((N, K)), (0.2 + torch.rand(M, groups, generator=g)) / 100,
            (0.2 + torch.rand(-(-N // 128), groups, generator=g)) / 100)


def run(a, b, sa, sb, out, pads=(0, 0, 0), offset=0, sa_m_fast=True, sb_n_fast=False, workspace=True):
    (M, K), N = a.shape, b.shape[0]

    def place(x, pad, fill):
        flat = torch.full((x.shape[0] * (x.shape[1] + pad) + offset,), fill, device="cuda").to(x.dtype)
        view = flat[offset:].view(x.shape[0], x.shape[1] + pad)
        view[:, :x.shape[1]] = x.cuda()
        return view
    # (what lies behind a row's K columns is NaN: no kernel may let it into a sum)
    da, db = place(a, pads[0], float("nan")), place(b, pads[1], float("nan"))
    ldc = N + pads[2]
    c = torch.full((M, ldc), 3.0, device="cuda", dtype=DT[out])
    dsa = (sa.t() if sa_m_fast else sa).contiguous().cuda()
    dsb = (sb.t() if sb_n_fast else sb).contiguous().cuda()
    op = ck.DeviceGemmBlockScaleF8(out)
    arg = op.MakeArgumentPointer(da.data_ptr(), db.data_ptr(), c, dsa, dsb, M, N, K, K + pads[0], K + pads[1], ldc,
                                 (1, M) if sa_m_fast else (sa.shape[1], 1), (1, sb.shape[0]) if sb_n_fast else (sb.shape[1], 1))
    assert op.IsSupportedArgument(arg), ck.capi.last_error()
    need = op.GetWorkSpaceSize(arg) if workspace else 0
    if need:
        op.SetWorkSpacePointer(arg, torch.full((need,), 0x7F, device="cuda", dtype=torch.uint8))
    op.MakeInvokerPointer().Run(arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    c = c.cpu()
    assert bool((c[:, N:] == 3).all()), "wrote behind the row"
    return c[:, :N]


def check(M, N, K, out="bf16", seed=None, **kw):
    a, b, sa, sb = operands(M, N, K, seed if seed is not None else M * 31 + N * 17 + K)
    got = run(a, b, sa, sb, out, **kw).double()
    want, mag, cut = sp.gemm(a, b, sa, sb)
    sums = (128 + sa.shape[1] + 4) * 2.0 ** -23 * mag + (0 if out == "f32" else cut)
    bound = sums + sp.HALF_STEP[DT[out]] * (want.abs() + sums) + 1e-30
    worst = ((got - want).abs() / bound).max()
    assert bool(((got - want).abs() <= bound).all()), (M, N, K, out, float(worst))


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 64, 65, 127, 128, 200])
@pytest.mark.parametrize("N,K", [(16, 128), (130, 256), (257, 400)])
def test_rows(M, N, K):
    check(M, N, K)


@pytest.mark.parametrize("N", [1, 15, 127, 128, 129, 255, 256, 300])
def test_columns(N):
    check(5, N, 272)
    check(140, N, 272, "f32")


@pytest.mark.parametrize("K", [16, 112, 128, 144, 1040, 2048, 4096, 11008])
def test_long_sums(K):
    check(3, 96, K, "f32")
    check(40, 160, K, "f16")


@pytest.mark.parametrize("M,N,K", [(256, 256, 512), (257, 511, 640), (600, 300, 1024), (1025, 130, 144), (300, 2049, 384), (2001, 1003, 1040)])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_tiles(M, N, K, out):
    check(M, N, K, out)


@pytest.mark.parametrize("M", [1, 30, 150])
@pytest.mark.parametrize("K,pads,offset", [(100, (0, 0, 0), 0), (129, (0, 0, 1), 0), (256, (1, 0, 0), 0), (256, (0, 5, 3), 0),
                                           (256, (16, 32, 8), 0), (256, (0, 0, 0), 1), (7, (0, 0, 0), 0), (1, (0, 0, 0), 0),
                                           (1000, (8, 8, 0), 0)])
def test_any_extent_stride_and_address(M, K, pads, offset):
    check(M, 70, K, pads=pads, offset=offset)


@pytest.mark.parametrize("sa_m_fast", [True, False])
@pytest.mark.parametrize("sb_n_fast", [True, False])
@pytest.mark.parametrize("M", [4, 70, 300])
def test_scale_strides(M, sa_m_fast, sb_n_fast):
    check(M, 390, 640, sa_m_fast=sa_m_fast, sb_n_fast=sb_n_fast)


@pytest.mark.parametrize("M,N,K", [(1, 64, 8192), (16, 128, 11008), (64, 200, 4096), (130, 128, 8192)])
def test_with_and_without_the_workspace(M, N, K):
    check(M, N, K, "f32", workspace=True)
    check(M, N, K, "f32", workspace=False)


def test_no_columns_to_sum_over():
    c = torch.full((3, 5), 2.0, device="cuda", dtype=torch.bfloat16)
    op = ck.DeviceGemmBlockScaleF8("bf16")
    op.MakeInvokerPointer().Run(op.MakeArgumentPointer(0, 0, c, 0, 0, 3, 5, 0, 0, 0, 5, (1, 3), (0, 1)),
                                ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert bool((c == 0).all())


def test_nan_and_infinite_scales_reach_their_rows_only():
    a, b, sa, sb = operands(150, 140, 384, 77)
    a[3, 130] = float("nan")
    sa[60, 1] = float("inf")
    c = run(a, b, sa, sb, "f32")
    assert bool(c[3].isnan().all())
    assert not bool(c[60].isfinite().any())
    rest = [i for i in range(150) if i not in (3, 60)]
    assert bool(c[rest].isfinite().all())


def test_exact_sums_come_out_exactly():
    # small whole numbers, scales powers of two: every partial sum is exact in fp32, whatever its order
    g = sp.gen(3)
    for M, N, K in ((5, 40, 1024), (70, 130, 512), (300, 260, 640)):
        a = torch.randint(-3, 4, (M, K), generator=g).float().to(torch.float8_e4m3fn)
        b = torch.randint(-3, 4, (N, K), generator=g).float().to(torch.float8_e4m3fn)
        groups = -(-K // 128)
        sa = torch.exp2(torch.randint(-2, 3, (M, groups), generator=g).float())
        sb = torch.exp2(torch.randint(-2, 3, (-(-N // 128), groups), generator=g).float())
        want = sp.gemm(a, b, sa, sb)[0]
        assert torch.equal(run(a, b, sa, sb, "f32").double(), want)
        # (products within 2^-4 ... 9 of each other: nothing lies under the 8-bit instruction's grid either)
        assert torch.equal(run(a, b, sa, sb, "bf16"), want.to(torch.bfloat16))


@pytest.mark.parametrize("M,K", [(5, 256), (20, 256), (100, 512), (70, 264)])
def test_products_that_cancel(M, K):
    """Eights of +P, -P and six products of 1, scales 1. fp32 outputs: exactly 6 an eight. 16-bit outputs: the same where 1 lies on the
    grid (P = 64: 2^-7); for P = 448^2 (16) each 1 is lost, less than 2^-13 P."""
    ones = lambda n: torch.ones(n, -(-K // 128))
    for p in (8.0, 448.0):
        a, b = torch.ones(M, K), torch.ones(40, K)
        a[:, ::8], a[:, 1::8], b[:, ::8], b[:, 1::8] = p, p, p, -p
        a, b = a.to(torch.float8_e4m3fn), b.to(torch.float8_e4m3fn)
        want = 6.0 * (K // 8)
        assert bool((run(a, b, ones(M), ones(1), "f32") == want).all())
        for out in ("bf16", "f16"):
            got = run(a, b, ones(M), ones(1), out).float()
            rounded = float(torch.tensor(want).to(DT[out]))
            assert bool((got == rounded).all() if p == 8.0 else ((got >= 0) & (got <= rounded)).all()), (p, out, got.unique())


def check_norm(M, N, K, out):
    """The 2-norm of the error, over outputs of normal operands: half a step of each output, fp32's roundings as in check, and of the
    cut products the root of their squares' sum (seven of an eight by less than 2^-13 of its largest; a cut goes towards zero, so that its sign is
    the product's own, and these are independent)."""
    a, b, sa, sb = operands(M, N, K, M + N + K)
    got = run(a, b, sa, sb, out).double()
    want, mag, _ = sp.gemm(a, b, sa, sb)
    wide = lambda x, s: (x.double() * s)[:, :K // 8 * 8].view(x.shape[0], -1, 8).abs().amax(dim=2) ** 2
    cut = 7 * 2.0 ** -26 * (wide(a, sa.repeat_interleave(128, dim=1)[:, :K]) @
                            wide(b, sb.repeat_interleave(128, dim=1)[:, :K].repeat_interleave(128, dim=0)[:N]).t())
    bound = sp.HALF_STEP[DT[out]] * want.norm() + (128 + sa.shape[1] + 4) * 2.0 ** -23 * mag.norm()
    if out != "f32":
        bound += cut.sum().sqrt()
    assert float((got - want).norm()) <= float(bound), (float((got - want).norm() / want.norm()), float(bound / want.norm()))


@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [(9, 700, 1024), (30, 300, 512), (200, 300, 512), (40, 200, 2048), (100, 200, 1000)])
def test_error_in_the_2_norm(M, N, K, out):
    check_norm(M, N, K, out)


@pytest.mark.parametrize("out", ["f16", "bf16"])
@pytest.mark.parametrize("M", [6, 30, 150])
def test_nan_and_infinite_scales_in_16_bit_outputs(M, out):
    a, b, sa, sb = operands(M, 140, 384, 78)
    a[3, 130] = float("nan")
    sa[5, 1] = float("inf")
    c = run(a, b, sa, sb, out)
    assert bool(c[3].isnan().all()) and not bool(c[5].isfinite().any())
    rest = [i for i in range(M) if i not in (3, 5)]
    assert bool(c[rest].isfinite().all())


def on(tile, M, N, K, out, runs=1, workspace=1 << 40):
    """This problem runs on that tile (the plan of 16-byte aligned operands)."""
    types = {"f32": ck.capi.TYPE_F32, "f16": ck.capi.TYPE_F16, "bf16": ck.capi.TYPE_BF16}
    got = ck.capi.gemm_f8_plan(M, N, K, c_type=types[out], workspace_bytes=workspace)
    assert got[:2] == tile and (got[2] == runs or runs is None and got[2] > 1), got


@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,N,K,tile", [
    (1, 300, 400, (16, 16)), (16, 130, 272, (16, 16)), (17, 200, 1040, (32, 32)), (32, 47, 144, (32, 32)),
    (33, 300, 400, (64, 128)), (2001, 1003, 1040, (64, 128)),
    (1025, 2100, 512, (128, 128)), (2049, 1300, 400, (128, 128)), (1153, 1922, 144, (128, 128)),    # one row, two columns in the last tiles
    (1300, 2049, 128, (128, 128)), (9001, 1100, 16, (128, 128))])                                   # a single group, of 16 columns
def test_every_kernel(M, N, K, tile, out):
    on(tile, M, N, K, out)
    check(M, N, K, out)


@pytest.mark.parametrize("out", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(3841, 3844, 144), (3900, 3300, 400), (4000, 3960, 272), (3970, 3970, 16)])
def test_the_largest_tile(M, N, K, out):
    """256 x 256, with one row, four columns, and no column of the right half (so no scale of its block either) in the last tiles."""
    on((256, 256), M, N, K, out)
    check(M, N, K, out)


@pytest.mark.parametrize("M,N,K", [(64, 200, 4096), (130, 128, 8192), (70, 390, 2064), (33, 4096, 11008)])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_runs_of_k(M, N, K, out):
    on((64, 128), M, N, K, out, runs=None)
    check(M, N, K, out)
    on((64, 128), M, N, K, out, workspace=0)


@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("M,N,tile", [(1025, 2100, (128, 128)), (3841, 3844, (256, 256))])
def test_large_tiles_exactly(M, N, tile, out):
    """Small whole numbers, scales powers of two: every sum is exact, whatever the order; twice the same bits; rows with a NaN or an infinite
    scale keep it to themselves; the scales' other strides."""
    if out == "f32" and tile == (256, 256):
        tile = (128, 128)
    K, g = 400, sp.gen(M + N)
    on(tile, M, N, K, out)
    a, b = (torch.randint(-3, 4, (n, K), generator=g).float().to(torch.float8_e4m3fn) for n in (M, N))
    sa, sb = (torch.exp2(torch.randint(-2, 3, (n, 4), generator=g).float()) for n in (M, -(-N // 128)))
    want = sp.gemm(a, b, sa, sb)[0].to(DT[out])
    got = run(a, b, sa, sb, out)
    assert torch.equal(got, want) and torch.equal(run(a, b, sa, sb, out, sa_m_fast=False, sb_n_fast=True, pads=(16, 32, 3)), want)
    a[M - 1, 130], sa[700, 1] = float("nan"), float("inf")
    got = run(a, b, sa, sb, out)
    assert bool(got[M - 1].isnan().all()) and not bool(got[700].isfinite().any())
    rest = torch.ones(M, dtype=torch.bool)
    rest[[M - 1, 700]] = False
    assert torch.equal(got[rest], want[rest])


@pytest.mark.parametrize("M,N,K,out", [(1025, 2100, 512, "f16"), (1025, 2100, 512, "f32"), (3900, 3300, 400, "f16"), (3900, 3300, 400, "bf16")])
def test_error_of_large_tiles_in_the_2_norm(M, N, K, out):
    check_norm(M, N, K, out)
