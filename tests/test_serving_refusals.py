"""What the 8-bit serving operators refuse, answered by pure host logic: no kernel is launched."""
import ctypes as C

import pytest

import composable_kernel_amd as ck
from composable_kernel_amd import capi

L = None


@pytest.fixture(autouse=True)
def _lib():
    global L
    L = capi.lib()


def cache(type_=capi.TYPE_E4M3, blocks=8, size=16, heads=2, dim=64, head=None, token=None, scale=None, block=None, p=4096):
    token = dim if token is None else token
    head = size * token if head is None else head
    return capi.KvCache8Desc(p, p, p, p, type_, blocks, size, heads, dim, head, token, heads if scale is None else scale,
                             heads * size * dim if block is None else block)


@pytest.mark.parametrize("args,want", [
    ((4, 256, 256, 256, 1, 4, capi.TYPE_BF16), capi.OK),
    ((0, 0, 0, 0, 0, 0, capi.TYPE_F32), capi.OK),
    ((1, 300, 0, 0, 0, 1, capi.TYPE_F16), capi.OK),
    ((-1, 256, 256, 256, 1, 4, capi.TYPE_BF16), capi.INVALID_VALUE),
    ((4, 256, 256, 256, 1, 4, capi.TYPE_E4M3), capi.INVALID_VALUE),
    ((4, 256, 255, 256, 1, 4, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((4, 256, 256, 255, 1, 4, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((4, 256, 256, 256, 1, 3, capi.TYPE_BF16), capi.UNSUPPORTED),     # two scales on one element
    ((4, 256, 256, 256, 0, 4, capi.TYPE_BF16), capi.UNSUPPORTED),
])
def test_quantize(args, want):
    assert L.ckx_quantize_blocks_f8_is_supported(*args) == want
    if want != capi.OK:
        assert L.ckx_quantize_blocks_f8(0, 0, 0, *args, None) == want and capi.last_error()


def test_quantize_pointers():
    ok = (4, 256, 256, 256, 1, 4, capi.TYPE_BF16)
    assert L.ckx_quantize_blocks_f8(0, 4096, 4096, *ok, None) == capi.INVALID_VALUE
    assert L.ckx_quantize_blocks_f8(4097, 4096, 4096, *ok, None) == capi.UNSUPPORTED
    assert L.ckx_quantize_blocks_f8(4096, 4096, 4098, *ok, None) == capi.UNSUPPORTED
    assert L.ckx_quantize_blocks_f8(0, 0, 0, 0, *ok[1:], None) == capi.OK      # nothing to do


@pytest.mark.parametrize("args,want", [
    ((4, 8, 256, 256, 256, 8, 1, 4, 2, 1, capi.TYPE_BF16), capi.OK),
    ((4, 8, 0, 0, 0, 8, 0, 0, 0, 0, capi.TYPE_BF16), capi.OK),
    ((4, 8, 256, 256, 256, 8, 1, 4, 2, 1, capi.TYPE_I8), capi.INVALID_VALUE),
    ((4, -8, 256, 256, 256, 8, 1, 4, 2, 1, capi.TYPE_BF16), capi.INVALID_VALUE),
    ((4, 8, 256, 255, 256, 8, 1, 4, 2, 1, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((4, 8, 256, 256, 255, 8, 1, 4, 2, 1, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((4, 8, 256, 256, 256, 7, 1, 4, 2, 1, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((4, 8, 256, 256, 256, 8, -1, 4, 2, 1, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((4, 8, 256, 1 << 24, 256, 8, 1, 4, 2, 1, capi.TYPE_BF16), capi.UNSUPPORTED),
])
def test_gemm(args, want):
    assert L.ckx_gemm_f8_blockscale_is_supported(*args) == want
    if want != capi.OK:
        assert L.ckx_gemm_f8_blockscale(0, 0, 0, 0, 0, *args, None, 0, None) == want and capi.last_error()


def test_gemm_pointers():
    ok = (4, 8, 256, 256, 256, 8, 1, 4, 2, 1, capi.TYPE_BF16)
    p = 4096
    for k in range(5):
        ptrs = [p] * 5
        ptrs[k] = 0
        assert L.ckx_gemm_f8_blockscale(*ptrs, *ok, None, 0, None) == capi.INVALID_VALUE
    assert L.ckx_gemm_f8_blockscale(p, p, p + 1, p, p, *ok, None, 0, None) == capi.UNSUPPORTED
    assert L.ckx_gemm_f8_blockscale(p, p, p, p + 2, p, *ok, None, 0, None) == capi.UNSUPPORTED
    assert L.ckx_gemm_f8_blockscale(p, p, p, p, p, *ok, p + 4, 64, None) == capi.INVALID_VALUE
    assert L.ckx_gemm_f8_blockscale(0, 0, 0, 0, 0, 0, *ok[1:], None, 0, None) == capi.OK


@pytest.mark.parametrize("args,want", [
    ((4, 16, 8, 8, 64, 16), capi.OK),
    ((0, 0, 0, 0, 0, 128), capi.OK),
    ((8192, 16, 8, 8, 64, 16), capi.OK),
    ((8193, 16, 8, 8, 64, 16), capi.UNSUPPORTED),
    ((4, 16, 8, 7, 64, 16), capi.UNSUPPORTED),
    ((4, 16, 8, 8, 64, 24), capi.UNSUPPORTED),
    ((4, -1, 8, 8, 64, 16), capi.INVALID_VALUE),
])
def test_tables(args, want):
    assert L.ckx_kv_cache_tables_is_supported(*args) == want
    if want != capi.OK:
        assert L.ckx_kv_cache_tables(*[4096] * 8, *args, None) == want and capi.last_error()


def test_tables_pointers():
    ok = (4, 16, 8, 8, 64, 16)
    p = [4096 * (i + 1) for i in range(8)]
    for k in range(8):
        assert L.ckx_kv_cache_tables(*[0 if i == k else x for i, x in enumerate(p)], *ok, None) == capi.INVALID_VALUE
        assert L.ckx_kv_cache_tables(*[x + 1 if i == k else x for i, x in enumerate(p)], *ok, None) == capi.UNSUPPORTED
    # the lengths are read by every workgroup while the new ones are written
    assert L.ckx_kv_cache_tables(*[p[0] if i == 5 else x for i, x in enumerate(p)], *ok, None) == capi.INVALID_VALUE
    assert L.ckx_kv_cache_tables(*[p[6] + 12 if i == 7 else x for i, x in enumerate(p)], *ok, None) == capi.INVALID_VALUE


BAD_CACHES = [
    (dict(type_=capi.TYPE_BF16), capi.INVALID_VALUE),
    (dict(blocks=-1), capi.INVALID_VALUE),
    (dict(size=24, head=1536), capi.UNSUPPORTED),
    (dict(size=256), capi.UNSUPPORTED),
    (dict(dim=72), capi.UNSUPPORTED),
    (dict(dim=144), capi.UNSUPPORTED),
    (dict(dim=0), capi.UNSUPPORTED),
    (dict(token=48), capi.UNSUPPORTED),
    (dict(token=72), capi.UNSUPPORTED),
    (dict(head=512), capi.UNSUPPORTED),              # heads on each other
    (dict(block=1024), capi.UNSUPPORTED),
    (dict(scale=1), capi.UNSUPPORTED),
    (dict(heads=1, token=1 << 27, head=0, block=1 << 32), capi.UNSUPPORTED),
    (dict(blocks=1 << 28), capi.UNSUPPORTED),        # slot numbers past 31 bits
]


@pytest.mark.parametrize("bad,want", BAD_CACHES)
def test_caches(bad, want):
    c = cache(**bad)
    assert L.ckx_kv_cache_store8_is_supported(C.byref(c), 4, 128, 64, 128, 64, capi.TYPE_BF16) == want
    assert L.ckx_paged_attention8_is_supported(C.byref(c), 2, 4, 4, 64, 4, 4, 256, 64, 256, 64, 0.125, 1, capi.TYPE_BF16) == want
    assert L.ckx_paged_attention8_workspace_bytes(C.byref(c), 2, 4, 4, 64, 4) == 0


def test_cache_layouts():
    for c in (cache(), cache(token=128, head=64), cache(heads=1, head=0), cache(token=80, head=1280, block=2560), cache(blocks=1, block=0, scale=0)):
        assert L.ckx_kv_cache_store8_is_supported(C.byref(c), 4, 128, 64, 128, 64, capi.TYPE_BF16) == capi.OK
    assert L.ckx_kv_cache_store8_is_supported(None, 4, 128, 64, 128, 64, capi.TYPE_BF16) == capi.INVALID_VALUE


@pytest.mark.parametrize("args,want", [
    ((4, 128, 64, 192, 64, capi.TYPE_F16), capi.OK),
    ((-4, 128, 64, 128, 64, capi.TYPE_F16), capi.INVALID_VALUE),
    ((4, 128, 64, 128, 64, capi.TYPE_F32), capi.INVALID_VALUE),
    ((4, 124, 60, 128, 64, capi.TYPE_F16), capi.UNSUPPORTED),
    ((4, 128, 64, 120, 64, capi.TYPE_F16), capi.UNSUPPORTED),
    ((4, 132, 64, 128, 64, capi.TYPE_F16), capi.UNSUPPORTED),
])
def test_store(args, want):
    c = cache()
    assert L.ckx_kv_cache_store8_is_supported(C.byref(c), *args) == want
    if want != capi.OK:
        assert L.ckx_kv_cache_store8(4096, 4096, 4096, C.byref(c), *args, None) == want


def test_store_pointers():
    args, c = (4, 128, 64, 128, 64, capi.TYPE_F16), cache()
    for k in range(3):
        p = [4096] * 3
        p[k] = 0
        assert L.ckx_kv_cache_store8(*p, C.byref(c), *args, None) == capi.INVALID_VALUE
    assert L.ckx_kv_cache_store8(4104, 4096, 4096, C.byref(c), *args, None) == capi.UNSUPPORTED
    bad = cache(p=0)
    assert L.ckx_kv_cache_store8(4096, 4096, 4096, C.byref(bad), *args, None) == capi.INVALID_VALUE
    bad = cache(p=4104)
    assert L.ckx_kv_cache_store8(4096, 4096, 4096, C.byref(bad), *args, None) == capi.UNSUPPORTED


GOOD = dict(batch=2, tokens=4, heads=4, kv=64, blocks=4, st=4, qt=256, qh=64, ot=256, oh=64, scale=0.125, causal=1, t=capi.TYPE_BF16)


@pytest.mark.parametrize("change,want", [
    ({}, capi.OK),
    (dict(batch=0, tokens=0), capi.OK),
    (dict(batch=-1), capi.INVALID_VALUE),
    (dict(kv=-1), capi.INVALID_VALUE),
    (dict(t=capi.TYPE_F32), capi.INVALID_VALUE),
    (dict(causal=2), capi.INVALID_VALUE),
    (dict(scale=float("nan")), capi.INVALID_VALUE),
    (dict(scale=float("inf")), capi.INVALID_VALUE),
    (dict(heads=3), capi.UNSUPPORTED),
    (dict(st=3), capi.UNSUPPORTED),
    (dict(qt=248), capi.UNSUPPORTED),
    (dict(oh=60), capi.UNSUPPORTED),
    (dict(blocks=1 << 28, st=1 << 28), capi.UNSUPPORTED),
    (dict(tokens=1 << 30, batch=1 << 20), capi.UNSUPPORTED),
])
def test_attention(change, want):
    c, a = cache(), {**GOOD, **change}
    assert L.ckx_paged_attention8_is_supported(C.byref(c), *a.values()) == want
    if want != capi.OK:
        assert L.ckx_paged_attention8(*[4096] * 5, C.byref(c), *a.values(), None, 0, None) == want and capi.last_error()


def test_attention_pointers_and_workspace():
    c, a = cache(), list(GOOD.values())
    for k in range(5):
        p = [4096] * 5
        p[k] = 0
        assert L.ckx_paged_attention8(*p, C.byref(c), *a, None, 0, None) == capi.INVALID_VALUE
    assert L.ckx_paged_attention8(4104, 4096, 4096, 4096, 4096, C.byref(c), *a, None, 0, None) == capi.UNSUPPORTED
    long = {**GOOD, "batch": 1, "tokens": 1, "kv": 8192, "blocks": 512, "st": 512}
    need = L.ckx_paged_attention8_workspace_bytes(C.byref(c), 1, 1, 4, 8192, 512)
    assert need > 0
    for p, n in ((0, need), (4096, need - 1)):
        assert L.ckx_paged_attention8(*[4096] * 5, C.byref(c), *long.values(), p, n, None) == capi.UNSUPPORTED
        assert "workspace" in capi.last_error()
    assert L.ckx_paged_attention8(*[4096] * 5, C.byref(c), *long.values(), 4100, need, None) == capi.INVALID_VALUE


def test_python_operators_check_types():
    import torch
    x = torch.zeros(4, 256)
    op = ck.DeviceBlockQuantizeF8("bf16")
    with pytest.raises(TypeError):
        op.MakeArgumentPointer(x, 0, 0, 4, 256, 256, 256, 1, 4)
    bad = op.MakeArgumentPointer(0, 0, 0, 4, 256, 8, 256, 1, 4)
    assert not op.IsSupportedArgument(bad)
    with pytest.raises(RuntimeError, match="DeviceBlockQuantizeF8"):
        op.MakeInvokerPointer().Run(bad)
    with pytest.raises(TypeError):
        ck.DeviceGemmBlockScaleF8.GetInstances()
    k = torch.zeros(4, 2, 16, 64, dtype=torch.int8)
    s = torch.ones(4, 2)
    assert ck.KvCache8(k, k.clone(), s, s.clone()).desc.type == capi.TYPE_I8
    with pytest.raises(TypeError):
        ck.KvCache8(k.float(), k.float(), s, s)
    with pytest.raises(ValueError):
        ck.KvCache8(k, k[:3], s, s)
    with pytest.raises(ValueError):
        ck.KvCache8(k, k, s, s[:, :1])


def test_python_operators_refuse_host_memory_and_wide_sizes():
    import torch
    x = torch.zeros(4, 256)
    q, scale = torch.zeros(4, 256, dtype=torch.float8_e4m3fn), torch.zeros(4, 2)
    op = ck.DeviceBlockQuantizeF8("f32")
    host = op.MakeArgumentPointer(x, q, scale, 4, 256, 256, 256, 2, 1)
    assert op.IsSupportedArgument(host)
    with pytest.raises(ValueError, match="one GPU"):
        op.MakeInvokerPointer().Run(host)
    mixed = op.MakeArgumentPointer(torch.zeros(4, 256, device="meta"), q, scale, 4, 256, 256, 256, 2, 1)
    with pytest.raises(ValueError, match="one GPU"):
        op.MakeInvokerPointer().Run(mixed)
    for wide in (2 ** 31, 2 ** 32 + 4, -2 ** 31 - 1):
        with pytest.raises(OverflowError):
            op.MakeArgumentPointer(0, 0, 0, wide, 256, 256, 256, 1, 4)
        with pytest.raises(OverflowError):
            ck.DeviceKvCacheTables().MakeArgumentPointer(*[0] * 8, 4, 8, 4, 4, wide, 16)


def test_largest_sizes():
    gemm = lambda M, N, K, lda=16, ldb=16, ldc=0: L.ckx_gemm_f8_blockscale_is_supported(M, N, K, lda, ldb, max(ldc, N), 1, M, 1, 1, capi.TYPE_BF16)
    assert gemm(1, 1, 1 << 30) == capi.OK and gemm(1, 1, (1 << 30) + 16) == capi.UNSUPPORTED
    assert gemm(1, (1 << 26) - 16, 16) == capi.OK and gemm(1, 1 << 26, 16) == capi.UNSUPPORTED
    assert gemm(1 << 28, 128, 16) == capi.OK and gemm(1 << 29, 128, 16) == capi.UNSUPPORTED
    c = cache()
    store = lambda n: L.ckx_kv_cache_store8_is_supported(C.byref(c), n, 128, 64, 128, 64, capi.TYPE_F16)
    assert store(1 << 29) == capi.OK and store((1 << 29) + 1) == capi.UNSUPPORTED
    attend = lambda **k: L.ckx_paged_attention8_is_supported(C.byref(c), *{**GOOD, **k}.values())
    most = 0x7fff0000 // 16
    assert attend(blocks=most, st=most) == capi.OK and attend(blocks=most + 1, st=most + 1) == capi.UNSUPPORTED
    assert L.ckx_paged_attention8_workspace_bytes(C.byref(c), 1, 1, 4, 1 << 20, most + 1) == 0
    assert attend(scale=3e38) == capi.INVALID_VALUE and attend(scale=2e38) == capi.OK


def test_cache_strides_past_32_bits_are_refused():
    """Heads (or scales) further apart than the descriptor's 32 bits say: cut to them, a kernel would read and write elsewhere."""
    import torch
    blank = lambda shape, strides, t: torch.empty_strided(shape, strides, dtype=t, device="meta")
    scale = blank((2, 2), (2, 1), torch.float32)
    codes = lambda head, token=64: blank((2, 2, 16, 64), (1 << 45, head, token, 1), torch.int8)
    for k in (codes((1 << 32) + 1024), codes(1 << 31), codes(1 << 40, (1 << 32) + 64)):
        with pytest.raises(OverflowError):
            ck.KvCache8(k, k, scale, scale)
    wide = blank((2, 2), ((1 << 32) + 2, 1), torch.float32)
    with pytest.raises(OverflowError):
        ck.KvCache8(codes(1024), codes(1024), wide, wide)
    far = ck.KvCache8(codes((1 << 31) - 16), codes((1 << 31) - 16), scale, scale)       # (blocks have 64 bits)
    assert far.desc.stride_head == (1 << 31) - 16 and far.desc.stride_block == 1 << 45
    one = blank((2, 1, 16, 64), (1 << 45, 1 << 40, 64, 1), torch.int8)                  # (a single head's stride is never used)
    assert L.ckx_kv_cache_store8_is_supported(C.byref(ck.KvCache8(one, one, scale[:, :1], scale[:, :1]).desc), 4, 64, 64, 64, 64,
                                              capi.TYPE_BF16) == capi.OK


def test_gemm_plan():
    plan = capi.gemm_f8_plan
    assert plan(1, 11008, 4096) == (16, 16, 1) and plan(32, 11008, 4096) == (32, 32, 1)
    assert plan(4096, 11008, 4096) == (256, 256, 1) and plan(4096, 11008, 4096, c_type=capi.TYPE_F32) == (128, 128, 1)
    assert plan(64, 4096, 8192)[2] == 1                                              # (runs of K need their workspace)
    need = L.ckx_gemm_f8_blockscale_workspace_bytes(64, 4096, 8192)
    tile, runs = plan(64, 4096, 8192, workspace_bytes=need)[:2], plan(64, 4096, 8192, workspace_bytes=need)[2]
    assert tile == (64, 128) and runs > 1 and need == 4 * 64 * 4096 * runs
    for odd in (dict(K=4097), dict(lda=4104), dict(ldb=4104)):
        assert plan(**{**dict(M=64, N=4096, K=4096), **odd}) == (128, 128, 0)
    assert plan(1, 4096, 4096, lda=0) == (16, 16, 1)                                  # (a single row's stride is never used)
    assert plan(0, 8, 16) == plan(8, 0, 16) == (0, 0, 0) and plan(8, 8, 0) == (128, 128, 0)
    for bad in (dict(M=-1), dict(c_type=capi.TYPE_I8), dict(lda=1), dict(workspace_bytes=-1)):
        with pytest.raises(capi.CkxError):
            plan(**{**dict(M=8, N=8, K=16), **bad})
    one = C.c_int(0)
    assert L.ckx_gemm_f8_blockscale_plan(8, 8, 16, 16, 16, 8, capi.TYPE_BF16, 0, C.byref(one), C.byref(one), None) == capi.INVALID_VALUE
