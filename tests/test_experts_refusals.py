"""What the int8 linear and mixture-of-experts operators refuse, answered by pure host logic: no kernel is launched."""
import ctypes as C

import pytest

import composable_kernel_amd as ck
from composable_kernel_amd import capi

L = None
P = 1 << 20


@pytest.fixture(autouse=True)
def _lib():
    global L
    L = capi.lib()


def route(tokens=64, experts=16, top_k=2, stride=None, groups=1, top_groups=1, best=1, scoring=capi.SCORE_SOFTMAX, renormalise=1,
          x_type=capi.TYPE_F32, scale=1.0):
    return capi.RouteDesc(tokens, experts, top_k, experts if stride is None else stride, groups, top_groups, best, scoring, renormalise, x_type, scale)


@pytest.mark.parametrize("desc,want", [
    (route(), capi.OK),
    (route(tokens=0), capi.OK),
    (route(tokens=1, stride=0), capi.OK),
    (route(experts=1024, top_k=32), capi.OK),
    (route(experts=64, groups=64, top_groups=64, best=2), capi.OK),
    (route(tokens=1 << 24, top_k=1), capi.OK),
    (route(tokens=-1), capi.INVALID_VALUE),
    (route(top_k=-1), capi.INVALID_VALUE),
    (route(x_type=capi.TYPE_I8), capi.INVALID_VALUE),
    (route(scoring=2), capi.INVALID_VALUE),
    (route(renormalise=2), capi.INVALID_VALUE),
    (route(scale=float("nan")), capi.INVALID_VALUE),
    (route(scale=float("inf")), capi.INVALID_VALUE),
    (route(best=0), capi.INVALID_VALUE),
    (route(best=3), capi.INVALID_VALUE),
    (route(experts=0, top_k=0), capi.UNSUPPORTED),
    (route(experts=1025), capi.UNSUPPORTED),
    (route(top_k=0), capi.UNSUPPORTED),
    (route(top_k=17), capi.UNSUPPORTED),
    (route(experts=64, top_k=33), capi.UNSUPPORTED),
    (route(groups=3), capi.UNSUPPORTED),
    (route(groups=0), capi.UNSUPPORTED),
    (route(experts=130, groups=65), capi.UNSUPPORTED),
    (route(groups=4, top_groups=5), capi.UNSUPPORTED),
    (route(groups=4, top_groups=0), capi.UNSUPPORTED),
    (route(tokens=(1 << 23) + 1), capi.UNSUPPORTED),
    (route(stride=15), capi.UNSUPPORTED),
    (route(tokens=1, stride=-1), capi.UNSUPPORTED),
])
def test_route(desc, want):
    assert L.ckx_route_experts_is_supported(C.byref(desc)) == want
    if want != capi.OK:
        ptrs = [P * (i + 1) for i in range(8)]
        assert L.ckx_route_experts(*ptrs, C.byref(desc), 0, 0, None) == want and capi.last_error()
        assert L.ckx_route_experts_workspace_bytes(C.byref(desc)) == 0


def test_route_pointers():
    d = route()
    need = L.ckx_route_experts_workspace_bytes(C.byref(d))
    ok = [P * (i + 1) for i in range(8)]  # logits, bias, number, ids, weights, offsets, rows, places
    ws = (P * 9, need) if need else (0, 0)

    def call(change, ws=ws, d=d):
        return L.ckx_route_experts(*[change.get(i, p) for i, p in enumerate(ok)], C.byref(d), *ws, None)

    for i in (0, 3, 4, 5, 6, 7):
        assert call({i: 0}) == capi.INVALID_VALUE, i
    for i in range(8):
        assert call({i: ok[i] + 2}) == capi.UNSUPPORTED, i
    # an output on an input, two outputs on each other
    assert call({3: ok[0] + 64 * 16 * 4 - 4}) == capi.INVALID_VALUE
    assert call({7: ok[1] + 15 * 4}) == capi.INVALID_VALUE
    assert call({5: ok[2] - 16 * 4}) == capi.INVALID_VALUE
    assert call({4: ok[3] + 64 * 2 * 4 - 4}) == capi.INVALID_VALUE
    assert call({7: ok[6]}) == capi.INVALID_VALUE
    # nothing to do
    assert L.ckx_route_experts(*[0] * 8, C.byref(route(tokens=0)), 0, 0, None) == capi.OK
    assert L.ckx_route_experts(*ok, None, 0, 0, None) == capi.INVALID_VALUE
    many = route(tokens=5000)
    need = L.ckx_route_experts_workspace_bytes(C.byref(many))
    assert need > 0
    assert call({}, (0, 0), many) == capi.UNSUPPORTED and call({}, (P * 9, need - 1), many) == capi.UNSUPPORTED
    assert call({}, (P * 9 + 8, need), many) == capi.INVALID_VALUE


@pytest.mark.parametrize("args,want", [
    ((4, 256, 256, 256, capi.TYPE_BF16), capi.OK),
    ((0, 0, 0, 0, capi.TYPE_F32), capi.OK),
    ((1, 300, 0, 0, capi.TYPE_F16), capi.OK),
    ((-1, 256, 256, 256, capi.TYPE_BF16), capi.INVALID_VALUE),
    ((4, -256, 256, 256, capi.TYPE_BF16), capi.INVALID_VALUE),
    ((4, 256, 256, 256, capi.TYPE_I8), capi.INVALID_VALUE),
    ((4, 256, 255, 256, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((4, 256, 256, 255, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((1, 256, -1, 256, capi.TYPE_BF16), capi.UNSUPPORTED),
])
def test_quantize(args, want):
    assert L.ckx_quantize_tokens_i8_is_supported(*args) == want
    if want != capi.OK:
        assert L.ckx_quantize_tokens_i8(P, P, P, *args, None) == want and capi.last_error()


def test_quantize_pointers():
    ok = (4, 256, 256, 256, capi.TYPE_BF16)
    for i in range(3):
        assert L.ckx_quantize_tokens_i8(*[0 if j == i else P for j in range(3)], *ok, None) == capi.INVALID_VALUE
    assert L.ckx_quantize_tokens_i8(P + 1, P, P, *ok, None) == capi.UNSUPPORTED
    assert L.ckx_quantize_tokens_i8(P, P, P + 2, *ok, None) == capi.UNSUPPORTED
    assert L.ckx_quantize_tokens_i8(0, 0, 0, 0, *ok[1:], None) == capi.OK


MOST = 131071


@pytest.mark.parametrize("args,want", [
    ((4, 8, 256, 256, 256, 8, 0, capi.TYPE_BF16), capi.OK),
    ((4, 8, 0, 0, 0, 8, 1, capi.TYPE_F32), capi.OK),
    ((1, 1, MOST, 0, 0, 0, 0, capi.TYPE_F16), capi.OK),
    ((0, 0, 0, 0, 0, 0, 0, capi.TYPE_F16), capi.OK),
    ((1 << 22, 128, 16, 16, 16, 128, 0, capi.TYPE_F16), capi.OK),
    ((-4, 8, 256, 256, 256, 8, 0, capi.TYPE_BF16), capi.INVALID_VALUE),
    ((4, -8, 256, 256, 256, 8, 0, capi.TYPE_BF16), capi.INVALID_VALUE),
    ((4, 8, -1, 256, 256, 8, 0, capi.TYPE_BF16), capi.INVALID_VALUE),
    ((4, 8, 256, 256, 256, 8, 2, capi.TYPE_BF16), capi.INVALID_VALUE),
    ((4, 8, 256, 256, 256, 8, 0, capi.TYPE_E4M3), capi.INVALID_VALUE),
    ((4, 8, MOST + 1, MOST + 1, MOST + 1, 8, 0, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((4, 8, 256, 255, 256, 8, 0, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((4, 8, 256, 256, 255, 8, 0, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((4, 1, 256, 256, 255, 8, 1, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((4, 8, 256, 256, 256, 7, 0, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((1, 8, 256, -1, 256, 8, 0, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((1, 8, 256, 256, 256, -8, 0, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((4, 0x40000000, 16, 16, 16, 0x40000000, 1, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((0x7fffffff, 8192, 16, 16, 16, 8192, 0, capi.TYPE_BF16), capi.UNSUPPORTED),
])
def test_gemm(args, want):
    assert L.ckx_gemm_i8_tokenscale_is_supported(*args) == want
    if want != capi.OK:
        assert L.ckx_gemm_i8_tokenscale(*[P] * 6, *args, None, 0, None) == want and capi.last_error()


def test_gemm_pointers():
    ok = (4, 8, 256, 256, 256, 8, 0, capi.TYPE_BF16)
    for i in range(5):                                # (the bias may be null)
        assert L.ckx_gemm_i8_tokenscale(*[0 if j == i else P for j in range(6)], *ok, None, 0, None) == capi.INVALID_VALUE
    for i in (2, 3, 4, 5):
        assert L.ckx_gemm_i8_tokenscale(*[P + 1 if j == i else P for j in range(6)], *ok, None, 0, None) == capi.UNSUPPORTED
    assert L.ckx_gemm_i8_tokenscale(*[P] * 6, *ok, P + 4, 64, None) == capi.INVALID_VALUE
    assert L.ckx_gemm_i8_tokenscale(*[P] * 6, *ok, P, -1, None) == capi.INVALID_VALUE
    assert L.ckx_gemm_i8_tokenscale(*[0] * 6, 0, *ok[1:], None, 0, None) == capi.OK


def experts(rows=64, rows_a=32, experts=8, N=96, K=128, a=None, b=None, c=None, per=2, gated=0, c_type=capi.TYPE_BF16, batch=None):
    return capi.ExpertsDesc(rows, rows_a, experts, N, K, K if a is None else a, K if b is None else b, N if c is None else c, per, gated, c_type, 0,
                            N * K if batch is None else batch)


@pytest.mark.parametrize("desc,want", [
    (experts(), capi.OK),
    (experts(rows=0), capi.OK),
    (experts(experts=0), capi.OK),
    (experts(K=0), capi.OK),
    (experts(batch=0), capi.OK),                     # every expert the same matrix
    (experts(rows=1 << 24, experts=1024), capi.OK),
    (experts(rows=-1), capi.INVALID_VALUE),
    (experts(rows_a=-1), capi.INVALID_VALUE),
    (experts(experts=-1), capi.INVALID_VALUE),
    (experts(N=-1), capi.INVALID_VALUE),
    (experts(per=0), capi.INVALID_VALUE),
    (experts(gated=3), capi.INVALID_VALUE),
    (experts(c_type=capi.TYPE_I8), capi.INVALID_VALUE),
    (experts(K=MOST + 1), capi.UNSUPPORTED),
    (experts(experts=1025), capi.UNSUPPORTED),
    (experts(rows=(1 << 24) + 1), capi.UNSUPPORTED),
    (experts(a=127), capi.UNSUPPORTED),
    (experts(b=127), capi.UNSUPPORTED),
    (experts(c=95), capi.UNSUPPORTED),
    (experts(batch=-1), capi.UNSUPPORTED),
    (experts(rows=1 << 24, N=1 << 20), capi.UNSUPPORTED),
])
def test_experts(desc, want):
    assert L.ckx_experts_gemm_i8_is_supported(C.byref(desc)) == want
    if want != capi.OK:
        assert L.ckx_experts_gemm_i8(*[P] * 8, C.byref(desc), None) == want and capi.last_error()


def test_experts_pointers():
    d = experts()
    for i in (0, 1, 2, 3, 4, 6):                     # (the biases and the rows may be null)
        assert L.ckx_experts_gemm_i8(*[0 if j == i else P for j in range(8)], C.byref(d), None) == capi.INVALID_VALUE
    for i in (2, 3, 4, 5, 6, 7):
        assert L.ckx_experts_gemm_i8(*[P + 1 if j == i else P for j in range(8)], C.byref(d), None) == capi.UNSUPPORTED
    assert L.ckx_experts_gemm_i8(*[0] * 8, C.byref(experts(rows=0)), None) == capi.OK
    assert L.ckx_experts_gemm_i8(*[0] * 8, C.byref(experts(experts=0)), None) == capi.OK
    assert L.ckx_experts_gemm_i8(*[P] * 8, None, None) == capi.INVALID_VALUE


@pytest.mark.parametrize("args,want", [
    ((4, 2, 8, 96, 96, 96, 96, capi.TYPE_BF16), capi.OK),
    ((4, 0, 0, 96, 96, 96, 96, capi.TYPE_F32), capi.OK),
    ((1, 2, 1, 96, 0, 0, 0, capi.TYPE_F16), capi.OK),
    ((4, 2, 8, 96, 96, 0, 96, capi.TYPE_F16), capi.OK),    # one row for all
    ((-1, 2, 8, 96, 96, 96, 96, capi.TYPE_BF16), capi.INVALID_VALUE),
    ((4, -2, 8, 96, 96, 96, 96, capi.TYPE_BF16), capi.INVALID_VALUE),
    ((4, 2, 8, 96, 96, 96, 96, capi.TYPE_I8), capi.INVALID_VALUE),
    ((4, 2, 8, 96, 95, 96, 96, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((4, 2, 8, 96, 96, 96, 95, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((4, 2, 8, 96, 96, -1, 96, capi.TYPE_BF16), capi.UNSUPPORTED),
    ((1 << 20, 17, 8, 96, 96, 96, 96, capi.TYPE_BF16), capi.UNSUPPORTED),
])
def test_combine(args, want):
    assert L.ckx_experts_combine_is_supported(*args) == want
    if want != capi.OK:
        assert L.ckx_experts_combine(*[P] * 5, *args, None) == want and capi.last_error()


def test_combine_pointers():
    ok = (4, 2, 8, 96, 96, 96, 96, capi.TYPE_BF16)
    for i in (0, 1, 2, 4):                           # (add may be null)
        assert L.ckx_experts_combine(*[0 if j == i else P for j in range(5)], *ok, None) == capi.INVALID_VALUE
    for i in range(5):
        assert L.ckx_experts_combine(*[P + 1 if j == i else P * (j + 1) for j in range(5)], *ok, None) == capi.UNSUPPORTED
    # add in place, but with other rows
    assert L.ckx_experts_combine(P, P, P, P * 3, P * 3, 4, 2, 8, 96, 96, 0, 96, capi.TYPE_BF16, None) == capi.INVALID_VALUE
    assert L.ckx_experts_combine(0, 0, 0, 0, 0, 0, *ok[1:], None) == capi.OK


def test_plans():
    """Each kernel has sizes that it is chosen for."""
    plan = capi.gemm_i8_plan
    assert plan(0, 8, 16) == (0, 0, 0) and plan(8, 0, 16) == (0, 0, 0)
    assert plan(1, 4096, 4096) == (16, 16, 1) and plan(1, 4096, 4096, gated=True) == (16, 32, 1) and plan(16, 4096, 16384) == (16, 16, 1)
    assert plan(40, 4096, 4096) == (32, 32, 1)
    assert plan(512, 4096, 4096)[::2] == (64, 1)
    assert plan(1024, 4096, 4096)[0] == 128
    assert plan(8192, 8192, 8192) == (256, 256, 1)
    # K of odd length, strides that are no multiples of 16, and no K at all: the kernel for any call
    assert plan(64, 64, 100)[2] == 0 and plan(64, 64, 96, lda=100)[2] == 0 and plan(64, 64, 96, ldb=104)[2] == 0 and plan(64, 64, 0)[2] == 0
    # few tiles and a long K: runs of it, which take a workspace
    need = L.ckx_gemm_i8_tokenscale_workspace_bytes(128, 256, 16384, 0)
    tile_m, tile_n, runs = plan(128, 256, 16384, workspace_bytes=need)
    assert runs > 1 and need == 4 * 128 * 256 * runs and plan(128, 256, 16384)[2] == 1
    few = lambda **kw: capi.experts_gemm_i8_plan(experts(**kw))
    assert few(rows=0) == (0, 0, 0) and few(experts=0) == (0, 0, 0)
    assert few(rows=8, K=4096) == (16, 16, 1) and few(rows=8, K=4096, gated=1) == (16, 32, 1)
    assert few(rows=256, N=4096, K=4096)[:2] == (64, 128) and few(rows=512, N=4096, K=512)[:2] == (128, 128)
    assert few(rows=2048, N=4096, K=4096) == (256, 256, 1)
    assert few(K=136)[2] == 0 and few(batch=96 * 128 + 8)[2] == 0
    # rows gathered from all of A have to lie within 2 GiB, and rows in order need not
    far = experts(rows=2048, rows_a=1 << 20, K=4096)
    assert capi.experts_gemm_i8_plan(far, gathered=True)[2] == 0 and capi.experts_gemm_i8_plan(far, gathered=False)[2] == 1


def test_plan_refusals():
    one = C.c_int(0)
    r = C.byref(one)
    assert L.ckx_gemm_i8_tokenscale_plan(4, 8, 256, 256, 256, 8, 0, capi.TYPE_BF16, 0, r, r, None) == capi.INVALID_VALUE
    assert L.ckx_gemm_i8_tokenscale_plan(4, 8, 256, 256, 256, 8, 0, capi.TYPE_BF16, -1, r, r, r) == capi.INVALID_VALUE
    assert L.ckx_gemm_i8_tokenscale_plan(4, 8, 256, 255, 256, 8, 0, capi.TYPE_BF16, 0, r, r, r) == capi.UNSUPPORTED
    assert L.ckx_experts_gemm_i8_plan(C.byref(experts()), 2, r, r, r) == capi.INVALID_VALUE
    assert L.ckx_experts_gemm_i8_plan(None, 0, r, r, r) == capi.INVALID_VALUE
    assert L.ckx_experts_gemm_i8_plan(C.byref(experts()), 0, r, None, r) == capi.INVALID_VALUE


def test_operators_of_python():
    """What the classes refuse themselves: other types, other element operations."""
    with pytest.raises(KeyError):
        ck.DeviceRouteExperts("f32", Scoring="tanh")
    with pytest.raises(TypeError):
        ck.DeviceRouteExperts().MakeArgumentPointer(*[None] * 8, 4, 8, 2, 8, weight_element_op=ck.AddRelu())
    import torch
    x = torch.zeros(4, 8)
    with pytest.raises(TypeError):
        ck.DeviceTokenQuantizeI8("bf16").MakeArgumentPointer(x, None, None, 4, 8, 8, 8)
    op = ck.DeviceGemmTokenScaleI8("bf16")
    arg = op.MakeArgumentPointer(*[None] * 6, 4, 8, 256, 255, 256, 8)
    assert not op.IsSupportedArgument(arg) and "leading dimension" in capi.last_error()
