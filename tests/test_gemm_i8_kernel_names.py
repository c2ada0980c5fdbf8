"""Which kernel a token-scaled int8 product is given, by name (pure host logic)."""
import ctypes as C
import random

import pytest

from composable_kernel_amd import capi

NAMES = {"direct16x16": (16, 16), "direct16x16 eight waves": (16, 16), "direct32x32": (32, 32), "tile64x128": (64, 128), "tile128x128": (128, 128),
         "tile128x128 two a CU": (128, 128), "tile256x256": (256, 256), "any16x16": (16, 16), "any128x128": (128, 128)}


@pytest.mark.parametrize("M,N,K,gated,name", [
    (1, 4096, 4096, False, "direct16x16"), (16, 4096, 16384, True, "direct16x16 eight waves"), (40, 4096, 4096, False, "direct32x32"),
    (512, 4096, 4096, False, "tile64x128"), (1024, 4096, 4096, False, "tile128x128"), (2048, 4096, 128, False, "tile128x128 two a CU"),
    (8192, 8192, 8192, False, "tile256x256"), (8, 64, 100, False, "any16x16"), (200, 64, 100, True, "any128x128")])
def test_dense(M, N, K, gated, name):
    assert capi.gemm_i8_kernel(M, N, K, gated=gated) == name
    m, n, runs = capi.gemm_i8_plan(M, N, K, gated=gated)
    assert (m, n) == (NAMES[name][0], NAMES[name][1] * (2 if gated and NAMES[name] == (16, 16) else 1))


def experts(rows, E, N, K, gated=0):
    return capi.ExpertsDesc(rows, rows, E, N, K, K, K, N, 1, gated, capi.TYPE_BF16, 0, N * K)


@pytest.mark.parametrize("desc,name", [
    (experts(8, 8, 96, 4096), "direct16x16"), (experts(300, 3, 1030, 1040), "tile64x128"), (experts(512, 64, 4096, 4096), "tile64x128 two a CU"),
    (experts(2000, 3, 1030, 400), "tile128x128 two a CU"), (experts(16384, 8, 4096, 4096), "tile256x256"), (experts(8, 8, 64, 100), "any16x16")])
def test_experts(desc, name):
    assert capi.experts_gemm_i8_kernel(desc) == name


def test_nothing_to_do_and_refusals():
    L = capi.lib()
    assert capi.gemm_i8_kernel(0, 8, 16) == "" and capi.experts_gemm_i8_kernel(experts(0, 8, 64, 128)) == ""
    assert L.ckx_gemm_i8_tokenscale_kernel_name(4, 8, 256, 255, 256, 8, 0, capi.TYPE_BF16, 0) is None and "leading dimension" in capi.last_error()
    assert L.ckx_gemm_i8_tokenscale_kernel_name(4, 8, 256, 256, 256, 8, 0, capi.TYPE_BF16, -1) is None
    assert L.ckx_experts_gemm_i8_kernel_name(None, 0) is None
    assert L.ckx_experts_gemm_i8_kernel_name(C.byref(experts(8, 8, 64, 128)), 2) is None
    with pytest.raises(capi.CkxError):
        capi.gemm_i8_kernel(4, 8, 256, lda=255)


THREADS = {"any128x128": 256, "direct16x16": 256, "direct16x16 eight waves": 512, "direct32x32": 512, "tile64x128": 512, "tile128x128 two a CU": 512,
           "tile128x128": 512, "tile64x128 two a CU": 256, "any16x16": 256}


def test_launches_of_the_largest_problems():
    """Whatever problem is supported, the launch of its kernel has fewer than 2^32 threads."""
    rng, some = random.Random(5), 0
    for _ in range(30000):
        gated, E = rng.random() < 0.5, int(2 ** rng.uniform(0, 10)) if rng.random() < 0.6 else 0
        most = 24 if E else 31
        M = min(2 ** most, int(2 ** rng.uniform(most - 12, most + 0.01)))
        if rng.random() < 0.3:
            M = int(2 ** rng.uniform(0, most - 12))
        N = min(2 ** 30 - 1, int(2 ** min(30.0, rng.uniform(0, 40 - M.bit_length()))))
        K = min(131071, int(2 ** rng.uniform(0, 17))) // 16 * 16 + (1 if rng.random() < 0.1 else 0)
        if E:
            desc = experts(M, E, N, K, int(gated))
            if capi.lib().ckx_experts_gemm_i8_is_supported(C.byref(desc)) != capi.OK:
                continue
            name, (m, n, runs) = capi.experts_gemm_i8_kernel(desc, False), capi.experts_gemm_i8_plan(desc, False)
        else:
            ws = 2 ** 62 if rng.random() < 0.5 else 0
            if M == 2 ** 31 or capi.lib().ckx_gemm_i8_tokenscale_is_supported(M, N, K, K, K, N, int(gated), capi.TYPE_BF16) != capi.OK:
                continue
            name, (m, n, runs) = capi.gemm_i8_kernel(M, N, K, gated=gated, workspace_bytes=ws), capi.gemm_i8_plan(M, N, K, gated=gated, workspace_bytes=ws)
        rows = M // m + min(E, M) if E else -(-M // m)
        threads = rows * -(-N * (1 + gated) // n) * max(1, runs) * THREADS.get(name, 0)
        assert threads < 2 ** 32, (E, M, N, K, gated, name, runs)
        some += threads > 2 ** 30
    assert some > 100
