"""The C++ classes of the int8 linear and mixture-of-experts operators, through the profiler's commands: the product it writes is checked
against the plain forms on inputs made again from the same seeds, and what the profiler verifies itself has to pass."""
import numpy as np
import pytest
import torch

import experts_plain as ep
from composable_kernel_amd.host_tensor import splitmix64, uniform_f16
from test_serving_host_gpu import DT, SEED, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("c_type,gated", [(1, 0), (2, 1)])
@pytest.mark.parametrize("M,N,K", [(1, 384, 512), (100, 200, 272), (130, 72, 100), (512, 640, 1024)])
def test_gemm_i8_tokenscale(c_type, gated, M, N, K, tmp_path):
    out, dump = _run(["gemm_i8_tokenscale", c_type, 0, 1, 0, 1, M, N, K, gated, 2], tmp_path)
    assert "DeviceTokenQuantizeI8" in out and "DeviceGemmTokenScaleI8" in out and out.count("Perf:") == 2
    wide = N * (1 + gated)
    x = torch.from_numpy(uniform_f16((M, K), -1, 1, SEED + 15))
    w = torch.from_numpy((splitmix64(SEED + 16, wide * K) >> np.uint64(56)).astype(np.uint8)).view(torch.int8).view(wide, K)
    sw = torch.from_numpy((1.0 / (4096 << (splitmix64(SEED + 17, wide) >> np.uint64(62)).astype(np.int64))).astype(np.float32))
    q, s = ep.quantize(x)
    got = torch.from_numpy(np.fromfile(dump, np.int16)).view(DT[c_type]).view(M, N)
    ep.near(got, *ep.scaled(q, w, s, sw, None, bool(gated), DT[c_type]))


@pytest.mark.parametrize("c_type,init,M,N,K,gated", [(1, 1, 3, 300, 1000, 0), (2, 1, 600, 520, 512, 1), (2, 2, 40, 128, 4096, 0), (1, 0, 20, 40, 128, 1)])
def test_gemm_i8_tokenscale_verified(c_type, init, M, N, K, gated, tmp_path):
    out, dump = _run(["gemm_i8_tokenscale", c_type, 1, init, 0, 0, M, N, K, gated], tmp_path)
    assert f"verified DeviceTokenQuantizeI8: {min(M, 256) * (K + 1)} values" in out
    assert f"verified DeviceGemmTokenScaleI8: {min(M * N, 4096)} values" in out and "Error" not in out and "Perf" not in out
    assert bool(np.fromfile(dump, np.int16).any()) == (init > 0)


@pytest.mark.parametrize("scores,init,time,T,E,k,H,I", [(1, 1, 0, 1, 8, 2, 512, 256), (2, 1, 1, 300, 16, 4, 256, 384), (1, 1, 0, 64, 60, 6, 200, 72),
                                                        (2, 0, 0, 5, 3, 3, 64, 64), (1, 2, 1, 4000, 8, 2, 256, 128)])
def test_experts_i8_verified(scores, init, time, T, E, k, H, I, tmp_path):
    out, dump = _run(["experts_i8", scores, 1, init, 0, time, T, E, k, H, I, 2], tmp_path)
    assert f"verified DeviceRouteExperts: {2 * min(T, 1024) * k + E + 1 + T * k} values" in out
    assert f"verified DeviceExpertsGemmI8, gated: {min(T * k * I, 4096)} values" in out
    assert f"verified DeviceExpertsGemmI8: {min(T * k * H, 4096)} values" in out
    assert f"verified DeviceExpertsCombine: {min(T * H, 8192)} values" in out
    assert out.count("verified DeviceTokenQuantizeI8") == 2 and "Error" not in out and out.count("Perf:") == (6 if time else 0)
    assert bool(np.fromfile(dump, np.int16).any()) == (init > 0)
