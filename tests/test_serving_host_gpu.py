"""The C++ classes of the 8-bit serving operators, through the profiler's commands: the tensors they write are checked against the
plain forms on inputs made again from the same seeds."""
import os
import subprocess

import numpy as np
import pytest
import torch

import serving_plain as sp
from composable_kernel_amd.host_tensor import splitmix64, uniform_f16

pytestmark = pytest.mark.gpu
BIN = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "composable_kernel_amd", "bin", "ckx_profiler")
SEED = 0xC0FFEE
DT = {1: torch.float16, 2: torch.bfloat16}


def _run(args, tmp_path):
    if not os.path.exists(BIN):
        pytest.fail(f"{BIN} is not built (python -m composable_kernel_amd.build)")
    dump = str(tmp_path / "out.bin")
    r = subprocess.run([BIN] + [str(a) for a in args], env=dict(os.environ, CKX_PROFILER_DUMP=dump), stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True, timeout=100)
    assert r.returncode == 0, r.stdout
    return r.stdout, dump


@pytest.mark.parametrize("c_type", [1, 2])
@pytest.mark.parametrize("M,N,K", [(1, 384, 512), (100, 200, 272), (512, 640, 1024)])
def test_gemm_f8_blockscale(c_type, M, N, K, tmp_path):
    out, dump = _run(["gemm_f8_blockscale", c_type, 0, 1, 0, 1, M, N, K, 2], tmp_path)
    assert "DeviceBlockQuantizeF8" in out and "DeviceGemmBlockScaleF8" in out and out.count("Perf:") == 2
    x = torch.from_numpy(uniform_f16((M, K), -1, 1, SEED + 10))
    codes = (splitmix64(SEED + 11, N * K) >> np.uint64(56)).astype(np.uint8)
    codes[(codes & 127) == 127] = 0
    w = torch.from_numpy(codes).view(torch.float8_e4m3fn).view(N, K)
    groups, nb = -(-K // 128), -(-N // 128)
    sw = splitmix64(SEED + 12, nb * groups) >> np.uint64(62)
    sw = torch.from_numpy((1.0 / (64 << sw.astype(np.int64))).astype(np.float32)).view(nb, groups)
    q, s = sp.quantize(x)
    want, mag, cut = sp.gemm(q, w, s, sw)
    got = torch.from_numpy(np.fromfile(dump, np.int16)).view(DT[c_type]).view(M, N).double()
    bound = sp.HALF_STEP[DT[c_type]] * want.abs() + (128 + groups + 4) * 2.0 ** -23 * mag + 1.01 * cut + 2.0 ** -25
    assert bool(((got - want).abs() <= bound).all()), float((got - want).abs().max())


@pytest.mark.parametrize("cache,B,ctx,new,heads,kv,D,size,causal", [(1, 3, 0, 1, 4, 2, 64, 16, 1), (1, 4, 50, 1, 8, 2, 128, 16, 1),
                                                                 (2, 2, 33, 40, 4, 4, 64, 32, 1), (1, 2, 20, 70, 6, 2, 80, 16, 0)])
def test_paged_attention8(cache, B, ctx, new, heads, kv, D, size, causal, tmp_path):
    out, dump = _run(["paged_attention8", cache, 0, 1, 0, 1, B, ctx, new, heads, kv, D, size, causal, 2], tmp_path)
    assert all(n in out for n in ("DeviceKvCacheTables", "DeviceKvCacheStore8", "DevicePagedAttention8"))
    # the same two steps on plain caches, sequence after sequence: where a block lies does not matter
    code, width = (torch.float8_e4m3fn, torch.int8)[cache - 1], -(-(ctx + new) // size)
    codes = [torch.zeros(B * width, kv, size, D).to(code) for _ in range(2)]
    scales = [torch.zeros(B * width, kv) for _ in range(2)]
    row = (heads + 2 * kv) * D
    for at, n, seed in ((0, ctx, SEED + 13), (ctx, new, SEED + 14)):
        qkv = torch.from_numpy(uniform_f16((B * n, row), -1, 1, seed)) if n else torch.zeros(0, row, dtype=torch.float16)
        slots = [b * width * size + at + i for b in range(B) for i in range(n)]
        for i in range(2):
            x = qkv[:, (heads + i * kv) * D:(heads + (i + 1) * kv) * D].reshape(-1, kv, D)
            sp.store(codes[i], scales[i], x, slots)
    table = torch.arange(B * width, dtype=torch.int32).view(B, width)
    q, scale = qkv[:, :heads * D].reshape(-1, heads, D), float(np.float32(1) / np.sqrt(np.float32(D)))
    o, mag, big = sp.attention(q, table, [b * new for b in range(B + 1)], [ctx + new] * B, *codes, *scales, scale, bool(causal))
    got = torch.from_numpy(np.fromfile(dump, np.float16)).view(B * new, heads, D).double()
    bound = sp.attention_bound(o, mag, big, torch.float16, D, ctx + new) + 2.0 ** -25 + sp.small_products(scales[1], code, ctx + new)
    assert bool(((got - o).abs() <= bound).all()), float((got - o).abs().max())


@pytest.mark.parametrize("c_type,init,M,N,K", [(1, 1, 3, 300, 1000), (2, 1, 600, 520, 512), (2, 2, 40, 128, 4096), (1, 0, 20, 40, 128)])
def test_gemm_f8_blockscale_verified(c_type, init, M, N, K, tmp_path):
    out, dump = _run(["gemm_f8_blockscale", c_type, 1, init, 0, 0, M, N, K], tmp_path)
    assert f"verified DeviceBlockQuantizeF8: {min(M, 256) * (K + -(-K // 128))} values" in out
    assert f"verified DeviceGemmBlockScaleF8: {min(M * N, 4096)} values" in out and "Error" not in out and "Perf" not in out
    assert bool(np.fromfile(dump, np.int16).any()) == (init > 0)


@pytest.mark.parametrize("cache,init,time,B,ctx,new,heads,kv,D,size,causal", [
    (1, 1, 0, 3, 500, 1, 8, 2, 128, 16, 1), (2, 1, 1, 2, 33, 90, 4, 4, 64, 32, 1), (1, 1, 1, 2, 20, 70, 6, 2, 80, 16, 0), (2, 0, 0, 2, 5, 3, 4, 2, 64, 16, 1)])
def test_paged_attention8_verified(cache, init, time, B, ctx, new, heads, kv, D, size, causal, tmp_path):
    out, dump = _run(["paged_attention8", cache, 1, init, 0, time, B, ctx, new, heads, kv, D, size, causal, 2], tmp_path)
    assert "verified DeviceKvCacheTables" in out and f"verified DeviceKvCacheStore8: {2 * min(B * new, 512) * kv * D} values" in out
    assert f"verified DevicePagedAttention8: {min(B * new * heads, 256) * D} values" in out and "Error" not in out
    assert bool(np.fromfile(dump, np.int16).any()) == (init > 0)
