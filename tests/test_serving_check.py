"""The host checks behind the profiler's verification of the 8-bit serving operators, on the CPU: what the plain forms in 64 bits give
passes, and a planted mistake is counted."""
import os
import subprocess

import numpy as np
import pytest
import torch

import serving_plain as sp

HOST = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "composable_kernel_amd", "host")
SOURCE = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include "ckx/serving_check.hpp"
template <typename T>
std::vector<T> load(const char* name)
{
    std::vector<T> v;
    FILE* f = std::fopen(name, "rb");
    T x;
    while(f && std::fread(&x, sizeof(T), 1, f) == 1)
        v.push_back(x);
    if(f)
        std::fclose(f);
    return v;
}
int main(int argc, char** argv)
{
    int p[12] = {};
    for(int i = 2; i < argc; ++i)
        p[i - 2] = std::atoi(argv[i]);
    std::size_t n = 0, bad = 0;
    if(!std::strcmp(argv[1], "codes"))
    {
        const auto x = load<double>("x"), y = load<double>("y");
        for(std::size_t i = 0; i < x.size(); ++i, ++n)
            bad += ckx::e4m3_value(ckx::e4m3_code(x[i])) != y[i];
    }
    else if(!std::strcmp(argv[1], "quantise"))
    {
        const auto x = load<double>("x");
        const int K  = p[1];
        bad = ckx::quantise_errors([&](std::size_t m, int k) { return x[m * K + k]; }, load<uint8_t>("q").data(), load<float>("s").data(), p[0], K, n);
    }
    else if(!std::strcmp(argv[1], "gemm"))
    {
        const auto c = load<double>("c");
        const int N  = p[1];
        bad = ckx::gemm_f8_errors([&](std::size_t m, std::size_t j) { return c[m * N + j]; }, load<uint8_t>("a").data(), load<uint8_t>("b").data(),
                                  load<float>("sa").data(), load<float>("sb").data(), p[0], N, p[2], 0x1p-11, n);
    }
    else
    {
        const auto k = load<uint8_t>("k"), v = load<uint8_t>("v");
        const auto ks = load<float>("ks"), vs = load<float>("vs");
        const auto table = load<int32_t>("table");
        const auto x = load<double>("x"), o = load<double>("o");
        const int H = p[1], D = p[3], fresh = p[8], group = p[9];
        const ckx::Cache8View c{k.data(), v.data(), ks.data(), vs.data(), table.data(), p[0], H, p[2], D, p[4], p[5], p[6], p[7] != 0};
        if(!c.sound())
            bad = n = 1;
        else if(!std::strcmp(argv[1], "store"))
            bad = ckx::store8_errors([&](int b, int i, int h, int d, int value) { return x[((std::size_t)(value * p[4] + b) * fresh + i) * H * D + h * D + d]; }, c, fresh, n);
        else
        {
            auto at = [&](const std::vector<double>& y) { return [&](int b, int i, int h, int d) { return y[((std::size_t)(b * fresh + i) * H * group + h) * D + d]; }; };
            bad = ckx::attention8_errors(at(x), at(o), c, fresh, group, 1.0 / std::sqrt((double)D), p[10] != 0, n);
        }
    }
    std::printf("%zu %zu\n", bad, n);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("check")
    (d / "check.cpp").write_text(SOURCE)
    r = subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-I", HOST, str(d / "check.cpp"), "-o", str(d / "check")], stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0 and "warning" not in r.stdout, r.stdout
    return str(d / "check")


@pytest.fixture
def check(program, tmp_path):
    def _check(what, *sizes, **arrays):
        for name, x in arrays.items():
            (x if isinstance(x, np.ndarray) else x.contiguous().view(torch.uint8).numpy() if x.dtype in sp.QMAX else x.contiguous().numpy()
             ).tofile(tmp_path / name)
        r = subprocess.run([program, what] + [str(int(s)) for s in sizes], cwd=tmp_path, stdout=subprocess.PIPE, text=True, timeout=60)
        assert r.returncode == 0
        return tuple(int(x) for x in r.stdout.split())
    return _check


def test_codes(check):
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    x = codes[~codes.isnan()].double().sort().values
    x = torch.cat([x, (x[1:] + x[:-1]) / 2, (x[1:] * 0.51 + x[:-1] * 0.49), torch.tensor([-0.0, 2.0 ** -11, -2.0 ** -10, 1e-30])])
    assert check("codes", x=x, y=x.float().to(torch.float8_e4m3fn).double()) == (0, x.numel())


@pytest.mark.parametrize("M,K", [(3, 300), (700, 40)])
def test_quantiser(check, M, K):
    x = sp.normal(sp.gen(1), (M, K), torch.float16)
    q, s = sp.quantize(x)
    bad, n = check("quantise", M, K, x=x.double(), q=q, s=s.t())
    assert bad == 0 and n == min(M, 256) * (K + -(-K // 128))
    wrong = q.view(torch.uint8).clone()
    wrong[0, K - 1] ^= 1
    assert check("quantise", M, K, x=x.double(), q=wrong.numpy(), s=s.t())[0] == 1
    s[M - 1, 0] *= 1 + 2.0 ** -22
    assert check("quantise", M, K, x=x.double(), q=q, s=s.t())[0] == 1


@pytest.mark.parametrize("M,N,K", [(5, 130, 300), (90, 200, 128)])
def test_product(check, M, N, K):
    g = sp.gen(2)
    code = lambda n: sp.normal(g, (n, K), scale=100.0).clamp(-448, 448).to(torch.float8_e4m3fn)
    groups = -(-K // 128)
    a, b, sa, sb = code(M), code(N), torch.rand(M, groups, generator=g) / 50, torch.rand(-(-N // 128), groups, generator=g) / 50
    c = sp.gemm(a, b, sa, sb)[0].half().double()
    size = dict(a=a, b=b, sa=sa.t(), sb=sb)
    assert check("gemm", M, N, K, c=c, **size) == (0, min(M * N, 4096))
    c[M - 1, N - 1] += c.abs().mean()
    assert check("gemm", M, N, K, c=c, **size)[0] == 1
    assert check("gemm", M, N, K, c=torch.full_like(c, float("nan")), **size)[0] == min(M * N, 4096)


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("causal", [True, False])
def test_store_and_attention(check, code, causal):
    B, H, group, D, size, ctx, fresh = 2, 2, 3, 32, 16, 21, 14
    g, kv = sp.gen(3), ctx + fresh
    width = -(-kv // size)
    cache = [torch.zeros(B * width, H, size, D).to(code) for _ in range(2)] + [torch.zeros(B * width, H) for _ in range(2)]
    table = torch.randperm(B * width, generator=g).int().view(B, width)
    for at, n in ((0, ctx), (ctx, fresh)):
        x = [sp.normal(g, (B, n, H, D), torch.float16) for _ in range(2)]
        slots = [int(table[b, (at + i) // size]) * size + (at + i) % size for b in range(B) for i in range(n)]
        for i in range(2):
            sp.store(cache[i], cache[2 + i], x[i].view(-1, H, D), slots)
    sizes = (B * width, H, size, D, B, width, kv, code == torch.int8, fresh, group, causal)
    view = dict(k=cache[0], v=cache[1], ks=cache[2], vs=cache[3], table=table)
    kept = torch.stack(x).double()
    assert check("store", *sizes, x=kept, **view) == (0, 2 * B * fresh * H * D)
    kept[1, B - 1, 3, 1, 5] += 0.5
    assert check("store", *sizes, x=kept, **view)[0] == 1
    q = sp.normal(g, (B * fresh, H * group, D), torch.float16)
    o = sp.attention(q, table, [0, fresh, 2 * fresh], [kv] * B, *cache, D ** -0.5, causal)[0].half().double()
    n = B * fresh * H * group * D
    assert n < 256 * D
    assert check("attention", *sizes, x=q.double(), o=o, **view) == (0, n)
    o[B * fresh - 1, H * group - 1, D - 1] += 0.05
    assert check("attention", *sizes, x=q.double(), o=o, **view)[0] == 1
    other = sizes[:-1] + (not causal,)
    assert check("attention", *other, x=q.double(), o=o, **view)[0] > n // 4       # (the other mask)
    view["table"] = table.clone()
    view["table"][1, 0] = B * width
    assert check("attention", *sizes, x=q.double(), o=o, **view) == (1, 1)
