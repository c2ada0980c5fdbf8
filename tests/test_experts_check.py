"""The host checks behind the profiler's verification of the int8 linear and mixture-of-experts operators, on the CPU: what the plain forms
in 64 bits give passes, and a planted mistake is counted."""
import os
import subprocess

import pytest
import torch

import experts_plain as ep

HOST = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "composable_kernel_amd", "host")
SOURCE = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include "ckx/experts_check.hpp"
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
    const auto x = load<double>("x");
    if(!std::strcmp(argv[1], "quantise"))
        bad = ckx::token_quantise_errors([&](std::size_t m, int k) { return x[m * p[1] + k]; }, load<int8_t>("q").data(), load<float>("s").data(), p[0], p[1], n);
    else if(!std::strcmp(argv[1], "route"))
    {
        const auto ids = load<int32_t>("ids"), offsets = load<int32_t>("offsets"), rows = load<int32_t>("rows"), places = load<int32_t>("places");
        const auto w = load<float>("w");
        bad = ckx::route_errors([&](std::size_t t, int e) { return x[t * p[1] + e]; },
                                ckx::RouteView{ids.data(), offsets.data(), rows.data(), places.data(), w.data(), p[0], p[1], p[2], p[3] != 0, p[4] != 0}, n);
    }
    else if(!std::strcmp(argv[1], "gemm"))
    {
        const auto a = load<int8_t>("a"), b = load<int8_t>("b");
        const auto sa = load<float>("sa"), sb = load<float>("sb");
        const auto expert = load<int32_t>("expert"), row = load<int32_t>("row");
        bad = ckx::gemm_i8_errors([&](std::size_t m, std::size_t j) { return x[m * p[1] + j]; },
                                  [&](std::size_t m, std::size_t& r, std::size_t& e) { r = row[m], e = expert[m]; },
                                  ckx::GemmI8View{a.data(), b.data(), sa.data(), sb.data(), p[0], p[1], p[2], p[3] != 0}, 0x1p-11, n);
    }
    else
    {
        const auto y = load<double>("y");
        const auto places = load<int32_t>("places");
        const auto w = load<float>("w");
        bad = ckx::combine_errors([&](std::size_t t, std::size_t j) { return x[t * p[3] + j]; }, [&](std::size_t i, std::size_t j) { return y[i * p[3] + j]; },
                                  places.data(), w.data(), p[0], p[1], p[2], p[3], 0x1p-11, n);
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
        for name, t in arrays.items():
            t.contiguous().numpy().tofile(tmp_path / name)
        r = subprocess.run([program, what] + [str(int(s)) for s in sizes], cwd=tmp_path, stdout=subprocess.PIPE, text=True, timeout=60)
        assert r.returncode == 0
        return tuple(int(v) for v in r.stdout.split())
    return _check


@pytest.mark.parametrize("M,K", [(3, 300), (700, 40)])
def test_quantiser(check, M, K):
    x = ep.normal(ep.gen(1), (M, K), torch.float16)
    q, s = ep.quantize(x)
    assert check("quantise", M, K, x=x.double(), q=q, s=s) == (0, min(M, 256) * (K + 1))
    wrong = q.clone()
    wrong[0, K - 1] ^= 1
    assert check("quantise", M, K, x=x.double(), q=wrong, s=s)[0] == 1
    s[M - 1] *= 1 + 2.0 ** -22
    assert check("quantise", M, K, x=x.double(), q=q, s=s)[0] == 1


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [False, True])
def test_router(check, scoring, renormalise):
    T, E, k = 50, 20, 3
    x = ep.normal(ep.gen(2), (T, E), torch.float16)
    x[7] = 0.5
    ids, w, offsets, rows, places = ep.route(x, None, k, scoring, renormalise)
    size = (T, E, k, scoring == "sigmoid", renormalise)
    good = dict(x=x.double(), ids=ids, w=w.float(), offsets=offsets, rows=rows, places=places)
    assert check("route", *size, **good) == (0, 2 * T * k + E + 1 + T * k)
    wrong = {n: t.clone() for n, t in good.items()}
    wrong["w"][T - 1, k - 1] *= 1 + 2.0 ** -22
    assert check("route", *size, **wrong)[0] == 1
    wrong = {n: t.clone() for n, t in good.items()}
    wrong["rows"][[0, 1]] = wrong["rows"][[1, 0]]
    assert check("route", *size, **wrong)[0] == 2
    wrong = {n: t.clone() for n, t in good.items()}
    wrong["ids"][5, [0, 1]] = wrong["ids"][5, [1, 0]]
    assert check("route", *size, **wrong)[0] >= 2


@pytest.mark.parametrize("gated", [False, True])
def test_product(check, gated):
    M, N, K, E, R = 60, 70, 90, 3, 25
    g = ep.gen(3)
    wide = N * (2 if gated else 1)
    a, b = ep.codes(g, (R, K)), ep.codes(g, (E, wide, K))
    sa, sb = torch.rand(R, generator=g) / 50, torch.rand(E, wide, generator=g) / 50
    row, expert = torch.randint(0, R, (M,), generator=g, dtype=torch.int32), torch.randint(0, E, (M,), generator=g, dtype=torch.int32)
    c = torch.stack([ep.scaled(a[r:r + 1], b[e], sa[r:r + 1], sb[e], None, gated, torch.float16)[0][0] for r, e in zip(row.tolist(), expert.tolist())])
    keep = c.abs().amax() / 30000
    sb /= keep ** (0.5 if gated else 1)              # (fp16 has to hold the outputs)
    c = torch.stack([ep.scaled(a[r:r + 1], b[e], sa[r:r + 1], sb[e], None, gated, torch.float16)[0][0] for r, e in zip(row.tolist(), expert.tolist())])
    args = dict(a=a, b=b, sa=sa, sb=sb, row=row, expert=expert)
    x = c.half().double()
    assert check("gemm", M, N, K, gated, x=x, **args) == (0, min(M * N, 4096))
    x[M - 1, N - 1] += x.abs().mean()
    assert check("gemm", M, N, K, gated, x=x, **args)[0] == 1
    assert check("gemm", M, N, K, gated, x=torch.full_like(x, float("nan")), **args)[0] == min(M * N, 4096)


def test_sums(check):
    T, k, R, N = 30, 4, 50, 100
    g = ep.gen(4)
    y, w = ep.normal(g, (R, N), torch.float16), torch.rand(T, k, generator=g)
    places = torch.randint(-1, R + 1, (T, k), generator=g, dtype=torch.int32)
    x = ep.combine(y, places, w, None, torch.float16)[0].half().double()
    assert check("combine", T, k, R, N, x=x, y=y.double(), places=places, w=w) == (0, T * N)
    x[T - 1, N - 1] += 0.01
    assert check("combine", T, k, R, N, x=x, y=y.double(), places=places, w=w)[0] == 1
