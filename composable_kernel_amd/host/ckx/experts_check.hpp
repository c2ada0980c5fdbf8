// Plain host forms in 64 bits of the int8 linear and mixture-of-experts operators (include/ckx.h), over a sample of the outputs, as
// serving_check.hpp has them for the other 8-bit operators: every function returns how many of the values it looked at are further
// from the plain form than the operator's stated roundings allow.
#pragma once

#include "ckx/serving_check.hpp"

namespace ckx {

// x(m, k) -> double; codes [M, K], scales [M]: bit for bit
template <typename X>
std::size_t token_quantise_errors(X x, const int8_t* q, const float* scale, int M, int K, std::size_t& checked)
{
    std::size_t bad = 0;
    for(std::size_t m : places((std::size_t)M, 256))
    {
        double most = std::ldexp(1.0, -100);
        for(int k = 0; k < K; ++k)
            most = std::max(most, std::fabs(x(m, k)));
        bad += scale[m] != (float)most / 127.0f;
        for(int k = 0; k < K; ++k)
            bad += q[m * K + k] != (int)std::nearbyint((float)(x(m, k) * 127.0 / most));
        checked += (std::size_t)K + 1;
    }
    return bad;
}

// x(t, e) -> double, finite; no bias, no groups. Ids and tables as they are, weights to half a step of fp32.
struct RouteView
{
    const int32_t *ids, *offsets, *rows, *places;
    const float* weights;
    int tokens, experts, top_k;
    bool sigmoid, renormalise;
};
template <typename X>
std::size_t route_errors(X x, const RouteView& r, std::size_t& checked)
{
    std::size_t bad = 0;
    std::vector<double> s(r.experts);
    std::vector<int> order(r.experts);
    for(std::size_t t : places((std::size_t)r.tokens, 1024))
    {
        double top = -INFINITY, all = 0, sum = 0;
        for(int e = 0; e < r.experts; ++e)
            order[e] = e, top = std::max(top, x(t, e));
        for(int e = 0; e < r.experts; ++e)
            all += s[e] = r.sigmoid ? 1 / (1 + std::exp(-x(t, e))) : std::exp(x(t, e) - top);
        std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return x(t, a) > x(t, b); });
        for(int e = 0; e < r.experts && !r.sigmoid; ++e)
            s[e] /= all;
        for(int j = 0; j < r.top_k; ++j)
            sum += s[order[j]];
        for(int j = 0; j < r.top_k; ++j)
        {
            const double want = s[order[j]] / (r.renormalise ? sum : 1.0);
            bad += r.ids[t * r.top_k + j] != order[j];
            bad += !(std::fabs(r.weights[t * r.top_k + j] - want) <= std::ldexp(want, -24) * (1 + 1e-6));
        }
        checked += 2 * (std::size_t)r.top_k;
    }
    // the tables of all ids
    const int pairs = r.tokens * r.top_k;
    std::vector<int32_t> next(r.experts + 1, 0);
    for(int i = 0; i < pairs; ++i)
        if(r.ids[i] >= 0 && r.ids[i] < r.experts)
            ++next[r.ids[i] + 1];
    for(int e = 0; e < r.experts; ++e)
        next[e + 1] += next[e];
    for(int e = 0; e <= r.experts; ++e)
        bad += r.offsets[e] != next[e];
    for(int i = 0; i < pairs; ++i)
    {
        const bool there   = r.ids[i] >= 0 && r.ids[i] < r.experts;
        const int32_t want = there ? next[r.ids[i]]++ : -1;
        bad += r.places[i] != want || (there && r.rows[want] != i);
    }
    checked += (std::size_t)r.experts + 1 + pairs;
    return bad;
}

// C [M, N] of codes: c(m, n) -> double, rounded by `half_step`; from(m, row of A, expert); b [experts, N (gated: 2 N), K]
struct GemmI8View
{
    const int8_t *a, *b;
    const float *sa, *sb;
    int M, N, K;
    bool gated;
};
template <typename C, typename From>
std::size_t gemm_i8_errors(C c, From from, const GemmI8View& v, double half_step, std::size_t& checked)
{
    std::size_t bad = 0;
    const double u  = std::ldexp(1.0, -24);
    for(std::size_t at : places((std::size_t)v.M * v.N, 4096))
    {
        const std::size_t m = at / v.N, n = at % v.N;
        std::size_t row = 0, expert = 0;
        from(m, row, expert);
        double d[2] = {};
        for(int h = 0; h <= (v.gated ? 1 : 0); ++h)
        {
            const std::size_t j = expert * v.N * (v.gated ? 2 : 1) + h * v.N + n;
            int64_t sum         = 0;
            for(int k = 0; k < v.K; ++k)
                sum += (int)v.a[row * v.K + k] * v.b[j * v.K + k];
            d[h] = (double)sum * v.sa[row] * v.sb[j];
        }
        // three roundings of a product; of silu 1.1 times its argument's error and (8 + |argument|) of its own, of the product one more
        double want = d[0], err = 3.01 * u * std::fabs(d[0]);
        if(v.gated)
        {
            const double s = d[0] / (1 + std::exp(-d[0])), es = 1.1 * err + std::fabs(s) * (8 + std::fabs(d[0])) * u + std::ldexp(1.0, -112);
            want = s * d[1];
            err  = es * std::fabs(d[1]) * (1 + 4 * u) + std::fabs(want) * 4.1 * u;
        }
        bad += !(std::fabs(c(m, n) - want) <= err + half_step * (std::fabs(want) + err) + std::ldexp(1.0, -25));
        ++checked;
    }
    return bad;
}

// out(t, n) -> double: the sums of a token's rows y(i, n), weighted; no add
template <typename O, typename Y>
std::size_t combine_errors(O out, Y y, const int32_t* place, const float* weights, int tokens, int top_k, int rows, int N, double half_step,
                           std::size_t& checked)
{
    std::size_t bad = 0;
    for(std::size_t at : places((std::size_t)tokens * N, 8192))
    {
        const std::size_t t = at / N, n = at % N;
        double want = 0, size = 0;
        for(int j = 0; j < top_k; ++j)
        {
            const int i = place[t * top_k + j];
            if(i < 0 || i >= rows)
                continue;
            const double x = (double)weights[t * top_k + j] * y((std::size_t)i, n);
            want += x, size += std::fabs(x);
        }
        const double sums = (top_k + 1) * std::ldexp(size, -24);
        bad += !(std::fabs(out(t, n) - want) <= sums + half_step * (std::fabs(want) + sums) + std::ldexp(1.0, -25));
        ++checked;
    }
    return bad;
}

} // namespace ckx
