// Plain host forms of the 8-bit serving operators (include/ckx.h) in 64 bits, over a sample of the outputs: what the profiler's
// verification compares with. No HIP: everything is in host memory. Every function returns how many of the values it looked at are
// further from the plain form than the operator's stated roundings allow.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <vector>

namespace ckx {

inline double e4m3_value(uint8_t c)
{
    const int e = c >> 3 & 15, m = c & 7;
    if((c & 127) == 127)
        return NAN;
    const double v = e == 0 ? std::ldexp(m, -9) : std::ldexp(8 + m, e - 10);
    return c & 128 ? -v : v;
}

// the code whose value is nearest to x, |x| <= 448; ties to even
inline uint8_t e4m3_code(double x)
{
    const double a = std::fabs(x);
    int e          = -6;
    if(a > 0)
    {
        std::frexp(a, &e); // a = f * 2^e, 1/2 <= f < 1
        e = std::max(e - 1, -6);
    }
    const int steps = (int)std::nearbyint(std::ldexp(a, 3 - e)); // eighths of 2^e: 0 ... 16
    const int code  = ((e + 6) << 3) + steps;                    // (a subnormal number has e = -6 and steps under 8; 16 carries)
    return (uint8_t)((std::signbit(x) ? 128 : 0) | code);
}

// at most `most` of `n` places, spread over all of them
inline std::vector<std::size_t> places(std::size_t n, std::size_t most)
{
    std::vector<std::size_t> at(std::min(n, most));
    for(std::size_t i = 0; i < at.size(); ++i)
        at[i] = n <= most ? i : (std::size_t)((double)i * (double)(n - 1) / (double)(most - 1));
    return at;
}

// x(m, k) -> double; codes [M, K], scales [groups, M]: bit for bit
template <typename X>
std::size_t quantise_errors(X x, const uint8_t* q, const float* scale, int M, int K, std::size_t& checked)
{
    std::size_t bad = 0;
    for(std::size_t m : places((std::size_t)M, 256))
        for(int g = 0; g * 128 < K; ++g)
        {
            const int end = std::min(K, (g + 1) * 128);
            double most   = std::ldexp(1.0, -100);
            for(int k = g * 128; k < end; ++k)
                most = std::max(most, std::fabs(x(m, k)));
            bad += scale[(std::size_t)g * M + m] != (float)most / 448.0f;
            for(int k = g * 128; k < end; ++k)
                bad += q[m * K + k] != e4m3_code((float)(x(m, k) * 448.0 / most));
            checked += (std::size_t)(end - g * 128) + 1;
        }
    return bad;
}

// c(m, n) -> double, rounded by `half_step` of its size; a [M, K], b [N, K] codes, sa [groups, M], sb [ceil(N / 128), groups].
// Allowed beside the output's rounding: fp32 sums, and what the 8-bit instruction cuts of eight neighbouring products.
template <typename C>
std::size_t gemm_f8_errors(C c, const uint8_t* a, const uint8_t* b, const float* sa, const float* sb, int M, int N, int K, double half_step,
                           std::size_t& checked)
{
    double value[256];
    for(int i = 0; i < 256; ++i)
        value[i] = e4m3_value((uint8_t)i);
    const int groups = (K + 127) / 128;
    std::size_t bad  = 0;
    for(std::size_t at : places((std::size_t)M * N, 4096))
    {
        const std::size_t m = at / N, n = at % N;
        double want = 0, size = 0, cut = 0;
        for(int k0 = 0; k0 < K; k0 += 8)
        {
            const double s = (double)sa[(std::size_t)(k0 / 128) * M + m] * sb[(n / 128) * groups + k0 / 128];
            double most    = 0;
            for(int k = k0; k < std::min(K, k0 + 8); ++k)
            {
                const double p = value[a[m * K + k]] * value[b[n * K + k]] * s;
                want += p, size += std::fabs(p), most = std::max(most, std::fabs(p));
            }
            cut += 7 * std::ldexp(most, -13);
        }
        const double sums = cut + (132 + groups) * std::ldexp(size, -23);
        bad += !(std::fabs(c(m, n) - want) <= sums + half_step * (std::fabs(want) + sums) + std::ldexp(1.0, -25));
        ++checked;
    }
    return bad;
}

// A cache [blocks, heads, block_size, dim] with scales [blocks, heads] and the tables of `batch` sequences [batch, width], `kv` tokens each.
struct Cache8View
{
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int32_t* table;
    int blocks, heads, block_size, dim, batch, width, kv;
    bool int8;
    double most() const { return int8 ? 127 : 448; }
    double value(uint8_t c) const { return int8 ? (double)(int8_t)c : e4m3_value(c); }
    int block(int b, int t) const { return table[(std::size_t)b * width + t / block_size]; }
    std::size_t at(int b, int t, int h) const
    {
        return (((std::size_t)block(b, t) * heads + h) * block_size + t % block_size) * dim;
    }
    std::size_t scale_at(int b, int t, int h) const { return (std::size_t)block(b, t) * heads + h; }
    bool sound() const // every block that a sequence has lies in the cache
    {
        for(int b = 0; b < batch; ++b)
            for(int t = 0; t < kv; t += block_size)
                if(block(b, t) < 0 || block(b, t) >= blocks)
                    return false;
        return true;
    }
};

// x(b, i, h, d, value) -> double: the last `fresh` tokens' keys and values. Their codes are rounded once; the
// quotient before that and the scale are fp32, half a step of which (2^-24) counts by the value.
template <typename X>
std::size_t store8_errors(X x, const Cache8View& c, int fresh, std::size_t& checked)
{
    std::size_t bad = 0;
    for(std::size_t at : places((std::size_t)c.batch * fresh, 512))
    {
        const int b = (int)(at / fresh), i = (int)(at % fresh), t = c.kv - fresh + i;
        for(int h = 0; h < c.heads; ++h)
            for(int d = 0; d < c.dim; ++d)
                for(int value = 0; value < 2; ++value)
                {
                    const double s    = (value ? c.vs : c.ks)[c.scale_at(b, t, h)], want = x(b, i, h, d, value);
                    const double got  = c.value((value ? c.v : c.k)[c.at(b, t, h) + d]) * s;
                    const double step = c.int8 ? s / 2 : std::max(std::fabs(want) / 16, std::ldexp(s, -10));
                    bad += !(std::fabs(got - want) <= step + std::ldexp(std::fabs(want), -23));
                    ++checked;
                }
    }
    return bad;
}

// q(b, i, h, d) -> double, o(b, i, h, d) -> double (fp16): the last `fresh` tokens' attention, `group` query heads a cache head
template <typename Q, typename O>
std::size_t attention8_errors(Q q, O o, const Cache8View& c, int fresh, int group, double scale, bool causal, std::size_t& checked)
{
    std::size_t bad = 0;
    const int heads = c.heads * group;
    std::vector<double> p, sum(c.dim), size(c.dim);
    for(std::size_t at : places((std::size_t)c.batch * fresh * heads, 256))
    {
        const int h = (int)(at % heads), i = (int)(at / heads % fresh), b = (int)(at / heads / fresh), hk = h / group;
        const int see = causal ? c.kv - fresh + i + 1 : c.kv;
        double top = -INFINITY, big = 0, largest = 0, all = 0;
        p.assign(see, 0.0);
        for(int t = 0; t < see; ++t)
        {
            const std::size_t key = c.at(b, t, hk);
            const double s        = c.ks[c.scale_at(b, t, hk)] * scale;
            double dot = 0, abs = 0;
            for(int d = 0; d < c.dim; ++d)
            {
                const double x = q(b, i, h, d) * c.value(c.k[key + d]);
                dot += x, abs += std::fabs(x);
            }
            p[t] = dot * s, top = std::max(top, p[t]), big = std::max(big, abs * std::fabs(s));
            largest = std::max(largest, std::fabs((double)c.vs[c.scale_at(b, t, hk)]));
        }
        std::fill(sum.begin(), sum.end(), 0.0);
        std::fill(size.begin(), size.end(), 0.0);
        for(int t = 0; t < see; ++t)
        {
            const double w = std::exp(p[t] - top), s = c.vs[c.scale_at(b, t, hk)];
            const std::size_t value = c.at(b, t, hk);
            all += w;
            for(int d = 0; d < c.dim; ++d)
            {
                const double x = w * s * c.value(c.v[value + d]);
                sum[d] += x, size[d] += std::fabs(x);
            }
        }
        // a summand: half a step of fp16, its score's fp32 roundings (twice: in the sum of the probabilities too), the sums' own; fp16's
        // subnormal numbers in a probability and in the output
        const double rel = std::ldexp(1.0, -11) + 2 * (c.dim + 4) * std::ldexp(big, -23) + 2 * (see + 16) * std::ldexp(1.0, -23);
        for(int d = 0; d < c.dim; ++d)
        {
            const double want = all > 0 ? sum[d] / all : 0.0, mag = all > 0 ? size[d] / all : 0.0;
            bad += !(std::fabs(o(b, i, h, d) - want) <=
                     std::ldexp(std::fabs(want), -11) + mag * rel + see * std::ldexp(c.most() * largest, -25) + std::ldexp(1.0, -25));
            ++checked;
        }
    }
    return bad;
}

} // namespace ckx
