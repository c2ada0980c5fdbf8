// Each token's experts, their weights, and the experts' rows in order (formula: include/ckx.h, ckx_route_experts).
//
// A wave takes a token; lane l holds the experts l * EPL ... l * EPL + EPL - 1, so that the lowest lane of a tie has the lowest
// expert. What decides the order is compared as whole numbers that rise with the value: the bits of the fp32 logit where there is no
// bias (both scores rise with it), those of the 64-bit sum of score and bias otherwise, whose upper halves settle all but ties. A pick
// is one maximum over the wave.
// The tables are a stable counting sort of the tokens * top_k pairs. Up to kOneGroup tokens one workgroup does all of it; otherwise
// each workgroup leaves the counts of its tokens in the workspace and a second launch adds them up and places the pairs. Nothing in it depends on
// the order in which waves run.
#include "experts.hpp"
#include "f8.hpp"

namespace ckx {

namespace {

constexpr int kWaves = 16, kThreads = kWaves * 64;
constexpr int kOneGroup = 64, kMostChunks = 256;

// numbers that rise with the value; none of them is 0
__device__ __forceinline__ uint32_t rising(float x)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t rising(double x)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}

// over the wave's lanes
template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v)
{
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
    return v > o ? v : o;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
    v = max_dpp<0x111>(v); // from 1, 2, 4, 8 lanes below in the row of 16
    v = max_dpp<0x112>(v);
    v = max_dpp<0x114>(v);
    v = max_dpp<0x118>(v);
    v = max_dpp<0x142>(v); // the last lane of a row to the next row
    v = max_dpp<0x143>(v); // lane 31 to the upper half
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for(int d = 1; d < 64; d *= 2)
        v += __shfl_xor(v, d, 64);
    return v;
}
// the lowest lane that holds the largest of the numbers (hi, lo); -1: all are 0
template <bool WIDE>
__device__ __forceinline__ int best_lane(uint32_t hi, uint32_t lo)
{
    const uint32_t top = wave_max(hi);
    if(top == 0)
        return -1;
    uint64_t who = __ballot(hi == top);
    if(WIDE && (who & (who - 1)))
    {
        const uint32_t low = wave_max(hi == top ? lo : 0u);
        who                = __ballot(hi == top && lo == low);
    }
    return (int)__builtin_ctzll(who);
}

struct Pick
{
    int expert;
    float x;
};

// WIDE: there are biases. ALL: every expert's score is needed (biases, sums of two in a group, a softmax that is not renormalised).
template <typename X, int EPL, bool WIDE, bool ALL>
__device__ __forceinline__ void route_token(const RouteArgs& p, int64_t t, int lane, double* values, const float (&bias)[EPL], const int (&group)[EPL])
{
    constexpr float kLargest = 3.402823466e38f;
    const X* const row       = reinterpret_cast<const X*>(p.x) + t * p.stride_x;
    float x[EPL];
    uint32_t hi[EPL], lo[EPL];
    bool there[EPL];
    uint32_t most = 0;
#pragma unroll
    for(int i = 0; i < EPL; ++i)
    {
        const int e = lane * EPL + i;
        float v     = e < p.experts ? (float)row[e] : -__builtin_inff();
        there[i]    = v > -__builtin_inff() && bias[i] > -__builtin_inff(); // (a NaN is not)
        x[i]        = there[i] ? __builtin_fminf(v, kLargest) + 0.0f : -__builtin_inff(); // (-0 is 0)
        hi[i]       = there[i] ? rising(x[i]) : 0u;
        lo[i]       = 0;
        most        = hi[i] > most ? hi[i] : most;
    }
    most              = wave_max(most);
    const float x_max = most ? __builtin_bit_cast(float, most & 0x80000000u ? most ^ 0x80000000u : ~most) : 0.0f;
    double total      = 1.0;
    double value[EPL];
    if constexpr(ALL)
    {
        double sum = 0.0;
#pragma unroll
        for(int i = 0; i < EPL; ++i)
        {
            const double d = there[i] ? exp(p.sigmoid ? -(double)x[i] : (double)x[i] - (double)x_max) : 0.0;
            value[i]       = p.sigmoid ? 1.0 / (1.0 + d) : d;
            sum += d;
        }
        if(!p.sigmoid)
        {
            total = wave_sum(sum);
            total = total > 0.0 ? total : 1.0;
#pragma unroll
            for(int i = 0; i < EPL; ++i)
                value[i] /= total;
        }
        if constexpr(WIDE)
#pragma unroll
            for(int i = 0; i < EPL; ++i)
            {
                value[i] += (double)__builtin_fminf(bias[i], kLargest);
                const uint64_t key = there[i] ? rising(value[i]) : 0;
                hi[i] = (uint32_t)(key >> 32), lo[i] = (uint32_t)key;
            }
    }
    if(p.groups > 1)
    {
        const int size = p.experts / p.groups;
#pragma unroll
        for(int i = 0; i < EPL; ++i)
            if(lane * EPL + i < p.experts)
                values[lane * EPL + i] = !there[i] ? -__builtin_inf() : (ALL && (WIDE || p.group_best == 2)) ? value[i] : (double)x[i];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        double first = -__builtin_inf(), second = -__builtin_inf();
        if(lane < p.groups)
            for(int i = 0; i < size; ++i)
            {
                const double v = values[lane * size + i];
                second         = v > first ? first : v > second ? v : second;
                first          = v > first ? v : first;
            }
        __builtin_amdgcn_wave_barrier();
        const bool any     = first > -__builtin_inf();
        const double sum   = p.group_best == 2 && second > -__builtin_inf() ? first + second : first;
        uint64_t key       = any ? rising(sum + 0.0) : 0;
        uint64_t stays     = 0;
        for(int j = 0; j < p.top_groups; ++j)
        {
            const int best = best_lane<true>((uint32_t)(key >> 32), (uint32_t)key);
            if(best < 0)
                break;
            stays |= 1ull << best;
            key = lane == best ? 0 : key;
        }
#pragma unroll
        for(int i = 0; i < EPL; ++i)
            if(!(stays >> group[i] & 1))
                hi[i] = lo[i] = 0;
    }
    // the picks: lane j keeps the j-th
    Pick mine{-1, 0.0f};
    for(int j = 0; j < p.top_k; ++j)
    {
        uint32_t bh = hi[0], bl = lo[0];
        float bx = x[0];
        int at   = 0;
#pragma unroll
        for(int i = 1; i < EPL; ++i)
            if(hi[i] > bh || (WIDE && hi[i] == bh && lo[i] > bl))
                bh = hi[i], bl = lo[i], bx = x[i], at = i;
        const int best = best_lane<WIDE>(bh, bl);
        if(best < 0)
            break;
        const int e   = best * EPL + __builtin_amdgcn_readlane(at, best);
        const float v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, bx), best));
        if(lane == j)
            mine = Pick{e, v};
#pragma unroll
        for(int i = 0; i < EPL; ++i)
            if(lane * EPL + i == e)
                hi[i] = lo[i] = 0;
    }
    double w = 0.0;
    if(mine.expert >= 0)
    {
        const double d = exp(p.sigmoid ? -(double)mine.x : (double)mine.x - (double)x_max);
        w              = p.sigmoid ? 1.0 / (1.0 + d) : d / total;
    }
    if(p.renormalise)
    {
        const double sum = wave_sum(w);
        w                = sum > 0.0 ? w / sum : 0.0;
    }
    if(lane < p.top_k)
    {
        p.ids[t * p.top_k + lane]     = mine.expert;
        p.weights[t * p.top_k + lane] = (float)(w * (double)p.scale);
    }
}

// sums of the counts before each expert, over the workgroup: base[e] for e < experts; returns the sum of all
__device__ __forceinline__ int sums_before(int* base, int count, int experts, int* parts)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int v = count;
#pragma unroll
    for(int d = 1; d < 64; d *= 2)
    {
        const int o = __shfl_up(v, d, 64);
        v += lane >= d ? o : 0;
    }
    if(lane == 63)
        parts[wave] = v;
    __syncthreads();
    int before = 0, all = 0;
    for(int w = 0; w < kWaves; ++w)
    {
        const int n = parts[w];
        before += w < wave ? n : 0;
        all += n;
    }
    if((int)threadIdx.x < experts)
        base[threadIdx.x] = before + v - count;
    __syncthreads();
    return all;
}

// the pairs [from, to) to their places: base[e] is where the next row of expert e goes. 1024 pairs at a time, 64 a wave; cells:
// [kWaves][experts] numbers.
__device__ __forceinline__ void place_pairs(const RouteArgs& p, int64_t from, int64_t to, int* base, int* cells)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int bits = 32 - __builtin_clz(p.experts | 1);
    for(int64_t at = from; at < to; at += kThreads)
    {
        for(int i = threadIdx.x; i < kWaves * p.experts; i += kThreads)
            cells[i] = 0;
        __syncthreads();
        const int64_t pair = at + threadIdx.x;
        const int e        = pair < to ? p.ids[pair] : -1;
        uint64_t same      = __ballot(e >= 0);
        for(int b = 0; b < bits; ++b)
        {
            const uint64_t set = __ballot(e >> b & 1);
            same &= (e >> b & 1) ? set : ~set;
        }
        const int rank = (int)__builtin_popcountll(same & ((1ull << lane) - 1));
        if(e >= 0 && rank == 0)
            cells[wave * p.experts + e] = (int)__builtin_popcountll(same);
        __syncthreads();
        if((int)threadIdx.x < p.experts)
        {
            int next = base[threadIdx.x];
            for(int w = 0; w < kWaves; ++w)
            {
                const int n                          = cells[w * p.experts + threadIdx.x];
                cells[w * p.experts + threadIdx.x] = next;
                next += n;
            }
            base[threadIdx.x] = next;
        }
        __syncthreads();
        if(pair < to)
        {
            const int place = e >= 0 ? cells[wave * p.experts + e] + rank : -1;
            p.places[pair]  = place;
            if(e >= 0)
                p.rows[place] = (int)pair;
        }
        __syncthreads();
    }
}

// LDS: [kWaves][experts] doubles (groups) or numbers (tables)
template <typename X, int EPL, bool WIDE, bool ALL>
__global__ __launch_bounds__(kThreads) void route_kernel(RouteArgs p)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t ckx_route_lds[];
    __shared__ int counts[kMostExperts], parts[kWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t first = (int64_t)blockIdx.x * p.chunk_tokens;
    const int64_t last  = first + p.chunk_tokens < p.tokens ? first + p.chunk_tokens : p.tokens;
    const int live      = p.live ? max(0, min(*p.live, p.tokens)) : p.tokens;
    double* const values = reinterpret_cast<double*>(ckx_route_lds) + wave * p.experts;
    float bias[EPL];
    int group[EPL];
#pragma unroll
    for(int i = 0; i < EPL; ++i)
    {
        const int e = lane * EPL + i;
        bias[i]     = WIDE && e < p.experts ? p.bias[e] : 0.0f;
        group[i]    = p.groups > 1 && e < p.experts ? e / (p.experts / p.groups) : 0;
    }
    if(p.offsets)
    {
        for(int e = threadIdx.x; e < p.experts; e += kThreads)
            counts[e] = 0;
        __syncthreads();
    }
    for(int64_t t = first + wave; t < last; t += kWaves)
    {
        if(t < live)
            route_token<X, EPL, WIDE, ALL>(p, t, lane, values, bias, group);
        else if(lane < p.top_k)
            p.ids[t * p.top_k + lane] = -1, p.weights[t * p.top_k + lane] = 0.0f;
        if(p.offsets && lane < p.top_k)
        {
            const int e = p.ids[t * p.top_k + lane]; // (the lane's own)
            if(e >= 0)
                atomicAdd(&counts[e], 1);
        }
    }
    if(!p.offsets)
        return;
    __syncthreads();
    const int count = (int)threadIdx.x < p.experts ? counts[threadIdx.x] : 0;
    if(p.chunks > 1)
    {
        if((int)threadIdx.x < p.experts)
            p.ws[(int64_t)blockIdx.x * p.experts + threadIdx.x] = count;
        return;
    }
    const int all = sums_before(counts, count, p.experts, parts);
    if((int)threadIdx.x < p.experts)
        p.offsets[threadIdx.x] = counts[threadIdx.x];
    if(threadIdx.x == 0)
        p.offsets[p.experts] = all;
    const int64_t pairs = (int64_t)p.tokens * p.top_k;
    for(int64_t i = all + threadIdx.x; i < pairs; i += kThreads)
        p.rows[i] = -1;
    place_pairs(p, 0, pairs, counts, reinterpret_cast<int*>(ckx_route_lds));
}

__global__ __launch_bounds__(kThreads) void route_tables_kernel(RouteArgs p)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t ckx_route_lds[];
    __shared__ int mine[kMostExperts], totals[kMostExperts], parts[kWaves];
    for(int e = threadIdx.x; e < p.experts; e += kThreads)
        mine[e] = totals[e] = 0;
    __syncthreads();
    // (threads in rows of `wide`, a chunk each)
    int wide = 64;
    while(wide < p.experts)
        wide *= 2;
    const int e = threadIdx.x & (wide - 1);
    if(e < p.experts)
    {
        int before = 0, all = 0;
#pragma unroll 8
        for(int c = threadIdx.x / wide; c < p.chunks; c += kThreads / wide)
        {
            const int n = p.ws[(int64_t)c * p.experts + e];
            before += c < (int)blockIdx.x ? n : 0;
            all += n;
        }
        atomicAdd(&mine[e], before);
        atomicAdd(&totals[e], all);
    }
    __syncthreads();
    const int total = (int)threadIdx.x < p.experts ? totals[threadIdx.x] : 0;
    const int all   = sums_before(totals, total, p.experts, parts);
    if((int)threadIdx.x < p.experts)
    {
        mine[threadIdx.x] += totals[threadIdx.x];
        if(blockIdx.x == 0)
            p.offsets[threadIdx.x] = totals[threadIdx.x];
    }
    if(blockIdx.x == 0 && threadIdx.x == 0)
        p.offsets[p.experts] = all;
    const int64_t pairs = (int64_t)p.tokens * p.top_k, a_chunk = (int64_t)p.chunk_tokens * p.top_k;
    const int64_t from = blockIdx.x * a_chunk, to = from + a_chunk < pairs ? from + a_chunk : pairs;
    for(int64_t i = (from > all ? from : all) + threadIdx.x; i < to; i += kThreads)
        p.rows[i] = -1;
    __syncthreads();
    place_pairs(p, from, to, mine, reinterpret_cast<int*>(ckx_route_lds));
}

template <typename F>
hipError_t allow_lds(F* kernel, size_t bytes)
{
    return bytes > 65536 ? hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes)
                         : hipSuccess;
}

template <typename X, int EPL, bool WIDE, bool ALL>
hipError_t launch(const RouteArgs& a, hipStream_t s)
{
    const size_t cells = a.offsets ? (size_t)kWaves * a.experts * 4 : 0;
    const size_t lds   = a.groups > 1 ? (size_t)kWaves * a.experts * 8 : a.chunks == 1 ? cells : 0;
    hipError_t e       = allow_lds(&route_kernel<X, EPL, WIDE, ALL>, lds);
    if(e != hipSuccess)
        return e;
    hipLaunchKernelGGL((route_kernel<X, EPL, WIDE, ALL>), dim3(a.chunks), dim3(kThreads), lds, s, a);
    e = hipGetLastError();
    if(e != hipSuccess || a.chunks == 1 || !a.offsets)
        return e;
    if((e = allow_lds(&route_tables_kernel, cells)) != hipSuccess)
        return e;
    hipLaunchKernelGGL(route_tables_kernel, dim3(a.chunks), dim3(kThreads), cells, s, a);
    return hipGetLastError();
}

template <typename X, int EPL>
hipError_t launch_form(const RouteArgs& a, hipStream_t s)
{
    if(a.bias)
        return launch<X, EPL, true, true>(a, s);
    const bool all = (a.groups > 1 && a.group_best == 2) || (!a.sigmoid && !a.renormalise);
    return all ? launch<X, EPL, false, true>(a, s) : launch<X, EPL, false, false>(a, s);
}

template <typename X>
hipError_t launch_any(const RouteArgs& a, hipStream_t s)
{
    return a.experts <= 64    ? launch_form<X, 1>(a, s)
           : a.experts <= 128 ? launch_form<X, 2>(a, s)
           : a.experts <= 256 ? launch_form<X, 4>(a, s)
           : a.experts <= 512 ? launch_form<X, 8>(a, s)
                              : launch_form<X, 16>(a, s);
}

void cut(int tokens, int& chunk_tokens, int& chunks)
{
    chunk_tokens = tokens, chunks = 1;
    if(tokens > kOneGroup)
    {
        chunk_tokens = (int)(((int64_t)tokens + kMostChunks - 1) / kMostChunks);
        chunk_tokens = (chunk_tokens + kWaves - 1) / kWaves * kWaves;
        chunks       = (int)(((int64_t)tokens + chunk_tokens - 1) / chunk_tokens);
    }
}

} // namespace

int64_t route_workspace(int tokens, int experts)
{
    int per, chunks;
    cut(tokens, per, chunks);
    return chunks > 1 ? 4ll * chunks * experts : 0;
}

hipError_t route_launch(RouteArgs a, int x_type, hipStream_t s)
{
    cut(a.tokens, a.chunk_tokens, a.chunks);
    return x_type == CKX_TYPE_F32 ? launch_any<float>(a, s) : x_type == CKX_TYPE_F16 ? launch_any<_Float16>(a, s) : launch_any<__bf16>(a, s);
}

} // namespace ckx
