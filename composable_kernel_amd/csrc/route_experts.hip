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

constexpr int kWaves = 8, kThreads = kWaves * 64; // (16 experts a lane take more registers than 16 waves leave)
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

// ---- four tokens a wave: up to 256 experts and 16 picks, groups that are whole lanes -----------------------------------------------
// Sixteen lanes take a token, EPL experts a lane one after the other. Its values stay what they are, fp32 logits where there is no bias
// and 64-bit sums otherwise: the largest of 16 values in a lane is 15 instructions, that of a row of lanes four rotations, and the lowest
// expert of those that hold it another four.
template <int CTRL>
__device__ __forceinline__ int row_dpp(int v)
{
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false);
}
template <int CTRL>
__device__ __forceinline__ float row_dpp(float v)
{
    return __builtin_bit_cast(float, row_dpp<CTRL>(__builtin_bit_cast(int, v)));
}
template <int CTRL>
__device__ __forceinline__ double row_dpp(double v)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)row_dpp<CTRL>((int)(uint32_t)b) | (uint64_t)(uint32_t)row_dpp<CTRL>((int)(uint32_t)(b >> 32)) << 32);
}
__device__ __forceinline__ float most_of(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ double most_of(double a, double b) { return __builtin_fmax(a, b); }
__device__ __forceinline__ float least_of(float a, float b) { return __builtin_fminf(a, b); }
__device__ __forceinline__ double least_of(double a, double b) { return __builtin_fmin(a, b); }
// of the row's sixteen lanes, in all of them (rotations by 8, 4, 2 and 1 lanes)
template <typename V>
__device__ __forceinline__ V row_most(V v)
{
    v = most_of(v, row_dpp<0x128>(v));
    v = most_of(v, row_dpp<0x124>(v));
    v = most_of(v, row_dpp<0x122>(v));
    return most_of(v, row_dpp<0x121>(v));
}
__device__ __forceinline__ int row_least(int v)
{
    v = min(v, row_dpp<0x128>(v));
    v = min(v, row_dpp<0x124>(v));
    v = min(v, row_dpp<0x122>(v));
    return min(v, row_dpp<0x121>(v));
}
__device__ __forceinline__ double row_sum(double v)
{
    v += row_dpp<0x128>(v);
    v += row_dpp<0x124>(v);
    v += row_dpp<0x122>(v);
    return v + row_dpp<0x121>(v);
}

// x[i] = exp(x[i]) in 64 bits: 2^n times the series of exp over half a step to either side of zero, whose term behind the last kept is
// under 2^-52 of the sum. Coefficient by coefficient over all of them, so that each is in a register once and no sum waits for the last;
// the library's function takes three times the instructions, one value after the other.
template <int N>
__device__ __forceinline__ void exp_all(double (&x)[N])
{
    constexpr double c[] = {1.0 / 479001600.0, 1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0,
                            1.0 / 120.0,       1.0 / 24.0,       1.0 / 6.0,       0.5,            1.0,           1.0};
    double y[N];
    int n[N];
#pragma unroll
    for(int i = 0; i < N; ++i)
    {
        x[i]           = __builtin_fmin(__builtin_fmax(x[i], -745.2), 709.78); // (exp of less is 0; of more: the callers look)
        const double m = __builtin_rint(x[i] * 1.4426950408889634074);
        x[i]           = __builtin_fma(-m, 6.93147180369123816490e-01, x[i]); // (ln 2 in two parts)
        x[i]           = __builtin_fma(-m, 1.90821492927058770002e-10, x[i]);
        n[i]           = (int)m;
        y[i]           = 1.0 / 6227020800.0;
    }
#pragma unroll
    for(int k = 0; k < 13; ++k)
#pragma unroll
        for(int i = 0; i < N; ++i)
            y[i] = __builtin_fma(y[i], x[i], c[k]);
#pragma unroll
    for(int i = 0; i < N; ++i)
        x[i] = __builtin_ldexp(y[i], n[i]);
}
// 1 / x for x >= 1: two of Newton's steps from the instruction's estimate
__device__ __forceinline__ double reciprocal(double x)
{
    double y = __builtin_amdgcn_rcp(x);
    y        = __builtin_fma(__builtin_fma(-x, y, 1.0), y, y);
    return __builtin_fma(__builtin_fma(-x, y, 1.0), y, y);
}

// the lane's experts [lane * EPL ... ) of a row of logits, -infinity behind the last
template <typename X, int EPL>
__device__ __forceinline__ void load_logits(const X* row, int first, int experts, float (&x)[EPL])
{
    struct __attribute__((packed)) All
    {
        X v[EPL];
    };
    if(first + EPL <= experts)
    {
        const All a = *reinterpret_cast<const All*>(row + first);
#pragma unroll
        for(int i = 0; i < EPL; ++i)
            x[i] = (float)a.v[i];
    }
    else
#pragma unroll
        for(int i = 0; i < EPL; ++i)
            x[i] = first + i < experts ? (float)row[first + i] : -__builtin_inff();
}

// V: float, there are no biases; double: there are. ALL as above. `live`: of the lane's row of lanes.
template <typename X, int EPL, typename V, bool ALL>
__device__ __forceinline__ void route_tokens(const RouteArgs& p, int64_t t, bool live, int lane, const float (&bias)[EPL], int (&ids)[1])
{
    constexpr bool WIDE      = sizeof(V) == 8;
    constexpr float kLargest = 3.402823466e38f;
    constexpr V kNone        = -(V)__builtin_inff();
    const int first          = lane * EPL;
    const X* const row       = reinterpret_cast<const X*>(p.x) + (live ? t : 0) * p.stride_x;
    float x[EPL];
    load_logits(row, first, p.experts, x);
    auto there = [&](int i) { return x[i] > -__builtin_inff(); };
    float most = -__builtin_inff();
#pragma unroll
    for(int i = 0; i < EPL; ++i)
    {
        x[i] = __builtin_fminf(live && there(i) && bias[i] > -__builtin_inff() ? x[i] : -__builtin_inff(), kLargest); // (a NaN is out)
        most = __builtin_fmaxf(most, x[i]);
    }
    const float x_max = row_most(most);
    V value[EPL];      // by which experts are ordered
    double score[EPL]; // ALL: s, or s + bias
    double total = 1.0;
    if constexpr(ALL)
    {
        // (-infinity, which is out, goes the way of a number: to 0 or behind its own check)
        const double at = p.sigmoid ? 0.0 : (double)__builtin_fmaxf(x_max, -kLargest), sign = p.sigmoid ? -1.0 : 1.0;
#pragma unroll
        for(int i = 0; i < EPL; ++i)
            score[i] = sign * (double)__builtin_fmaxf(x[i], -kLargest) - at;
        exp_all(score);
        if(p.sigmoid)
        {
#pragma unroll
            for(int i = 0; i < EPL; ++i)
                score[i] = x[i] < -709.78f ? 0.0 : reciprocal(1.0 + score[i]); // (the exponential is past the range)
        }
        else
        {
            double sum = 0.0;
#pragma unroll
            for(int i = 0; i < EPL; ++i)
            {
                score[i] = there(i) ? score[i] : 0.0;
                sum += score[i];
            }
            total            = row_sum(sum);
            total            = total > 0.0 ? total : 1.0;
            const double one = reciprocal(total); // (at least 1, the largest's own)
#pragma unroll
            for(int i = 0; i < EPL; ++i)
                score[i] *= one;
        }
    }
#pragma unroll
    for(int i = 0; i < EPL; ++i)
    {
        if constexpr(WIDE)
        {
            score[i] += (double)__builtin_fminf(bias[i], kLargest);
            value[i] = there(i) ? score[i] : kNone;
        }
        else
            value[i] = x[i];
    }
    if(p.groups > 1)
    {
        // the group's lanes all come to hold its value
        const int lanes = p.experts / p.groups / EPL, mine = lane / lanes;
        auto best_two   = [&](auto of) {
            using S  = decltype(of(0));
            S a = -(S)__builtin_inff(), b = -(S)__builtin_inff();
            auto with = [&](S v) {
                b = most_of(b, least_of(a, v));
                a = most_of(a, v);
            };
#pragma unroll
            for(int i = 0; i < EPL; ++i)
                with(of(i));
            // another lane's two: both go in
            auto other = [&](S c, S d) {
                with(c);
                with(d);
            };
            if(lanes > 1)
                other(row_dpp<0xb1>(a), row_dpp<0xb1>(b)); // the neighbour in a pair of lanes
            if(lanes > 2)
                other(row_dpp<0x4e>(a), row_dpp<0x4e>(b)); // the other pair of four
            if(lanes > 4)
                other(row_dpp<0x141>(a), row_dpp<0x141>(b)); // eight lanes mirrored: the other four
            return p.group_best == 2 && b > -(S)__builtin_inff() ? (double)(a + b) : (double)a;
        };
        double of;
        if constexpr(ALL && !WIDE)
            of = p.group_best == 2 ? best_two([&](int i) { return there(i) ? score[i] : -__builtin_inf(); }) : best_two([&](int i) { return (double)value[i]; });
        else
            of = best_two([&](int i) { return value[i]; });
        bool stays = false;
        for(int j = 0; j < p.top_groups; ++j)
        {
            const double top = row_most(of);
            const int which  = row_least(of == top ? mine : 64);
            const bool won   = which == mine && top > -__builtin_inf();
            stays |= won;
            of = won ? -__builtin_inf() : of;
        }
#pragma unroll
        for(int i = 0; i < EPL; ++i)
            value[i] = stays ? value[i] : kNone;
    }
    // the picks: lane j keeps the j-th
    int expert = -1;
    for(int j = 0; j < p.top_k; ++j)
    {
        V best = value[0];
#pragma unroll
        for(int i = 1; i < EPL; ++i)
            best = most_of(best, value[i]);
        const V top = row_most(best);
        int at      = kMostExperts;
#pragma unroll
        for(int i = EPL - 1; i >= 0; --i)
            at = value[i] == top ? first + i : at;
        const int e = row_least(at);
        if(lane == j && top > kNone)
            expert = e;
#pragma unroll
        for(int i = 0; i < EPL; ++i)
            value[i] = first + i == e ? kNone : value[i];
    }
    double w = 0.0;
    if(expert >= 0)
    {
        const float v  = __builtin_fminf((float)row[expert], kLargest);
        const double d = exp(p.sigmoid ? -(double)v : (double)v - (double)x_max);
        w              = p.sigmoid ? 1.0 / (1.0 + d) : d / total;
    }
    if(p.renormalise)
    {
        const double sum = row_sum(w);
        w                = sum > 0.0 ? w / sum : 0.0;
    }
    ids[0] = expert;
    if(t < p.tokens && lane < p.top_k)
    {
        p.ids[t * p.top_k + lane]     = expert;
        p.weights[t * p.top_k + lane] = (float)(w * (double)p.scale);
    }
}

// whether the kernel of four tokens a wave takes a call, EPL experts a lane
int row_experts(const RouteArgs& a)
{
    int epl = 1;
    while(epl * 16 < a.experts)
        epl *= 2;
    const int size = a.experts / a.groups, lanes = size / epl;
    const bool whole = a.groups == 1 || (size % epl == 0 && (lanes & (lanes - 1)) == 0 && lanes <= 8);
    return epl <= 16 && a.top_k <= 16 && whole ? epl : 0;
}

// base[e]: from the counts of each expert to the sums of those before it, over the workgroup; returns the sum of all
__device__ __forceinline__ int sums_before(int* base, int experts, int* parts)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int all = 0;
    for(int e0 = 0; e0 < experts; e0 += kThreads)
    {
        const int e     = e0 + (int)threadIdx.x;
        const int count = e < experts ? base[e] : 0;
        int v           = count;
#pragma unroll
        for(int d = 1; d < 64; d *= 2)
        {
            const int o = __shfl_up(v, d, 64);
            v += lane >= d ? o : 0;
        }
        if(lane == 63)
            parts[wave] = v;
        __syncthreads();
        int before = all;
        for(int w = 0; w < kWaves; ++w)
        {
            const int n = parts[w];
            before += w < wave ? n : 0;
            all += n;
        }
        if(e < experts)
            base[e] = before + v - count;
        __syncthreads();
    }
    return all;
}

// the pairs [from, to) to their places: base[e] is where the next row of expert e goes. 512 pairs at a time, 64 a wave; cells:
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
        for(int x = threadIdx.x; x < p.experts; x += kThreads)
        {
            int n[kWaves], next = base[x];
#pragma unroll
            for(int w = 0; w < kWaves; ++w)
                n[w] = cells[w * p.experts + x];
#pragma unroll
            for(int w = 0; w < kWaves; ++w)
            {
                cells[w * p.experts + x] = next;
                next += n[w];
            }
            base[x] = next;
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

// ROWS: four tokens a wave. LDS: [kWaves][experts] doubles (one token a wave, groups) or numbers (tables)
template <typename X, bool ROWS, int EPL, bool WIDE, bool ALL>
__global__ __launch_bounds__(kThreads) void route_kernel(RouteArgs p)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t ckx_route_lds[];
    __shared__ int counts[kMostExperts], parts[kWaves];
    const int lane = threadIdx.x & (ROWS ? 15 : 63), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t first = (int64_t)blockIdx.x * p.chunk_tokens;
    const int64_t last  = first + p.chunk_tokens < p.tokens ? first + p.chunk_tokens : p.tokens;
    const int live      = p.live ? max(0, min(*p.live, p.tokens)) : p.tokens;
    double* const values = reinterpret_cast<double*>(ckx_route_lds) + wave * p.experts;
    float bias[EPL] = {};
    int group[EPL];
    if constexpr(WIDE)
        load_logits(p.bias, lane * EPL, p.experts, bias);
#pragma unroll
    for(int i = 0; i < EPL; ++i)
    {
        const int e = lane * EPL + i;
        group[i]    = !ROWS && p.groups > 1 && e < p.experts ? e / (p.experts / p.groups) : 0;
    }
    if(p.offsets)
    {
        for(int e = threadIdx.x; e < p.experts; e += kThreads)
            counts[e] = 0;
        __syncthreads();
    }
    if constexpr(ROWS)
        for(int64_t t0 = first + wave * 4; t0 < last; t0 += kWaves * 4)
        {
            const int64_t t = t0 + (threadIdx.x >> 4 & 3);
            int expert[1];
            route_tokens<X, EPL, typename std::conditional<WIDE, double, float>::type, ALL>(p, t < last ? t : p.tokens, t < last && t < live, lane, bias, expert);
            if(p.offsets && expert[0] >= 0)
                atomicAdd(&counts[expert[0]], 1);
        }
    else
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
    if(p.chunks > 1)
    {
        for(int e = threadIdx.x; e < p.experts; e += kThreads)
            p.ws[(int64_t)blockIdx.x * p.experts + e] = counts[e];
        return;
    }
    const int all = sums_before(counts, p.experts, parts);
    for(int e = threadIdx.x; e < p.experts; e += kThreads)
        p.offsets[e] = counts[e];
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
    // (threads in rows of `wide`, a chunk each, four experts a thread)
    int wide = 16;
    while(wide * 4 < p.experts)
        wide *= 2;
    const int e0 = (threadIdx.x & (wide - 1)) * 4, per = kThreads / wide;
    if(e0 < p.experts)
    {
        const int left = p.experts - e0;
        i32x4 before = {0, 0, 0, 0}, all = {0, 0, 0, 0};
#pragma unroll 8
        for(int c = threadIdx.x / wide; c < p.chunks; c += per)
        {
            const int* at = p.ws + (int64_t)c * p.experts + e0;
            i32x4 n       = {0, 0, 0, 0};
            if(left >= 4)
                n = load_vec<i32x4>(at);
            else
                n = i32x4{at[0], left > 1 ? at[1] : 0, left > 2 ? at[2] : 0, 0};
            before += c < (int)blockIdx.x ? n : i32x4{0, 0, 0, 0};
            all += n;
        }
#pragma unroll
        for(int i = 0; i < 4; ++i)
            if(i < left)
            {
                atomicAdd(&mine[e0 + i], before[i]);
                atomicAdd(&totals[e0 + i], all[i]);
            }
    }
    __syncthreads();
    const int all = sums_before(totals, p.experts, parts);
    for(int e = threadIdx.x; e < p.experts; e += kThreads)
    {
        mine[e] += totals[e];
        if(blockIdx.x == 0)
            p.offsets[e] = totals[e];
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

template <typename X, bool ROWS, int EPL, bool WIDE, bool ALL>
hipError_t launch(const RouteArgs& a, hipStream_t s)
{
    const size_t cells = a.offsets ? (size_t)kWaves * a.experts * 4 : 0;
    const size_t lds   = !ROWS && a.groups > 1 ? (size_t)kWaves * a.experts * 8 : a.chunks == 1 ? cells : 0;
    hipError_t e       = allow_lds(&route_kernel<X, ROWS, EPL, WIDE, ALL>, lds);
    if(e != hipSuccess)
        return e;
    hipLaunchKernelGGL((route_kernel<X, ROWS, EPL, WIDE, ALL>), dim3(a.chunks), dim3(kThreads), lds, s, a);
    e = hipGetLastError();
    if(e != hipSuccess || a.chunks == 1 || !a.offsets)
        return e;
    if((e = allow_lds(&route_tables_kernel, cells)) != hipSuccess)
        return e;
    hipLaunchKernelGGL(route_tables_kernel, dim3(a.chunks), dim3(kThreads), cells, s, a);
    return hipGetLastError();
}

template <typename X, bool ROWS, int EPL>
hipError_t launch_form(const RouteArgs& a, hipStream_t s)
{
    if(a.bias)
        return launch<X, ROWS, EPL, true, true>(a, s);
    const bool all = (a.groups > 1 && a.group_best == 2) || (!a.sigmoid && !a.renormalise);
    return all ? launch<X, ROWS, EPL, false, true>(a, s) : launch<X, ROWS, EPL, false, false>(a, s);
}

template <typename X>
hipError_t launch_any(const RouteArgs& a, hipStream_t s)
{
    switch(row_experts(a))
    {
    case 1: return launch_form<X, true, 1>(a, s);
    case 2: return launch_form<X, true, 2>(a, s);
    case 4: return launch_form<X, true, 4>(a, s);
    case 8: return launch_form<X, true, 8>(a, s);
    case 16: return launch_form<X, true, 16>(a, s);
    default: break;
    }
    return a.experts <= 256 ? launch_form<X, false, 4>(a, s) : launch_form<X, false, 16>(a, s);
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
