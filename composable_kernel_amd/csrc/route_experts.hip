// Each token's experts, their weights, and the experts' rows in order (formula: include/ckx.h, ckx_route_experts).
//
// A wave takes a token; lane l holds the experts l * EPL ... l * EPL + EPL - 1, so that the lowest lane of a tie has the lowest
// expert. What decides the order is compared as whole numbers that rise with the value: the bits of the fp32 logit where there is no
// bias (both scores rise with it), those of the 64-bit sum of score and bias otherwise, whose upper halves settle all but ties. A pick
// is one maximum over the wave.
// The tables are a stable counting sort of the tokens * top_k pairs. For few tokens one workgroup does all of it; otherwise
// each workgroup leaves the counts of its tokens in the workspace and a second launch adds them up and places the pairs. Nothing in it depends on
// the order in which waves run.
// 16384 tokens of 256 experts, sigmoid, biases, groups, eight each: 27.4 to 30 us, of them 19 to 21 for the scores and picks (1690 vector instructions a wave of
// four tokens, 40 % of the cycles, the rest their order) and 8.5 for the tables; 64 experts 14.2, one token 5.7 with its launch.
#include "experts.hpp"
#include "f8.hpp"

namespace ckx {

namespace {

constexpr int kWaves = 16, kThreads = kWaves * 64; // of a workgroup, at most
constexpr int kTableWaves = 8, kTableThreads = kTableWaves * 64;
constexpr int kOneGroup = 64, kMostChunks = 256;
__host__ __device__ constexpr int counts_row(int experts, bool bytes) { return bytes ? (experts + 15) / 16 : (experts + 3) / 4; } // in pieces of 16 bytes
constexpr int kByteCount = 255; // tokens of a workgroup up to which its counts are bytes (an expert has a token once)

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

struct Pick
{
    int expert;
    float x;
};

// WIDE: there are biases. ALL: every expert's score is needed (biases, sums of two in a group, a softmax that is not renormalised).
template <typename X, int EPL, bool WIDE, bool ALL>
__device__ __forceinline__ int route_token(const RouteArgs& p, int64_t t, int lane, double* values)
{
    constexpr float kLargest = 3.402823466e38f;
    const X* const row       = reinterpret_cast<const X*>(p.x) + t * p.stride_x;
    float x[EPL], bias[EPL] = {};
    if constexpr(WIDE)
        load_logits(p.bias, lane * EPL, p.experts, bias);
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
            if(!(stays >> min((lane * EPL + i) / size, 63) & 1))
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
    return mine.expert;
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
__device__ __forceinline__ uint32_t row_dpp(uint32_t v)
{
    return (uint32_t)row_dpp<CTRL>((int)v);
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
__device__ __forceinline__ uint32_t most_of(uint32_t a, uint32_t b) { return max(a, b); }
__device__ __forceinline__ float most_of(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ double most_of(double a, double b) { return __builtin_fmax(a, b); }
__device__ __forceinline__ float least_of(float a, float b) { return __builtin_fminf(a, b); }
__device__ __forceinline__ double least_of(double a, double b) { return __builtin_fmin(a, b); }
// keys that are `gone` become 0. Comparisons first: a mask that the instruction before has written costs two waits, which the compiler's
// pairs of comparison and choice pay for each key.
__device__ __forceinline__ void clear_four(uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d, uint32_t gone)
{
    uint64_t m0, m1, m2, m3;
    asm("v_cmp_ne_u32_e64 %4, %0, %8\n\tv_cmp_ne_u32_e64 %5, %1, %8\n\tv_cmp_ne_u32_e64 %6, %2, %8\n\tv_cmp_ne_u32_e64 %7, %3, %8\n\t"
        "v_cndmask_b32_e64 %0, 0, %0, %4\n\tv_cndmask_b32_e64 %1, 0, %1, %5\n\tv_cndmask_b32_e64 %2, 0, %2, %6\n\tv_cndmask_b32_e64 %3, 0, %3, %7"
        : "+v"(a), "+v"(b), "+v"(c), "+v"(d), "=&s"(m0), "=&s"(m1), "=&s"(m2), "=&s"(m3)
        : "v"(gone));
}
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
template <typename V>
__device__ __forceinline__ V row_sum(V v)
{
    v += row_dpp<0x128>(v);
    v += row_dpp<0x124>(v);
    v += row_dpp<0x122>(v);
    return v + row_dpp<0x121>(v);
}

// groups of the row that stand before the lane's own, `lanes` lanes each
__device__ __forceinline__ int groups_before(float of, int group, int lanes)
{
    int before = 0;
    static_for<15>([&](auto r) {
        constexpr int BY = decltype(r)::value + 1;
        if((BY & (lanes - 1)) == 0)
        {
            const float v = row_dpp<0x120 + BY>(of);
            const int g   = row_dpp<0x120 + BY>(group);
            before += (int)(v > of) | ((int)(v == of) & (int)(g < group));
        }
    });
    return before;
}
// the best and the next of a group of `lanes` lanes, from the lane's own
template <typename V>
__device__ __forceinline__ void group_two(V& best, V& next, int lanes)
{
    auto with = [&](V c, V d) {
        next = most_of(most_of(next, d), least_of(best, c));
        best = most_of(best, c);
    };
    if(lanes > 1)
        with(row_dpp<0xb1>(best), row_dpp<0xb1>(next)); // the neighbour in a pair of lanes
    if(lanes > 2)
        with(row_dpp<0x4e>(best), row_dpp<0x4e>(next)); // the other pair of four
    if(lanes > 4)
        with(row_dpp<0x141>(best), row_dpp<0x141>(next)); // eight lanes mirrored: the other four
}
template <typename V, int EPL>
__device__ __forceinline__ V group_value(const RouteArgs& p, const V (&v)[EPL], int lanes)
{
    constexpr V kNone = -(V)__builtin_inff(), kLowest = (V)-3.402823466e38f;
    V best = kNone, next = kNone;
#pragma unroll
    for(int i = 0; i < EPL; ++i)
    {
        next = most_of(next, least_of(best, v[i]));
        best = most_of(best, v[i]);
    }
    group_two(best, next, lanes);
    // (two biases near the type's lowest value, as masks have them, are past it together: the group is there all the same. Its order among such
    // groups is in doubt, since the room that their sums are given is infinite)
    return p.group_best == 2 && next > kNone ? most_of(best + next, kLowest) : best;
}

// WIDE and ALL as above; `live`: of the lane's row of lanes. Scores in fp32 find the token's experts; those, one a lane, are computed in
// 64 bits (their weights need that anyway), one more than asked for, and put in order by them; the last that counts has to lie further above
// the next expert, and the groups that stay above the others, than the fp32 scores may be off. Where one does not, the row is `in_doubt`,
// nothing is written, and the wave takes the token by itself (route_token): one 4.5 us at the end of a launch; all of 16384 tokens of 256 experts (a peaked softmax with
// biases of zero) 51 us, none 28.
// How far: sigmoid, with t = exp(-x) off by (|x| + 3) 2^-24 of itself (x log2 e rounded, the power of two, its rounding) and s (1 - s) |x|
// under 0.23, s is off by less than 4 * 2^-24; softmax, p |x - max| under 0.37, and the sum of at most 16 + 4 terms in a row off by 20 *
// 2^-24: 27 * 2^-24; and half a step each for the biases' and the groups' sums.
// any_off: there are biases that are -infinity or no numbers.
template <typename X, int EPL, bool WIDE, bool ALL>
__device__ __forceinline__ int route_tokens(const RouteArgs& p, const X* row, float (&x)[EPL], int64_t t, bool live, int lane, const float (&bias)[EPL], bool any_off,
                                            uint64_t& doubt)
{
    constexpr float kLargest = 3.402823466e38f, kNone = -__builtin_inff();
    const int first = lane * EPL;
    if(WIDE && any_off)
#pragma unroll
        for(int i = 0; i < EPL; ++i)
            x[i] = bias[i] > kNone ? x[i] : kNone;
    float most = kNone;
#pragma unroll
    for(int i = 0; i < EPL; ++i)
        most = __builtin_fmaxf(most, x[i]);
    const float x_max = row_most(most);
    bool in_doubt     = x_max > kLargest; // (infinities are what the definition makes of them)
    const float off   = p.sigmoid ? 0x1p-21f : 0x1p-19f; // of a score
    float value[EPL];                                    // by which experts are ordered
    float score[EPL];                                    // s, or s + bias; -infinity: not available (a NaN is not)
    float total = 1.0f;
    if constexpr(ALL)
    {
        constexpr float kLog2e = 1.4426950408889634f;
        if(p.sigmoid)
        {
#pragma unroll
            for(int i = 0; i < EPL; ++i)
            {
                const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x[i] * -kLog2e)) + bias[i];
                score[i]      = x[i] > kNone ? s : kNone;
            }
        }
        else
        {
            const float at = __builtin_fmaxf(x_max, -kLargest);
            float sum      = 0.0f;
#pragma unroll
            for(int i = 0; i < EPL; ++i)
            {
                score[i] = x[i] > kNone ? __builtin_amdgcn_exp2f((x[i] - at) * kLog2e) : 0.0f;
                sum += score[i];
            }
            total           = row_sum(sum);
            const float one = __builtin_amdgcn_rcpf(total);
#pragma unroll
            for(int i = 0; i < EPL; ++i)
                score[i] = x[i] > kNone ? score[i] * one + bias[i] : kNone;
        }
    }
#pragma unroll
    for(int i = 0; i < EPL; ++i)
        value[i] = WIDE ? score[i] : (x[i] > kNone ? x[i] + 0.0f : kNone); // (-0 is 0)
    if(p.groups > 1)
    {
        const int lanes   = p.experts / p.groups / EPL, mine = lane / lanes;
        const bool by_sum = ALL && !WIDE && p.group_best == 2;
        float of;
        if(by_sum)
            of = group_value(p, score, lanes);
        else
            of = group_value(p, value, lanes);
        const bool stays = (int)(of > kNone) & (int)(groups_before(of, mine, lanes) < p.top_groups);
        if(WIDE || by_sum)
        {
            const float low = -row_most(stays ? -of : kNone), high = row_most(stays ? kNone : of);
            in_doubt |= !(low - high > 4 * off + 0x1p-20f * (__builtin_fabsf(low) + __builtin_fabsf(high))) && high > kNone;
        }
#pragma unroll
        for(int i = 0; i < EPL; ++i)
            value[i] = stays ? value[i] : kNone;
    }
    // the picks: lane j keeps the j-th. Keys rise with the value but for its last four bits, whose place the expert's number in its lane
    // takes (the lower one above); lanes compare them without it. Keys up to that of -infinity stand for none.
    constexpr uint32_t kNoKey = 0x007fffffu;
    uint32_t key[EPL], next;
#pragma unroll
    for(int i = 0; i < EPL; ++i)
        key[i] = (rising(value[i]) & ~15u) | (uint32_t)(15 - i);
    auto most_key = [&]() {
        uint32_t best = key[0];
#pragma unroll
        for(int i = 1; i < EPL; ++i)
            best = max(best, key[i]);
        return best;
    };
    const int picks = min(p.top_k + 1, 16); // (one more than asked for, which has to prove to be the next)
    int expert      = -1;
    for(int j = 0; j < picks; ++j)
    {
        const uint32_t best = most_key();
        next                = row_most(best | 15u);
        const int mine      = (best | 15u) == next ? first + 15 - (int)(best & 15u) : kMostExperts;
        const int e         = row_least(mine);
        expert              = (int)(lane == j) & (int)(next > kNoKey) ? e : expert;
        const uint32_t gone = mine == e ? best : 0u;
#pragma unroll
        for(int i = 0; i + 3 < EPL; i += 4)
            clear_four(key[i], key[i + 1], key[i + 2], key[i + 3], gone);
        if constexpr(EPL < 4)
#pragma unroll
            for(int i = 0; i < EPL; ++i)
                key[i] = key[i] == gone ? 0u : key[i];
    }
    next                = row_most(most_key() | 15u); // of what is left
    const bool any_next = next > kNoKey;
    const float above   = __builtin_bit_cast(float, next & 0x80000000u ? next ^ 0x80000000u : ~next); // the most that its value can be
    expert              = live ? expert : -1;
    const float v  = expert >= 0 ? __builtin_fminf((float)row[expert], kLargest) : 0.0f;
    const double d = exp(p.sigmoid ? -(double)v : (double)v - (double)x_max);
    const double s = expert < 0 ? 0.0 : p.sigmoid ? 1.0 / (1.0 + d) : d / (double)total; // (the softmax's fp32 sum leaves the weights, which are renormalised)
    int place      = lane; // among the picks
    if(WIDE || sizeof(X) == 4) // (16-bit logits: a key holds all of them, ties are in their order)
    {
        const double mine   = expert < 0 ? -__builtin_inf() : WIDE ? s + (double)__builtin_fminf(p.bias[expert], kLargest) : (double)v;
        const double room   = WIDE ? (double)off + 0x1p-22 * __builtin_fabs((double)above) : 0.0, slack = WIDE && !p.sigmoid ? 2 * (double)off : 0.0;
        const double before = row_dpp<0x121>(mine); // (the lane below; the first has none)
        const int number    = row_dpp<0x121>(expert);
        const bool turned   = (int)(lane > 0) & (int)(expert >= 0) & ((int)(mine > before - slack) | ((int)(mine == before) & (int)(expert < number)));
        if(__ballot(turned) != 0)
        {
            if(WIDE && !p.sigmoid)
                in_doubt |= turned; // (these values are no better than the sum)
            else
            {
                int rank = 0;
                static_for<15>([&](auto r) {
                    const double o = row_dpp<0x121 + decltype(r)::value>(mine);
                    const int n    = row_dpp<0x121 + decltype(r)::value>(expert);
                    rank += (int)(n >= 0) & ((int)(o > mine) | ((int)(o == mine) & (int)(n < expert)));
                });
                place = expert >= 0 ? rank : lane;
            }
        }
        in_doubt |= (int)(place == p.top_k - 1) & (int)any_next & (int)!(mine > (double)above + room);
    }
    const bool picked = place < p.top_k && lane < picks;
    doubt           = __ballot((int)in_doubt & (int)live);
    const bool mean = (doubt >> (threadIdx.x & 48) & 0xffff) != 0;
    double w        = picked ? s : 0.0;
    if(p.renormalise)
    {
        const double sum = row_sum(w);
        w                = sum > 0.0 ? w / sum : 0.0;
    }
    if(t < p.tokens && picked && !mean)
    {
        p.ids[t * p.top_k + place]     = expert;
        p.weights[t * p.top_k + place] = (float)(w * (double)p.scale);
    }
    return mean || !picked ? -1 : expert;
}

// whether the kernel of four tokens a wave takes a call, EPL experts a lane
int row_experts(const RouteArgs& a)
{
    int epl = 1;
    while(epl * 16 < a.experts)
        epl *= 2;
    const int size = a.experts / a.groups, lanes = size / epl;
    const bool whole = a.groups == 1 || (size % epl == 0 && (lanes & (lanes - 1)) == 0 && lanes <= 8);
    // (a softmax that is not renormalised needs its sum in 64 bits)
    return epl <= 16 && a.top_k <= 16 && whole && (a.sigmoid || a.renormalise) ? epl : 0;
}

// base[e]: from the counts of each expert to the sums of those before it, over the workgroup; returns the sum of all
__device__ __forceinline__ int sums_before(int* base, int experts, int* parts, int waves)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int all = 0;
    for(int e0 = 0; e0 < experts; e0 += waves * 64)
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
        for(int w = 0; w < waves; ++w)
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

// the pairs [from, to) to their places: base[e] is where the next row of expert e goes. 64 pairs a wave at a time; cells: [waves][experts]
// numbers.
__device__ __forceinline__ void place_pairs(const RouteArgs& p, int from, int to, int* base, int* cells, int waves)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int bits = 32 - __builtin_clz(p.experts | 1);
    for(int at = from; at < to; at += waves * 64)
    {
        const int pair = at + (int)threadIdx.x, e = pair < to ? p.ids[pair] : -1;
        for(int i = threadIdx.x; i < waves * p.experts; i += waves * 64)
            cells[i] = 0;
        __syncthreads();
        uint64_t same = __ballot(e >= 0);
#pragma unroll 1
        for(int b = 0; b < bits; ++b)
        {
            const uint64_t set = __ballot(e >> b & 1);
            same &= (e >> b & 1) ? set : ~set;
        }
        const int rank = (int)__builtin_popcountll(same & ((1ull << lane) - 1));
        if(e >= 0 && rank == 0)
            cells[wave * p.experts + e] = (int)__builtin_popcountll(same);
        __syncthreads();
        for(int x = threadIdx.x; x < p.experts; x += waves * 64)
        {
            int next = base[x];
#pragma unroll 1
            for(int* c = cells + x; c < cells + waves * p.experts; c += p.experts)
            {
                const int n = *c;
                *c          = next;
                next += n;
            }
            base[x] = next;
        }
        __syncthreads();
        if(pair < to)
        {
            const int place = e >= 0 ? cells[wave * p.experts + e] + rank : -1;
            p.places[pair]  = place;
            if(e >= 0)
                p.rows[place] = pair;
        }
        __syncthreads();
    }
}

// ROWS: four tokens a wave. LDS: [waves][experts] doubles (groups) or numbers (tables)
template <typename X, bool ROWS, int EPL, bool WIDE, bool ALL>
__global__ __launch_bounds__(kThreads) void route_kernel(RouteArgs p)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t ckx_route_lds[];
    __shared__ int counts[kMostExperts], parts[kWaves];
    const int waves = (int)blockDim.x / 64;
    const int lane = threadIdx.x & (ROWS ? 15 : 63), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t first = (int64_t)blockIdx.x * p.chunk_tokens;
    const int64_t last  = first + p.chunk_tokens < p.tokens ? first + p.chunk_tokens : p.tokens;
    const int live      = p.live ? max(0, min(*p.live, p.tokens)) : p.tokens;
    double* const values = reinterpret_cast<double*>(ckx_route_lds) + wave * p.experts;
    auto count = [&](int e) {
        if(p.offsets && e >= 0)
            atomicAdd(&counts[e], 1);
    };
    auto clear = [&]() {
        if(!p.offsets)
            return;
        for(int e = threadIdx.x; e < p.experts; e += waves * 64)
            counts[e] = 0;
        __syncthreads();
    };
    if constexpr(ROWS)
    {
        // (the first logits are asked for before anything is waited for; rows of lanes without a token read the first one's)
        const int l64     = threadIdx.x & 63;
        auto row_of       = [&](int64_t t) { return reinterpret_cast<const X*>(p.x) + (t < last ? t : first) * p.stride_x; };
        float bias[EPL]   = {}, x[EPL];
        int64_t t         = first + wave * 4 + (l64 >> 4);
        load_logits(row_of(t), lane * EPL, p.experts, x);
        if constexpr(WIDE)
            load_logits(p.bias, lane * EPL, p.experts, bias);
        clear();
        bool off = false;
        if constexpr(WIDE)
#pragma unroll
            for(int i = 0; i < EPL; ++i)
            {
                off |= !(bias[i] > -__builtin_inff());
                bias[i] = bias[i] > 3.402823466e38f ? 3.402823466e38f : bias[i]; // (a NaN stays one)
            }
        const bool any_off = __ballot(off) != 0;
        for(int64_t t0 = first + wave * 4; t0 < last; t0 += waves * 4, t += waves * 4)
        {
            uint64_t doubt;
            count(route_tokens<X, EPL, WIDE, ALL>(p, row_of(t), x, t < last ? t : p.tokens, t < last && t < live, lane, bias, any_off, doubt));
            for(int row = 0; row < 4; ++row)
                if(doubt >> (16 * row) & 0xffff)
                    count(route_token<X, (EPL + 3) / 4, WIDE, ALL>(p, t0 + row, l64, values));
            if(t0 + waves * 4 < last)
                load_logits(row_of(t + waves * 4), lane * EPL, p.experts, x);
        }
    }
    else
    {
        clear();
        for(int64_t t = first + wave; t < last; t += waves)
        {
            if(t < live)
                count(route_token<X, EPL, WIDE, ALL>(p, t, lane, values));
            else if(lane < p.top_k)
                p.ids[t * p.top_k + lane] = -1, p.weights[t * p.top_k + lane] = 0.0f;
        }
    }
    if(!p.offsets)
        return;
    __syncthreads();
    if(p.chunks > 1)
    {
        const bool bytes = p.chunk_tokens <= kByteCount;
        uint8_t* const to = static_cast<uint8_t*>(p.ws) + (int64_t)blockIdx.x * counts_row(p.experts, bytes) * 16;
        for(int e = threadIdx.x; e < p.experts; e += waves * 64)
        {
            if(bytes)
                to[e] = (uint8_t)counts[e];
            else
                reinterpret_cast<int*>(to)[e] = counts[e];
        }
        return;
    }
    const int all = sums_before(counts, p.experts, parts, waves);
    for(int e = threadIdx.x; e < p.experts; e += waves * 64)
        p.offsets[e] = counts[e];
    if(threadIdx.x == 0)
        p.offsets[p.experts] = all;
    const int pairs = p.tokens * p.top_k;
    for(int i = all + threadIdx.x; i < pairs; i += waves * 64)
        p.rows[i] = -1;
    place_pairs(p, 0, pairs, counts, reinterpret_cast<int*>(ckx_route_lds), waves);
}

// The counts of all workgroups' tokens are asked for in pieces of 16 bytes, a few a thread and all of them at once: the launch before wrote them through
// other XCDs' L2s, so that each round of loads takes as long as memory. Bytes are added in pairs of 16 bits (an expert has at most
// kMostChunks * kByteCount tokens).
template <bool BYTES>
__global__ __launch_bounds__(kTableThreads) void route_tables_kernel(RouteArgs p)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t ckx_route_lds[]; // [kTableWaves][experts]
    __shared__ int mine[kMostExperts], totals[kMostExperts], parts[kTableWaves];
    constexpr int N = BYTES ? 8 : 4; // sums of a piece
    const int pairs = p.tokens * p.top_k, a_chunk = p.chunk_tokens * p.top_k;
    const int from = blockIdx.x * a_chunk, to = min(from + a_chunk, pairs);
    const int row = counts_row(p.experts, BYTES);
    for(int i = threadIdx.x; i < row * N; i += kTableThreads)
        mine[i] = totals[i] = 0;
    int wide = 0; // threads that a row of counts takes, a power of two
    while(1 << wide < row)
        ++wide;
    const int piece = threadIdx.x & ((1 << wide) - 1), step = kTableThreads >> wide;
    __syncthreads();
    if(piece < row) // (lanes of the same piece are all in or out)
    {
        int before[N] = {}, all[N] = {};
        const u32x4* at = reinterpret_cast<const u32x4*>(p.ws) + piece;
#pragma unroll 8
        for(int c = threadIdx.x >> wide; c < p.chunks; c += step)
        {
            const u32x4 w    = at[c * row];
            const uint32_t m = c < (int)blockIdx.x ? ~0u : 0u;
#pragma unroll
            for(int i = 0; i < N; ++i)
            {
                const uint32_t v = BYTES ? (w[i / 2] >> (8 * (i & 1))) & 0x00ff00ffu : w[i & 3];
                all[i] += v;
                before[i] += v & m;
            }
        }
        // (the lanes of a wave that hold the same piece first: one address takes one of them at a time)
        for(int d = 1 << wide; d < 64; d *= 2)
#pragma unroll
            for(int i = 0; i < N; ++i)
            {
                all[i] += __shfl_xor(all[i], d, 64);
                before[i] += __shfl_xor(before[i], d, 64);
            }
        if((threadIdx.x & 63) >> min(wide, 6) == 0)
#pragma unroll
            for(int i = 0; i < N; ++i)
            {
                atomicAdd(&totals[piece * N + i], all[i]);
                atomicAdd(&mine[piece * N + i], before[i]);
            }
    }
    __syncthreads();
    if constexpr(BYTES)
    {
        // (the pairs apart: expert e in half e / 2 % 2 of sum e / 4 * 2 + e % 2)
        int a[kMostExperts / kTableThreads], b[kMostExperts / kTableThreads];
#pragma unroll
        for(int i = 0; i < kMostExperts / kTableThreads; ++i)
        {
            const int e = threadIdx.x + i * kTableThreads, k = min(e / 4 * 2 + e % 2, row * N - 1), by = e / 2 % 2 * 16;
            a[i] = mine[k] >> by & 0xffff, b[i] = totals[k] >> by & 0xffff;
        }
        __syncthreads();
#pragma unroll
        for(int i = 0; i < kMostExperts / kTableThreads; ++i)
            mine[threadIdx.x + i * kTableThreads] = a[i], totals[threadIdx.x + i * kTableThreads] = b[i];
        __syncthreads();
    }
    const int all = sums_before(totals, p.experts, parts, kTableWaves);
    for(int e = threadIdx.x; e < p.experts; e += kTableThreads)
    {
        mine[e] += totals[e];
        if(blockIdx.x == 0)
            p.offsets[e] = totals[e];
    }
    if(blockIdx.x == 0 && threadIdx.x == 0)
        p.offsets[p.experts] = all;
    for(int i = max(from, all) + threadIdx.x; i < to; i += kTableThreads)
        p.rows[i] = -1;
    __syncthreads();
    place_pairs(p, from, to, mine, reinterpret_cast<int*>(ckx_route_lds), kTableWaves);
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
    // as many waves as the workgroup's tokens take; of a single workgroup eight at most: its tables wait for all of them at each step
    const int per = ROWS ? 4 : 1, want = (a.chunk_tokens + per - 1) / per, most = a.chunks > 1 ? kWaves : 8;
    const int waves    = want < 4 ? 4 : want > most ? most : want;
    const size_t cells = a.offsets && a.chunks == 1 ? (size_t)waves * a.experts * 4 : 0, sums = a.groups > 1 ? (size_t)waves * a.experts * 8 : 0;
    const size_t lds   = sums > cells ? sums : cells;
    hipError_t e       = allow_lds(&route_kernel<X, ROWS, EPL, WIDE, ALL>, lds);
    if(e != hipSuccess)
        return e;
    hipLaunchKernelGGL((route_kernel<X, ROWS, EPL, WIDE, ALL>), dim3(a.chunks), dim3(waves * 64), lds, s, a);
    e = hipGetLastError();
    if(e != hipSuccess || a.chunks == 1 || !a.offsets)
        return e;
    const size_t tables = (size_t)kTableWaves * a.experts * 4;
    const auto kernel   = a.chunk_tokens <= kByteCount ? &route_tables_kernel<true> : &route_tables_kernel<false>;
    if((e = allow_lds(kernel, tables)) != hipSuccess)
        return e;
    hipLaunchKernelGGL(kernel, dim3(a.chunks), dim3(kTableThreads), tables, s, a);
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
    return a.experts <= 256 ? launch_form<X, false, 4>(a, s) : a.experts <= 512 ? launch_form<X, false, 8>(a, s) : launch_form<X, false, 16>(a, s);
}

// One workgroup up to 64 tokens of up to 8192 logits together, and up to 16 tokens of any: 64 tokens of 64 experts 8.8 us (two launches 9.6),
// 32 tokens of 256 with groups 11.3 (11.8; 64 tokens: 16.7, 12.0), 16 of 1024 19.9 (21.5; 24: 26.2).
void cut(int tokens, int experts, int& chunk_tokens, int& chunks)
{
    chunk_tokens = tokens, chunks = 1;
    if(tokens > kOneGroup || (tokens > 16 && tokens * experts > 8192))
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
    cut(tokens, experts, per, chunks);
    return chunks > 1 ? 16ll * chunks * counts_row(experts, per <= kByteCount) : 0;
}

hipError_t route_launch(RouteArgs a, int x_type, hipStream_t s)
{
    // tables of no tokens: the kernel asks for a first row of logits all the same and looks at none of it; the offsets have the room
    if(a.tokens == 0)
        a.x = a.offsets;
    cut(a.tokens, a.experts, a.chunk_tokens, a.chunks);
    return x_type == CKX_TYPE_F32 ? launch_any<float>(a, s) : x_type == CKX_TYPE_F16 ? launch_any<_Float16>(a, s) : launch_any<__bf16>(a, s);
}

} // namespace ckx
