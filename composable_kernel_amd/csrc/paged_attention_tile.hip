// Attention over the 8-bit cache for prompts: many query rows per sequence, so that the cache is converted once for 128 of them.
//
// One workgroup takes 128 query rows (the heads of one group times consecutive tokens), 32 a wave, and walks the cached tokens in
// steps of 64 with running maxima and sums. The codes of the next step are on their way into registers while one is multiplied;
// they are converted (keys to the type of q, values to fp16) on their way into LDS, values transposed by byte permutes, two
// stages, one barrier a step.
//   scores   S^T = K Q^T, v_mfma_f32_32x32x16: lane (row l % 32 of q, h = l / 32) gets tokens 8x + 4h + y (x, y < 4) of each 32
//   output   O^T = V^T P^T: 16 tokens an instruction, the lane's own probabilities as its operand: slots of half h are tokens
//            {4h .. 4h + 3, 8 + 4h .. + 3} of each 16, which the values' rows in LDS are ordered by. The rows themselves (elements of
//            d) are ordered so that a lane ends with 16 neighbouring elements of each 32.
// LDS rows of 16-byte chunks, chunk c of row r at c ^ (r & 15) (keys of 128), c ^ (r & 7) (keys of 64), c ^ ((r ^ r / 4) & 7)
// (values): eight neighbouring rows never meet on a bank, neither for the writes nor for the reads.
// What bounds it are vector instructions: 13 for each of a lane's scores for int8, 11 for e4m3 (heads of 128, counted).
// Multiply-add, exponential (which takes the time of four), sum, half a conversion and half a maximum are the softmax's. A lane
// converts 64 codes a step for its 32 scores, 1.5 instructions each for int8 and 0.5 for e4m3, and transposes its values by 16
// byte permutes. The rest is addresses, scales and masks. The matrix instructions wait for them and hardly run beside them: 4
// sequences of 4096 and 1024 new tokens, 32 / 8 heads of 128, int8 303 us, 0.66 PFLOP/s, vector instructions active 51 % of the
// launch, matrix cores busy 27 %; e4m3 284 us, 46 and 28 %. LDS is active 24 % of it, a seventh of that conflicts. Fragments
// further ahead, and the output's matrix instructions between the exponentials, are level; a copy of the loop without masks gives
// heads of 64 a tenth and spills at 128.
#include "paged_attention.hpp"

namespace ckx {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kStep = 64, kRows = 128;

template <typename T>
__device__ __forceinline__ f32x16 mfma32(const i32x4& a, const i32x4& b, const f32x16& c)
{
    if constexpr(std::is_same<T, __bf16>::value)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// f over the two lanes l, l ^ 32
template <typename F>
__device__ __forceinline__ float over_halves(float x, F&& f)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto a     = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    return f(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
}

template <typename T, int CODE, int DP>
__global__ __launch_bounds__(256, 2) void attention_tile_kernel(AttentionArgs p)
{
    constexpr int KC = DP / 8, KK = DP / 16, DT = DP / 32; // chunks of a key row; instructions along d; output tiles
    constexpr int K_TILE = kStep * DP * 2, V_TILE = DP * kStep * 2, STAGE = K_TILE + V_TILE;
    __shared__ __align__(16) uint8_t lds[2 * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const int D = p.cache.head_dim;

    // the last tiles first: with the causal mask they have the most to do
    int id              = (int)(gridDim.x - 1 - blockIdx.x);
    const int split     = id % p.splits;
    id /= p.splits;
    const int per_tile  = p.cache.num_heads * p.head_tiles;
    const int head_tile = id % per_tile;
    const TileOf tile   = tile_of(p, id / per_tile);
    if(!tile.live)
        return;
    const int kvh = head_tile / p.head_tiles, h0 = (head_tile - kvh * p.head_tiles) * p.tile_heads;
    const int row = wave * 32 + r, rt = row / p.tile_heads, rh = h0 + (row - rt * p.tile_heads);
    const bool row_live = rt < p.tile_tokens && tile.first + rt < tile.q_len && rh < p.group;
    const int head      = kvh * p.group + rh;
    const int64_t token = tile.q0 + tile.first + rt;
    const int see       = row_live ? (p.causal ? tile.kv - (tile.of - 1 - (tile.first + rt)) : tile.kv) : 0;
    const int last      = min(tile.first + p.tile_tokens, tile.q_len) - 1;
    const int most      = max(p.causal ? tile.kv - (tile.of - 1 - last) : tile.kv, 0);
    // the share of the cached tokens: an even number of steps
    const int all_steps = (most + kStep - 1) / kStep, per = ((all_steps + p.splits - 1) / p.splits + 1) & ~1;
    const int begin = min(split * per, (all_steps + 1) & ~1), steps = min(begin + per, all_steps);
    // the least and the most that a live row of this wave sees
    int least = row_live ? see : 0x7fffffff, furthest = see;
#pragma unroll
    for(int d = 1; d < 64; d *= 2)
        least = min(least, __shfl_xor(least, d)), furthest = max(furthest, __shfl_xor(furthest, d));
    least = __builtin_amdgcn_readfirstlane(least), furthest = __builtin_amdgcn_readfirstlane(furthest);

    i32x4 qf[KK];
#pragma unroll
    for(int k = 0; k < KK; ++k)
    {
        qf[k] = i32x4{0, 0, 0, 0};
        if(row_live && 16 * k < D)
            qf[k] = *reinterpret_cast<const i32x4*>(reinterpret_cast<const T*>(p.q) + token * p.sq_t + (int64_t)head * p.sq_h + 16 * k + 8 * h);
        // (a negative score scale: its sign goes here, so that the largest score is the largest product)
        if(p.scale < 0.0f)
            qf[k] ^= (int)0x80008000;
    }

    // Block numbers and scales of a step: lane b (and 4 + b) has those of its b-th 16 tokens, keys (values). They are asked for a
    // step, the numbers two steps ahead, in front of the codes' loads: through the scalar cache every wait for an LDS read would
    // wait for them as well.
    const int* const table = p.table + (int64_t)tile.b * p.stride_table;
    const float* const scales = (lane & 4 ? p.cache.p_v_scale : p.cache.p_k_scale) + kvh;
    auto blocks_of = [&](int step) {
        const int t = step * kStep + 16 * (lane & 3);
        const int b = t < most ? table[t >> p.block_shift] : -1;
        return b >= 0 && b < p.cache.num_blocks ? b : -1; // (-1: no such block)
    };
    auto scales_of = [&](int blocks) { return blocks >= 0 ? scales[(int64_t)blocks * p.cache.stride_scale] : 0.0f; };
    const uint8_t* const kc = reinterpret_cast<const uint8_t*>(p.cache.p_k) + (int64_t)kvh * p.cache.stride_head;
    const uint8_t* const vc = reinterpret_cast<const uint8_t*>(p.cache.p_v) + (int64_t)kvh * p.cache.stride_head;
    const int in_block      = (1 << p.block_shift) - 1;

    // A wave brings 16 tokens of a step, all of one block. Keys: lane (token l / 4, quarter l % 4 of the row). Values: eight
    // tokens (as above) times four (two) elements
    constexpr int KB = DP / 64, VL = DP / 4;            // 16-byte loads of a lane's quarter; lanes of a value row's four elements
    constexpr int VG = 64 / VL;                         // token halves side by side in a wave (DP 128: 2; DP 64: 4, two of them idle)
    u32x4 kb[2][KB]; // (of even and odd steps)
    uint32_t vb[2][8];
    const int kt = lane >> 2, kq = lane & 3;
    const int vh = lane / VL, vd = (lane % VL) * 4;     // half, element
    // (columns behind head_dim repeat its last ones: q is zero there, and no one stores such an element of the output)
    uint32_t k_off[KB];
#pragma unroll
    for(int j = 0; j < KB; ++j)
        k_off[j] = (uint32_t)kt * p.cache.stride_token + min(kq * (DP / 4) + 16 * j, D - 16);
    const uint32_t v_off = (uint32_t)(4 * (vh & 1)) * p.cache.stride_token + min(vd, D - 4);
    auto fetch = [&](int step, int block, auto odd) {
        constexpr int S = decltype(odd)::value;
        if(block < 0)
        {
#pragma unroll
            for(int j = 0; j < KB; ++j)
                kb[S][j] = u32x4{0, 0, 0, 0};
#pragma unroll
            for(int i = 0; i < 8; ++i)
                vb[S][i] = 0;
            return;
        }
        const int64_t at       = (int64_t)block * p.cache.stride_block + (int64_t)((step * kStep + wave * 16) & in_block) * p.cache.stride_token;
        const uint8_t* const k = kc + at;
        const uint8_t* const v = vc + at;
#pragma unroll
        for(int j = 0; j < KB; ++j)
            kb[S][j] = *reinterpret_cast<const u32x4*>(k + k_off[j]);
#pragma unroll
        for(int i = 0; i < 8; ++i)
            vb[S][i] = *reinterpret_cast<const uint32_t*>(v + (int64_t)(8 * (i >> 2) + (i & 3)) * p.cache.stride_token + v_off);
    };
    // element 32 j + 16 a + 4 x + y lies in row 32 j + 8 x + 4 a + y
    const int krow = wave * 16 + kt, vrow = (vd & ~31) + (((vd >> 2) & 3) << 3) + (((vd >> 4) & 1) << 2);
    const uint32_t k_write = krow * (DP * 2) + (((kq * (KC / 4)) ^ (krow & (KC - 1))) << 4);
    const uint32_t v_write = K_TILE + vrow * (kStep * 2) + (((2 * wave + vh) ^ ((vrow ^ (vrow >> 2)) & 7)) << 4);
    // In pieces (2 KB chunks of keys, 4 of values), so that a wave converts the next step's between the matrix instructions of its
    // scores: heads of 64, 8 x (1024 + 256) 50.9 -> 44.3 us, heads of 128, 4 x (4096 + 1024) e4m3 292 -> 285. The stage was last read a
    // step ago.
    uint32_t k_to, v_to, v_lo[4], v_hi[4];
    auto deposit_begin = [&](int step, auto odd) {
        constexpr int S = decltype(odd)::value;
        const int t = step * kStep + wave * 16;
        if(t + 16 > most) // (what lies behind the last token is no value: zero, whatever its bytes are)
        {
#pragma unroll
            for(int i = 0; i < 8; ++i)
                vb[S][i] = t + 8 * (i >> 2) + 4 * vh + (i & 3) < most ? vb[S][i] : 0;
        }
        k_to = k_write + (step & 1) * STAGE, v_to = v_write + (step & 1) * STAGE;
        asm volatile("" : "+v"(k_to), "+v"(v_to));
    };
    constexpr int PIECES = 2 * KB + 4;
    auto deposit_piece = [&](int n, auto odd) {
        constexpr int S = decltype(odd)::value;
        if(n < 2 * KB) // (+ kq * KC / 4, whose bits are higher ones)
            *reinterpret_cast<i32x4*>(lds + (k_to ^ (uint32_t)(n << 4))) =
                codes8<CODE, T>(kb[S][n / 2][2 * (n & 1)], kb[S][n / 2][2 * (n & 1) + 1]);
        else if(DP == 128 || vh < 2)
        {
            const int i = n - 2 * KB;
            if(i == 0)
            {
                transpose4(vb[S][0], vb[S][1], vb[S][2], vb[S][3], v_lo);
                transpose4(vb[S][4], vb[S][5], vb[S][6], vb[S][7], v_hi);
            }
            *reinterpret_cast<i32x4*>(lds + (v_to ^ (uint32_t)(i << 4)) + i * (kStep * 2)) = codes8<CODE, _Float16>(v_lo[i], v_hi[i]);
        }
    };
    auto deposit = [&](int step, auto odd) {
        deposit_begin(step, odd);
#pragma unroll
        for(int n = 0; n < PIECES; ++n)
            deposit_piece(n, odd);
    };

    // A block with a negative scale: what the wave has put of it into LDS changes sign (exactly: 16-bit floats), the scale counts by its
    // size. Behind the step's work, where the branch parts nothing that is scheduled together.
    auto negate = [&](int step, float scales) {
        const uint32_t mine = (uint32_t)__ballot(scales < 0.0f) >> wave; // bit 0: keys, 4: values
        if((mine & 0x11u) == 0)
            return;
        uint32_t k_old = k_write + (step & 1) * STAGE, v_old = v_write + (step & 1) * STAGE;
        asm volatile("" : "+v"(k_old), "+v"(v_old)); // (worked out here, not kept)
        if(mine & 1u)
#pragma unroll
            for(int n = 0; n < 2 * KB; ++n)
                *reinterpret_cast<i32x4*>(lds + (k_old ^ (uint32_t)(n << 4))) ^= (int)0x80008000;
        if((mine & 16u) && (DP == 128 || vh < 2))
#pragma unroll
            for(int i = 0; i < 4; ++i)
                *reinterpret_cast<i32x4*>(lds + (v_old ^ (uint32_t)(i << 4)) + i * (kStep * 2)) ^= (int)0x80008000;
    };

    const uint32_t k_read = r * (DP * 2) + ((h ^ (r & (KC - 1))) << 4), v_read = K_TILE + r * (kStep * 2) + ((h ^ ((r ^ (r >> 2)) & 7)) << 4);
    f32x16 o[DT];
#pragma unroll
    for(int j = 0; j < DT; ++j)
#pragma unroll
        for(int i = 0; i < 16; ++i)
            o[j][i] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f;
    // The value scale that the row's sums are relative to, the largest finite one (by its size) that it has seen, and its logarithm;
    // `low`: the least of them among the wave's rows (steps that all rows see whole leave them one), under which no scale raises any.
    constexpr float kLeast = 1.9259299443872359e-34f; // (2^-112: a score's sum relative to it stays finite)
    float top = kLeast, top_log = -112.0f, low = kLeast;

    auto lane_of = [](auto x, int from) {
        return __builtin_bit_cast(decltype(x), __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), from));
    };
    std::integral_constant<int, 0> even;
    std::integral_constant<int, 1> odd;
    // of this step and the two behind it; their codes are fetched two steps ahead
    int blocks = blocks_of(begin), blocks1 = blocks_of(begin + 1), blocks2 = blocks_of(begin + 2);
    float scale = scales_of(blocks), scale1 = scales_of(blocks1);
    fetch(begin, lane_of(blocks, wave), even);
    fetch(begin + 1, lane_of(blocks1, wave), odd);
    deposit(begin, even);
    negate(begin, scale);
    __syncthreads();
    auto one_step = [&](int step, auto mine, auto other) {
        const uint32_t there = (uint32_t)__ballot(blocks >= 0) & 15u; // (a bit for each 16 tokens)
        // (behind the last step: no block, nothing read)
        const float scale2 = scales_of(blocks2);
        const int blocks3  = blocks_of(step + 3);
        fetch(step + 2, lane_of(blocks2, wave), mine);
        const int t0 = step * kStep;
        auto multiply = [&](bool whole) {
            // chunk 2 k + h of a row: k's bits flip those of k = 0. (Worked out in every step: kept over the loop, the addresses are
            // twelve registers that the kernel has not got.)
            uint32_t k_at = k_read + (step & 1) * STAGE, v_at = v_read + (step & 1) * STAGE;
            asm volatile("" : "+v"(k_at), "+v"(v_at));
            // The value scales go into the exponent, exp2(score - m + log2(scale / top)), which saves a multiplication a score; the
            // sum of the probabilities takes them out again, 16 tokens at a time. All scales enter by their size (negate).
            const float size = __builtin_fabsf(scale);
            float keep_v     = 1.0f;
            if(__any((lane & 4) && size > low))
            {
                float next = top;
#pragma unroll
                for(int b = 0; b < 4; ++b)
                {
                    const float v = lane_of(size, 4 + b);
                    next          = __builtin_fmaxf(next, __builtin_isfinite(v) && see - t0 > 16 * b ? v : 0.0f);
                }
                keep_v = top / next;
                top = next, top_log = __builtin_amdgcn_logf(next);
                float x = see > t0 ? next : __builtin_inff(); // (rows that are through do not count)
#pragma unroll
                for(int d = 1; d < 32; d *= 2)
                    x = __builtin_fminf(x, __shfl_xor(x, d));
                low = lane_of(x, 0);
            }
            // (Under 2^-40 of a row's top every product is zero in fp16. Lifted to that, no probability sinks under fp32's normal numbers
            // on the way to the sum, and no 1 / w is infinite.)
            const float least_w = __builtin_fmaxf(low * 0x1p-40f, 0x1p-125f), w = size < least_w ? least_w : size;
            const float w_logs = __builtin_amdgcn_logf(w), w_invs = __builtin_amdgcn_rcpf(w);
            // (fp32's least number in place of zero: no -inf times zero, and no score of a tiny scale changes. NaN stays.)
            const float cs = size * __builtin_fabsf(p.scale), c_least = cs < 0x1p-149f ? 0x1p-149f : cs;
            float c[4], w_log[4], w_inv[4];
#pragma unroll
            for(int b = 0; b < 4; ++b)
                c[b] = lane_of(c_least, b), w_log[b] = lane_of(w_logs, 4 + b), w_inv[b] = lane_of(w_invs, 4 + b);
            deposit_begin(step + 1, other);
            f32x16 s[2];
            constexpr int DQ = 2; // fragments DQ pairs of instructions ahead: an LDS read takes about as long as three of them
            i32x4 kf[DQ + 1][2];
            auto read_k = [&](int k) {
#pragma unroll
                for(int u = 0; u < 2; ++u)
                    kf[k % (DQ + 1)][u] = *reinterpret_cast<const i32x4*>(lds + (k_at ^ (uint32_t)(k << 5)) + u * 32 * DP * 2);
            };
#pragma unroll
            for(int k = 0; k < DQ; ++k)
                read_k(k);
#pragma unroll
            for(int k = 0; k < KK; ++k)
            {
                if(k + DQ < KK)
                    read_k(k + DQ);
#pragma unroll
                for(int u = 0; u < 2; ++u)
                    s[u] = mfma32<T>(kf[k % (DQ + 1)][u], qf[k], k == 0 ? f32x16(0.0f) : s[u]);
#pragma unroll
                for(int n = k * PIECES / KK; n < (k + 1) * PIECES / KK; ++n)
                    deposit_piece(n, other);
                __builtin_amdgcn_sched_barrier(0);
            }
            const int reach = see - t0 - 4 * h;
            if(!whole)
            {
                // (a branch: without these the compiler masks every step)
                asm volatile("" : "+v"(s[0]));
                asm volatile("" : "+v"(s[1]));
#pragma unroll
                for(int u = 0; u < 2; ++u)
#pragma unroll
                    for(int i = 0; i < 16; ++i)
                    {
                        const int t = 32 * u + 8 * (i >> 2) + (i & 3);
                        s[u][i]     = (there >> (2 * u + (i >> 3)) & 1) && t < reach ? s[u][i] : -__builtin_inff();
                    }
            }
            // (the maximum is there for the range only: of the unscaled scores of 16 tokens, then scaled; and it is raised only by
            // leaps, 2^6 or more, so that the sums are seldom rescaled: no probability exceeds 2^6 then)
            float most_s = -__builtin_inff();
#pragma unroll
            for(int b = 0; b < 4; ++b)
            {
                float x = s[b >> 1][8 * (b & 1)];
#pragma unroll
                for(int i = 1; i < 8; ++i)
                    x = __builtin_elementwise_maximum(x, s[b >> 1][8 * (b & 1) + i]);
                most_s = __builtin_elementwise_maximum(most_s, x == -__builtin_inff() ? x : x * c[b]); // (-inf: nothing seen, whatever the scale is)
            }
            // (maximum, which a NaN wins: one instruction for three values where fmaxf makes every one a quiet number first. A row with a NaN
            // among its scores raises no maximum any more; it is NaN.)
            most_s = over_halves(most_s, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
            float keep_o = keep_v;
            if(__any(most_s > m + 6.0f))
            {
                // (the rows that leap, no others: a row's bits are its own)
                float now = most_s > m + 6.0f ? most_s : m;
                asm volatile("" : "+v"(now)); // (in the branch: left to itself the compiler chooses outside of it, every step)
                const float keep = __builtin_amdgcn_exp2f(m - (now == -__builtin_inff() ? 0.0f : now));
                m = now;
                l *= keep;
                keep_o *= keep;
            }
            if(__any(keep_o != 1.0f))
            {
#pragma unroll
                for(int j = 0; j < DT; ++j)
                    o[j] *= keep_o;
            }
            const float zero = (m == -__builtin_inff() ? 0.0f : m) + top_log; // (nothing seen yet)
            i32x4 vf[2][DT];
            auto read_v = [&](int k) {
#pragma unroll
                for(int j = 0; j < DT; ++j)
                    vf[k & 1][j] = *reinterpret_cast<const i32x4*>(lds + (v_at ^ (uint32_t)(k << 5)) + j * 32 * kStep * 2);
            };
            i32x4 pf[4];
            float sums = 0.0f; // over top
#pragma unroll
            for(int b = 0; b < 4; ++b)
            {
                // a masked score is -inf and its probability zero, but for scales that are no numbers: they are kept from rows
                // that see none of the lane's eight tokens
                const bool sees  = whole || reach > 16 * b;
                const float cb   = sees ? c[b] : 1.0f, bias = sees ? w_log[b] - zero : 0.0f;
                float pr[8], sum = 0.0f;
#pragma unroll
                for(int i = 0; i < 8; ++i)
                {
                    pr[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b >> 1][8 * (b & 1) + i], cb, bias));
                    sum += pr[i];
                }
                sums  = __builtin_fmaf(sum, sees ? w_inv[b] : 0.0f, sums);
                pf[b] = i32x4{(int)pack_f16(pr[0], pr[1]), (int)pack_f16(pr[2], pr[3]), (int)pack_f16(pr[4], pr[5]), (int)pack_f16(pr[6], pr[7])};
            }
            l = __builtin_fmaf(sums, top, l);
            read_v(0);
#pragma unroll
            for(int k = 0; k < 4; ++k)
            {
                if(k < 3)
                    read_v(k + 1);
#pragma unroll
                for(int j = 0; j < DT; ++j)
                    o[j] = mfma32<_Float16>(vf[k & 1][j], pf[k], o[j]);
            }
        };
        if(t0 < furthest)
            multiply(t0 + kStep <= least && there == 15u);
        else
            deposit(step + 1, other);
        negate(step + 1, scale1);
        blocks = blocks1, blocks1 = blocks2, blocks2 = blocks3;
        scale = scale1, scale1 = scale2;
        __syncthreads();
    };
    for(int step = begin; step < steps; step += 2)
    {
        one_step(step, even, odd);
        if(step + 1 < steps)
            one_step(step + 1, odd, even);
    }

    l = over_halves(l, [](float a, float b) { return a + b; });
    if(!row_live)
        return;
    if(p.splits > 1)
    {
        const int64_t at = (token * p.heads + head) * p.splits + split;
#pragma unroll
        for(int j = 0; j < DT; ++j)
#pragma unroll
            for(int e = 0; e < 16; e += 4)
                *reinterpret_cast<f32x4*>(p.ws + at * DP + 32 * j + 16 * h + e) =
                    f32x4{o[j][e] * top, o[j][e + 1] * top, o[j][e + 2] * top, o[j][e + 3] * top};
        if(h == 0)
        {
            float* const ml = p.ws + attention_rows(p) * p.splits * DP + at * 2;
            ml[0] = m, ml[1] = l;
        }
        return;
    }
    const float f = l == 0.0f ? 0.0f : top / l; // (a row that sees nothing: zero)
    T* const to   = reinterpret_cast<T*>(p.o) + token * p.so_t + (int64_t)head * p.so_h;
    typedef T tx8 __attribute__((ext_vector_type(8)));
#pragma unroll
    for(int j = 0; j < DT; ++j)
#pragma unroll
        for(int e = 0; e < 2; ++e)
        {
            const int d = 32 * j + 16 * h + 8 * e;
            tx8 x;
#pragma unroll
            for(int i = 0; i < 8; ++i)
                x[i] = (T)(o[j][8 * e + i] * f);
            if(d < D)
                *reinterpret_cast<tx8*>(to + d) = x;
        }
}

template <typename T, int CODE>
hipError_t launch(const AttentionArgs& a, hipStream_t s)
{
    const dim3 grid((unsigned)((int64_t)a.tiles * a.cache.num_heads * a.head_tiles * a.splits));
    if(a.cache.head_dim <= 64)
        hipLaunchKernelGGL((attention_tile_kernel<T, CODE, 64>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((attention_tile_kernel<T, CODE, 128>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

} // namespace

hipError_t attention_tile_launch(const AttentionArgs& a, bool f16, hipStream_t s)
{
    if(a.cache.type == CKX_TYPE_E4M3)
        return f16 ? launch<_Float16, CODE_E4M3>(a, s) : launch<__bf16, CODE_E4M3>(a, s);
    return f16 ? launch<_Float16, CODE_I8>(a, s) : launch<__bf16, CODE_I8>(a, s);
}

} // namespace ckx
