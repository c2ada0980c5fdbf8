// Attention over the 8-bit cache for prompts: many query rows per sequence, so that the cache is converted once for 128 of them.
//
// One workgroup takes 128 query rows (the heads of one group times consecutive tokens), 32 a wave, and walks the cached tokens in
// steps of 64 with running maxima and sums. The codes of the next step are on their way into registers while one is multiplied; they are
// converted (keys to the type of q, values to fp16) on their way into LDS, values transposed by byte permutes, two stages, one
// barrier a step.
//   scores   S^T = K Q^T, v_mfma_f32_32x32x16: lane (row l % 32 of q, h = l / 32) gets tokens 8x + 4h + y (x, y < 4) of each 32
//   output   O^T = V^T P^T: 16 tokens an instruction, the lane's own probabilities as its operand: slots of half h are tokens
//            {4h .. 4h + 3, 8 + 4h .. + 3} of each 16, which the values' rows in LDS are ordered by. The rows themselves (elements of
//            d) are ordered so that a lane ends with 16 neighbouring elements of each 32.
// LDS rows of 16-byte chunks, chunk c of row r at c ^ (r & 15) (keys of 128), c ^ (r & 7) (keys of 64), c ^ ((r ^ r / 4) & 7)
// (values): eight neighbouring rows never meet on a bank, neither for the writes nor for the reads.
// What bounds it are vector instructions: 8 a score (the exponential counts four), about as many cycles as the matrix
// instructions take, and the two share the SIMD's issue.
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
    const int see       = row_live ? (p.causal ? tile.kv - (tile.q_len - 1 - (tile.first + rt)) : tile.kv) : 0;
    const int last      = min(tile.first + p.tile_tokens, tile.q_len) - 1;
    const int most      = max(p.causal ? tile.kv - (tile.q_len - 1 - last) : tile.kv, 0);
    const int steps     = (most + kStep - 1) / kStep;
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
    }

    // uniform loads through the scalar cache
    typedef const __attribute__((address_space(4))) int* int_ptr;
    typedef const __attribute__((address_space(4))) float* float_ptr;
    const int_ptr table  = (int_ptr)(p.table + (int64_t)tile.b * p.stride_table);
    const float_ptr ksp = (float_ptr)(p.cache.p_k_scale + kvh), vsp = (float_ptr)(p.cache.p_v_scale + kvh);
    // number of the block that holds token t, -1 for none
    auto block_of = [&](int t) {
        const int b = t < most ? table[t >> p.block_shift] : -1;
        return b >= 0 && b < p.cache.num_blocks ? b : -1;
    };
    const uint8_t* const kc = reinterpret_cast<const uint8_t*>(p.cache.p_k) + (int64_t)kvh * p.cache.stride_head;
    const uint8_t* const vc = reinterpret_cast<const uint8_t*>(p.cache.p_v) + (int64_t)kvh * p.cache.stride_head;
    const int in_block      = (1 << p.block_shift) - 1;

    // A wave brings 16 tokens of a step, all of one block. Keys: lane (token l / 4, quarter l % 4 of the row). Values: eight
    // tokens (as above) times four (two) elements
    constexpr int KB = DP / 64, VL = DP / 4;            // 16-byte loads of a lane's quarter; lanes of a value row's four elements
    constexpr int VG = 64 / VL;                         // token halves side by side in a wave (DP 128: 2; DP 64: 4, two of them idle)
    u32x4 kb[KB];
    uint32_t vb[8];
    const int kt = lane >> 2, kq = lane & 3;
    const int vh = lane / VL, vd = (lane % VL) * 4;     // half, element
    auto fetch = [&](int step, int block) {
        const int t = step * kStep + wave * 16;
#pragma unroll
        for(int j = 0; j < KB; ++j)
            kb[j] = u32x4{0, 0, 0, 0};
#pragma unroll
        for(int i = 0; i < 8; ++i)
            vb[i] = 0;
        if(block < 0)
            return;
        const uint8_t* const k = kc + (int64_t)block * p.cache.stride_block + (int64_t)((t & in_block) + kt) * p.cache.stride_token;
        const uint8_t* const v = vc + (int64_t)block * p.cache.stride_block + (int64_t)(t & in_block) * p.cache.stride_token + vd;
#pragma unroll
        for(int j = 0; j < KB; ++j)
            if(kq * (DP / 4) + 16 * j < D)
                kb[j] = *reinterpret_cast<const u32x4*>(k + kq * (DP / 4) + 16 * j);
        if(vh < 2 && vd < D)
        {
#pragma unroll
            for(int i = 0; i < 8; ++i)
            {
                const int at = 8 * (i >> 2) + 4 * vh + (i & 3);
                if(t + at < most) // (what lies behind the last token is no value: zero, whatever its bytes are)
                    vb[i] = *reinterpret_cast<const uint32_t*>(v + (int64_t)at * p.cache.stride_token);
            }
        }
    };
    auto deposit = [&](int stage) {
        uint8_t* const kl = lds + stage * STAGE;
        uint8_t* const vl = kl + K_TILE;
        const int krow    = wave * 16 + kt;
#pragma unroll
        for(int j = 0; j < KB; ++j)
#pragma unroll
            for(int e = 0; e < 2; ++e)
            {
                const int c = kq * (KC / 4) + 2 * j + e;
                *reinterpret_cast<i32x4*>(kl + krow * (DP * 2) + ((c ^ (krow & (KC - 1))) << 4)) = codes8<CODE, T>(kb[j][2 * e], kb[j][2 * e + 1]);
            }
        if(vh < 2)
        {
            uint32_t lo[4], hi[4];
            transpose4(vb[0], vb[1], vb[2], vb[3], lo);
            transpose4(vb[4], vb[5], vb[6], vb[7], hi);
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                // element 32 j + 16 a + 4 x + y lies in row 32 j + 8 x + 4 a + y
                const int vrow = (vd & ~31) + (((vd >> 2) & 3) << 3) + (((vd >> 4) & 1) << 2) + i, c = 2 * wave + vh;
                *reinterpret_cast<i32x4*>(vl + vrow * (kStep * 2) + ((c ^ ((vrow ^ (vrow >> 2)) & 7)) << 4)) = codes8<CODE, _Float16>(lo[i], hi[i]);
            }
        }
    };

    f32x16 o[DT];
#pragma unroll
    for(int j = 0; j < DT; ++j)
#pragma unroll
        for(int i = 0; i < 16; ++i)
            o[j][i] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f;
    ValueScale unit;

    int mine = block_of(wave * 16);
    fetch(0, mine);
    mine = block_of(kStep + wave * 16);
    deposit(0);
    __syncthreads();
    for(int step = 0; step < steps; ++step)
    {
        const bool more = step + 1 < steps;
        if(more)
        {
            fetch(step + 1, mine);
            mine = block_of((step + 2) * kStep + wave * 16);
        }
        const int t0 = step * kStep;
        if(t0 < furthest)
        {
            const uint8_t* const kl = lds + (step & 1) * STAGE;
            const uint8_t* const vl = kl + K_TILE;
            float c[4], vs[4];
            bool whole = t0 + kStep <= least;
            bool there[4];
#pragma unroll
            for(int b = 0; b < 4; ++b)
            {
                const int block = block_of(t0 + 16 * b);
                there[b]        = block >= 0;
                whole &= there[b];
                c[b]  = there[b] ? ksp[(int64_t)block * p.cache.stride_scale] * p.scale : 0.0f;
                vs[b] = there[b] ? vsp[(int64_t)block * p.cache.stride_scale] : 0.0f;
            }
            f32x16 s[2];
#pragma unroll
            for(int u = 0; u < 2; ++u)
            {
#pragma unroll
                for(int i = 0; i < 16; ++i)
                    s[u][i] = 0.0f;
                const int krow = 32 * u + r;
#pragma unroll
                for(int k = 0; k < KK; ++k)
                    s[u] = mfma32<T>(*reinterpret_cast<const i32x4*>(kl + krow * (DP * 2) + (((2 * k + h) ^ (krow & (KC - 1))) << 4)), qf[k], s[u]);
            }
            float top = -__builtin_inff();
#pragma unroll
            for(int u = 0; u < 2; ++u)
#pragma unroll
                for(int i = 0; i < 16; ++i)
                    s[u][i] *= c[2 * u + (i >> 3)];
            if(!whole)
            {
#pragma unroll
                for(int u = 0; u < 2; ++u)
#pragma unroll
                    for(int i = 0; i < 16; ++i)
                    {
                        const int t = t0 + 32 * u + 8 * (i >> 2) + 4 * h + (i & 3);
                        s[u][i]     = there[2 * u + (i >> 3)] && t < see ? s[u][i] : -__builtin_inff();
                    }
            }
#pragma unroll
            for(int u = 0; u < 2; ++u)
#pragma unroll
                for(int i = 0; i < 16; ++i)
                    top = __builtin_fmaxf(top, s[u][i]);
            const float now  = __builtin_fmaxf(m, over_halves(top, [](float a, float b) { return __builtin_fmaxf(a, b); }));
            const float zero = now == -__builtin_inff() ? 0.0f : now; // (nothing seen yet: exp2(-inf - 0) = 0)
            const float keep = __builtin_amdgcn_exp2f(m - zero);
            m                = now;
            const float keep_o = keep * unit.take(vs[0], vs[1]) * unit.take(vs[2], vs[3]);
            if(__any(keep_o != 1.0f))
            {
                l *= keep;
#pragma unroll
                for(int j = 0; j < DT; ++j)
                    o[j] *= keep_o;
            }
            float w[4];
#pragma unroll
            for(int b = 0; b < 4; ++b)
                w[b] = unit.of(vs[b]);
            i32x4 pf[4];
#pragma unroll
            for(int u = 0; u < 2; ++u)
            {
                float pr[16];
#pragma unroll
                for(int i = 0; i < 16; ++i)
                {
                    pr[i] = __builtin_amdgcn_exp2f(s[u][i] - zero);
                    l += pr[i];
                    pr[i] *= w[2 * u + (i >> 3)];
                }
                if(!whole) // (masked: no value scale, which may be an infinity or NaN, gets into the sum)
                {
#pragma unroll
                    for(int i = 0; i < 16; ++i)
                        pr[i] = s[u][i] == -__builtin_inff() ? 0.0f : pr[i];
                }
#pragma unroll
                for(int k = 0; k < 2; ++k)
                    pf[2 * u + k] = i32x4{(int)pack_f16(pr[8 * k], pr[8 * k + 1]), (int)pack_f16(pr[8 * k + 2], pr[8 * k + 3]),
                                          (int)pack_f16(pr[8 * k + 4], pr[8 * k + 5]), (int)pack_f16(pr[8 * k + 6], pr[8 * k + 7])};
            }
#pragma unroll
            for(int j = 0; j < DT; ++j)
            {
                const int vrow = 32 * j + r;
#pragma unroll
                for(int k = 0; k < 4; ++k)
                    o[j] = mfma32<_Float16>(*reinterpret_cast<const i32x4*>(vl + vrow * (kStep * 2) + (((2 * k + h) ^ ((vrow ^ (vrow >> 2)) & 7)) << 4)),
                                            pf[k], o[j]);
            }
        }
        if(more)
            deposit((step + 1) & 1);
        __syncthreads();
    }

    l = over_halves(l, [](float a, float b) { return a + b; });
    if(!row_live)
        return;
    const float f = l == 0.0f ? 0.0f : unit.top / l; // (a row that sees nothing: zero)
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
    const dim3 grid((unsigned)(a.tiles * a.cache.num_heads * a.head_tiles));
    if(a.cache.head_dim <= 64)
        hipLaunchKernelGGL((attention_tile_kernel<T, CODE, 64>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((attention_tile_kernel<T, CODE, 128>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

} // namespace

hipError_t attention_tile_launch(const AttentionArgs& a, int q_type, hipStream_t s)
{
    if(a.cache.type == CKX_TYPE_E4M3)
        return q_type == CKX_TYPE_F16 ? launch<_Float16, CODE_E4M3>(a, s) : launch<__bf16, CODE_E4M3>(a, s);
    return q_type == CKX_TYPE_F16 ? launch<_Float16, CODE_I8>(a, s) : launch<__bf16, CODE_I8>(a, s);
}

} // namespace ckx
