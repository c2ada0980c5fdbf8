// Attention over the 8-bit cache for few query rows per sequence (single tokens, a handful): the cache is read once, straight
// into registers.
//
// One workgroup takes 16 query rows (the heads of one group, times as many tokens as fit) and a share of the cached tokens; its
// waves take 32 tokens each in turn with running maxima and sums of their own and are joined through LDS at the end. Shares of
// one row are joined by a second launch.
//   scores   S^T = K Q^T, v_mfma_f32_16x16x32: lane (row l % 16 of q, g = l / 16) gets tokens 4g .. 4g + 3 of each 16
//   output   O^T = V^T P^T, the same instruction over 32 tokens: the lane's own probabilities are its operand, so V's lanes take tokens
//            {4g .. 4g + 3, 16 + 4g .. + 3} as well, eight (four) neighbouring elements of d each, transposed by byte permutes
//            in registers. MFMA j's row c stands for element c * E + j (E elements a lane): the lane ends with a contiguous
//            stretch of the output row.
// What bounds it is the cache's bytes: 64 sequences of 8192, 32 / 8 heads of 128, e4m3 157.7 us, 5.1 TB/s (reads alone reach 6.35
// on this card, 127 us; the waves wait 41 % of their time, vector instructions are active 31 % of the launch, the matrix cores 6
// %); int8, whose codes take three times the instructions to convert, 180 us. One sequence of 1000 11.2 us, of which the first
// loads, one behind the other (lengths, table, codes), are about four and the joining launch 3.4. The next 32 tokens' codes (8 KB
// a wave for heads of 128) are on their way while the present ones are multiplied; block numbers and scales of 32 such turns are
// fetched at once, a lane each.
// The number of shares is one for the call. Sequences of very different lengths, enough of them to fill the CUs, leave the
// longest to one workgroup a head: one of 131072 among 31 of 1000 844 us, where its bytes take 52.
#include "paged_attention.hpp"

namespace ckx {

namespace {

// query rows of a sequence (tokens x heads of a group), on average, past which the kernel for prompts takes over; it / this one, us:
// 16 sequences of 4096, 32 / 8 heads of 128: 48 rows 82 / 59, 72 rows 82 / 80, 120 rows 89 / 114; 64 of 1000, 96 rows 65 / 131;
// 16 of 2000, 16 / 16 heads of 64: 96 rows 66 / 56, 192 rows 93 / 101
constexpr int kPromptRows = 80;
constexpr int NW          = 8; // waves (four, with three workgroups a CU: 64 sequences of 8192 170 us against 159)

template <typename T>
__device__ __forceinline__ f32x4 mfma_qk(const i32x4& k, const i32x4& q, const f32x4& c)
{
    if constexpr(std::is_same<T, __bf16>::value)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
}

// DP: head_dim rounded up to 64 or 128
template <typename T, int CODE, int DP>
__global__ __launch_bounds__(NW * 64, 2) void attention_rows_kernel(AttentionArgs p)
{
    constexpr int KJ = DP / 64;  // 16-byte loads of a key row's lane
    constexpr int E  = DP / 16;  // elements of a value row's lane
    __shared__ float part[NW][16][DP + 4];
    __shared__ float part_m[NW][16], part_l[NW][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int D = p.cache.head_dim;

    int id           = blockIdx.x;
    const int split  = id % p.splits;
    id /= p.splits;
    const int head_tile = id % (p.cache.num_heads * p.head_tiles);
    const TileOf tile   = tile_of(p, id / (p.cache.num_heads * p.head_tiles));
    if(!tile.live)
        return;
    const int kvh = head_tile / p.head_tiles, h0 = (head_tile - kvh * p.head_tiles) * p.tile_heads;
    // the lane's query row
    const int rt = r / p.tile_heads, rh = h0 + (r - rt * p.tile_heads);
    const bool row_live = rt < p.tile_tokens && tile.first + rt < tile.q_len && rh < p.group;
    const int head      = kvh * p.group + rh;
    const int64_t token = tile.q0 + tile.first + rt;
    const int behind    = tile.of - 1 - (tile.first + rt); // query tokens behind the row's
    const int see       = row_live ? (p.causal ? tile.kv - behind : tile.kv) : 0;
    const int last      = min(tile.first + p.tile_tokens, tile.q_len) - 1;
    const int most      = max(p.causal ? tile.kv - (tile.of - 1 - last) : tile.kv, 0); // what the tile's furthest row sees

    // the share: whole steps of 32 tokens; the wave's turns among them
    const int steps = (most + 31) / 32, per = (steps + p.splits - 1) / p.splits;
    const int step0 = min(split * per, steps), step1 = min(step0 + per, steps);
    const int turns = max(step1 - step0 - wave + NW - 1, 0) / NW;

    const int* const table  = p.table + (int64_t)tile.b * p.stride_table;
    const uint8_t* const kc = reinterpret_cast<const uint8_t*>(p.cache.p_k) + (int64_t)kvh * p.cache.stride_head;
    const uint8_t* const vc = reinterpret_cast<const uint8_t*>(p.cache.p_v) + (int64_t)kvh * p.cache.stride_head;
    const int in_block      = (1 << p.block_shift) - 1;
    auto first_of           = [&](int turn) { return (step0 + wave + NW * turn) * 32; }; // token
    // lane 2 x + h: block and scales of the 16 tokens h of turn (32 n + x); -1: no such block
    int blocks  = -1;
    float ks_of = 0.0f, vs_of = 0.0f;
    auto look_up = [&](int turn) {
        const int t = first_of(turn + (lane >> 1)) + 16 * (lane & 1);
        blocks      = turn + (lane >> 1) < turns && t < most ? table[t >> p.block_shift] : -1;
        blocks      = blocks < p.cache.num_blocks ? blocks : -1;
        ks_of = vs_of = 0.0f;
        if(blocks >= 0)
        {
            ks_of = p.cache.p_k_scale[(int64_t)blocks * p.cache.stride_scale + kvh];
            vs_of = p.cache.p_v_scale[(int64_t)blocks * p.cache.stride_scale + kvh];
        }
    };
    // (columns behind head_dim repeat its last ones: q is zero there, and no one stores such an element of the output)
    uint32_t k_off[KJ];
#pragma unroll
    for(int j = 0; j < KJ; ++j)
        k_off[j] = (uint32_t)r * p.cache.stride_token + min(64 * j + 16 * g, D - 16);
    const uint32_t v_off = (uint32_t)(4 * g) * p.cache.stride_token + min(r * E, D - E);
    struct Turn
    {
        u32x4 kb[2][KJ];
        uint32_t vb[8][E / 4];
        float ks[2], vs[2];
        bool there[2];
    };
    auto lane_of = [](auto x, int from) {
        return __builtin_bit_cast(decltype(x), __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), from));
    };
    // (the first turn's codes are asked for before its scales are waited for; in the loop that order costs registers and 6 % for int8)
    auto scales_to = [&](Turn& x, int turn) {
#pragma unroll
        for(int h = 0; h < 2; ++h)
            x.ks[h] = lane_of(ks_of, 2 * (turn & 31) + h), x.vs[h] = lane_of(vs_of, 2 * (turn & 31) + h);
    };
    auto fetch = [&](Turn& x, int turn, auto first) {
        if((turn & 31) == 0)
            look_up(turn);
#pragma unroll
        for(int h = 0; h < 2; ++h)
        {
            const int from  = 2 * (turn & 31) + h;
            const int block = lane_of(blocks, from);
            x.there[h]      = block >= 0;
            if constexpr(!decltype(first)::value)
                x.ks[h] = lane_of(ks_of, from), x.vs[h] = lane_of(vs_of, from);
            if(block < 0)
            {
#pragma unroll
                for(int j = 0; j < KJ; ++j)
                    x.kb[h][j] = u32x4{0, 0, 0, 0};
#pragma unroll
                for(int i = 0; i < 4; ++i)
#pragma unroll
                    for(int e = 0; e < E / 4; ++e)
                        x.vb[4 * h + i][e] = 0;
                continue;
            }
            const int64_t at       = (int64_t)block * p.cache.stride_block + (int64_t)((first_of(turn) + 16 * h) & in_block) * p.cache.stride_token;
            const uint8_t* const k = kc + at;
            const uint8_t* const v = vc + at;
#pragma unroll
            for(int j = 0; j < KJ; ++j)
                x.kb[h][j] = *reinterpret_cast<const u32x4*>(k + k_off[j]);
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                const uint8_t* const vi = v + (int64_t)i * p.cache.stride_token + v_off;
                if constexpr(E == 8)
                {
                    const u32x2 y = *reinterpret_cast<const u32x2*>(vi);
                    x.vb[4 * h + i][0] = y[0], x.vb[4 * h + i][1] = y[1];
                }
                else
                    x.vb[4 * h + i][0] = *reinterpret_cast<const uint32_t*>(vi);
            }
        }
        if constexpr(decltype(first)::value)
        {
            __builtin_amdgcn_sched_barrier(0);
            scales_to(x, turn);
        }
    };

    Turn even, odd;
    if(turns > 0)
        fetch(even, 0, std::true_type{});
    i32x4 qf[KJ][2];
#pragma unroll
    for(int j = 0; j < KJ; ++j)
#pragma unroll
        for(int h = 0; h < 2; ++h)
        {
            const int d = 64 * j + 16 * g + 8 * h;
            qf[j][h]    = i32x4{0, 0, 0, 0};
            if(row_live && d < D)
                qf[j][h] = *reinterpret_cast<const i32x4*>(reinterpret_cast<const T*>(p.q) + token * p.sq_t + (int64_t)head * p.sq_h + d);
        }

    f32x4 acc[E];
#pragma unroll
    for(int j = 0; j < E; ++j)
        acc[j] = f32x4{0, 0, 0, 0};
    float m = -__builtin_inff(), l = 0.0f;
    ValueScale unit;

    auto multiply = [&](Turn& x, int turn) {
        const int t0 = first_of(turn);
        if(t0 + 32 > most) // (what lies behind the last token is no value: zero, whatever its bytes are)
        {
#pragma unroll
            for(int i = 0; i < 8; ++i)
#pragma unroll
                for(int e = 0; e < E / 4; ++e)
                    x.vb[i][e] = t0 + 16 * (i >> 2) + 4 * g + (i & 3) < most ? x.vb[i][e] : 0;
        }
        float s[8], top = -__builtin_inff();
#pragma unroll
        for(int h = 0; h < 2; ++h)
        {
            f32x4 y = {0, 0, 0, 0};
#pragma unroll
            for(int j = 0; j < KJ; ++j)
            {
                y = mfma_qk<T>(codes8<CODE, T>(x.kb[h][j][0], x.kb[h][j][1]), qf[j][0], y);
                y = mfma_qk<T>(codes8<CODE, T>(x.kb[h][j][2], x.kb[h][j][3]), qf[j][1], y);
            }
            const float c = x.ks[h] * p.scale;
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                const bool seen = x.there[h] && t0 + 16 * h + 4 * g + i < see;
                s[4 * h + i]    = seen ? y[i] * c : -__builtin_inff();
                top             = __builtin_fmaxf(top, s[4 * h + i]);
            }
        }
        top = max_over_rows(top);
        // (the maximum is there for the range only and raised only by leaps, 2^6 or more: the sums are seldom rescaled)
        float keep_o   = 1.0f;
        const float v0 = t0 < see ? __builtin_fabsf(x.vs[0]) : 0.0f, v1 = t0 + 16 < see ? __builtin_fabsf(x.vs[1]) : 0.0f; // (no block: zero)
        if(__any(v0 > unit.top || v1 > unit.top))
            keep_o = unit.take(v0, v1);
        if(__any(top > m + 6.0f))
        {
            // (the rows that leap, no others: a row's bits are its own)
            float now = top > m + 6.0f ? top : m;
            asm volatile("" : "+v"(now)); // (in the branch: left to itself the compiler chooses outside of it, every turn)
            const float keep = __builtin_amdgcn_exp2f(m - (now == -__builtin_inff() ? 0.0f : now));
            m = now;
            l *= keep;
            keep_o *= keep;
        }
        if(__any(keep_o != 1.0f))
        {
#pragma unroll
            for(int j = 0; j < E; ++j)
                acc[j] *= keep_o;
        }
        const float zero = m == -__builtin_inff() ? 0.0f : m; // (nothing seen yet: exp2(-inf - 0) = 0)
        const float w[2] = {unit.of(x.vs[0]), unit.of(x.vs[1])};
        float pr[8];
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            pr[i] = __builtin_amdgcn_exp2f(s[i] - zero);
            l += pr[i];
            // (masked: no value scale, which may be an infinity or NaN, gets into the sum)
            pr[i] = s[i] == -__builtin_inff() ? 0.0f : pr[i] * w[i >> 2];
        }
        const i32x4 pf = {(int)pack_f16(pr[0], pr[1]), (int)pack_f16(pr[2], pr[3]), (int)pack_f16(pr[4], pr[5]),
                          (int)pack_f16(pr[6], pr[7])};
#pragma unroll
        for(int e = 0; e < E / 4; ++e)
        {
            uint32_t lo[4], hi[4];
            transpose4(x.vb[0][e], x.vb[1][e], x.vb[2][e], x.vb[3][e], lo);
            transpose4(x.vb[4][e], x.vb[5][e], x.vb[6][e], x.vb[7][e], hi);
#pragma unroll
            for(int j = 0; j < 4; ++j)
                acc[4 * e + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    __builtin_bit_cast(f16x8, (codes8<CODE, _Float16>(lo[j], hi[j]))), __builtin_bit_cast(f16x8, pf), acc[4 * e + j], 0, 0, 0);
        }
    };
    for(int turn = 0; turn < turns; turn += 2)
    {
        if(turn + 1 < turns)
            fetch(odd, turn + 1, std::false_type{});
        multiply(even, turn);
        if(turn + 2 < turns)
            fetch(even, turn + 2, std::false_type{});
        if(turn + 1 < turns)
            multiply(odd, turn + 1);
    }

    // the waves' sums. Lane (r, g) holds elements (4g + i) * E + j of row r at acc[j][i].
    l = sum_over_rows(l);
    if(g == 0)
        part_m[wave][r] = m, part_l[wave][r] = l;
#pragma unroll
    for(int j = 0; j < E; ++j)
#pragma unroll
        for(int i = 0; i < 4; ++i)
            part[wave][r][(4 * g + i) * E + j] = acc[j][i] * unit.top;
    __syncthreads();
    // thread (row, 16 of them a row) joins E elements
    if(threadIdx.x >= 256)
        return;
    const int row = threadIdx.x >> 4, c = threadIdx.x & 15;
    const int jt = row / p.tile_heads, jh = h0 + (row - jt * p.tile_heads);
    if(jt >= p.tile_tokens || tile.first + jt >= tile.q_len || jh >= p.group || c * E >= D)
        return;
    float top = -__builtin_inff();
#pragma unroll
    for(int w = 0; w < NW; ++w)
        top = __builtin_fmaxf(top, part_m[w][row]);
    const float zero = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f, o[E];
#pragma unroll
    for(int e = 0; e < E; ++e)
        o[e] = 0.0f;
#pragma unroll
    for(int w = 0; w < NW; ++w)
    {
        const float f = __builtin_amdgcn_exp2f(part_m[w][row] - zero);
        sum += part_l[w][row] * f;
#pragma unroll
        for(int e = 0; e < E; ++e)
            o[e] += part[w][row][c * E + e] * f;
    }
    const int64_t out_token = tile.q0 + tile.first + jt, out_head = kvh * p.group + jh;
    if(p.splits == 1)
    {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum; // (a row that sees nothing: zero)
        T* const to = reinterpret_cast<T*>(p.o) + out_token * p.so_t + out_head * p.so_h + c * E;
        typedef T tx __attribute__((ext_vector_type(E)));
        tx x;
#pragma unroll
        for(int e = 0; e < E; ++e)
            x[e] = (T)(o[e] * inv);
        *reinterpret_cast<tx*>(to) = x;
    }
    else
    {
        const int64_t at = (out_token * p.heads + out_head) * p.splits + split;
        float* const to  = p.ws + at * DP + c * E;
#pragma unroll
        for(int e = 0; e < E; e += 4)
            *reinterpret_cast<f32x4*>(to + e) = f32x4{o[e], o[e + 1], o[e + 2], o[e + 3]};
        if(c == 0)
        {
            float* const ml = p.ws + attention_rows(p) * p.splits * DP + at * 2;
            ml[0] = top, ml[1] = sum;
        }
    }
}

// joins the shares of a query row: 16 lanes a row. Rows outside the sequences (cu_q) are left alone.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs p)
{
    constexpr int E = DP / 16;
    const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int c       = threadIdx.x & 15;
    if(row >= attention_rows(p) || c * E >= p.cache.head_dim)
        return;
    const int64_t token = row / p.heads, head = row - token * p.heads;
    if(token < p.cu_q[0] || token >= p.cu_q[p.batch])
        return;
    const float* const ml = p.ws + attention_rows(p) * p.splits * DP + row * p.splits * 2;
    const float* const at = p.ws + row * p.splits * DP + c * E;
    float top             = -__builtin_inff();
#pragma unroll 8
    for(int s = 0; s < p.splits; ++s)
        top = __builtin_fmaxf(top, ml[2 * s]);
    const float zero = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f, o[E];
#pragma unroll
    for(int e = 0; e < E; ++e)
        o[e] = 0.0f;
#pragma unroll 8
    for(int s = 0; s < p.splits; ++s)
    {
        const float f = __builtin_amdgcn_exp2f(ml[2 * s] - zero);
        sum += ml[2 * s + 1] * f;
#pragma unroll
        for(int e = 0; e < E; e += 4)
        {
            const f32x4 x = *reinterpret_cast<const f32x4*>(at + (int64_t)s * DP + e);
#pragma unroll
            for(int i = 0; i < 4; ++i)
                o[e + i] += x[i] * f;
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    typedef T tx __attribute__((ext_vector_type(E)));
    tx x;
#pragma unroll
    for(int e = 0; e < E; ++e)
        x[e] = (T)(o[e] * inv);
    *reinterpret_cast<tx*>(reinterpret_cast<T*>(p.o) + token * p.so_t + head * p.so_h + c * E) = x;
}

struct Plan
{
    int tile_tokens, tile_heads, head_tiles, tiles, splits;
    bool prompt;
};

Plan plan(const ckx_kv_cache8& c, int batch, int tokens, int heads, int max_kv, int max_blocks)
{
    Plan p;
    const int group = heads / c.num_heads;
    p.prompt        = (int64_t)tokens * group > (int64_t)kPromptRows * batch;
    const int rows  = p.prompt ? 128 : 16, most_heads = p.prompt ? 32 : 16;
    p.tile_heads    = group < most_heads ? group : most_heads;
    p.head_tiles    = (group + p.tile_heads - 1) / p.tile_heads;
    p.tile_tokens   = rows / p.tile_heads;
    p.tiles         = p.tile_tokens == 1 ? tokens : tokens / p.tile_tokens + batch;
    // Shares of the cached tokens, joined by a second launch, where the tiles alone leave CUs without work. Single tokens: one
    // workgroup a CU (what fits on one), none of under 256 tokens, a turn for each wave; 8 sequences of 8192: 30.5 us, 32.7 with two
    // a CU, 38.3 with three. Prompts: up to two a CU, none of under 128 tokens, two steps, and none under 1024 cached tokens, where the
    // second launch costs what the shares give (whole / shares of 128, heads of 128: 1 x 512 new 21.0 / 25.9 us, 1 x 1024 34.8 / 34.5,
    // 4 x (1000 + 100) 26.8 / 20.5; shares of 256 22.0).
    const int64_t groups  = (int64_t)(tokens < p.tiles ? tokens : p.tiles) * c.num_heads * p.head_tiles;
    const int64_t longest = (int64_t)max_blocks * c.block_size;
    const int64_t kv      = max_kv < longest ? max_kv : longest;
    int64_t splits        = p.prompt ? 512 / groups : (256 + groups - 1) / groups;
    const int64_t least   = p.prompt ? 128 : 256;
    if(splits > kv / least)
        splits = kv / least;
    if(p.prompt && kv < 1024)
        splits = 1;
    p.splits = (int)(splits < 1 ? 1 : splits > 64 ? 64 : splits);
    return p;
}

int padded(int head_dim) { return head_dim <= 64 ? 64 : 128; }

template <typename T, int CODE>
hipError_t launch_rows(const AttentionArgs& a, hipStream_t s)
{
    const dim3 grid((unsigned)((int64_t)a.tiles * a.cache.num_heads * a.head_tiles * a.splits));
    if(padded(a.cache.head_dim) == 64)
        hipLaunchKernelGGL((attention_rows_kernel<T, CODE, 64>), grid, dim3(NW * 64), 0, s, a);
    else
        hipLaunchKernelGGL((attention_rows_kernel<T, CODE, 128>), grid, dim3(NW * 64), 0, s, a);
    return hipGetLastError();
}

template <typename T>
hipError_t launch(const AttentionArgs& a, bool prompt, hipStream_t s)
{
    hipError_t e = prompt ? attention_tile_launch(a, std::is_same<T, _Float16>::value, s)
                   : a.cache.type == CKX_TYPE_E4M3 ? launch_rows<T, CODE_E4M3>(a, s)
                                                   : launch_rows<T, CODE_I8>(a, s);
    if(e != hipSuccess || a.splits == 1)
        return e;
    const dim3 grid((unsigned)((attention_rows(a) + 15) / 16));
    if(padded(a.cache.head_dim) == 64)
        hipLaunchKernelGGL((attention_join_kernel<T, 64>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((attention_join_kernel<T, 128>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

} // namespace

// a launch has fewer than 2^32 threads
bool attention_fits(const ckx_kv_cache8& c, int batch, int tokens, int heads, int max_kv, int max_blocks)
{
    const Plan p = plan(c, batch, tokens, heads, max_kv, max_blocks);
    return (int64_t)p.tiles * c.num_heads * p.head_tiles * p.splits < (1ll << 32) / (NW * 64);
}

int64_t attention_workspace(const ckx_kv_cache8& c, int batch, int tokens, int heads, int max_kv, int max_blocks)
{
    const Plan p = plan(c, batch, tokens, heads, max_kv, max_blocks);
    return p.splits == 1 ? 0 : (int64_t)tokens * heads * p.splits * (padded(c.head_dim) + 2) * 4;
}

hipError_t attention_launch(AttentionArgs a, int q_type, hipStream_t s)
{
    const Plan p  = plan(a.cache, a.batch, a.tokens, a.heads, a.max_kv, a.max_blocks);
    a.tile_tokens = p.tile_tokens, a.tile_heads = p.tile_heads, a.head_tiles = p.head_tiles, a.tiles = p.tiles, a.splits = p.splits;
    return q_type == CKX_TYPE_F16 ? launch<_Float16>(a, p.prompt, s) : launch<__bf16>(a, p.prompt, s);
}

} // namespace ckx
