// int8 GEMM with a scale for each token and channel, dense and for each expert's rows (formulas: include/ckx.h,
// ckx_gemm_i8_tokenscale and ckx_experts_gemm_i8).
#include <cmath>

#include "gemm_i8_big.hpp"

namespace ckx {

namespace {

// 16 bytes of which `left` are there, zeros behind them, any alignment
__device__ __forceinline__ i32x4 ragged16(const int8_t* at, int left)
{
    if(left >= 16)
        return load_vec<i32x4>(at);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for(int i = 0; i < 16; ++i)
        if(i < left)
            w[i >> 2] |= (uint32_t)(uint8_t)at[i] << (8 * (i & 3));
    return i32x4{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
}

// Any K, leading dimension and address: 128 rows x 128 rows of B, four waves of 64 x 64, the operands through registers into LDS, a K
// tile of 128 ahead: asked for in front of the products, put into LDS behind them. 128 / 4096 x 11008 x 4100: 40 / 317 us, where K = 4096 takes 14.5 / 148:
// unaligned vectors through registers.
template <typename T, bool GATED>
__global__ __launch_bounds__(256) void gemm_i8_any_kernel(GemmI8Args p)
{
    constexpr int BM = 128, BN = 128, TILE = 128 * 128;
    __shared__ __align__(16) uint8_t lds[2][2][TILE];
    __shared__ float sb[BN], bias[BN];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1, q = lane >> 4;
    I8Tile t;
    if(!i8_find_tile(p, (int)blockIdx.x, BM, t))
        return;
    const int n0 = t.tn * (GATED ? BN / 2 : BN);
    i8_load_scales<GATED>(p, t.expert, n0, BN, tid, 256, sb, bias);
    // a wave fills LDS rows wave * 32 ... + 31 of either tile, eight rows a load; chunk c of row r lies at c ^ (r & 7). Rows that are not there
    // take another's place: C does not have them, or their scale is 0
    const int8_t *ra[4], *rb[4];
    int row[4], m[4];
#pragma unroll
    for(int j = 0; j < 4; ++j)
        row[j] = wave * 32 + j * 8 + (lane >> 3);
    i8_rows_of_a(p, t, row, m);
#pragma unroll
    for(int j = 0; j < 4; ++j)
    {
        bool second;
        const int n = min(n0 + i8_col_of<GATED>((uint32_t)row[j], second), p.N - 1), kc = ((lane & 7) ^ (row[j] & 7)) * 16;
        rb[j]       = p.b + (int64_t)t.expert * p.batch_b + ((int64_t)n + (second ? p.N : 0)) * p.ldb + kc;
        ra[j]       = m[j] >= 0 ? p.a + (int64_t)m[j] * p.lda + kc : rb[j];
    }
    struct Rows
    {
        i32x4 a[4], b[4];
    };
    auto fetch = [&](Rows& x, int g) {
        if((g + 1) * 128 <= p.K)
        {
#pragma unroll
            for(int j = 0; j < 4; ++j)
                x.a[j] = load_vec<i32x4>(ra[j] + g * 128), x.b[j] = load_vec<i32x4>(rb[j] + g * 128);
        }
        else
#pragma unroll
            for(int j = 0; j < 4; ++j)
            {
                const int left = p.K - g * 128 - ((lane & 7) ^ (row[j] & 7)) * 16;
                x.a[j] = ragged16(ra[j] + g * 128, left), x.b[j] = ragged16(rb[j] + g * 128, left);
            }
    };
    auto put = [&](const Rows& x, int stage) {
        uint8_t* const at = &lds[stage][0][wave * 4096 + lane * 16];
#pragma unroll
        for(int j = 0; j < 4; ++j)
            *reinterpret_cast<i32x4*>(at + j * 1024) = x.a[j], *reinterpret_cast<i32x4*>(at + j * 1024 + TILE) = x.b[j];
    };
    i32x4 acc[4][4];
#pragma unroll
    for(int i = 0; i < 4; ++i)
#pragma unroll
        for(int j = 0; j < 4; ++j)
            acc[i][j] = i32x4{0, 0, 0, 0};
    Rows next;
    if(p.ksteps > 0)
    {
        fetch(next, 0);
        put(next, 0);
    }
    for(int g = 0; g < p.ksteps; ++g)
    {
        __syncthreads();
        if(g + 1 < p.ksteps)
            fetch(next, g + 1);
#pragma unroll
        for(int ks = 0; ks < 2; ++ks)
        {
            auto fragment = [&](const uint8_t* tile, int row) {
                return *reinterpret_cast<const i32x4*>(tile + row * 128 + (((ks * 4 + q) ^ (row & 7)) << 4));
            };
            i32x4 bf[4];
#pragma unroll
            for(int j = 0; j < 4; ++j)
                bf[j] = fragment(lds[g & 1][1], wn * 64 + j * 16 + (lane & 15));
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                const i32x4 af = fragment(lds[g & 1][0], wm * 64 + i * 16 + (lane & 15));
#pragma unroll
                for(int j = 0; j < 4; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j], af, acc[i][j], 0, 0, 0);
            }
        }
        if(g + 1 < p.ksteps)
            put(next, (g + 1) & 1); // (every wave has read it before this step's barrier)
    }
    __syncthreads(); // (K = 0: the scales)
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        const int r = wm * 64 + i * 16 + (lane & 15), m = t.m0 + r;
        if(r >= t.rows)
            continue;
        const int from = i8_row_of_a(p, t, r);
        i8_finish<T, GATED>(reinterpret_cast<T*>(p.c) + (int64_t)m * p.ldc, n0 + wn * (GATED ? 32 : 64), p.N, q, acc[i], from >= 0 ? p.sa[from] : 0.0f,
                            sb + wn * 64, bias + wn * 64);
    }
}

// BM rows x BN rows of B, WM x WN x KH waves, NST stages of operands in LDS: the loads of a K tile (128) are asked for NST - 1 tiles
// ahead. The way from the L2s into LDS bounds the steps: 70 to 80 GB/s a CU with any of these tiles (64 x 128: 24 KB in 0.29 to 0.33 us, 128
// x 128: 32 KB in 0.37 to 0.44), while LDS is active for 13 to 20 % of the time and the matrix cores for 16 to 25 %. To get there a SIMD needs two
// waves, or one's wait for its fragments shows. Either a CU holds two workgroups (KH = 1), or it holds one and KH = 2 waves share an output, one for
// each half of a K tile; then the next tile's fragments are read while the present are multiplied. 64 x 128 with both from 0.43 to 0.29 us a step (128
// rows of 4096 x 4096 17.5 to 13.5; two waves alone 14.0).
// The direct loads are inline assembly: the compiler, told of them, would wait for all of them before every LDS read of another
// stage. Its own LDS reads it waits for itself; the wait for the direct loads stands in front of the barrier.
// The bounds of a resource are checked against a lane's offset without the scalar one, which holds K: a lane whose columns lie behind K asks
// out of range, for A and for B, or it would read behind the last row's end.
template <typename T, bool GATED, int BM, int BN, int WM, int WN, int KH, int NST>
__global__ __launch_bounds__(WM* WN* KH * 64) void gemm_i8_tile_kernel(GemmI8Args p)
{
    constexpr int NW = WM * WN * KH, MT = BM / WM / 16, NG = BN / WN / 64, NLA = BM / 8 / NW, NLB = BN / 8 / NW, LPT = NLA + NLB, COLS = GATED ? BN / 2 : BN;
    constexpr int A_TILE = BM * 128, B_AT = NST * A_TILE, B_TILE = BN * 128, S_AT = B_AT + NST * B_TILE;
    static_assert(BN / WN % 64 == 0 && BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "");
    static_assert(KH == 1 || (MT % 2 == 0 && WM * WN * MT * NG * 4096 <= S_AT), "");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[]; // [A | B | scales of rows, of columns, biases]
    float* const s_row = reinterpret_cast<float*>(lds + S_AT);
    float* const s_col = s_row + BM;
    float* const s_bias = s_col + BN;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kh = wave / (WM * WN), wm = wave / WN % WM, wn = wave % WN, q = lane >> 4;
    I8Tile t;
    int run = 0;
    if(p.offsets)
    {
        if(!i8_expert_tile(p, (int)blockIdx.x, BM, t))
            return;
    }
    else
    {
        int tm; // (a run of K tiles takes the place of a batch)
        tile_of_block((int)blockIdx.x, p.tiles_m, p.tiles_n, p.ksplit, run, tm, t.tn);
        t.expert = 0, t.m0 = tm * BM, t.rows = min(BM, p.M - t.m0);
    }
    const int g0 = run * p.per, g1 = min(g0 + p.per, p.ksteps);
    const int n0 = t.tn * COLS;
    // resources that end with the last byte of what the tile may read; rows are counted from the tile's first, or from the first
    // of A (gathered) and of the expert's B (its halves lie apart)
    const int64_t a0 = p.rows ? 0 : t.m0, b0 = GATED ? 0 : n0;
    const int64_t rows_a = p.rows ? p.rows_a : min((int64_t)t.rows, (int64_t)p.rows_a - t.m0), rows_b = GATED ? 2 * (int64_t)p.N : min(BN, p.N - n0);
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.a + a0 * p.lda, rows_a > 0 ? (uint32_t)((rows_a - 1) * p.lda + p.K) : 0u);
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(p.b + (int64_t)t.expert * p.batch_b + b0 * p.ldb, (uint32_t)((rows_b - 1) * p.ldb + p.K));
    const uint32_t base = (uint32_t)(uintptr_t)(lds_ptr_t)lds;
    // a load fills eight rows, chunk c of row r at c ^ (r & 7)
    const int kc = ((lane & 7) ^ (lane >> 3)) * 16;
    uint32_t oa[NLA], ob[NLB];
#pragma unroll
    for(int j = 0; j < NLB; ++j)
    {
        bool second;
        const int n = n0 + i8_col_of<GATED>((uint32_t)((wave * NLB + j) * 8 + (lane >> 3)), second);
        ob[j]       = n < p.N ? (uint32_t)(n - b0 + (second ? p.N : 0)) * (uint32_t)p.ldb + kc : kOutOfRange;
    }
    int row[NLA], m[NLA];
#pragma unroll
    for(int j = 0; j < NLA; ++j)
        row[j] = (wave * NLA + j) * 8 + (lane >> 3);
    i8_rows_of_a(p, t, row, m);
#pragma unroll
    for(int j = 0; j < NLA; ++j)
        oa[j] = m[j] >= 0 ? (uint32_t)(m[j] - a0) * (uint32_t)p.lda + kc : kOutOfRange;
    auto load16 = [&](const __amdgpu_buffer_rsrc_t& r, uint32_t off, uint32_t k, uint32_t at) {
        asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(off), "s"(r), "s"(k), "s"(at));
    };
    // (tiles behind the last come as zeros: the counts of loads under way stay the same)
    auto load_all = [&](int g) {
        const uint32_t k = (uint32_t)g * 128, st = (uint32_t)g % NST;
        const bool in = (int)k + kc < p.K;
#pragma unroll
        for(int j = 0; j < NLA; ++j)
            load16(ra, in ? oa[j] : kOutOfRange, k, base + st * A_TILE + (wave * NLA + j) * 1024);
#pragma unroll
        for(int j = 0; j < NLB; ++j)
            load16(rb, in ? ob[j] : kOutOfRange, k, base + B_AT + st * B_TILE + (wave * NLB + j) * 1024);
    };
    for(int g = g0; g < g0 + NST - 1; ++g)
        load_all(g);
    // (behind the first loads: their waits are the compiler's, and count those too)
    i8_load_scales<GATED>(p, t.expert, n0, BN, tid, NW * 64, s_col, s_bias);
    for(int r = tid; r < BM; r += NW * 64)
    {
        const int m = i8_row_of_a(p, t, r);
        s_row[r]    = m >= 0 ? p.sa[m] : 0.0f;
    }
    i32x4 acc[MT][NG][4];
#pragma unroll
    for(int i = 0; i < MT; ++i)
#pragma unroll
        for(int j = 0; j < NG * 4; ++j)
            acc[i][j / 4][j % 4] = i32x4{0, 0, 0, 0};
    const int a_row = wm * (BM / WM) + (lane & 15), b_row = wn * NG * 64 + (lane & 15);
    const int a_lo = a_row * 128 + ((q ^ (a_row & 7)) << 4), b_lo = B_AT + b_row * 128 + ((q ^ (b_row & 7)) << 4);
    struct Fragments
    {
        i32x4 a[2 / KH][MT], b[2 / KH][NG * 4];
    };
    auto read = [&](Fragments& f, int g) {
        const uint8_t* const at = lds + g % NST * A_TILE;
        const uint8_t* const bt = lds + g % NST * B_TILE;
#pragma unroll
        for(int s = 0; s < 2 / KH; ++s)
        {
            const int half = (KH > 1 ? kh : s) * 64;
#pragma unroll
            for(int j = 0; j < NG * 4; ++j)
                f.b[s][j] = *reinterpret_cast<const i32x4*>(bt + (b_lo ^ half) + j * 2048);
#pragma unroll
            for(int i = 0; i < MT; ++i)
                f.a[s][i] = *reinterpret_cast<const i32x4*>(at + (a_lo ^ half) + i * 2048);
        }
    };
    auto multiply = [&](const Fragments& f) {
#pragma unroll
        for(int s = 0; s < 2 / KH; ++s)
#pragma unroll
            for(int i = 0; i < MT; ++i)
#pragma unroll
                for(int j = 0; j < NG * 4; ++j)
                    acc[i][j / 4][j % 4] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.b[s][j], f.a[s][i], acc[i][j / 4][j % 4], 0, 0, 0);
    };
    // until all of the workgroup's loads but those of `tiles` tiles have landed
    auto landed = [&](auto tiles) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(decltype(tiles)::value * LPT) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    if constexpr(KH > 1)
    {
        // the fragments of a tile are read while the one before is multiplied
        Fragments x, y;
        auto step = [&](const Fragments& now, Fragments& next, int g) {
            landed(std::integral_constant<int, NST - 3>());
            load_all(g + NST - 1); // (into the stage of the tile before, which every wave has multiplied before this barrier)
            read(next, g + 1);
            multiply(now);
        };
        landed(std::integral_constant<int, NST - 2>());
        read(x, g0);
        for(int g = g0; g < g1; g += 2)
        {
            step(x, y, g);
            if(g + 1 < g1)
                step(y, x, g + 1);
        }
    }
    else
        for(int g = g0; g < g1; ++g)
        {
            landed(std::integral_constant<int, NST - 2>());
            load_all(g + NST - 1); // (into the stage that every wave has read before this barrier)
            Fragments f;
            read(f, g);
            multiply(f);
        }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // (no load may land in LDS that is another workgroup's by then)
    __syncthreads();                                 // (a run without K tiles: the scales)
    constexpr int MINE = MT / KH;                    // fragment rows that the wave finishes
    i32x4 sum[MINE][NG][4];
    if constexpr(KH > 1)
    {
        // each of the two waves of an output hands the other half of its sums over
        i32x4* const there = reinterpret_cast<i32x4*>(lds) + ((wm * WN + wn) * KH + kh) * (MINE * NG * 4 * 64) + lane;
        i32x4* const here  = reinterpret_cast<i32x4*>(lds) + ((wm * WN + wn) * KH + 1 - kh) * (MINE * NG * 4 * 64) + lane;
#pragma unroll
        for(int i = 0; i < MINE; ++i)
#pragma unroll
            for(int j = 0; j < NG * 4; ++j)
            {
                here[(i * NG * 4 + j) * 64] = kh ? acc[i][j / 4][j % 4] : acc[MINE + i][j / 4][j % 4];
                sum[i][j / 4][j % 4]        = kh ? acc[MINE + i][j / 4][j % 4] : acc[i][j / 4][j % 4];
            }
        __syncthreads();
#pragma unroll
        for(int i = 0; i < MINE; ++i)
#pragma unroll
            for(int j = 0; j < NG * 4; ++j)
                sum[i][j / 4][j % 4] += there[(i * NG * 4 + j) * 64];
    }
    else
#pragma unroll
        for(int i = 0; i < MINE; ++i)
#pragma unroll
            for(int j = 0; j < NG * 4; ++j)
                sum[i][j / 4][j % 4] = acc[i][j / 4][j % 4];
#pragma unroll
    for(int i = 0; i < MINE; ++i)
    {
        const int r = wm * (BM / WM) + (kh * MINE + i) * 16 + (lane & 15);
        if(r >= t.rows)
            continue;
#pragma unroll
        for(int g = 0; g < NG; ++g)
        {
            const int at = wn * NG + g, n = n0 + at * (GATED ? 32 : 64);
            if(p.ksplit > 1)
            {
                int* const row = p.ws + ((int64_t)run * p.M + t.m0 + r) * p.N * (GATED ? 2 : 1);
#pragma unroll
                for(int h = 0; h < 2; ++h)
                {
                    const int c = n + 8 * q + (GATED ? 0 : 32 * h);
                    int* const to = row + (GATED && h ? p.N : 0);
                    store_room<4>(to + c, sum[i][g][2 * h], (p.N - c) * 4, false);
                    store_room<4>(to + c + 4, sum[i][g][2 * h + 1], (p.N - c - 4) * 4, false);
                }
            }
            else
                i8_finish<T, GATED>(reinterpret_cast<T*>(p.c) + (int64_t)(t.m0 + r) * p.ldc, n, p.N, q, sum[i][g], s_row[r], s_col + at * 64, s_bias + at * 64);
        }
    }
}

// C from the sums of the runs: four columns a thread
template <typename T, bool GATED>
__global__ __launch_bounds__(256) void gemm_i8_join_kernel(GemmI8Args p, int quads)
{
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t m  = id / quads;
    const int n      = (int)(id - m * quads) * 4;
    if(m >= p.M)
        return;
    const int64_t wide = (int64_t)p.N * (GATED ? 2 : 1);
    const float sa     = p.sa[m];
    T* const c         = reinterpret_cast<T*>(p.c) + m * p.ldc + n;
    float x[2][4];
#pragma unroll
    for(int h = 0; h < (GATED ? 2 : 1); ++h)
    {
        const int64_t col = n + (h ? p.N : 0);
        const int* at     = p.ws + m * wide + col;
        i32x4 v           = {0, 0, 0, 0};
        for(int r = 0; r < p.ksplit; ++r, at += (int64_t)p.M * wide)
            if(n + 4 <= p.N)
                v += load_vec<i32x4>(at);
            else
                for(int j = 0; n + j < p.N; ++j)
                    v[j] += at[j];
#pragma unroll
        for(int j = 0; j < 4; ++j)
            x[h][j] = n + j < p.N ? (float)v[j] * sa * p.sb[col + j] + (p.bias ? p.bias[col + j] : 0.0f) : 0.0f;
    }
    typedef T tx4 __attribute__((ext_vector_type(4)));
    tx4 out;
#pragma unroll
    for(int j = 0; j < 4; ++j)
        out[j] = (T)(GATED ? i8_silu<T>(x[0][j]) * x[1][j] : x[0][j]);
    if(n + 4 <= p.N)
        reinterpret_cast<AnyAlign<tx4>*>(c)->v = out;
    else
        for(int j = 0; n + j < p.N; ++j)
            c[j] = out[j];
}

// Few rows: a workgroup takes MT x NT tiles of 16 x 16 and its NW waves share the K tiles among them, each straight from memory into
// its registers (the next K tile's 32 bytes a lane and tile row are on their way while one is multiplied); the waves' sums meet in LDS.
// Nothing waits at a barrier until the end: what a product of few rows needs, which is bound by reading B once. Gated, the tiles of B
// come in pairs, a gate's and its partner's. ANY: any K, stride and address, 1 / 16 x 11008 x 4100 16 us.
template <typename T, bool GATED, int MT, int NT, int NW, bool ANY>
__global__ __launch_bounds__(NW * 64) void gemm_i8_direct_kernel(GemmI8Args p)
{
    constexpr int BM = MT * 16, COLS = NT * 16 / (GATED ? 2 : 1);
    static_assert(!GATED || NT % 2 == 0, "");
    __shared__ __align__(16) i32x4 sums[NW][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    I8Tile t;
    if(!i8_find_tile(p, (int)blockIdx.x, BM, t))
        return;
    const int n0 = t.tn * COLS;
    const int64_t a0 = p.rows ? 0 : t.m0, b0 = GATED ? 0 : n0;
    const int64_t rows_a = p.rows ? p.rows_a : min((int64_t)t.rows, (int64_t)p.rows_a - t.m0), rows_b = GATED ? 2 * (int64_t)p.N : min(COLS, p.N - n0);
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.a + a0 * p.lda, rows_a > 0 ? (uint32_t)((rows_a - 1) * p.lda + p.K) : 0u);
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(p.b + (int64_t)t.expert * p.batch_b + b0 * p.ldb, (uint32_t)((rows_b - 1) * p.ldb + p.K));
    struct Step
    {
        i32x4 a[MT][2], b[NT][2];
    };
    uint32_t oa[MT], ob[NT];
    const int8_t *pa[MT], *pb[NT]; // (ANY)
#pragma unroll
    for(int j = 0; j < NT; ++j)
    {
        const int n = n0 + (GATED ? j / 2 : j) * 16 + r;
        pb[j]       = p.b + (int64_t)t.expert * p.batch_b + (int64_t)(min(n, p.N - 1) + (GATED && (j & 1) ? p.N : 0)) * p.ldb + q * 16;
        ob[j]       = n < p.N ? (uint32_t)(n - b0 + (GATED && (j & 1) ? p.N : 0)) * (uint32_t)p.ldb + q * 16 : kOutOfRange;
    }
    int row[MT], m[MT];
#pragma unroll
    for(int i = 0; i < MT; ++i)
        row[i] = i * 16 + r;
    i8_rows_of_a(p, t, row, m);
#pragma unroll
    for(int i = 0; i < MT; ++i)
    {
        pa[i] = m[i] >= 0 ? p.a + (int64_t)m[i] * p.lda + q * 16 : pb[0]; // (a row that is not there: C does not have it, or its scale is 0)
        oa[i] = m[i] >= 0 ? (uint32_t)(m[i] - a0) * (uint32_t)p.lda + q * 16 : kOutOfRange;
    }
    auto load = [&](Step& x, int g) {
        if constexpr(ANY)
        {
            auto from = [&](auto whole, const int8_t* at, int h) {
                const int k = g * 128 + h * 64;
                if constexpr(decltype(whole)::value)
                    return load_vec<i32x4>(at + k);
                else
                    return ragged16(at + k, p.K - k - q * 16);
            };
            auto both = [&](auto whole) {
#pragma unroll
                for(int h = 0; h < 2; ++h)
                {
#pragma unroll
                    for(int j = 0; j < NT; ++j)
                        x.b[j][h] = from(whole, pb[j], h);
#pragma unroll
                    for(int i = 0; i < MT; ++i)
                        x.a[i][h] = from(whole, pa[i], h);
                }
            };
            if((g + 1) * 128 <= p.K)
                both(std::true_type{});
            else
                both(std::false_type{});
        }
        else
#pragma unroll
        for(int h = 0; h < 2; ++h)
        {
            const int k        = g * 128 + h * 64;
            const uint32_t out = k + q * 16 < p.K ? 0u : kOutOfRange; // (columns behind K, and tiles behind the last)
#pragma unroll
            for(int j = 0; j < NT; ++j)
                x.b[j][h] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rb, (int)(ob[j] | out), k, 0));
#pragma unroll
            for(int i = 0; i < MT; ++i)
                x.a[i][h] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(ra, (int)(oa[i] | out), k, 0));
        }
    };
    i32x4 acc[MT][NT];
#pragma unroll
    for(int i = 0; i < MT; ++i)
#pragma unroll
        for(int j = 0; j < NT; ++j)
            acc[i][j] = i32x4{0, 0, 0, 0};
    auto multiply = [&](const Step& x) {
#pragma unroll
        for(int h = 0; h < 2; ++h)
#pragma unroll
            for(int i = 0; i < MT; ++i)
#pragma unroll
                for(int j = 0; j < NT; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.b[j][h], x.a[i][h], acc[i][j], 0, 0, 0);
    };
    Step x, y;
    if(wave < p.ksteps)
        load(x, wave);
    for(int g = wave; g < p.ksteps; g += 2 * NW)
    {
        if(g + NW < p.ksteps)
            load(y, g + NW);
        multiply(x);
        if(g + 2 * NW < p.ksteps)
            load(x, g + 2 * NW);
        if(g + NW < p.ksteps)
            multiply(y);
    }
#pragma unroll
    for(int i = 0; i < MT; ++i)
#pragma unroll
        for(int j = 0; j < NT; ++j)
            sums[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    constexpr int PER = GATED ? 2 : 1;
    const int64_t at_b = (int64_t)t.expert * p.N * PER;
    for(int tile = wave; tile < MT * NT / PER; tile += NW)
    {
        const int i = tile / (NT / PER), j = tile % (NT / PER);
        const int m = i * 16 + r, n = n0 + j * 16 + 4 * q;
        if(m >= t.rows || n >= p.N)
            continue;
        const int from = i8_row_of_a(p, t, m);
        const float sa = from >= 0 ? p.sa[from] : 0.0f;
        float d[PER][4];
#pragma unroll
        for(int h = 0; h < PER; ++h)
        {
            i32x4 v = sums[0][i * NT + j * PER + h][lane];
#pragma unroll
            for(int w = 1; w < NW; ++w)
                v += sums[w][i * NT + j * PER + h][lane];
#pragma unroll
            for(int e = 0; e < 4; ++e)
            {
                const int64_t k = at_b + (h ? p.N : 0) + min(n + e, p.N - 1);
                d[h][e]         = (float)v[e] * sa * p.sb[k] + (p.bias ? p.bias[k] : 0.0f);
            }
        }
        typedef T tx4 __attribute__((ext_vector_type(4)));
        T* const c = reinterpret_cast<T*>(p.c) + (int64_t)(t.m0 + m) * p.ldc + n;
        tx4 out;
#pragma unroll
        for(int e = 0; e < 4; ++e)
            out[e] = (T)(GATED ? i8_silu<T>(d[0][e]) * d[PER - 1][e] : d[0][e]);
        if(n + 4 <= p.N)
            reinterpret_cast<AnyAlign<tx4>*>(c)->v = out;
        else
#pragma unroll
            for(int e = 0; e < 3; ++e)
                if(n + e < p.N)
                    c[e] = out[e];
    }
}

// tiles of BM rows that a launch has at most: each expert with rows ends in one that is not full
int64_t most_tiles_m(const GemmI8Args& a, int BM)
{
    return a.offsets ? a.M / BM + (a.experts < a.M ? a.experts : a.M) : ((int64_t)a.M + BM - 1) / BM;
}

void cut(GemmI8Args& a, int BM, int cols)
{
    a.tiles_m = (int)most_tiles_m(a, BM), a.tiles_n = (a.N + cols - 1) / cols;
}
template <typename T, bool GATED, int BM, int BN, int WM, int WN, int KH, int NST>
hipError_t launch_tiles(GemmI8Args& a, hipStream_t s)
{
    constexpr int kLds = NST * (BM + BN) * 128 + (BM + 2 * BN) * 4;
    auto* const kernel = &gemm_i8_tile_kernel<T, GATED, BM, BN, WM, WN, KH, NST>;
    hipError_t e       = kLds > 65536 ? hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds) : hipSuccess;
    if(e != hipSuccess)
        return e;
    cut(a, BM, GATED ? BN / 2 : BN);
    hipLaunchKernelGGL(kernel, dim3((unsigned)a.tiles_m * (unsigned)a.tiles_n * (unsigned)a.ksplit), dim3(WM * WN * KH * 64), kLds, s, a);
    e = hipGetLastError();
    if(e != hipSuccess || a.ksplit == 1)
        return e;
    const int quads = (a.N + 3) / 4;
    hipLaunchKernelGGL((gemm_i8_join_kernel<T, GATED>), dim3((unsigned)(((int64_t)a.M * quads + 255) / 256)), dim3(256), 0, s, a, quads);
    return hipGetLastError();
}
template <typename T, bool GATED, int MT, int NT, int NW, bool ANY = false>
hipError_t launch_direct(GemmI8Args& a, hipStream_t s)
{
    cut(a, MT * 16, NT * 16 / (GATED ? 2 : 1));
    hipLaunchKernelGGL((gemm_i8_direct_kernel<T, GATED, MT, NT, NW, ANY>), dim3((unsigned)a.tiles_m * (unsigned)a.tiles_n), dim3(NW * 64), 0, s, a);
    return hipGetLastError();
}

// Which kernel, and into how many runs K is cut. us of a step (a K tile) that one CU's tiles take, as measured (rows x 4096 x 4096):
//   64 x 128, four stages    0.29, all CUs busy 0.33         128 rows 13.5, 512: 15.6
//   128 x 128, four stages   0.37, all CUs busy 0.44         512: 18.7, 1024: 22.4, 2048: 43 (64 x 128: 28.8, 55)
//   128 x 128, two stages    0.57 to 0.63, two a CU 0.93 to 0.98     512: 22.4, 1024: 25, 2048: 35 to 38 (256 x 256: 39, 44)
//   256 x 256, four waves    1.05, all CUs busy 1.47         4096: 51.6 (128 x 128 66.3), 4096 x 11008: 145 (213)
// and about 4 us around the steps, which a second round pays again where a CU holds one workgroup. Runs cost 4 us more and their sums' way to the workspace
// and back.
// Up to 16 rows the direct kernel of one row tile, 11008 x 4096: 1 row 9.7 to 10.2, 16 rows 13.7 to 14.0 (64 x 128 tiles in two runs 14.7); 8 waves where K is
// long (4096 x 11008: 9.9 where four take 10.7). To 64 rows the direct kernel of two row tiles where its workgroups find a CU each, 4096 x 4096
// 10.5 us for 32 rows (11.8 in the best runs of tiles), 11008 x 4096 18 (13.5). To 128 rows the direct kernel of one row tile where N is short (its
// cost: TileCost): 102 rows of 343 x 2176 gated 6.4 us (six runs of 64 x 128 tiles 18.4), 80 of 640 x 6544 7.1 (13.7).
// Experts: experts_plan, by the rows that experts have on average, since the host knows no more.
struct Plan
{
    int kind; // below
    int ksplit, per;
};
enum
{
    kAny     = 0, // 128 x 128, any K, stride and address
    kDirect1 = 1, // 16 x 16, four waves
    kDirect8 = 2, // the same, eight waves
    kDirect2 = 3, // 32 x 32
    kTile64  = 4, // 64 x 128
    kTile128 = 5, // 128 x 128, two workgroups a CU
    kTile256 = 6, // 256 x 256
    kDeep128 = 7, // 128 x 128, four stages
    kPair64  = 8, // 64 x 128, two workgroups a CU, for experts: the loads of one fill the other's beginning and end
    kAnyFew  = 9  // 16 x 16, any K, stride and address
};
// of each kind: a workgroup's rows of A and of B (16 x 16, gated: twice as many of B), its threads
struct Shape
{
    const char* name;
    int rows, cols, threads;
};
constexpr Shape kShapes[] = {{"any128x128", 128, 128, 256},
                             {"direct16x16", 16, 16, 256},
                             {"direct16x16 eight waves", 16, 16, 512},
                             {"direct32x32", 32, 32, 512},
                             {"tile64x128", 64, 128, 512},
                             {"tile128x128 two a CU", 128, 128, 512},
                             {"tile256x256", 256, 256, 256},
                             {"tile128x128", 128, 128, 512},
                             {"tile64x128 two a CU", 64, 128, 256},
                             {"any16x16", 16, 16, 256}};
int rows_of_b(const GemmI8Args& a, int kind) { return kShapes[kind].cols * (a.gated && kShapes[kind].cols == 16 ? 2 : 1); }
// a launch has fewer than 2^32 threads (256 x 256 tiles: a workgroup a CU)
bool launch_fits(const GemmI8Args& a, int kind, int runs)
{
    const int64_t wide = (int64_t)a.N * (a.gated ? 2 : 1), cols = rows_of_b(a, kind);
    return kind == kTile256 || most_tiles_m(a, kShapes[kind].rows) * ((wide + cols - 1) / cols) * runs < (1ll << 32) / kShapes[kind].threads;
}

// whether the kernels of 16-byte vectors take a call: K, strides and addresses in whole vectors, and what a tile may read within 32-bit
// offsets (rows that are gathered from all of A, the halves of a gated B)
bool whole_vectors(const GemmI8Args& a)
{
    constexpr int64_t kMost = 0x7fff0000;
    const uint64_t odd      = reinterpret_cast<uintptr_t>(a.a) | reinterpret_cast<uintptr_t>(a.b) | (uint64_t)a.K | (uint64_t)(a.rows_a > 1 ? a.lda : 0) |
                         (uint64_t)((int64_t)a.N * (a.gated ? 2 : 1) > 1 ? a.ldb : 0) | (uint64_t)(a.experts > 1 ? a.batch_b : 0);
    const int64_t rows_a = a.rows ? a.rows_a : a.rows_a < 256 ? a.rows_a : 256, rows_b = a.gated ? 2 * (int64_t)a.N : a.N < 256 ? a.N : 256;
    return a.K > 0 && (odd & 15) == 0 && rows_a * a.lda <= kMost && rows_b * a.ldb <= kMost && a.K <= kMost;
}

// us = 2 + (work^3 + memory^3)^(1/3): memory the bytes that a launch cannot do without at the rate that the kernel reaches, work its rounds of tiles
// (slots at a time), each with what a tile's beginning and end take and its K tiles, which take longer the more slots are in use. Fitted to 310 products
// of 4 to 128 experts, 0.1 to 4800 rows each, K 256 to 4096: on average 2.8 % from the best of the five, where borders by rows and K alone were
// 18 % and up to 3.3 times (519 rows of 512 x 1040 in each of 4 experts: 10.4 us on 64 x 128 tiles, 23.4 on 256 x 256). Examples, 64 experts of 2816 x 4096
// gated: a row each 86 direct, 96 on 64 x 128; 8 rows 151, 137 (128 x 128: 156); 64 rows 185 on 64 x 128, 179 on 256 x 256. Where a call has fewer rows than M (a
// rank's slice of the offsets, a padded step) the choice is that of M: 8 of 64 such experts, 512 tokens of eight rows each 44 us, 31.5 with the slice's 533 rows alone; 64 tokens
// 21.9, 23.6.
struct TileCost
{
    int kind, slots;
    double end, step, busy, mb_per_us, uneven;
    double us(double tiles, int steps, double mb) const
    {
        const double n = tiles / slots, turns = n > 1 && n + uneven > 1 ? n + uneven : 1;
        const double work = turns * (end + steps * (step + busy * (n < 1 ? n : 1))), memory = mb / mb_per_us;
        return 2 + std::cbrt(work * work * work + memory * memory * memory);
    }
};
constexpr TileCost kExpertsCosts[] = {{kDirect1, 2048, 2.49, 0.04, 0.70, 5.27, -0.61}, {kPair64, 512, 3.88, 0.31, 0.58, 5.96, 0.25},
                                      {kTile128, 512, 3.33, 0.39, 0.93, 5.87, 0.21}, {kTile256, 256, 8.14, 0.70, 0.81, 6.13, 0.18},
                                      {kTile64, 256, 3.58, 0.24, 0.26, 5.60, 0.28}};
Plan experts_plan(const GemmI8Args& a, int steps)
{
    const double rows = (double)a.M / a.experts, used = a.experts * (1 - std::exp(-rows)), wide = (double)a.N * (a.gated ? 2 : 1);
    const double mb   = (used * wide * a.K + (double)(a.rows ? a.rows_a : a.M) * a.K + 2.0 * a.M * a.N) * 1e-6;
    Plan best{kTile256, 1, steps};
    double least = 1e300;
    for(const TileCost& c : kExpertsCosts)
    {
        if(!launch_fits(a, c.kind, 1))
            continue;
        const int high = kShapes[c.kind].rows, cols = rows_of_b(a, c.kind);
        double tiles   = rows > high / 2 ? a.M / (double)high + 0.5 * a.experts : used; // (an expert's last is half full)
        tiles          = (tiles > used ? tiles : used);
        const double us = c.us((tiles < a.M ? tiles : a.M) * std::ceil(wide / cols), steps, mb);
        if(us < least)
            least = us, best.kind = c.kind;
    }
    return best;
}

Plan plan(const GemmI8Args& a, int64_t workspace_bytes)
{
    const int steps = (int)(((int64_t)a.K + 127) / 128);
    if(!whole_vectors(a))
    {
        // (11008 x 4100: 16 rows 16 us on 16 x 16 tiles, 33 on 128 x 128; 32: 27, 34; 48: 38, 35; 64 experts of 2816 x 4100, 8 rows each: 201, 200)
        const double rows = (double)a.M / (a.offsets ? a.experts : 1);
        const int64_t n16 = most_tiles_m(a, 16) * ((a.N + 15) / 16);
        return Plan{a.K > 0 && (rows <= (a.offsets ? 8 : 16) || (rows <= 48 && n16 <= 2048)) ? kAnyFew : kAny, 1, steps};
    }
    if(a.offsets)
        return experts_plan(a, steps);
    if(a.M <= 16)
        return Plan{a.K > 8192 ? kDirect8 : kDirect1, 1, steps};
    const int64_t wide = (int64_t)a.N * (a.gated ? 2 : 1);
    auto tiles         = [&](int bm, int bn) { return ((int64_t)a.M + bm - 1) / bm * ((wide + bn - 1) / bn); };
    auto rounds        = [](int64_t n) { return (double)((n + 255) / 256); };
    const int64_t big  = tiles(256, 256);
    const double share = (double)big / (256 * rounds(big));
    Plan best{kTile256, 1, steps};
    double us    = 2 + rounds(big) * (2 + steps * (1.05 + 0.42 * share * share));
    auto compare = [&](double t, const Plan& p) {
        if(t < us && launch_fits(a, p.kind, p.ksplit))
            us = t, best = p;
    };
    if(a.M <= 128)
    {
        constexpr TileCost direct{kDirect1, 2048, 1.27, 0.08, 0.57, 5.3, 0.22};
        compare(direct.us((double)tiles(16, a.gated ? 32 : 16), steps, ((double)wide * a.K + (double)a.M * a.K + 2.0 * a.M * a.N) * 1e-6),
                Plan{a.K > 8192 ? kDirect8 : kDirect1, 1, steps});
    }
    if(a.M <= 64)
    {
        const double n = rounds(tiles(32, 32));
        compare(3.4 + steps * 0.2 * n * (n > 1 ? 1.13 : 1.0), Plan{kDirect2, 1, steps});
    }
    for(int ks = 1; ks <= 16 && ks * 2 <= (steps > 1 ? steps : 2); ++ks)
    {
        const int per     = (steps + ks - 1) / ks, runs = (steps + per - 1) / per;
        const double sums = runs > 1 ? 4.0 * a.M * wide * runs : 0.0, join = runs > 1 ? 4 + 2 * sums / 4e6 : 0.0;
        if(sums > (double)workspace_bytes)
            continue;
        const int64_t n64 = tiles(64, 128) * runs, n128 = tiles(128, 128) * runs, rest = n128 % 512;
        const double r64 = rounds(n64), s64 = (double)n64 / (256 * r64), r128 = rounds(n128), s128 = (double)n128 / (256 * r128);
        compare(join + r64 * (3.9 + 0.5 * s64 + per * (0.285 + 0.045 * s64)), Plan{kTile64, runs, per});
        compare(join + r128 * (4.8 + 4 * s128 * s128 + per * (0.365 + 0.08 * s128)), Plan{kDeep128, runs, per});
        compare(3.5 + join + per * (0.98 * (double)(n128 / 512) + (rest == 0 ? 0.0 : rest > 256 ? 0.93 : 0.52 + 0.13 * (double)rest / 256)),
                Plan{kTile128, runs, per});
    }
    return best;
}

template <typename T>
constexpr int type_of()
{
    return sizeof(T) == 4 ? CKX_TYPE_F32 : std::is_same<T, _Float16>::value ? CKX_TYPE_F16 : CKX_TYPE_BF16;
}

template <typename T, bool GATED>
hipError_t launch(GemmI8Args& a, int64_t workspace_bytes, hipStream_t s)
{
    const Plan w = plan(a, workspace_bytes);
    a.ksplit = w.ksplit, a.per = w.per;
    switch(w.kind)
    {
    case kDirect1: return launch_direct<T, GATED, 1, GATED ? 2 : 1, 4>(a, s);
    case kDirect8: return launch_direct<T, GATED, 1, GATED ? 2 : 1, 8>(a, s);
    case kDirect2: return launch_direct<T, GATED, 2, 2, 8>(a, s);
    case kTile64: return launch_tiles<T, GATED, 64, 128, 2, 2, 2, 4>(a, s);
    case kTile128: return launch_tiles<T, GATED, 128, 128, 4, 2, 1, 2>(a, s);
    case kAnyFew: return launch_direct<T, GATED, 1, GATED ? 2 : 1, 4, true>(a, s);
    case kPair64: return launch_tiles<T, GATED, 64, 128, 2, 2, 1, 3>(a, s);
    case kDeep128: return launch_tiles<T, GATED, 128, 128, 2, 2, 2, 4>(a, s);
    case kTile256: return gemm_i8_big_launch(a, type_of<T>(), most_tiles_m(a, 256), s);
    default: break;
    }
    cut(a, 128, GATED ? 64 : 128);
    hipLaunchKernelGGL((gemm_i8_any_kernel<T, GATED>), dim3((unsigned)a.tiles_m * (unsigned)a.tiles_n), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_form(GemmI8Args& a, int64_t workspace_bytes, hipStream_t s)
{
    return a.gated ? launch<T, true>(a, workspace_bytes, s) : launch<T, false>(a, workspace_bytes, s);
}

} // namespace

// a launch has fewer than 2^32 threads, 512 a workgroup at most: one for 64 x 128 outputs (experts: 128 x 128), and where the rows are
// few for 16 x 16. What is left then has a kernel always; plan() takes none whose launch does not fit (a short N has many tiles of few columns)
bool gemm_i8_scaled_fits(int M, int N, int gated, int experts)
{
    GemmI8Args a{};
    a.M = M, a.experts = experts;
    const int none     = 0;
    a.offsets          = experts ? &none : nullptr; // (says that there are experts)
    const bool few     = experts ? M < (int64_t)experts * 256 : M <= 128;
    const int64_t wide = (int64_t)N * (gated ? 2 : 1);
    return most_tiles_m(a, few ? 16 : experts ? 128 : 64) * (wide / (few ? 16 : 128) + 2) < (1ll << 32) / 512;
}

int64_t gemm_i8_scaled_workspace(int M, int N, int K, int gated)
{
    GemmI8Args a{};
    a.M = a.rows_a = M, a.N = N, a.K = (K + 15) / 16 * 16, a.gated = gated, a.lda = a.ldb = a.K;
    const Plan w = plan(a, INT64_MAX);
    return w.ksplit > 1 ? 4ll * M * N * (gated ? 2 : 1) * w.ksplit : 0;
}

const char* gemm_i8_scaled_plan(const GemmI8Args& a, int64_t workspace_bytes, int* tile_m, int* tile_n, int* k_runs)
{
    const Plan w = plan(a, workspace_bytes);
    *tile_m = kShapes[w.kind].rows, *tile_n = rows_of_b(a, w.kind), *k_runs = w.kind == kAny || w.kind == kAnyFew ? 0 : w.ksplit;
    return kShapes[w.kind].name;
}

hipError_t gemm_i8_scaled_launch(GemmI8Args a, int c_type, int64_t workspace_bytes, hipStream_t s)
{
    a.ksteps = (int)(((int64_t)a.K + 127) / 128);
    return c_type == CKX_TYPE_F32   ? launch_form<float>(a, workspace_bytes, s)
           : c_type == CKX_TYPE_F16 ? launch_form<_Float16>(a, workspace_bytes, s)
                                    : launch_form<__bf16>(a, workspace_bytes, s);
}

} // namespace ckx
