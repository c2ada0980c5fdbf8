// GEMM with e4m3 operands and a scale for each block of 128 (formula: include/ckx.h, ckx_gemm_f8_blockscale).
//
// 16-bit outputs: one matrix instruction covers a group: v_mfma_f32_16x16x128_f8f6f4 multiplies 16 rows by 16 columns over 128
// bytes of K, so its result, started from zero, is the group's sum, and acc += (sa * sb) * result is one multiply-add per value
// and group. The instruction is issued as D^T = B_frag x A_frag: a lane then holds one row m and four consecutive columns of a 16
// x 16 tile, so that the row's scale is one register, and the rows of B are permuted in LDS (b_row_to_col) so that four tiles
// leave the lane with 16 consecutive columns.
// That instruction adds the products of eight neighbours of K on a grid 2^-13 of the power of two under the largest among them
// (measured: what lies under it is cut towards zero; 1.5e-5 of C in the 2-norm for normal codes, where the output's own rounding
// is 2^-11 or 2^-8 of each value). It goes by the products, not by their sum: where large ones cancel it is more than the
// rounding, and the callers are told so. fp32 outputs take the codes converted to fp16 (exact) through v_mfma_f32_16x16x32_f16,
// whose sums are fp32: 4096 x 11008 x 4096 432 us, where 16-bit outputs take 178.
#include "f8.hpp"
#include "serving.hpp"

namespace ckx {

namespace {

// 16 bytes at column k of a row, zeros behind column K, any alignment
__device__ __forceinline__ i32x4 ragged16(const uint8_t* row, int k, int K, bool live)
{
    if(live && k + 16 <= K)
        return load_vec<i32x4>(row + k);
    uint32_t w[4] = {0, 0, 0, 0};
    if(live)
    {
#pragma unroll
        for(int i = 0; i < 16; ++i)
            if(k + i < K)
                w[i >> 2] |= (uint32_t)row[k + i] << (8 * (i & 3));
    }
    return i32x4{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
}

// the group's sums of a 16 x 16 tile
template <bool EXACT>
__device__ __forceinline__ f32x4 group_sum(const i32x8& b, const i32x8& a)
{
    f32x4 d = {0, 0, 0, 0};
    if constexpr(EXACT)
    {
#pragma unroll
        for(int i = 0; i < 4; ++i)
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, (codes8<CODE_E4M3, _Float16>(b[2 * i], b[2 * i + 1]))),
                                                       __builtin_bit_cast(f16x8, (codes8<CODE_E4M3, _Float16>(a[2 * i], a[2 * i + 1]))), d,
                                                       0, 0, 0);
        return d;
    }
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, d, 0, 0, 0, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ void store_cols16(T* row, int n0, int N, const f32x4 (&v)[4])
{
    if constexpr(sizeof(T) == 4)
    {
#pragma unroll
        for(int t = 0; t < 4; ++t)
            store_room<4>(row + n0 + 4 * t, v[t], (N - n0 - 4 * t) * 4, false);
    }
    else
    {
        typedef T tx8 __attribute__((ext_vector_type(8)));
#pragma unroll
        for(int h = 0; h < 2; ++h)
        {
            tx8 x;
#pragma unroll
            for(int j = 0; j < 4; ++j)
                x[j] = (T)v[2 * h][j], x[4 + j] = (T)v[2 * h + 1][j];
            store_room<2>(row + n0 + 8 * h, x, (N - n0 - 8 * h) * 2, false);
        }
    }
}

// Any K, leading dimension and address: 128 x 128 tiles, four waves of 64 x 64, the operands through registers into LDS. What bounds it
// are the loads, one group ahead and byte by byte behind the last whole 16 of K: 4096 x 11008 x 4100 807 us (the kernels below, K 4096: 178),
// and with few rows its few workgroups: 1 x 11008 x 4100 87 us, 9 times the direct kernel's time for K 4096.
template <typename T>
__global__ __launch_bounds__(256) void gemm_f8_ragged_kernel(GemmF8Args p)
{
    constexpr int BM = 128, BN = 128, TILE = 128 * 128;
    __shared__ __align__(16) uint8_t lds[2][2][TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1, q = lane >> 4;
    int batch, tm, tn;
    tile_of_block((int)blockIdx.x, p.tiles_m, p.tiles_n, 1, batch, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int rows = min(BM, p.M - m0), cols = min(BN, p.N - n0);
    const uint8_t* const a0 = p.a + (int64_t)m0 * p.lda;
    const uint8_t* const b0 = p.b + (int64_t)n0 * p.ldb;
    // a wave fills LDS rows wave * 32 ... + 31 of either tile, eight rows a load; chunk c of row r lies at c ^ (r & 7)
    auto load = [&](int stage, int g) {
#pragma unroll
        for(int j = 0; j < 4; ++j)
        {
            const int r = wave * 32 + j * 8 + (lane >> 3), c = (lane & 7) ^ (r & 7);
            const int k = g * kGroup + c * 16, rn = (int)b_row_to_col((uint32_t)r);
            uint8_t* const at = &lds[stage][0][(wave * 32 + j * 8) * 128 + lane * 16];
            *reinterpret_cast<i32x4*>(at)        = ragged16(a0 + (int64_t)r * p.lda, k, p.K, r < rows);
            *reinterpret_cast<i32x4*>(at + TILE) = ragged16(b0 + (int64_t)rn * p.ldb, k, p.K, rn < cols);
        }
    };
    auto fragment = [&](const uint8_t* tile, int row) {
        const uint8_t* r = tile + row * 128;
        const i32x4 lo = *reinterpret_cast<const i32x4*>(r + ((q ^ (row & 7)) << 4));
        const i32x4 hi = *reinterpret_cast<const i32x4*>(r + (((4 + q) ^ (row & 7)) << 4));
        return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };

    f32x4 acc[4][4];
#pragma unroll
    for(int i = 0; i < 4; ++i)
#pragma unroll
        for(int t = 0; t < 4; ++t)
            acc[i][t] = f32x4{0, 0, 0, 0};
    // the scales of the next group are asked for before its operands, so that none of their waits waits for those
    const float* const sb = p.sb + (int64_t)tn * p.sb_n;
    const float* sa[4];
    float next[4], next_b = 0.0f;
#pragma unroll
    for(int i = 0; i < 4; ++i)
        sa[i] = p.sa + (int64_t)(m0 + min(wm * 64 + i * 16 + (lane & 15), rows - 1)) * p.sa_m;
    auto load_scales = [&](int g) {
        next_b = sb[(int64_t)g * p.sb_g];
#pragma unroll
        for(int i = 0; i < 4; ++i)
            next[i] = sa[i][(int64_t)g * p.sa_g];
    };
    if(p.groups > 0)
    {
        load_scales(0);
        load(0, 0);
    }
    for(int g = 0; g < p.groups; ++g)
    {
        __syncthreads();
        float s[4];
#pragma unroll
        for(int i = 0; i < 4; ++i)
            s[i] = next[i] * next_b;
        if(g + 1 < p.groups)
        {
            load_scales(g + 1);
            load((g + 1) & 1, g + 1);
        }
        i32x8 bf[4];
#pragma unroll
        for(int t = 0; t < 4; ++t)
            bf[t] = fragment(lds[g & 1][1], wn * 64 + t * 16 + (lane & 15));
#pragma unroll
        for(int i = 0; i < 4; ++i)
        {
            const int r    = wm * 64 + i * 16 + (lane & 15);
            const i32x8 af = fragment(lds[g & 1][0], r);
#pragma unroll
            for(int t = 0; t < 4; ++t)
            {
                const f32x4 d = group_sum<sizeof(T) == 4>(bf[t], af);
#pragma unroll
                for(int j = 0; j < 4; ++j)
                    acc[i][t][j] = __builtin_fmaf(s[i], d[j], acc[i][t][j]);
            }
        }
    }
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        const int r = wm * 64 + i * 16 + (lane & 15), n = n0 + wn * 64 + 16 * q;
        if(r < rows && n < p.N)
            store_cols16(reinterpret_cast<T*>(p.c) + (int64_t)(m0 + r) * p.ldc, n, p.N, acc[i]);
    }
}

// BM x BN tiles, WM x WN waves, NST stages of operands in LDS: the loads of a group are asked for NST - 1 groups ahead. 256 x 256
// and 128 x 128 in two stages (133 KB; 67 KB, two workgroups a CU) where there are tiles enough, 64 x 128 in four otherwise: the
// time from a load to its data, about 1.1 us, is then spread over three groups instead of one. What bounds the large tiles is the
// multiply-adds that wait for each matrix result, beside the matrix instructions, and the clock: 4096 x 11008 x 4096 176 to 181
// us, 2.1 PFLOP/s (matrix cores busy 46 % of the launch, vector instructions active 35 %, no LDS conflicts), 8192 x 8192 x 8192
// 2.4 (plan() has the steps of each tile).
// The direct loads are inline assembly: the compiler, told of them, would wait for all of them before every LDS read of another
// stage. Its own LDS reads it waits for itself; the wait for the direct loads stands in front of the barrier.
template <typename T, int BM, int BN, int WM, int WN, int NST>
__global__ __launch_bounds__(WM* WN * 64) void gemm_f8_tile_kernel(GemmF8Args p)
{
    constexpr int NW = WM * WN, MT = BM / WM / 16, NLA = BM / 8 / NW, NLB = BN / 8 / NW, LPT = NLA + NLB + 1;
    constexpr int A_TILE = BM * 128, B_AT = NST * A_TILE, B_TILE = BN * 128, S_AT = B_AT + NST * B_TILE, S_TILE = BM * 4;
    static_assert(BN / WN == 64 && (NLB == 2 || NLB == 4) && BM % 64 == 0, "");
    __shared__ __align__(1024) uint8_t lds[S_AT + NST * S_TILE]; // [A | B | row scales], stage after stage
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN, q = lane >> 4;
    int run, tm, tn; // (a run of groups takes the place of a batch)
    tile_of_block((int)blockIdx.x, p.tiles_m, p.tiles_n, p.ksplit, run, tm, tn);
    const int g0 = run * p.per, g1 = min(g0 + p.per, p.groups);
    const int m0 = tm * BM, n0 = tn * BN;
    const int rows = min(BM, p.M - m0), cols = min(BN, p.N - n0);
    // a resource ends with the tile's last row: what is asked for behind it comes as zeros (the scalar offset takes part in the
    // range check)
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.a + (int64_t)m0 * p.lda, (uint32_t)(rows - 1) * p.lda + p.K);
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(p.b + (int64_t)n0 * p.ldb, (uint32_t)(cols - 1) * p.ldb + p.K);
    const __amdgpu_buffer_rsrc_t rs =
        make_rsrc(p.sa + (int64_t)m0 * p.sa_m, ((uint32_t)(rows - 1) * p.sa_m + (uint32_t)(p.groups - 1) * p.sa_g + 1) * 4);
    const uint32_t base = (uint32_t)(uintptr_t)(lds_ptr_t)lds;

    // a load fills eight rows, chunk c of row r at c ^ (r & 7). B's rows lie in b_row_to_col's order: within a wave's rows, eight
    // rows on are 32 columns on, sixteen are 4
    const int kc      = ((lane & 7) ^ (lane >> 3)) * 16;
    const int row0_a = wave * NLA * 8 + (lane >> 3), row0_b = wave * NLB * 8 + (lane >> 3);
    const uint32_t oa = (uint32_t)row0_a * p.lda + kc, ob = b_row_to_col((uint32_t)row0_b) * p.ldb + kc;
    const int sr      = (wave % (BM / 64)) * 64 + lane; // (several waves bring the same scales)
    const uint32_t os = sr < rows ? (uint32_t)sr * p.sa_m * 4 : kOutOfRange;
    auto load16 = [&](const __amdgpu_buffer_rsrc_t& r, uint32_t off, uint32_t k, uint32_t at) {
        asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(off), "s"(r), "s"(k), "s"(at));
    };
    // (groups behind the last come as zeros: the counts of loads under way stay the same)
    auto load_all = [&](int g) {
        const uint32_t k = (uint32_t)g * kGroup, st = (uint32_t)g % NST;
        const bool in = (int)k + kc < p.K; // (selected, not or-ed in: the sum with the scalar offset stays under 2^32)
#pragma unroll
        for(int j = 0; j < NLA; ++j)
            load16(ra, in ? oa : kOutOfRange, k + (uint32_t)(j * 8) * p.lda, base + st * A_TILE + (wave * NLA + j) * 1024);
#pragma unroll
        for(int j = 0; j < NLB; ++j)
            load16(rb, in ? ob : kOutOfRange, k + (uint32_t)((j & 1) * 32 + (j >> 1) * 4) * p.ldb, base + B_AT + st * B_TILE + (wave * NLB + j) * 1024);
        asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds" ::"v"(g < p.groups ? os : kOutOfRange), "s"(rs),
                     "s"((uint32_t)g * p.sa_g * 4), "s"(base + S_AT + st * S_TILE + (uint32_t)(wave % (BM / 64)) * 256));
    };
    const int a_row = wm * (BM / WM) + (lane & 15), b_row = wn * 64 + (lane & 15);
    const int a_lo = a_row * 128 + ((q ^ (a_row & 7)) << 4), a_hi = a_lo ^ 64;
    const int b_lo = B_AT + b_row * 128 + ((q ^ (b_row & 7)) << 4), b_hi = b_lo ^ 64;
    auto both = [](const uint8_t* lo, const uint8_t* hi) {
        const i32x4 x = *reinterpret_cast<const i32x4*>(lo), y = *reinterpret_cast<const i32x4*>(hi);
        return i32x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    };
    f32x4 acc[MT][4];
#pragma unroll
    for(int i = 0; i < MT; ++i)
#pragma unroll
        for(int t = 0; t < 4; ++t)
            acc[i][t] = f32x4{0, 0, 0, 0};
    // the column block's scales: through the scalar cache, which takes no part in the counts of vector loads
    const int sb_col = (n0 + wn * 64) >> 7;
    const auto* const sb = (const __attribute__((address_space(4))) float*)(p.sb + (int64_t)(sb_col <= (p.N - 1) >> 7 ? sb_col : 0) * p.sb_n);

    for(int g = g0; g < g0 + NST - 1; ++g)
        load_all(g);
    for(int g = g0; g < g1; ++g)
    {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 2) * LPT) : "memory"); // this group's
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        load_all(g + NST - 1); // (into the stage that every wave has read before this barrier)
        const float sb_now      = sb[(int64_t)g * p.sb_g];
        const int st            = g % NST;
        const uint8_t* const at = lds + st * A_TILE;
        const uint8_t* const bt = lds + st * B_TILE;
        const float* const sa   = reinterpret_cast<const float*>(lds + S_AT + st * S_TILE) + a_row;
        // matrix instruction k runs beside the multiply-adds of k - LAG
        constexpr int LAG = 2, NK = MT * 4;
        i32x8 af[2], bf[4];
        float s[2], x[2];
        f32x4 d[LAG + 1];
        af[0] = both(at + a_lo, at + a_hi);
        s[0]  = sa[0];
#pragma unroll
        for(int t = 0; t < 4; ++t)
            bf[t] = both(bt + b_lo + t * 2048, bt + b_hi + t * 2048);
        auto add = [&](int k, float y) {
            f32x4& c = acc[k >> 2][k & 3];
#pragma unroll
            for(int j = 0; j < 4; ++j)
                c[j] = __builtin_fmaf(y, d[k % (LAG + 1)][j], c[j]);
            asm volatile("" : "+v"(c)); // (here: left to itself the compiler keeps all results and adds them at the end)
        };
#pragma unroll
        for(int k = 0; k < NK + LAG; ++k)
        {
            if(k < NK && (k & 3) == 0)
            {
                const int i = k >> 2;
                x[i & 1]    = s[i & 1] * sb_now;
                if(i + 1 < MT)
                {
                    af[(i + 1) & 1] = both(at + a_lo + (i + 1) * 2048, at + a_hi + (i + 1) * 2048);
                    s[(i + 1) & 1]  = sa[(i + 1) * 16];
                }
            }
            if(k < NK)
                d[k % (LAG + 1)] = group_sum<sizeof(T) == 4>(bf[k & 3], af[(k >> 2) & 1]);
            __builtin_amdgcn_sched_barrier(0);
            if(k >= LAG)
                add(k - LAG, x[((k - LAG) >> 2) & 1]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // (no load may land in LDS that is another workgroup's by then)
#pragma unroll
    for(int i = 0; i < MT; ++i)
    {
        const int r = wm * (BM / WM) + i * 16 + (lane & 15), n = n0 + wn * 64 + 16 * q;
        if(r < rows && n < p.N)
        {
            if(p.ksplit > 1)
                store_cols16(p.ws + ((int64_t)run * p.M + m0 + r) * p.N, n, p.N, acc[i]);
            else
                store_cols16(reinterpret_cast<T*>(p.c) + (int64_t)(m0 + r) * p.ldc, n, p.N, acc[i]);
        }
    }
}

// C from the sums of the runs, added in order: four columns a thread
template <typename T>
__global__ __launch_bounds__(256) void gemm_f8_join_kernel(GemmF8Args p, int quads)
{
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t m  = id / quads;
    const int n      = (int)(id - m * quads) * 4;
    if(m >= p.M)
        return;
    const float* at = p.ws + m * p.N + n;
    T* const c      = reinterpret_cast<T*>(p.c) + m * p.ldc + n;
    if(n + 4 <= p.N)
    {
        f32x4 v = reinterpret_cast<const AnyAlign<f32x4>*>(at)->v;
        for(int r = 1; r < p.ksplit; ++r)
            v += reinterpret_cast<const AnyAlign<f32x4>*>(at + (int64_t)r * p.M * p.N)->v;
        typedef T tx4 __attribute__((ext_vector_type(4)));
        tx4 out;
#pragma unroll
        for(int j = 0; j < 4; ++j)
            out[j] = (T)v[j];
        reinterpret_cast<AnyAlign<tx4>*>(c)->v = out;
    }
    else
        for(int j = 0; n + j < p.N; ++j)
        {
            float v = at[j];
            for(int r = 1; r < p.ksplit; ++r)
                v += at[(int64_t)r * p.M * p.N + j];
            c[j] = (T)v;
        }
}

template <typename T, int BM, int BN, int WM, int WN, int NST>
hipError_t launch_tiles(GemmF8Args& a, hipStream_t s)
{
    a.tiles_m = (a.M + BM - 1) / BM, a.tiles_n = (a.N + BN - 1) / BN;
    hipLaunchKernelGGL((gemm_f8_tile_kernel<T, BM, BN, WM, WN, NST>), dim3((unsigned)a.tiles_m * (unsigned)a.tiles_n * (unsigned)a.ksplit),
                       dim3(WM * WN * 64), 0, s, a);
    hipError_t e = hipGetLastError();
    if(e != hipSuccess || a.ksplit == 1)
        return e;
    const int quads = (a.N + 3) / 4;
    hipLaunchKernelGGL((gemm_f8_join_kernel<T>), dim3((unsigned)(((int64_t)a.M * quads + 255) / 256)), dim3(256), 0, s, a, quads);
    return hipGetLastError();
}

// Few output tiles: a workgroup takes MT x NT tiles of 16 x 16 and its NW waves share the groups of K among them, each straight from
// memory into its registers (the next group's 32 bytes a lane and tile row are on their way while one is multiplied); the
// waves' sums meet in LDS. Nothing waits at a barrier until the end, and a CU has NW * 2 * (MT + NT) * 2 KB under way: what a
// product of few rows needs, which is bound by reading B once.
template <typename T, int MT, int NT, int NW>
__global__ __launch_bounds__(NW * 64) void gemm_f8_direct_kernel(GemmF8Args p)
{
    constexpr int BM = MT * 16, BN = NT * 16;
    __shared__ __align__(16) f32x4 sums[NW][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    int batch, tm, tn;
    tile_of_block((int)blockIdx.x, p.tiles_m, p.tiles_n, 1, batch, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int rows = min(BM, p.M - m0), cols = min(BN, p.N - n0);
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.a + (int64_t)m0 * p.lda, (uint32_t)(rows - 1) * p.lda + p.K);
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(p.b + (int64_t)n0 * p.ldb, (uint32_t)(cols - 1) * p.ldb + p.K);

    struct Group
    {
        i32x4 a[MT][2], b[NT][2];
        float sa[MT], sb;
    };
    uint32_t oa[MT], ob[NT];
#pragma unroll
    for(int i = 0; i < MT; ++i)
        oa[i] = i * 16 + r < rows ? (uint32_t)(i * 16 + r) * p.lda + q * 16 : kOutOfRange;
#pragma unroll
    for(int t = 0; t < NT; ++t)
        ob[t] = t * 16 + r < cols ? (uint32_t)(t * 16 + r) * p.ldb + q * 16 : kOutOfRange;
    const float* const sb = p.sb + (int64_t)(n0 >> 7) * p.sb_n;
    auto load = [&](Group& x, int g) {
#pragma unroll
        for(int h = 0; h < 2; ++h)
        {
            const int k        = g * kGroup + h * 64;
            const uint32_t out = k + q * 16 < p.K ? 0u : kOutOfRange; // (a group's columns behind K, and groups behind the last)
#pragma unroll
            for(int i = 0; i < MT; ++i)
                x.a[i][h] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(ra, (int)(oa[i] | out), k, 0));
#pragma unroll
            for(int t = 0; t < NT; ++t)
                x.b[t][h] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rb, (int)(ob[t] | out), k, 0));
        }
        const int gg = min(g, p.groups - 1);
        x.sb         = sb[(int64_t)gg * p.sb_g];
#pragma unroll
        for(int i = 0; i < MT; ++i)
            x.sa[i] = p.sa[(int64_t)(m0 + min(i * 16 + r, rows - 1)) * p.sa_m + (int64_t)gg * p.sa_g];
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for(int i = 0; i < MT; ++i)
#pragma unroll
        for(int t = 0; t < NT; ++t)
            acc[i][t] = f32x4{0, 0, 0, 0};
    auto joined = [](const i32x4(&x)[2]) { return i32x8{x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]}; };
    auto multiply = [&](const Group& x) {
#pragma unroll
        for(int i = 0; i < MT; ++i)
        {
            const float s = x.sa[i] * x.sb;
#pragma unroll
            for(int t = 0; t < NT; ++t)
            {
                const f32x4 d = group_sum<sizeof(T) == 4>(joined(x.b[t]), joined(x.a[i]));
#pragma unroll
                for(int j = 0; j < 4; ++j)
                    acc[i][t][j] = __builtin_fmaf(s, d[j], acc[i][t][j]);
            }
        }
    };
    Group x, y;
    if(wave < p.groups)
        load(x, wave);
    for(int g = wave; g < p.groups; g += 2 * NW)
    {
        if(g + NW < p.groups)
            load(y, g + NW);
        multiply(x);
        if(g + 2 * NW < p.groups)
            load(x, g + 2 * NW);
        if(g + NW < p.groups)
            multiply(y);
    }

#pragma unroll
    for(int i = 0; i < MT; ++i)
#pragma unroll
        for(int t = 0; t < NT; ++t)
            sums[wave][i * NT + t][lane] = acc[i][t];
    __syncthreads();
    for(int tile = wave; tile < MT * NT; tile += NW)
    {
        f32x4 v = sums[0][tile][lane];
#pragma unroll
        for(int w = 1; w < NW; ++w)
            v += sums[w][tile][lane];
        const int m = tile / NT * 16 + r, n = n0 + tile % NT * 16 + 4 * q;
        if(m < rows && n < p.N)
        {
            typedef T tx4 __attribute__((ext_vector_type(4)));
            T* const c = reinterpret_cast<T*>(p.c) + (int64_t)(m0 + m) * p.ldc + n;
            tx4 out;
#pragma unroll
            for(int j = 0; j < 4; ++j)
                out[j] = (T)v[j];
            if(n + 4 <= p.N)
                reinterpret_cast<AnyAlign<tx4>*>(c)->v = out;
            else
#pragma unroll
                for(int j = 0; j < 3; ++j)
                    if(n + j < p.N)
                        c[j] = out[j];
        }
    }
}

template <typename T, int MT, int NT, int NW>
hipError_t launch_direct(GemmF8Args& a, hipStream_t s)
{
    a.tiles_m = (a.M + MT * 16 - 1) / (MT * 16), a.tiles_n = (a.N + NT * 16 - 1) / (NT * 16);
    hipLaunchKernelGGL((gemm_f8_direct_kernel<T, MT, NT, NW>), dim3((unsigned)a.tiles_m * (unsigned)a.tiles_n), dim3(NW * 64), 0, s, a);
    return hipGetLastError();
}

// Which kernel, and into how many runs K is cut. us of a step (a group) that one CU's tiles take, as measured (K 4096, B streamed):
//   64 x 128, four stages    0.49, one workgroup a CU        512 x 4096: 19.4 us (128 x 128: 21.8, 256 x 256: 49.6)
//   128 x 128, two stages    0.58, two a CU 1.0              1024 x 4096: 23.7 (35.9, 50.1), 2048 x 4096: 35.5 (69.4, 52.4)
//   256 x 256, two stages    1.42, all CUs busy 1.75         4096 x 4096: 61.0 (140, 68.0), 8192 x 8192 x 8192: 460 (1068, 566)
// and about 4 us around the steps. A run costs 3 us more and its sums' way to the workspace and back. Between the direct kernel and the
// large tiles that leaves 1.6 to 3.2 times what the bytes or operations take: the loads of 64 x 128 tiles and of few 128 x 128 ones are
// longer than a step, and runs of K pay a second launch (64 x 11008 x 4096 16.3 us, 128 x 4096 x 11008 20.8, 1024 x 4096 x 4096 25.5).
// Up to 32 rows the direct kernel: one row of 11008 x 4096 9.7 us (reading the weights alone 8.7), 64 x 128 tiles 18.5; 16 rows 13.3, and
// past 16 the tiles draw level: 17 rows 14.9, 32 rows 17.7, 33 rows (tiles, two runs of K) 14.6.
struct Plan
{
    int kind; // 0: direct, up to 16 rows; 1: direct, up to 32; 2, 3, 4: the tiles above; kRagged
    int ksplit, per;
};
constexpr int kRagged = -1;

// whether the kernels of 16-byte vectors take K and the strides; `addresses`: those of A and B, or-ed
bool whole_vectors(int M, int N, int K, int lda, int ldb, uintptr_t addresses)
{
    return K > 0 && ((addresses | (uintptr_t)K | (uintptr_t)(M > 1 ? lda : 0) | (uintptr_t)(N > 1 ? ldb : 0)) & 15) == 0;
}

Plan plan(int M, int N, int K, bool exact, int64_t workspace_bytes)
{
    const int groups = (int)(((int64_t)K + kGroup - 1) / kGroup);
    Plan best{2, 1, groups};
    if(M <= 32)
    {
        best.kind = M <= 16 ? 0 : 1;
        return best;
    }
    auto tiles  = [&](int bm, int bn) { return ((int64_t)M + bm - 1) / bm * (((int64_t)N + bn - 1) / bn); };
    auto rounds = [](int64_t n, int64_t of) { return (double)((n + of - 1) / of); };
    const int64_t small = tiles(64, 128), mid = tiles(128, 128), big = tiles(256, 256);
    const double us_mid = 4 + groups * (1.0 * (double)(mid / 512) + (mid % 512 > 256 ? 1.0 : mid % 512 > 0 ? 0.58 : 0.0));
    const double us_big = 4 + groups * (big <= 128 ? 1.42 : 1.75 * rounds(big, 256));
    double us           = 4 + groups * 0.49 * rounds(small, 256);
    if(us_mid < us)
        us = us_mid, best.kind = 3;
    if(us_big < us && !exact) // (fp32 outputs: the 256 x 256 kernel has no registers for the conversions)
        us = us_big, best.kind = 4;
    for(int ks = 2; ks <= 16 && ks * 4 <= groups && small < 256; ++ks)
    {
        const int per     = (groups + ks - 1) / ks;
        const int runs    = (groups + per - 1) / per;
        const double sums = 4.0 * M * N * runs;
        const double t    = 7 + per * 0.49 * rounds(small * runs, 256) + 2 * sums / 4e6;
        if(t < us && sums <= (double)workspace_bytes)
            us = t, best = Plan{2, runs, per};
    }
    return best;
}

template <typename T>
hipError_t launch(GemmF8Args& a, int64_t workspace_bytes, hipStream_t s)
{
    // (the row scales of a tile are addressed through 32-bit offsets)
    const bool near = (int64_t)a.sa_m * 256 + (int64_t)a.sa_g * (a.groups + 4) < (1 << 29);
    if(!near || !whole_vectors(a.M, a.N, a.K, a.lda, a.ldb, reinterpret_cast<uintptr_t>(a.a) | reinterpret_cast<uintptr_t>(a.b)))
    {
        a.tiles_m = (a.M + 127) / 128, a.tiles_n = (a.N + 127) / 128;
        hipLaunchKernelGGL((gemm_f8_ragged_kernel<T>), dim3((unsigned)a.tiles_m * (unsigned)a.tiles_n), dim3(256), 0, s, a);
        return hipGetLastError();
    }
    constexpr bool exact = sizeof(T) == 4;
    const Plan p         = plan(a.M, a.N, a.K, exact, workspace_bytes);
    a.ksplit = p.ksplit, a.per = p.per;
    switch(p.kind)
    {
    case 0: return launch_direct<T, 1, 1, 8>(a, s);
    case 1: return launch_direct<T, 2, 2, 8>(a, s);
    case 2: return launch_tiles<T, 64, 128, 2, 2, 4>(a, s);
    case 3: return launch_tiles<T, 128, 128, 4, 2, 2>(a, s);
    default: break;
    }
    if constexpr(!exact)
        return launch_tiles<T, 256, 256, 2, 4, 2>(a, s);
    return hipErrorInvalidValue; // (not planned)
}

} // namespace

// a launch has fewer than 2^32 threads, 512 a workgroup at most: one for 16 columns (up to 32 rows) or for 64 x 128 outputs
bool gemm_f8_fits(int M, int N)
{
    const int64_t m = M <= 32 ? 2 : ((int64_t)M + 63) / 64, n = ((int64_t)N + (M <= 32 ? 15 : 127)) / (M <= 32 ? 16 : 128);
    return m * n < (1ll << 32) / 512;
}

int64_t gemm_f8_workspace(int M, int N, int K)
{
    const Plan p = plan(M, N, K, false, INT64_MAX);
    return p.ksplit > 1 ? 4ll * M * N * p.ksplit : 0;
}

void gemm_f8_plan(int M, int N, int K, int lda, int ldb, int c_type, int64_t workspace_bytes, int* tile_m, int* tile_n, int* k_runs)
{
    constexpr int m[] = {128, 16, 32, 64, 128, 256}, n[] = {128, 16, 32, 128, 128, 256};
    Plan p{kRagged, 0, 0};
    if(whole_vectors(M, N, K, lda, ldb, 0))
        p = plan(M, N, K, c_type == CKX_TYPE_F32, workspace_bytes);
    *tile_m = m[p.kind + 1], *tile_n = n[p.kind + 1], *k_runs = p.ksplit;
}

hipError_t gemm_f8_launch(GemmF8Args a, int c_type, int64_t workspace_bytes, hipStream_t s)
{
    a.groups = (int)(((int64_t)a.K + kGroup - 1) / kGroup);
    return c_type == CKX_TYPE_F32   ? launch<float>(a, workspace_bytes, s)
           : c_type == CKX_TYPE_F16 ? launch<_Float16>(a, workspace_bytes, s)
                                    : launch<__bf16>(a, workspace_bytes, s);
}

} // namespace ckx
