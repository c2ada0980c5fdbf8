// GEMM with e4m3 operands and a scale for each block of 128 (formula: include/ckx.h, ckx_gemm_f8_blockscale).
//
// 16-bit outputs: one matrix instruction covers a group: v_mfma_f32_16x16x128_f8f6f4 multiplies 16 rows by 16 columns over 128 bytes of K, so
// its result, started from zero, is the group's sum, and acc += (sa * sb) * result is one multiply-add per value and group. The
// instruction is issued as D^T = B_frag x A_frag: a lane then holds one row m and four consecutive columns of a 16 x 16 tile, so
// that the row's scale is one register, and the rows of B are permuted in LDS (b_row_to_col) so that four tiles leave the lane
// with 16 consecutive columns. That instruction adds the products of eight neighbours of K on a grid 2^-13 of the largest
// among them (measured: what lies under it is cut; 1.4e-5 of a group's sum in the 2-norm for normal codes). Against the output's own
// rounding, 2^-11 or 2^-8, that is nothing; fp32 outputs are worth more and take the codes converted to fp16 (exact) through
// v_mfma_f32_16x16x32_f16, whose sums are fp32, at half the rate.
#include "f8.hpp"
#include "serving.hpp"

namespace ckx {

namespace {

// 16 bytes at column k of a row, zeros behind column K: one element at a time, any alignment
__device__ __forceinline__ i32x4 ragged16(const uint8_t* row, int k, int K, bool live)
{
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

// 128 x 128 tiles, four waves of 64 x 64. WIDE: K, lda, ldb whole 16-byte vectors and aligned bases: operands go straight
// to LDS; otherwise through registers, a byte at a time.
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void gemm_f8_kernel(GemmF8Args p)
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
    // (a resource ends with the last row of the tile: rows behind it read as zeros)
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(a0, (uint32_t)(rows - 1) * p.lda + p.K);
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(b0, (uint32_t)(cols - 1) * p.ldb + p.K);

    // a wave fills LDS rows wave * 32 ... + 31 of either tile, eight rows a load; chunk c of row r lies at c ^ (r & 7)
    auto load = [&](int stage, int g) {
#pragma unroll
        for(int j = 0; j < 4; ++j)
        {
            const int r = wave * 32 + j * 8 + (lane >> 3), c = (lane & 7) ^ (r & 7);
            const int k = g * kGroup + c * 16, rn = (int)b_row_to_col((uint32_t)r);
            if constexpr(WIDE)
            {
                const uint32_t oa = r < rows && k < p.K ? (uint32_t)r * p.lda + k : kOutOfRange;
                const uint32_t ob = rn < cols && k < p.K ? (uint32_t)rn * p.ldb + k : kOutOfRange;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr_t)(lds[stage][0] + (wave * 32 + j * 8) * 128), 16, (int)oa, 0, 0, 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_ptr_t)(lds[stage][1] + (wave * 32 + j * 8) * 128), 16, (int)ob, 0, 0, 0);
            }
            else
            {
                uint8_t* const at = &lds[stage][0][(wave * 32 + j * 8) * 128 + lane * 16];
                *reinterpret_cast<i32x4*>(at)        = ragged16(a0 + (int64_t)r * p.lda, k, p.K, r < rows);
                *reinterpret_cast<i32x4*>(at + TILE) = ragged16(b0 + (int64_t)rn * p.ldb, k, p.K, rn < cols);
            }
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
    load(0, 0);
    for(int g = 0; g < p.groups; ++g)
    {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if(g + 1 < p.groups)
            load((g + 1) & 1, g + 1);
        const float sb = p.sb[(int64_t)tn * p.sb_n + (int64_t)g * p.sb_g];
        i32x8 bf[4];
#pragma unroll
        for(int t = 0; t < 4; ++t)
            bf[t] = fragment(lds[g & 1][1], wn * 64 + t * 16 + (lane & 15));
#pragma unroll
        for(int i = 0; i < 4; ++i)
        {
            const int r    = wm * 64 + i * 16 + (lane & 15);
            const i32x8 af = fragment(lds[g & 1][0], r);
            const float s  = r < rows ? p.sa[(int64_t)(m0 + r) * p.sa_m + (int64_t)g * p.sa_g] * sb : 0.0f;
#pragma unroll
            for(int t = 0; t < 4; ++t)
            {
                const f32x4 d = group_sum<sizeof(T) == 4>(bf[t], af);
#pragma unroll
                for(int j = 0; j < 4; ++j)
                    acc[i][t][j] = __builtin_fmaf(s, d[j], acc[i][t][j]);
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

template <typename T>
hipError_t launch(GemmF8Args& a, hipStream_t s)
{
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a.a) | reinterpret_cast<uintptr_t>(a.b) | (uintptr_t)a.K |
                           (uintptr_t)(a.M > 1 ? a.lda : 0) | (uintptr_t)(a.N > 1 ? a.ldb : 0);
    a.tiles_m = (a.M + 127) / 128, a.tiles_n = (a.N + 127) / 128;
    const dim3 grid((unsigned)a.tiles_m * (unsigned)a.tiles_n);
    if((bits & 15) == 0)
        hipLaunchKernelGGL((gemm_f8_kernel<T, true>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((gemm_f8_kernel<T, false>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

} // namespace

int64_t gemm_f8_workspace(int, int, int) { return 0; }

hipError_t gemm_f8_launch(GemmF8Args a, int c_type, int64_t, hipStream_t s)
{
    a.groups = (int)(((int64_t)a.K + kGroup - 1) / kGroup);
    return c_type == CKX_TYPE_F32 ? launch<float>(a, s) : c_type == CKX_TYPE_F16 ? launch<_Float16>(a, s) : launch<__bf16>(a, s);
}

} // namespace ckx
