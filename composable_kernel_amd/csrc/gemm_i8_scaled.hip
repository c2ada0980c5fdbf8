// int8 GEMM with a scale for each token and channel, dense and for each expert's rows (formulas: include/ckx.h,
// ckx_gemm_i8_tokenscale and ckx_experts_gemm_i8).
#include "gemm_i8_scaled.hpp"

namespace ckx {

namespace {

// 16 bytes at column k of a row, zeros behind column K, any alignment
__device__ __forceinline__ i32x4 ragged16(const int8_t* row, int k, int K, bool live)
{
    if(live && k + 16 <= K)
        return load_vec<i32x4>(row + k);
    uint32_t w[4] = {0, 0, 0, 0};
    if(live)
    {
#pragma unroll
        for(int i = 0; i < 16; ++i)
            if(k + i < K)
                w[i >> 2] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i & 3));
    }
    return i32x4{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
}

// Any K, leading dimension and address: 128 rows x 128 rows of B, four waves of 64 x 64, the operands through registers into LDS, a K
// tile of 128 ahead.
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
    // a wave fills LDS rows wave * 32 ... + 31 of either tile, eight rows a load; chunk c of row r lies at c ^ (r & 7)
    const int8_t *ra[4], *rb[4];
#pragma unroll
    for(int j = 0; j < 4; ++j)
    {
        const int r = wave * 32 + j * 8 + (lane >> 3);
        const int m = r < t.rows ? i8_row_of_a(p, t.m0 + r) : -1;
        ra[j]       = m >= 0 ? p.a + (int64_t)m * p.lda : nullptr;
        bool second;
        const int n = n0 + i8_col_of<GATED>((uint32_t)r, second);
        rb[j]       = n < p.N ? p.b + (int64_t)t.expert * p.batch_b + ((int64_t)n + (second ? p.N : 0)) * p.ldb : nullptr;
    }
    auto load = [&](int stage, int g) {
#pragma unroll
        for(int j = 0; j < 4; ++j)
        {
            const int r = wave * 32 + j * 8 + (lane >> 3), k = g * 128 + ((lane & 7) ^ (r & 7)) * 16;
            uint8_t* const at = &lds[stage][0][(wave * 32 + j * 8) * 128 + lane * 16];
            *reinterpret_cast<i32x4*>(at)        = ragged16(ra[j], k, p.K, ra[j] != nullptr);
            *reinterpret_cast<i32x4*>(at + TILE) = ragged16(rb[j], k, p.K, rb[j] != nullptr);
        }
    };
    i32x4 acc[4][4];
#pragma unroll
    for(int i = 0; i < 4; ++i)
#pragma unroll
        for(int j = 0; j < 4; ++j)
            acc[i][j] = i32x4{0, 0, 0, 0};
    if(p.ksteps > 0)
        load(0, 0);
    for(int g = 0; g < p.ksteps; ++g)
    {
        __syncthreads();
        if(g + 1 < p.ksteps)
            load((g + 1) & 1, g + 1);
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
    }
    __syncthreads(); // (K = 0: the scales)
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        const int r = wm * 64 + i * 16 + (lane & 15), m = t.m0 + r;
        if(r >= t.rows)
            continue;
        const int from = i8_row_of_a(p, m);
        i8_finish<T, GATED>(reinterpret_cast<T*>(p.c) + (int64_t)m * p.ldc, n0 + wn * (GATED ? 32 : 64), p.N, q, acc[i], from >= 0 ? p.sa[from] : 0.0f,
                            sb + wn * 64, bias + wn * 64);
    }
}

// tiles of BM rows that a launch has at most: each expert with rows ends in one that is not full
int64_t most_tiles_m(const GemmI8Args& a, int BM)
{
    return a.offsets ? a.M / BM + (a.experts < a.M ? a.experts : a.M) : ((int64_t)a.M + BM - 1) / BM;
}

template <typename T, bool GATED>
hipError_t launch(GemmI8Args& a, int64_t workspace_bytes, hipStream_t s)
{
    constexpr int COLS = GATED ? 64 : 128;
    a.tiles_m = (int)most_tiles_m(a, 128), a.tiles_n = (a.N + COLS - 1) / COLS;
    hipLaunchKernelGGL((gemm_i8_any_kernel<T, GATED>), dim3((unsigned)a.tiles_m * (unsigned)a.tiles_n), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_form(GemmI8Args& a, int64_t workspace_bytes, hipStream_t s)
{
    return a.gated ? launch<T, true>(a, workspace_bytes, s) : launch<T, false>(a, workspace_bytes, s);
}

} // namespace

bool gemm_i8_scaled_fits(int M, int N, int gated, int experts)
{
    GemmI8Args a{};
    a.M = M, a.experts = experts;
    const int most  = 0; // (offsets alone say that there are experts)
    a.offsets       = experts ? &most : nullptr;
    const int cols  = gated ? 64 : 128;
    return most_tiles_m(a, 128) * (((int64_t)N + cols - 1) / cols) < (1ll << 32) / 512;
}

int64_t gemm_i8_scaled_workspace(int, int, int, int) { return 0; }

hipError_t gemm_i8_scaled_launch(GemmI8Args a, int c_type, int64_t workspace_bytes, hipStream_t s)
{
    a.ksteps = (int)(((int64_t)a.K + 127) / 128);
    return c_type == CKX_TYPE_F32   ? launch_form<float>(a, workspace_bytes, s)
           : c_type == CKX_TYPE_F16 ? launch_form<_Float16>(a, workspace_bytes, s)
                                    : launch_form<__bf16>(a, workspace_bytes, s);
}

} // namespace ckx
