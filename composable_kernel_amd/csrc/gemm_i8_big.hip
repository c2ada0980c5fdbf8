// The token-scaled int8 GEMM and the experts' GEMM on 256 x 256 tiles of four waves (gemm_w4.hpp): where its tiles, the rows of A and B
// and the epilogue come from. 4096 x 11008 x 4096 in 148 us, 8192 x 8192 x 8192 in 387 (2.8 POP/s; a plain library product 2.5): matrix cores busy 56 to
// 61 % of the cycles at the clock that the power limit leaves, the rest a tile's beginning and end, where the CU's only workgroup waits for its first operands
// and its stores. The experts' rows of 64 experts, 32768 of 2816 x 4096 gated, 374: a fifth of it in tiles that are not full.
#include "gemm_i8_big.hpp"
#include "gemm_w4.hpp"
#include "tile_launch.hpp"

namespace ckx {

namespace {

template <typename T, bool GATED>
struct I8Big
{
    static constexpr bool kExt  = true;
    static constexpr int kTile  = 256, kCols = GATED ? 128 : 256;
    static constexpr int kLists = 3 * kTile * 4;              // scales of the tile's rows, of its columns, biases
    static constexpr int kBytes = kLists + 3 * kMostExperts * 4; // the experts' tiles
    const GemmI8Args& p;
    I8Tile t{};
    int n0 = 0;
    float asked[3];
    float s_row, s_col[16];
    const float* s_bias = nullptr;

    __device__ __forceinline__ explicit I8Big(const GemmI8Args& args) : p(args) {}
    __device__ __forceinline__ void begin(uint8_t* lds) const
    {
        if(!p.offsets)
            return;
        i8_list_tiles(p, kTile, reinterpret_cast<uint32_t*>(lds + kLists));
        __syncthreads();
    }
    __device__ __forceinline__ bool find(int unit, const uint8_t* lds)
    {
        if(p.offsets ? !i8_listed_tile(p, unit, kTile, reinterpret_cast<const uint32_t*>(lds + kLists), t) : unit >= p.tiles_m * p.tiles_n)
            return false;
        if(!p.offsets)
            i8_find_tile(p, unit, kTile, t);
        n0 = t.tn * kCols;
        return true;
    }
    // operands from the row on that offsets count from, and the bytes that may be read from there
    __device__ __forceinline__ int64_t first_a() const { return p.rows ? 0 : t.m0; }
    __device__ __forceinline__ int64_t first_b() const { return GATED ? 0 : n0; }
    __device__ __forceinline__ const uint8_t* a() const { return reinterpret_cast<const uint8_t*>(p.a) + first_a() * p.lda; }
    __device__ __forceinline__ const uint8_t* b() const { return reinterpret_cast<const uint8_t*>(p.b) + (int64_t)t.expert * p.batch_b + first_b() * p.ldb; }
    __device__ __forceinline__ uint32_t a_bytes() const
    {
        const int64_t rows = p.rows ? p.rows_a : min((int64_t)t.rows, (int64_t)p.rows_a - t.m0);
        return rows > 0 ? (uint32_t)((rows - 1) * p.lda + p.K) : 0u;
    }
    __device__ __forceinline__ uint32_t b_bytes() const
    {
        const int64_t rows = GATED ? 2 * (int64_t)p.N : min(kTile, p.N - n0);
        return (uint32_t)((rows - 1) * p.ldb + p.K);
    }
    // where rows r[...] of the tile begin; -1: there is none
    template <int N>
    __device__ __forceinline__ void rows_of_a(const int (&r)[N], int (&at)[N]) const
    {
        i8_rows_of_a(p, t, r, at);
#pragma unroll
        for(int j = 0; j < N; ++j)
            at[j] = at[j] >= 0 ? (int)((at[j] - first_a()) * p.lda) : -1;
    }
    __device__ __forceinline__ int row_of_b(uint32_t r) const
    {
        bool second;
        const int n = n0 + i8_col_of<GATED>(r, second);
        return n < p.N ? (int)((n - first_b() + (second ? p.N : 0)) * p.ldb) : -1;
    }
    // the scales: asked for in front of the tile's first operands, into LDS behind them, into registers in front of the epilogue
    __device__ __forceinline__ void ask(int tid)
    {
        const int m     = i8_row_of_a(p, t, tid);
        const int n     = n0 + (GATED ? (tid >> 6) * 32 + (tid & 31) : tid);
        const int64_t k = ((int64_t)t.expert * (GATED ? 2 : 1) + (GATED && (tid & 32) ? 1 : 0)) * p.N + n;
        asked[0]        = m >= 0 ? p.sa[m] : 0.0f;
        asked[1]        = n < p.N ? p.sb[k] : 0.0f;
        asked[2]        = n < p.N && p.bias ? p.bias[k] : 0.0f;
    }
    __device__ __forceinline__ void fill(uint8_t* lds, int tid)
    {
        float* const to = reinterpret_cast<float*>(lds);
#pragma unroll
        for(int i = 0; i < 3; ++i)
            to[i * kTile + tid] = asked[i];
    }
    // (of fragment row i, group g: 64 rows of B)
    __device__ __forceinline__ void fetch(const uint8_t* lds, int i, int g, int wm, int wn, int lane)
    {
        const float* const from = reinterpret_cast<const float*>(lds);
        const int at            = wn * 128 + g * 64 + 8 * (lane >> 4);
        s_row                   = from[wm * 128 + 16 * i + (lane & 15)];
#pragma unroll
        for(int j = 0; j < 16; ++j)
            s_col[j] = from[kTile + at + (j >> 3) * 32 + (j & 7)];
        s_bias = from + 2 * kTile + at;
    }
    // group g (64 rows of B) of fragment row i
    __device__ __forceinline__ void store(int i, int g, int wm, int wn, int lane, const i32x4 (&v)[4]) const
    {
        const int r = wm * 128 + 16 * i + (lane & 15), q = lane >> 4;
        if(r >= t.rows)
            return;
        T* const row = reinterpret_cast<T*>(p.c) + (int64_t)(t.m0 + r) * p.ldc;
        float x[2][8];
#pragma unroll
        for(int h = 0; h < 2; ++h)
        {
#pragma unroll
            for(int j = 0; j < 8; ++j)
                x[h][j] = (float)v[2 * h + (j >> 2)][j & 3] * s_row * s_col[8 * h + j];
            if(p.bias)
#pragma unroll
                for(int j = 0; j < 8; ++j)
                    x[h][j] += s_bias[32 * h + j];
        }
        if constexpr(GATED)
        {
#pragma unroll
            for(int j = 0; j < 8; ++j)
                x[0][j] = i8_silu<T>(x[0][j]) * x[1][j];
            i8_store8(row, n0 + (wn * 2 + g) * 32 + 8 * q, p.N, x[0]);
        }
        else
#pragma unroll
            for(int h = 0; h < 2; ++h)
                i8_store8(row, n0 + (wn * 2 + g) * 64 + 32 * h + 8 * q, p.N, x[h]);
    }
};

template <typename T, bool GATED>
__global__ __launch_bounds__(256) void gemm_i8_big_kernel(GemmI8Args p)
{
    extern __shared__ __attribute__((aligned(1024))) uint8_t ckx_smem[];
    GemmArgs g{};
    g.K = p.K;
    GemmW4<DT_I8, false, EPI_PASSTHROUGH, I8Big<T, GATED>>::run(g, ckx_smem, I8Big<T, GATED>(p));
}

template <typename T, bool GATED>
hipError_t launch(GemmI8Args& a, int64_t tiles, hipStream_t s)
{
    constexpr int kLds = GemmW4<DT_I8, false, EPI_PASSTHROUGH, I8Big<T, GATED>>::LDS;
    hipError_t e       = hipFuncSetAttribute(reinterpret_cast<const void*>(&gemm_i8_big_kernel<T, GATED>), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if(e != hipSuccess)
        return e;
    // one workgroup per CU (131 KB of LDS), a multiple of 8 so that a workgroup stays on its XCD over its tiles
    const int64_t most = num_cus() - num_cus() % 8;
    hipLaunchKernelGGL((gemm_i8_big_kernel<T, GATED>), dim3((unsigned)(tiles < most ? tiles : most)), dim3(256), kLds, s, a);
    return hipGetLastError();
}

} // namespace

hipError_t gemm_i8_big_launch(GemmI8Args& a, int c_type, int64_t tiles_m, hipStream_t s)
{
    const int cols = a.gated ? 128 : 256;
    a.tiles_m = (int)tiles_m, a.tiles_n = (a.N + cols - 1) / cols;
    const int64_t tiles = tiles_m * a.tiles_n;
    if(a.gated)
        return c_type == CKX_TYPE_F32 ? launch<float, true>(a, tiles, s) : c_type == CKX_TYPE_F16 ? launch<_Float16, true>(a, tiles, s) : launch<__bf16, true>(a, tiles, s);
    return c_type == CKX_TYPE_F32 ? launch<float, false>(a, tiles, s) : c_type == CKX_TYPE_F16 ? launch<_Float16, false>(a, tiles, s) : launch<__bf16, false>(a, tiles, s);
}

} // namespace ckx
