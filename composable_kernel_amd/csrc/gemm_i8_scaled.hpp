// What the kernels of the token-scaled int8 GEMM and of the experts' GEMM share: which rows and columns a workgroup has, how B's
// rows lie in LDS, and the epilogue.
//
// The matrix instruction is issued as D^T = B_frag x A_frag (v_mfma_i32_16x16x64_i8): a lane holds one row of C and four columns of
// each 16 x 16 tile. B's rows are ordered in LDS so that the four tiles of 64 rows leave a lane with two runs of eight consecutive
// columns: columns 8 q ... and 32 + 8 q ... of 64. Gated, the second run holds the same columns of the other half of B (the up
// projection beside the gate), and the workgroup's tile of C is half as wide.
#pragma once

#include "experts.hpp"
#include "f8.hpp"

namespace ckx {

// row r of a B tile in LDS -> column of C from the tile's first on; second: whether it is of B's second half
template <bool GATED>
__device__ __forceinline__ int i8_col_of(uint32_t r, bool& second)
{
    const uint32_t half = r >> 5 & 1, c = ((r & 15) >> 2) * 8 + (r >> 4 & 1) * 4 + (r & 3);
    second              = GATED && half;
    return (int)((r >> 6) * (GATED ? 32 : 64) + (GATED ? 0 : half * 32) + c);
}

struct I8Tile
{
    int m0, rows; // of C
    int tn;
    int expert;
};

// The tiles of a launch: a dense product's in the order of tile_of_block; the experts' by the rows that offsets give them now, dealt to
// the XCDs alike, each expert's tiles next to each other. False: there is no tile for this workgroup. The same for every lane.
__device__ __forceinline__ int i8_first_row(const GemmI8Args& p, int e) { return min(max(p.offsets[e], 0), p.M); }
// rows and tiles of the lane's expert of e0 ... e0 + 63, and the sum of the tiles up to it, `before` those of the experts before e0
__device__ __forceinline__ void i8_expert_tiles(const GemmI8Args& p, int e0, int BM, uint32_t before, int& lo, int& n, uint32_t& tiles, uint32_t& upto)
{
    const int lane = threadIdx.x & 63, e = e0 + lane;
    lo = n = 0;
    if(e < p.experts)
    {
        lo = i8_first_row(p, e);
        n  = max(i8_first_row(p, e + 1) - lo, 0);
    }
    tiles = (uint32_t)(n + BM - 1) / (uint32_t)BM;
    upto  = tiles;
#pragma unroll
    for(int d = 1; d < 64; d *= 2)
    {
        const uint32_t o = (uint32_t)__shfl_up((int)upto, d, 64);
        upto += lane >= d ? o : 0;
    }
    upto += before;
}
// the tile among `all` of a column of tiles that workgroup `block` takes, and its column
__device__ __forceinline__ bool i8_place_of(const GemmI8Args& p, int block, uint32_t all, uint32_t& tm, int& tn)
{
    const uint64_t nall = (uint64_t)all * (uint32_t)p.tiles_n;
    if((uint64_t)(uint32_t)block >= nall)
        return false;
    const uint32_t xcd = (uint32_t)block & 7, q = (uint32_t)(nall >> 3), r = (uint32_t)nall & 7;
    const uint32_t id  = xcd * q + (xcd < r ? xcd : r) + ((uint32_t)block >> 3);
    // (the tiles of one expert: columns outside, so that the tiles that share B's columns run together)
    constexpr uint32_t GM = 4;
    const uint32_t group = id / (GM * (uint32_t)p.tiles_n), first = group * GM, in = id - group * GM * (uint32_t)p.tiles_n;
    const uint32_t size  = min(GM, all - first);
    tm                   = first + in % size;
    tn                   = (int)(in / size);
    return true;
}
__device__ __forceinline__ bool i8_expert_tile(const GemmI8Args& p, int block, int BM, I8Tile& t)
{
    int lo, n;
    uint32_t tiles, upto, all = 0, tm;
    for(int e0 = 0; e0 < p.experts; e0 += 64)
    {
        i8_expert_tiles(p, e0, BM, all, lo, n, tiles, upto);
        all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    }
    if(!i8_place_of(p, block, all, tm, t.tn))
        return false;
    uint32_t before = 0;
    for(int e0 = 0; e0 < p.experts; e0 += 64)
    {
        if(p.experts > 64) // (otherwise they are at hand)
            i8_expert_tiles(p, e0, BM, before, lo, n, tiles, upto);
        const uint64_t who = __ballot(tm < upto);
        if(who)
        {
            const int w  = (int)__builtin_ctzll(who);
            const int in = ((int)tm - __builtin_amdgcn_readlane((int)(upto - tiles), w)) * BM;
            t.expert = e0 + w;
            t.m0     = __builtin_amdgcn_readlane(lo, w) + in;
            t.rows   = min(BM, __builtin_amdgcn_readlane(n, w) - in);
            return true;
        }
        before = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    }
    return false; // (not reached)
}
// the same for a workgroup that takes one tile after another: the sums, and the experts' first rows and their numbers, in LDS (3 * experts
// numbers)
__device__ __forceinline__ void i8_list_tiles(const GemmI8Args& p, int BM, uint32_t* list)
{
    const int lane = threadIdx.x & 63;
    uint32_t all   = 0;
    for(int e0 = 0; e0 < p.experts; e0 += 64) // (every wave for itself, the same numbers)
    {
        int lo, n;
        uint32_t tiles, upto;
        i8_expert_tiles(p, e0, BM, all, lo, n, tiles, upto);
        if(e0 + lane < p.experts)
            list[e0 + lane] = upto, list[p.experts + e0 + lane] = (uint32_t)lo, list[2 * p.experts + e0 + lane] = (uint32_t)n;
        all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    }
}
__device__ __forceinline__ bool i8_listed_tile(const GemmI8Args& p, int block, int BM, const uint32_t* list, I8Tile& t)
{
    const int lane = threadIdx.x & 63;
    uint32_t tm;
    if(!i8_place_of(p, block, (uint32_t)__builtin_amdgcn_readfirstlane((int)list[p.experts - 1]), tm, t.tn))
        return false;
    for(int e0 = 0; e0 < p.experts; e0 += 64)
    {
        const uint64_t who = __ballot(tm < list[min(e0 + lane, p.experts - 1)]);
        if(who)
        {
            const int e       = min(e0 + (int)__builtin_ctzll(who), p.experts - 1);
            const uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane(e > 0 ? (int)list[e - 1] : 0);
            const int lo = __builtin_amdgcn_readfirstlane((int)list[p.experts + e]), n = __builtin_amdgcn_readfirstlane((int)list[2 * p.experts + e]);
            const int in = (int)(tm - at) * BM;
            t.expert = e, t.m0 = lo + in, t.rows = min(BM, n - in);
            return true;
        }
    }
    return false; // (not reached)
}
__device__ __forceinline__ bool i8_find_tile(const GemmI8Args& p, int block, int BM, I8Tile& t)
{
    if(p.offsets)
        return i8_expert_tile(p, block, BM, t);
    int batch, tm;
    tile_of_block(block, p.tiles_m, p.tiles_n, 1, batch, tm, t.tn);
    t.expert = 0, t.m0 = tm * BM, t.rows = min(BM, p.M - t.m0);
    return true;
}
// rows of A that rows r[...] of a tile take; -1: none (behind the tile's last, or a row of zeros). The numbers are asked for all at once.
template <int N>
__device__ __forceinline__ void i8_rows_of_a(const GemmI8Args& p, const I8Tile& t, const int (&r)[N], int (&m)[N])
{
#pragma unroll
    for(int j = 0; j < N; ++j)
        m[j] = t.m0 + min(r[j], t.rows - 1);
    if(p.rows)
    {
#pragma unroll
        for(int j = 0; j < N; ++j)
            m[j] = p.rows[m[j]];
#pragma unroll
        for(int j = 0; j < N; ++j)
            m[j] = m[j] < 0 ? -1 : (int)((uint32_t)m[j] / (uint32_t)p.rows_per);
    }
#pragma unroll
    for(int j = 0; j < N; ++j)
        m[j] = r[j] < t.rows && m[j] < p.rows_a ? m[j] : -1;
}
__device__ __forceinline__ int i8_row_of_a(const GemmI8Args& p, const I8Tile& t, int r)
{
    const int one[1] = {r};
    int m[1];
    i8_rows_of_a(p, t, one, m);
    return m[0];
}

// x / (1 + exp(-x)): 16-bit outputs take the fast exponential and reciprocal, whose errors (a few 2^-24 of the value for |x| under 80)
// lie far under the output's rounding
template <typename T>
__device__ __forceinline__ float i8_silu(float x)
{
    if constexpr(sizeof(T) == 4)
        return x / (1.0f + expf(-x));
    else
        return x * __builtin_amdgcn_rcpf(1.0f + __expf(-x));
}

// eight consecutive columns of a row
template <typename T>
__device__ __forceinline__ void i8_store8(T* row, int n, int N, const float (&v)[8])
{
    if constexpr(sizeof(T) == 4)
    {
        store_room<4>(row + n, f32x4{v[0], v[1], v[2], v[3]}, (N - n) * 4, false);
        store_room<4>(row + n + 4, f32x4{v[4], v[5], v[6], v[7]}, (N - n - 4) * 4, false);
    }
    else
    {
        typedef T tx8 __attribute__((ext_vector_type(8)));
        tx8 x;
#pragma unroll
        for(int j = 0; j < 8; ++j)
            x[j] = (T)v[j];
        store_room<2>(row + n, x, (N - n) * 2, false);
    }
}
// the sums of eight columns with their scales (and biases) applied, in the formula's order
__device__ __forceinline__ void i8_scaled(const i32x4& a, const i32x4& b, float sa, const float* sb, const float* bias, float (&v)[8])
{
#pragma unroll
    for(int j = 0; j < 4; ++j)
    {
        v[j]     = (float)a[j] * sa * sb[j] + bias[j];
        v[4 + j] = (float)b[j] * sa * sb[4 + j] + bias[4 + j];
    }
}
// what a lane has of 64 columns (gated: 32 and their partners) of row `c_row`: sums of the four tiles; sb and bias: those of the 64
// rows of B in the order of the columns
template <typename T, bool GATED>
__device__ __forceinline__ void i8_finish(T* c_row, int n0, int N, int q, const i32x4 (&v)[4], float sa, const float* sb, const float* bias)
{
    float x[2][8];
#pragma unroll
    for(int h = 0; h < 2; ++h)
        i8_scaled(v[2 * h], v[2 * h + 1], sa, sb + 32 * h + 8 * q, bias + 32 * h + 8 * q, x[h]);
    if constexpr(GATED)
    {
#pragma unroll
        for(int j = 0; j < 8; ++j)
            x[0][j] = i8_silu<T>(x[0][j]) * x[1][j];
        i8_store8(c_row, n0 + 8 * q, N, x[0]);
    }
    else
    {
        i8_store8(c_row, n0 + 8 * q, N, x[0]);
        i8_store8(c_row, n0 + 32 + 8 * q, N, x[1]);
    }
}
// scales and biases of a tile's BN rows of B into LDS, in the order of i8_finish
template <bool GATED>
__device__ __forceinline__ void i8_load_scales(const GemmI8Args& p, int expert, int n0, int BN, int tid, int threads, float* sb, float* bias)
{
    const int64_t at = (int64_t)expert * p.N * (GATED ? 2 : 1);
    for(int i = tid; i < BN; i += threads)
    {
        const int n    = n0 + (GATED ? (i >> 6) * 32 + (i & 31) : i);
        const int64_t k = at + (GATED && (i & 32) ? p.N : 0) + n;
        sb[i]          = n < p.N ? p.sb[k] : 0.0f;
        bias[i]        = n < p.N && p.bias ? p.bias[k] : 0.0f;
    }
}

} // namespace ckx
