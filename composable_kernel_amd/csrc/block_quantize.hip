// Activations to e4m3 in groups of 128 columns (formula: include/ckx.h, ckx_quantize_blocks_f8).
//
// One pass over x: 16 lanes hold the 128 values of a group, eight each, so that the group's maximum crosses four lane exchanges
// and the codes leave from the registers they were read into. A workgroup takes 16 rows x 512 columns, 16 lanes a row: the scales
// of a group's 16 rows are written as one 64-byte piece where the scales' rows are next to each other. Rows at any address take
// the same wide accesses; only K's end goes element by element.
// Memory bounds it: 2 (or 4) bytes read and 1 written per value, and 1/32 byte of scales. bf16 8192 x 11008: 55.6 us, 4.9 TB/s of
// both together; reads alone (6.35 TB/s on this card) and writes alone (5.2) would take 46. The exact quotient costs 2.4 of it
// (53.2 with one multiplication in its place). fp32 11886 x 3388 43.5 us (107 where every row went element by element). 1 x 4096:
// the launch.
#include "f8.hpp"
#include "serving.hpp"

namespace ckx {

namespace {

constexpr int kRows = 16, kCols = 4; // of a workgroup's tile: rows, groups

template <typename T>
__global__ __launch_bounds__(256) void quantize_blocks_kernel(QuantArgs p, int col_tiles, int64_t tiles)
{
    const int lane = threadIdx.x & 15, row = threadIdx.x >> 4;
    const int groups = (p.K - 1) / kGroup + 1;
    for(int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x)
    {
        const int64_t tm = tile / col_tiles;
        const int g0     = (int)(tile - tm * col_tiles) * kCols;
        const int64_t m  = tm * kRows + row;
        if(m >= p.M)
            continue;
        const T* x = reinterpret_cast<const T*>(p.x) + m * p.sx;
        uint8_t* q = p.q + m * p.sq;
        float v[kCols][8];
#pragma unroll
        for(int c = 0; c < kCols; ++c)
        {
            const int64_t k = (int64_t)(g0 + c) * kGroup + lane * 8;
#pragma unroll
            for(int i = 0; i < 8; ++i)
                v[c][i] = 0.0f;
            if(k + 8 <= p.K)
                load8(x + k, v[c]);
            else
#pragma unroll
                for(int i = 0; i < 7; ++i)
                    if(k + i < p.K)
                        v[c][i] = (float)x[k + i];
        }
#pragma unroll
        for(int c = 0; c < kCols; ++c)
        {
            const int64_t k = (int64_t)(g0 + c) * kGroup + lane * 8;
            float amax      = kTinyAmax;
#pragma unroll
            for(int i = 0; i < 8; ++i)
                amax = __builtin_fmaxf(amax, __builtin_fabsf(v[c][i])); // (a NaN is passed over)
#pragma unroll
            for(int d = 1; d < 16; d *= 2)
                amax = __builtin_fmaxf(amax, __shfl_xor(amax, d, 16));
            const Quotient by = quotient_of<CODE_E4M3>(amax);
            uint32_t w[2];
#pragma unroll
            for(int h = 0; h < 2; ++h)
            {
                float t[4];
#pragma unroll
                for(int i = 0; i < 4; ++i)
                    t[i] = by.of<sizeof(T) == 2>(v[c][4 * h + i]);
                w[h] = codes_of<CODE_E4M3>(t[0], t[1], t[2], t[3]);
            }
            if(k + 8 <= p.K)
                reinterpret_cast<AnyAlign<u32x2>*>(q + k)->v = u32x2{w[0], w[1]};
            else
#pragma unroll
                for(int i = 0; i < 7; ++i)
                    if(k + i < p.K)
                        q[k + i] = (uint8_t)(w[i / 4] >> (8 * (i & 3)));
            if(lane == 0 && g0 + c < groups)
                p.scale[m * p.ss_m + (int64_t)(g0 + c) * p.ss_g] = amax / kE4m3Max;
        }
    }
}

template <typename T>
hipError_t launch(const QuantArgs& a, hipStream_t s)
{
    const int groups    = (a.K - 1) / kGroup + 1;
    const int col_tiles = (groups + kCols - 1) / kCols;
    const int64_t tiles = ((int64_t)a.M + kRows - 1) / kRows * col_tiles;
    const int grid      = (int)(tiles < (1 << 20) ? tiles : (1 << 20));
    hipLaunchKernelGGL((quantize_blocks_kernel<T>), dim3(grid), dim3(256), 0, s, a, col_tiles, tiles);
    return hipGetLastError();
}

} // namespace

hipError_t quantize_blocks_launch(const QuantArgs& a, int x_type, hipStream_t s)
{
    return x_type == CKX_TYPE_F32   ? launch<float>(a, s)
           : x_type == CKX_TYPE_F16 ? launch<_Float16>(a, s)
                                    : launch<__bf16>(a, s);
}

} // namespace ckx
