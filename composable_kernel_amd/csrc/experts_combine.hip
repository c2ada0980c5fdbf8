// The weighted sum of a token's rows (formula: include/ckx.h, ckx_experts_combine): eight columns a thread, the token's rows one
// after the other in fp32, so that the order of the sum is the order of its experts. Memory bounds it.
#include "experts.hpp"
#include "f8.hpp"

namespace ckx {

namespace {

template <typename T>
__global__ __launch_bounds__(256) void experts_combine_kernel(CombineArgs p, int col_tiles, int64_t tiles)
{
    for(int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x)
    {
        const int64_t t = tile / col_tiles;
        const int64_t n = ((tile - t * col_tiles) * 256 + threadIdx.x) * 8;
        if(n >= p.N)
            continue;
        const bool whole = n + 8 <= p.N;
        auto load = [&](const T* row, float(&v)[8]) {
            if(whole)
                load8(row + n, v);
            else
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    v[i] = n + i < p.N ? (float)row[n + i] : 0.0f;
        };
        float sum[8] = {};
        if(p.add)
            load(reinterpret_cast<const T*>(p.add) + t * p.sadd, sum);
        for(int j = 0; j < p.top_k; ++j)
        {
            const int row = p.places[t * p.top_k + j];
            if((unsigned)row >= (unsigned)p.rows)
                continue;
            const float w = p.weights[t * p.top_k + j];
            float v[8];
            load(reinterpret_cast<const T*>(p.y) + (int64_t)row * p.sy, v);
#pragma unroll
            for(int i = 0; i < 8; ++i)
                sum[i] = __builtin_fmaf(w, v[i], sum[i]);
        }
        T* const out = reinterpret_cast<T*>(p.out) + t * p.sout + n;
        typedef T tx8 __attribute__((ext_vector_type(8)));
        tx8 o;
#pragma unroll
        for(int i = 0; i < 8; ++i)
            o[i] = (T)sum[i];
        if(whole)
            reinterpret_cast<AnyAlign<tx8>*>(out)->v = o;
        else
#pragma unroll
            for(int i = 0; i < 7; ++i)
                if(n + i < p.N)
                    out[i] = o[i];
    }
}

template <typename T>
hipError_t launch(const CombineArgs& a, hipStream_t s)
{
    const int col_tiles = (int)(((int64_t)a.N + 2047) / 2048);
    const int64_t tiles = (int64_t)a.tokens * col_tiles;
    hipLaunchKernelGGL((experts_combine_kernel<T>), dim3((unsigned)(tiles < (1 << 20) ? tiles : (1 << 20))), dim3(256), 0, s, a, col_tiles, tiles);
    return hipGetLastError();
}

} // namespace

hipError_t combine_launch(const CombineArgs& a, int type, hipStream_t s)
{
    return type == CKX_TYPE_F32 ? launch<float>(a, s) : type == CKX_TYPE_F16 ? launch<_Float16>(a, s) : launch<__bf16>(a, s);
}

} // namespace ckx
