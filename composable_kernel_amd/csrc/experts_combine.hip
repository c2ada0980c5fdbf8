// The weighted sum of a token's rows (formula: include/ckx.h, ckx_experts_combine): eight columns a thread, the token's rows one
// after the other in fp32, so that the order of the sum is the order of its experts. Memory bounds it: 8192 tokens of eight rows of 4096 bf16
// 130 us, 5.2 TB/s, waves wait 89 % of their time; two rows each 40.8, 4.9. A row's last columns that are no eight are one thread's, one after the other: 4095 columns
// 167 us; 16 tokens 9.9 (4096: 3.0).
#include "experts.hpp"
#include "f8.hpp"

namespace ckx {

namespace {

constexpr int kBatch = 8; // rows that are under way together

// numbers that are the same for all lanes, through the scalar cache
template <typename T>
using Uniform = const __attribute__((address_space(4))) T*;

template <typename T>
struct Eight // consecutive elements, as they lie in memory
{
    u32x4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p)
    {
#pragma unroll
        for(int i = 0; i < (int)(sizeof(T) / 2); ++i)
            w[i] = load_vec<u32x4>(p + i * (16 / (int)sizeof(T)));
    }
    __device__ __forceinline__ float operator[](int i) const
    {
        typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
        constexpr int PER = 16 / (int)sizeof(T);
        return (float)__builtin_bit_cast(vec, w[i / PER])[i % PER];
    }
};

template <typename T>
__global__ __launch_bounds__(256) void experts_combine_kernel(CombineArgs p, int col_tiles, int64_t tiles)
{
    for(int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x)
    {
        const int64_t t = tile / col_tiles;
        const int64_t n = ((tile - t * col_tiles) * 256 + threadIdx.x) * 8;
        const Uniform<int> places    = (Uniform<int>)(p.places + t * p.top_k);
        const Uniform<float> weights = (Uniform<float>)(p.weights + t * p.top_k);
        const T* const y             = reinterpret_cast<const T*>(p.y) + n;
        const T* const add           = reinterpret_cast<const T*>(p.add) + t * p.sadd + n;
        T* const out                 = reinterpret_cast<T*>(p.out) + t * p.sout + n;
        if(n + 8 <= p.N)
        {
            float sum[8] = {};
            Eight<T> a;
            if(p.add)
                a.load(add);
            for(int j0 = 0; j0 < p.top_k; j0 += kBatch)
            {
                // the rows of a batch are all asked for before the first is used
                Eight<T> v[kBatch];
                int row[kBatch];
                float w[kBatch];
#pragma unroll
                for(int j = 0; j < kBatch; ++j)
                {
                    const int at = j0 + j < p.top_k ? j0 + j : j0;
                    row[j]       = j0 + j < p.top_k ? places[at] : -1;
                    w[j]         = weights[at];
                }
#pragma unroll
                for(int j = 0; j < kBatch; ++j)
                    if((unsigned)row[j] < (unsigned)p.rows)
                        v[j].load(y + (int64_t)row[j] * p.sy);
                if(j0 == 0 && p.add)
#pragma unroll
                    for(int i = 0; i < 8; ++i)
                        sum[i] = a[i];
#pragma unroll
                for(int j = 0; j < kBatch; ++j)
                    if((unsigned)row[j] < (unsigned)p.rows)
#pragma unroll
                        for(int i = 0; i < 8; ++i)
                            sum[i] = __builtin_fmaf(w[j], v[j][i], sum[i]);
            }
            if(p.top_k == 0 && p.add)
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    sum[i] = a[i];
            typedef T tx8 __attribute__((ext_vector_type(8)));
            tx8 o;
#pragma unroll
            for(int i = 0; i < 8; ++i)
                o[i] = (T)sum[i];
            reinterpret_cast<AnyAlign<tx8>*>(out)->v = o;
        }
        else
            for(int i = 0; n + i < p.N; ++i) // the row's end, one thread
            {
                float sum = p.add ? (float)add[i] : 0.0f;
                for(int j = 0; j < p.top_k; ++j)
                    if((unsigned)places[j] < (unsigned)p.rows)
                        sum = __builtin_fmaf(weights[j], (float)y[(int64_t)places[j] * p.sy + i], sum);
                out[i] = (T)sum;
            }
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
