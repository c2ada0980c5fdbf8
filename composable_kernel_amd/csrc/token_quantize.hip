// Activations to int8 with one scale per token (formula: include/ckx.h, ckx_quantize_tokens_i8).
//
// One pass: a row lies in the registers of its threads between its maximum and its codes (eight elements at a time, rows of up to
// 16384; longer ones are read again). 64 threads a row where it is short, 256 otherwise, whose maxima meet in LDS.
#include "experts.hpp"
#include "f8.hpp"

namespace ckx {

namespace {

constexpr int kMostChunks = 8; // of eight elements that a thread holds

// eight elements from column k on, zeros behind the row's end
template <typename T>
__device__ __forceinline__ void load_row8(const T* x, int64_t k, int K, float (&v)[8])
{
#pragma unroll
    for(int i = 0; i < 8; ++i)
        v[i] = 0.0f;
    if(k + 8 <= K)
        load8(x + k, v);
    else
#pragma unroll
        for(int i = 0; i < 7; ++i)
            if(k + i < K)
                v[i] = (float)x[k + i];
}
template <typename T>
__device__ __forceinline__ void store_row8(int8_t* q, int64_t k, int K, const float (&v)[8], const Quotient& by, bool finite)
{
    uint32_t w[2];
#pragma unroll
    for(int h = 0; h < 2; ++h)
    {
        float t[4];
#pragma unroll
        for(int i = 0; i < 4; ++i)
            t[i] = by.of<sizeof(T) == 2>(v[4 * h + i]);
        w[h] = finite ? codes_of<CODE_I8>(t[0], t[1], t[2], t[3]) : 0u;
    }
    if(k + 8 <= K)
        reinterpret_cast<AnyAlign<u32x2>*>(q + k)->v = u32x2{w[0], w[1]};
    else
#pragma unroll
        for(int i = 0; i < 7; ++i)
            if(k + i < K)
                q[k + i] = (int8_t)(w[i / 4] >> (8 * (i & 3)));
}
// the larger of two sizes, NaN where one is (sizes as bits: infinities lie above every number, NaNs above them)
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }

// NT threads a row, CH chunks of eight a thread (0: any number, the row is read twice)
template <typename T, int NT, int CH>
__global__ __launch_bounds__(256) void quantize_tokens_kernel(TokenQuantArgs p)
{
    constexpr int ROWS = 256 / NT;
    __shared__ uint32_t parts[4];
    const int tid = threadIdx.x % NT;
    for(int64_t m = (int64_t)blockIdx.x * ROWS + threadIdx.x / NT; m < p.M; m += (int64_t)gridDim.x * ROWS)
    {
        const T* const x = reinterpret_cast<const T*>(p.x) + m * p.sx;
        int8_t* const q  = p.q + m * p.sq;
        float v[CH > 0 ? CH : 1][8];
        uint32_t most = 0;
        auto count = [&](const float(&t)[8]) {
#pragma unroll
            for(int i = 0; i < 8; ++i)
                most = larger(most, __builtin_bit_cast(uint32_t, t[i]) & 0x7fffffffu);
        };
        if constexpr(CH > 0)
        {
#pragma unroll
            for(int c = 0; c < CH; ++c)
                load_row8(x, ((int64_t)c * NT + tid) * 8, p.K, v[c]);
#pragma unroll
            for(int c = 0; c < CH; ++c)
                count(v[c]);
        }
        else
            for(int64_t k = (int64_t)tid * 8; k < p.K; k += NT * 8)
            {
                load_row8(x, k, p.K, v[0]);
                count(v[0]);
            }
#pragma unroll
        for(int d = 1; d < 64; d *= 2)
            most = larger(most, (uint32_t)__shfl_xor((int)most, d, 64));
        if constexpr(NT > 64)
        {
            if((threadIdx.x & 63) == 0)
                parts[threadIdx.x >> 6] = most;
            __syncthreads();
            most = larger(larger(parts[0], parts[1]), larger(parts[2], parts[3]));
            __syncthreads(); // (the next row's maxima go to the same places)
        }
        const bool finite   = most < 0x7f800000u;
        const float amax    = __builtin_fmaxf(__builtin_bit_cast(float, most), kTinyAmax);
        const Quotient by   = quotient_of<CODE_I8>(finite ? amax : 1.0f);
        if constexpr(CH > 0)
        {
#pragma unroll
            for(int c = 0; c < CH; ++c)
            {
                const int64_t k = ((int64_t)c * NT + tid) * 8;
                if(k < p.K)
                    store_row8<T>(q, k, p.K, v[c], by, finite);
            }
        }
        else
            for(int64_t k = (int64_t)tid * 8; k < p.K; k += NT * 8)
            {
                load_row8(x, k, p.K, v[0]);
                store_row8<T>(q, k, p.K, v[0], by, finite);
            }
        if(tid == 0)
            p.scale[m] = finite ? amax / kI8Max : __builtin_nanf("");
    }
}

template <typename T, int NT, int CH>
hipError_t launch(const TokenQuantArgs& a, hipStream_t s)
{
    const int64_t groups = ((int64_t)a.M + 256 / NT - 1) / (256 / NT);
    hipLaunchKernelGGL((quantize_tokens_kernel<T, NT, CH>), dim3((unsigned)(groups < (1 << 20) ? groups : (1 << 20))), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_any(const TokenQuantArgs& a, hipStream_t s)
{
    const int64_t chunks = ((int64_t)a.K + 7) / 8;
    if(chunks <= 64)
        return launch<T, 64, 1>(a, s);
    if(chunks <= 128)
        return launch<T, 64, 2>(a, s);
    if(chunks <= 256)
        return launch<T, 256, 1>(a, s);
    if(chunks <= 512)
        return launch<T, 256, 2>(a, s);
    if(chunks <= 1024)
        return launch<T, 256, 4>(a, s);
    if(chunks <= 256 * 6)
        return launch<T, 256, 6>(a, s);
    if(chunks <= 256 * kMostChunks)
        return launch<T, 256, kMostChunks>(a, s);
    return launch<T, 256, 0>(a, s);
}

} // namespace

hipError_t quantize_tokens_launch(const TokenQuantArgs& a, int x_type, hipStream_t s)
{
    return x_type == CKX_TYPE_F32   ? launch_any<float>(a, s)
           : x_type == CKX_TYPE_F16 ? launch_any<_Float16>(a, s)
                                    : launch_any<__bf16>(a, s);
}

} // namespace ckx
