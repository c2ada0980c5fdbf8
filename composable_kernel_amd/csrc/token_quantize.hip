// Activations to int8 with one scale per token (formula: include/ckx.h, ckx_quantize_tokens_i8).
//
// One pass: a row lies in the registers of its threads between its maximum and its codes (eight elements at a time, rows of up to
// 16384; longer ones are read again). 64 threads a row where it is short, 256 otherwise, whose maxima meet in LDS. Memory bounds it: bf16 8192 x
// 11008 in 49.5 us, 5.5 TB/s of reads and writes (a plain copy of 2 GiB 5.0 to 5.7); fp32 8192 x 4096 31.5, 5.3. Loads that stood behind a branch each
// took 67 us for the first.
#include "experts.hpp"
#include "f8.hpp"

namespace ckx {

namespace {

constexpr int kMostChunks = 8; // of eight elements that a thread holds

// eight elements as they lie in memory. `most`: the largest of their sizes as bits, where infinities lie above every number and NaNs
// above them: two 16-bit values at a time.
template <typename T>
struct Row8
{
    u32x4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* x)
    {
#pragma unroll
        for(int i = 0; i < (int)(sizeof(T) / 2); ++i)
            w[i] = load_vec<u32x4>(x + i * (16 / (int)sizeof(T)));
    }
    __device__ __forceinline__ uint32_t most(uint32_t m) const
    {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for(int i = 0; i < (int)(sizeof(T) / 2); ++i)
#pragma unroll
            for(int j = 0; j < 4; ++j)
            {
                if constexpr(sizeof(T) == 4)
                    m = max(m, w[i][j] & 0x7fffffffu);
                else
                    m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, w[i][j] & 0x7fff7fffu)));
            }
        return m;
    }
    __device__ __forceinline__ float operator[](int i) const
    {
        typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
        constexpr int PER = 16 / (int)sizeof(T);
        return (float)__builtin_bit_cast(vec, w[i / PER])[i % PER];
    }
};
// the size that bits stand for
template <typename T>
__device__ __forceinline__ float size_of(uint32_t bits)
{
    if constexpr(sizeof(T) == 4)
        return __builtin_bit_cast(float, bits);
    else
        return (float)__builtin_bit_cast(T, (uint16_t)bits);
}
// (1.5 * 2^23 added: the sum's unit is 1, rounded to even, and its low byte the code)
template <typename T>
__device__ __forceinline__ uint32_t code_bits(float x, const Quotient& by)
{
    return __builtin_bit_cast(uint32_t, by.of<sizeof(T) == 2>(x) + 12582912.0f);
}
template <typename T>
__device__ __forceinline__ void store_codes(int8_t* q, const Row8<T>& v, const Quotient& by, bool finite)
{
    uint32_t c[8], w[2];
#pragma unroll
    for(int i = 0; i < 8; ++i)
        c[i] = code_bits<T>(v[i], by);
#pragma unroll
    for(int h = 0; h < 2; ++h)
        w[h] = finite ? (uint32_t)pack4_low_bytes((int)c[4 * h], (int)c[4 * h + 1], (int)c[4 * h + 2], (int)c[4 * h + 3]) : 0u;
    reinterpret_cast<AnyAlign<u32x2>*>(q)->v = u32x2{w[0], w[1]};
}

// NT threads a row, CH chunks of eight a thread (0: any number, the row is read twice). Every thread loads all its chunks, the row's last
// in place of those behind it, so that nothing stands between the loads; what is left of the row after its whole chunks, seven elements
// at most, is one element each for the first threads.
template <typename T, int NT, int CH>
__global__ __launch_bounds__(256) void quantize_tokens_kernel(TokenQuantArgs p)
{
    constexpr int ROWS = 256 / NT, N = CH > 0 ? CH : 1;
    __shared__ uint32_t parts[2][4];
    const int tid = threadIdx.x % NT, chunks = p.K / 8, rest = p.K % 8;
    int turn      = 0;
    for(int64_t m = (int64_t)blockIdx.x * ROWS + threadIdx.x / NT; m < p.M; m += (int64_t)gridDim.x * ROWS, turn ^= 1)
    {
        const T* const x = reinterpret_cast<const T*>(p.x) + m * p.sx;
        int8_t* const q  = p.q + m * p.sq;
        Row8<T> v[N];
        uint32_t most = 0;
        T last        = (T)0.0f;
        if(tid < rest)
            last = x[(int64_t)chunks * 8 + tid];
        if constexpr(CH > 0)
        {
            if(chunks > 0)
            {
#pragma unroll
                for(int c = 0; c < CH; ++c)
                    v[c].load(x + min(c * NT + tid, chunks - 1) * 8);
#pragma unroll
                for(int c = 0; c < CH; ++c)
                    most = v[c].most(most);
            }
        }
        else
            for(int c = tid; c < chunks; c += NT)
            {
                v[0].load(x + (int64_t)c * 8);
                most = v[0].most(most);
            }
        if constexpr(sizeof(T) == 2)
            most = max(max(most & 0xffffu, most >> 16), __builtin_bit_cast(uint16_t, last) & 0x7fffu);
        else
            most = max(most, __builtin_bit_cast(uint32_t, last) & 0x7fffffffu);
#pragma unroll
        for(int d = 1; d < 64; d *= 2)
            most = max(most, (uint32_t)__shfl_xor((int)most, d, 64));
        if constexpr(NT > 64)
        {
            // (a row's maxima have their places until the row after next: one barrier a row)
            if((threadIdx.x & 63) == 0)
                parts[turn][threadIdx.x >> 6] = most;
            __syncthreads();
            most = max(max(parts[turn][0], parts[turn][1]), max(parts[turn][2], parts[turn][3]));
        }
        const float size  = size_of<T>(most);
        const bool finite = size < __builtin_inff(); // (a NaN is not)
        const float amax  = __builtin_fmaxf(finite ? size : 1.0f, kTinyAmax);
        const Quotient by = quotient_of<CODE_I8>(amax);
        if constexpr(CH > 0)
        {
#pragma unroll
            for(int c = 0; c < CH; ++c)
                if(c * NT + tid < chunks)
                    store_codes(q + (c * NT + tid) * 8, v[c], by, finite);
        }
        else
            for(int c = tid; c < chunks; c += NT)
            {
                v[0].load(x + (int64_t)c * 8);
                store_codes(q + (int64_t)c * 8, v[0], by, finite);
            }
        if(tid < rest)
            q[(int64_t)chunks * 8 + tid] = finite ? (int8_t)code_bits<T>((float)last, by) : (int8_t)0;
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
