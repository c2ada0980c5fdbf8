// The cache of 8-bit blocks: tables of a step from the requests' lengths, and the store of new tokens (formulas:
// include/ckx.h, ckx_kv_cache_tables and ckx_kv_cache_store8).
#include "f8.hpp"
#include "serving.hpp"

namespace ckx {

namespace {

// ---------------------------------------------------------------------------------------------------- tables
// One launch: every workgroup sums the lengths of all sequences for itself (8 bytes a sequence, out of L2 after the first
// workgroup; 8192 at most, their two running sums in LDS), then takes its share of the tokens and of the new blocks and finds
// the sequence of each by bisection. The alternative, one workgroup that sums and a second launch that fills, costs the second
// launch. What bounds it is that latency: the bytes are few. 64 sequences 5.4 us, 1024 with 256 new tokens each 6.6.
constexpr int kTablesThreads = 256, kTokensPerGroup = 4 * kTablesThreads;

__device__ __forceinline__ int blocks_of(int tokens, int shift) { return (int)(((int64_t)tokens + (1 << shift) - 1) >> shift); }

// the last b in [0, n) with sums[b] <= x (sums ascending, sums[0] <= x)
__device__ __forceinline__ int last_at_most(const int* sums, int n, int x)
{
    int lo = 0, hi = n;
    while(hi - lo > 1)
    {
        const int mid = (lo + hi) >> 1;
        if(sums[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

__global__ __launch_bounds__(kTablesThreads) void kv_tables_kernel(TablesArgs p)
{
    __shared__ int cu[kMaxTableSequences + 1], base[kMaxTableSequences + 1];
    __shared__ int part[2][kTablesThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // a thread's stretch of sequences: its own sums, then those of the threads before it
    const int per = (p.batch + kTablesThreads - 1) / kTablesThreads;
    const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
    int tokens = 0, blocks = 0;
    for(int b = b0; b < b1; ++b)
    {
        const int c = max(p.context[b], 0), n = max(p.fresh[b], 0);
        cu[b] = tokens, base[b] = blocks;
        tokens += n;
        blocks += blocks_of(c + n, p.block_shift) - blocks_of(c, p.block_shift);
        if(blockIdx.x == 0)
            p.kv_lens[b] = c + n;
    }
    int t = tokens, k = blocks;
    for(int d = 1; d < 64; d *= 2)
    {
        const int tt = __shfl_up(t, d), kk = __shfl_up(k, d);
        if(lane >= d)
            t += tt, k += kk;
    }
    if(lane == 63)
        part[0][wave] = t, part[1][wave] = k;
    __syncthreads();
    int t0 = t - tokens, k0 = k - blocks, all_tokens = 0, all_blocks = 0;
    for(int w = 0; w < kTablesThreads / 64; ++w)
    {
        if(w < wave)
            t0 += part[0][w], k0 += part[1][w];
        all_tokens += part[0][w], all_blocks += part[1][w];
    }
    for(int b = b0; b < b1; ++b)
    {
        cu[b] += t0, base[b] += k0;
        if(blockIdx.x == 0)
            p.cu[b] = cu[b];
    }
    if(tid == 0)
    {
        cu[p.batch] = all_tokens, base[p.batch] = all_blocks;
        if(blockIdx.x == 0)
            p.cu[p.batch] = all_tokens, p.used[0] = all_blocks;
    }
    __syncthreads();

    // the table's new columns: new block f of all belongs to sequence b
    for(int f = blockIdx.x * kTablesThreads + tid; f < all_blocks && f < p.num_free; f += gridDim.x * kTablesThreads)
    {
        const int b   = last_at_most(base, p.batch, f);
        const int col = blocks_of(max(p.context[b], 0), p.block_shift) + f - base[b];
        if((unsigned)col < (unsigned)p.max_blocks) // (unsigned: sums past 31 bits lead nowhere outside)
            p.table[(int64_t)b * p.stride_table + col] = p.free[f];
    }
    // the slots, four neighbours a thread, whose sequence is looked for once; a new block comes from the free list itself, not from
    // the table that another workgroup is writing
    const int64_t x0 = (int64_t)blockIdx.x * kTokensPerGroup + tid * 4;
    if(x0 >= p.num_slots)
        return;
    int b = x0 < all_tokens ? last_at_most(cu, p.batch, (int)x0) : 0;
    int slot[4];
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        const int64_t x = x0 + i;
        slot[i]         = -1;
        if(x < all_tokens)
        {
            while(cu[b + 1] <= (int)x)
                ++b;
            const int c = max(p.context[b], 0), pos = c + (int)x - cu[b], col = pos >> p.block_shift;
            const int had = blocks_of(c, p.block_shift);
            int block     = -1;
            if((unsigned)col < (unsigned)p.max_blocks)
            {
                if(col < had)
                    block = p.table[(int64_t)b * p.stride_table + col];
                else if((unsigned)(base[b] + col - had) < (unsigned)p.num_free)
                    block = p.free[base[b] + col - had];
            }
            if(block >= 0 && block <= 0x7fffffff >> p.block_shift) // (a number without a 32-bit slot is no block)
                slot[i] = (block << p.block_shift) + (pos & ((1 << p.block_shift) - 1));
        }
    }
    if(x0 + 4 <= p.num_slots)
        reinterpret_cast<AnyAlign<i32x4>*>(p.slots + x0)->v = i32x4{slot[0], slot[1], slot[2], slot[3]};
    else
#pragma unroll
        for(int i = 0; i < 3; ++i)
            if(x0 + i < p.num_slots)
                p.slots[x0 + i] = slot[i];
}

// ---------------------------------------------------------------------------------------------------- store
// One wave takes a run (the new tokens of one block) of one head, keys or values: a pass for the maximum, the block's scale,
// the older codes if the scale grew, and a pass that writes the codes. Which runs begin among a wave's
// `span` tokens comes out of one comparison of neighbouring slots, so that no list of runs is needed. The first 16 (32) tokens of
// a run stay in registers between the passes. Memory bounds it (2 bytes read, 1 written per element): 4 x 4096 tokens of 8 heads of
// 128 in 19.4 us, 4.1 TB/s (13.4 at the rates that reads and writes alone reach); 64 tokens, latency: 5.3 with the launch.
constexpr int kKept = 4; // vectors a lane keeps

template <typename T, int CODE>
__global__ __launch_bounds__(256) void kv_store_kernel(StoreArgs p, int span)
{
    const int lane  = threadIdx.x & 63;
    const int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int first = (int)(u * span);
    if(u * span >= p.tokens)
        return;
    const int head   = blockIdx.y >> 1;
    const bool value = blockIdx.y & 1;
    const int shift = p.block_shift, size = 1 << shift;
    const int64_t slots = (int64_t)p.cache.num_blocks << shift;
    const T* x          = reinterpret_cast<const T*>(value ? p.v : p.k) + (int64_t)head * (value ? p.sv_h : p.sk_h);
    const int64_t xt    = value ? p.sv_t : p.sk_t;
    uint8_t* codes      = reinterpret_cast<uint8_t*>(value ? p.cache.p_v : p.cache.p_k) + (int64_t)head * p.cache.stride_head;
    float* scales       = (value ? p.cache.p_v_scale : p.cache.p_k_scale) + head;
    // block of token t's slot, -1 for a token that is skipped or not there
    auto block_of = [&](int64_t t) {
        if(t < 0 || t >= p.tokens)
            return -1;
        const int s = p.slots[t];
        return s < 0 || s >= slots ? -1 : s >> shift;
    };
    // lane l: the block of token first - 1 + l
    const int near = block_of((int64_t)first - 1 + lane);
    const int before = __shfl_up(near, 1); // (by all lanes: one that takes no part gives nothing)
    uint64_t leads   = __ballot(lane >= 1 && lane <= span && near >= 0 && near != before);

    const int per_token = p.cache.head_dim >> 3;      // lanes of eight elements
    const int at_once   = 64 / per_token;             // tokens
    const int my = lane / per_token, d = (lane - my * per_token) * 8;
    const bool active = my < at_once;
    while(leads)
    {
        const int i = __builtin_ctzll(leads); // (the lane)
        leads &= leads - 1;
        const int64_t t0 = (int64_t)first - 1 + i;
        const int block  = __builtin_amdgcn_readfirstlane(__shfl(near, i));
        const int begin  = p.slots[t0] & (size - 1);
        // tokens of the run, at most a block's: as far as the lanes see, then on from there
        int count = __builtin_ctzll(~(__ballot(near == block) >> i)); // (i >= 1: the shift brings zeros)
        if(count >= 64 - i)
            for(count = 64 - i; count < size; count += 64)
            {
                const uint64_t out = __ballot(block_of(t0 + count + lane) != block);
                if(out)
                {
                    count += __builtin_ctzll(out);
                    break;
                }
            }
        count = min(count, size);

        float amax = kTinyAmax;
        bool nan   = false;
        typedef T tx8 __attribute__((ext_vector_type(8)));
        tx8 kept[kKept];
#pragma unroll
        for(int c = 0; c < kKept; ++c)
        {
            const int n = c * at_once + my;
            kept[c]     = tx8{0, 0, 0, 0, 0, 0, 0, 0};
            if(active && n < count)
                kept[c] = *reinterpret_cast<const tx8*>(x + (t0 + n) * xt + d);
        }
        auto look = [&](const tx8& v) {
#pragma unroll
            for(int j = 0; j < 8; ++j)
            {
                amax = __builtin_fmaxf(amax, __builtin_fabsf((float)v[j]));
                nan |= v[j] != v[j];
            }
        };
#pragma unroll
        for(int c = 0; c < kKept; ++c)
            look(kept[c]);
#pragma unroll 4
        for(int n = kKept * at_once; n < count; n += at_once)
            if(active && n + my < count)
                look(*reinterpret_cast<const tx8*>(x + (t0 + n + my) * xt + d));
        for(int s = 1; s < 64; s *= 2)
            amax = __builtin_fmaxf(amax, __shfl_xor(amax, s));
        const float fresh = __any(nan) ? __builtin_nanf("") : amax / (CODE == CODE_E4M3 ? kE4m3Max : kI8Max);
        float* const at   = scales + (int64_t)block * p.cache.stride_scale;
        uint8_t* const to = codes + (int64_t)block * p.cache.stride_block;
        float now         = fresh;
        Quotient by       = quotient_of<CODE>(fresh == fresh ? amax : fresh);
        auto put = [&](int token, const float(&v)[8]) { // (a NaN has no code: the scale says it)
            float w[8];
#pragma unroll
            for(int j = 0; j < 8; ++j)
                w[j] = v[j] == v[j] ? v[j] : 0.0f;
            *reinterpret_cast<u32x2*>(to + (int64_t)token * p.cache.stride_token + d) =
                u32x2{codes_of<CODE>(w[0], w[1], w[2], w[3]), codes_of<CODE>(w[4], w[5], w[6], w[7])};
        };
        if(begin > 0)
        {
            const float old = *at;
            now             = old != old || __builtin_fabsf(old) >= fresh ? old : fresh; // (a scale of either sign, by its size)
            if(now == old || old != old)
                by = Quotient(1.0f, old);
            else
            {
                const float ratio = old / now;
                for(int n = 0; n < begin; n += at_once)
                    if(active && n + my < begin)
                    {
                        const u32x2 c = *reinterpret_cast<const u32x2*>(to + (int64_t)(n + my) * p.cache.stride_token + d);
                        float v[8];
#pragma unroll
                        for(int j = 0; j < 8; ++j)
                            v[j] = code_value<CODE>(c[j >> 2], j & 3) * ratio;
                        put(n + my, v);
                    }
            }
        }
        if(lane == 0)
            *at = now;
        auto write = [&](int n, const tx8& raw) {
            float v[8];
#pragma unroll
            for(int j = 0; j < 8; ++j)
                v[j] = by.of<true>((float)raw[j]);
            put(p.slots[t0 + n] & (size - 1), v);
        };
#pragma unroll
        for(int c = 0; c < kKept; ++c)
            if(active && c * at_once + my < count)
                write(c * at_once + my, kept[c]);
#pragma unroll 4
        for(int n = kKept * at_once; n < count; n += at_once)
            if(active && n + my < count)
                write(n + my, *reinterpret_cast<const tx8*>(x + (t0 + n + my) * xt + d));
    }
}

template <typename T, int CODE>
hipError_t launch_store(const StoreArgs& a, hipStream_t s)
{
    // Tokens a wave looks at, us with 1 / 4 / 16 of them (8 heads of 128). Single tokens of as many sequences: 64 5.0 / 6.9 / 22, 512
    // 7.6 / 8.2 / 21, 1024 12.1 / 10.9 / 21, 4096 43 / 35 / 37; prompts: 512 5.2 / 4.8 / 5.7, 1024 9.5 / 4.8 / 5.4, 4096 14.3 / 9.6 / 8.8,
    // 4 of 4096 37 / 25 / 19
    const int span      = a.tokens <= 512 ? 1 : a.tokens <= 4096 ? 4 : 16;
    const int64_t units = ((int64_t)a.tokens + span - 1) / span;
    hipLaunchKernelGGL((kv_store_kernel<T, CODE>), dim3((unsigned)((units + 3) / 4), (unsigned)a.cache.num_heads * 2), dim3(256), 0, s,
                       a, span);
    return hipGetLastError();
}

} // namespace

hipError_t kv_tables_launch(const TablesArgs& a, hipStream_t s)
{
    const int64_t groups = ((int64_t)a.num_slots + kTokensPerGroup - 1) / kTokensPerGroup;
    hipLaunchKernelGGL(kv_tables_kernel, dim3((unsigned)(groups > 0 ? groups : 1)), dim3(kTablesThreads), 0, s, a);
    return hipGetLastError();
}

hipError_t kv_store_launch(const StoreArgs& a, int x_type, hipStream_t s)
{
    if(a.cache.type == CKX_TYPE_E4M3)
        return x_type == CKX_TYPE_F16 ? launch_store<_Float16, CODE_E4M3>(a, s) : launch_store<__bf16, CODE_E4M3>(a, s);
    return x_type == CKX_TYPE_F16 ? launch_store<_Float16, CODE_I8>(a, s) : launch_store<__bf16, CODE_I8>(a, s);
}

} // namespace ckx
