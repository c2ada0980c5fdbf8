// Attention over a cache of 8-bit blocks (formula: include/ckx.h, ckx_paged_attention8): what its kernels share.
//
// The scales stay out of the products: a block's key scale multiplies the finished score q . codes, its value scale the
// probability, so that the matrix instructions run on the codes themselves, converted exactly to 16 bits (keys to the type of q,
// values to fp16). What is rounded is probability * value scale, to fp16 (2^-11 of each summand, independent from token to
// token), taken relative to the largest value scale that the row has met so far: without that, a scale of 2^-10 would put most of
// a row's products under fp16's normal numbers; bf16 would not need it, but rounds by 2^-8. Products under 2^-14 of that largest
// scale lose bits one by one, 2^-25 of it at most. Beside an fp16 output's own rounding it shows (2.9e-4 of the output where the
// plain form has 2.1e-4), beside bf16's by a percent.
#pragma once

#include "f8.hpp"
#include "serving.hpp"

namespace ckx {

// maximum / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48 (all of them get it). The halves of a swap go through scalars: a bit
// cast of a vector's element reads element 0.
template <typename F>
__device__ __forceinline__ float over_rows(float x, F&& f)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto a     = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    const uint32_t v = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
    const auto b     = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const uint32_t b0 = b[0], b1 = b[1];
    return f(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}
__device__ __forceinline__ float max_over_rows(float x)
{
    return over_rows(x, [](float a, float b) { return __builtin_fmaxf(a, b); });
}
__device__ __forceinline__ float sum_over_rows(float x)
{
    return over_rows(x, [](float a, float b) { return a + b; });
}

// round to nearest even
__device__ __forceinline__ uint32_t pack_f16(float a, float b)
{
    return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
}

// The value scale that a row's output sums are relative to: the largest finite one, by its size, of the blocks that the row has seen so far (a block
// that it does not see, however large, would cost it bits). take() returns what the sums so far are to be multiplied by, of() a
// scale relative to it (an infinity or NaN stays one).
struct ValueScale
{
    float top = kLeast, inv = 1.0f / kLeast;
    static constexpr float kLeast = 7.5e-37f; // (2^-120: no scale under it is told from zero)
    __device__ __forceinline__ float take(float a, float b)
    {
        a                = __builtin_isfinite(a) ? a : 0.0f;
        b                = __builtin_isfinite(b) ? b : 0.0f;
        const float next = __builtin_fmaxf(top, __builtin_fmaxf(a, b));
        if(next == top)
            return 1.0f;
        const float keep = top / next;
        top = next, inv = 1.0f / next;
        return keep;
    }
    __device__ __forceinline__ float of(float x) const { return x * inv; }
};

// four bytes of each of four tokens -> per element the four tokens' bytes
__device__ __forceinline__ void transpose4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t (&o)[4])
{
    const uint32_t ab0 = __builtin_amdgcn_perm(b, a, 0x05010400u), ab1 = __builtin_amdgcn_perm(b, a, 0x07030602u);
    const uint32_t cd0 = __builtin_amdgcn_perm(d, c, 0x05010400u), cd1 = __builtin_amdgcn_perm(d, c, 0x07030602u);
    o[0] = __builtin_amdgcn_perm(cd0, ab0, 0x05040100u), o[1] = __builtin_amdgcn_perm(cd0, ab0, 0x07060302u);
    o[2] = __builtin_amdgcn_perm(cd1, ab1, 0x05040100u), o[3] = __builtin_amdgcn_perm(cd1, ab1, 0x07060302u);
}

// What a tile is about: its sequence, its tokens and how far they see. The sequence is found by all lanes at once: sequence b's
// tiles begin at cu[b] / tile_tokens + b (cu[b] with one token a tile), which leaves every sequence enough of them. (64 sequences a
// round, each waiting for the one before: 1024 of 1000 tokens 493 us, where their bytes take 333.)
struct TileOf
{
    int b, q0, q_len, first; // sequence, its first row of q, its query tokens as far as q reaches, the tile's first token among them
    int of;                  // all its query tokens: what their places are counted by
    int kv;                  // cached tokens, as far as the table reaches
    bool live;
};
__device__ __forceinline__ TileOf tile_of(const AttentionArgs& p, int tile)
{
    const int lane = threadIdx.x & 63;
    TileOf t;
    t.b = 0, t.live = false, t.q0 = t.q_len = t.of = t.first = t.kv = 0;
    for(int b0 = 0; b0 < p.batch; b0 += 64)
    {
        // all three at once: what the sequence's lane has is handed on, not loaded again
        const int b = b0 + lane, at = min(b, p.batch - 1);
        const int begin = p.cu_q[at], end = p.cu_q[at + 1], kv = p.kv_lens[at];
        const int c = min(max(begin, 0), p.tokens), start = p.tile_tokens == 1 ? c : c / p.tile_tokens + b;
        const int n = __popcll(__ballot(b < p.batch && start <= tile)); // sequences that begin at or before the tile
        if(n > 0)
        {
            t.b     = b0 + n - 1;
            t.q0    = __builtin_amdgcn_readlane(c, n - 1);
            t.of    = max(__builtin_amdgcn_readlane(end, n - 1), t.q0) - t.q0;
            t.q_len = min(t.of, p.tokens - t.q0);
            t.first = (tile - __builtin_amdgcn_readlane(start, n - 1)) * p.tile_tokens;
            t.live  = t.first >= 0 && t.first < t.q_len;
            t.kv    = min(max(__builtin_amdgcn_readlane(kv, n - 1), 0), p.max_blocks << p.block_shift);
        }
        if(n < 64)
            break;
    }
    return t;
}

// sums of one share of the cached tokens, per query row: what the second pass joins
__host__ __device__ inline int64_t attention_rows(const AttentionArgs& p) { return (int64_t)p.tokens * p.heads; }

hipError_t attention_tile_launch(const AttentionArgs& a, bool f16, hipStream_t s); // paged_attention_tile.hip

} // namespace ckx
