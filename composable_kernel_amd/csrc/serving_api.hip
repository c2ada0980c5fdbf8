// C ABI of the 8-bit serving operators (include/ckx.h): argument checks and launch. The checks are pure host logic.
#include <hip/hip_runtime.h>

#include <cmath>

#include "api_error.hpp"
#include "serving.hpp"

namespace {

using ckx::api_fail;

bool half_type(int t) { return t == CKX_TYPE_F16 || t == CKX_TYPE_BF16; }
bool float_type(int t) { return t == CKX_TYPE_F32 || half_type(t); }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

constexpr float kLog2e        = 1.4426950408889634f;
constexpr int64_t kMostCached = 0x7fff0000; // (token numbers are rounded up to whole steps in 32 bits)

int block_shift(int size)
{
    return size == 16 ? 4 : size == 32 ? 5 : size == 64 ? 6 : size == 128 ? 7 : -1;
}

int check_cache(const ckx_kv_cache8* c)
{
    if(!c)
        return api_fail(CKX_INVALID_VALUE, "null cache");
    if(c->num_blocks < 0 || c->num_heads < 0 || c->head_dim < 0)
        return api_fail(CKX_INVALID_VALUE, "negative size");
    if(c->type != CKX_TYPE_E4M3 && c->type != CKX_TYPE_I8)
        return api_fail(CKX_INVALID_VALUE, "the cache holds e4m3 or int8 codes");
    if(block_shift(c->block_size) < 0)
        return api_fail(CKX_UNSUPPORTED, "block_size is 16, 32, 64 or 128");
    if(c->head_dim == 0 || c->head_dim % 16 || c->head_dim > 128)
        return api_fail(CKX_UNSUPPORTED, "head_dim is a multiple of 16 up to 128");
    if((int64_t)c->num_blocks * c->block_size > 0x7fffffffll)
        return api_fail(CKX_UNSUPPORTED, "slot numbers are 32-bit: at most 2^31 - 1 slots");
    if(c->stride_block % 16 || c->stride_head % 16 || c->stride_token % 16)
        return api_fail(CKX_UNSUPPORTED, "cache strides are multiples of 16");
    if((int64_t)c->block_size * c->stride_token > 0x7fffffffll)
        return api_fail(CKX_UNSUPPORTED, "the tokens of a block span 2 GiB");
    if(c->stride_block < 0 || c->stride_head < 0 || c->stride_token < c->head_dim || c->stride_scale < 0)
        return api_fail(CKX_UNSUPPORTED, "cache strides: tokens at least head_dim apart, none negative");
    // every (block, head, token) has bytes of its own: the three strides nest, heads and tokens in either order
    const int64_t hd = c->head_dim, tok = (int64_t)(c->block_size - 1) * c->stride_token,
                  head = c->num_heads > 1 ? (int64_t)(c->num_heads - 1) * c->stride_head : 0;
    const bool heads_outside = c->num_heads <= 1 || c->stride_head >= tok + hd;
    const bool heads_inside  = c->num_heads <= 1 || (c->stride_head >= hd && c->stride_token >= head + hd);
    if(!heads_outside && !heads_inside)
        return api_fail(CKX_UNSUPPORTED, "cache strides: two tokens or heads share bytes");
    if(c->num_blocks > 1 && (c->stride_block < head + tok + hd || c->stride_scale < c->num_heads))
        return api_fail(CKX_UNSUPPORTED, "cache strides: two blocks share bytes or scales");
    return CKX_OK;
}

int check_cache_pointers(const ckx_kv_cache8* c)
{
    if(!c->p_k || !c->p_v || !c->p_k_scale || !c->p_v_scale)
        return api_fail(CKX_INVALID_VALUE, "null cache pointer");
    if(!aligned16(c->p_k) || !aligned16(c->p_v))
        return api_fail(CKX_UNSUPPORTED, "the cache must be 16-byte aligned");
    if(!aligned4(c->p_k_scale) || !aligned4(c->p_v_scale))
        return api_fail(CKX_UNSUPPORTED, "the scales must be aligned to their element size");
    return CKX_OK;
}

// rows of `heads` heads of `dim` elements: strides in whole 16-byte vectors, no two rows on the same elements
bool rows_apart(int64_t st, int64_t sh, int heads, int dim)
{
    if(st < 0 || sh < 0 || st % 8 || sh % 8)
        return false;
    if(heads > 1 && sh < dim)
        return false;
    return st >= (heads > 1 ? (heads - 1) * sh : 0) + dim;
}

} // namespace

extern "C" {

int ckx_quantize_blocks_f8_is_supported(int32_t M, int32_t K, int32_t stride_x, int32_t stride_q, int32_t stride_scale_m,
                                        int32_t stride_scale_g, int x_type)
{
    if(M < 0 || K < 0)
        return api_fail(CKX_INVALID_VALUE, "negative size");
    if(!float_type(x_type))
        return api_fail(CKX_INVALID_VALUE, "x is fp32, fp16 or bf16");
    if(M > 1 && (stride_x < K || stride_q < K))
        return api_fail(CKX_UNSUPPORTED, "row strides are at least K");
    const int64_t groups = ((int64_t)K + 127) / 128;
    if(stride_scale_m < 0 || stride_scale_g < 0 || (M > 1 && stride_scale_m < 1) || (groups > 1 && stride_scale_g < 1) ||
       (M > 1 && groups > 1 && stride_scale_m < (groups - 1) * stride_scale_g + 1 &&
        stride_scale_g < (int64_t)(M - 1) * stride_scale_m + 1))
        return api_fail(CKX_UNSUPPORTED, "scale strides: two scales share an element");
    return CKX_OK;
}

int ckx_quantize_blocks_f8(const void* p_x, void* p_q, float* p_scale, int32_t M, int32_t K, int32_t stride_x,
                           int32_t stride_q, int32_t stride_scale_m, int32_t stride_scale_g, int x_type, void* stream)
{
    int st = ckx_quantize_blocks_f8_is_supported(M, K, stride_x, stride_q, stride_scale_m, stride_scale_g, x_type);
    if(st != CKX_OK)
        return st;
    if(M == 0 || K == 0)
        return CKX_OK;
    if(!p_x || !p_q || !p_scale)
        return api_fail(CKX_INVALID_VALUE, "null operand pointer");
    if((reinterpret_cast<uintptr_t>(p_x) & (x_type == CKX_TYPE_F32 ? 3 : 1)) || !aligned4(p_scale))
        return api_fail(CKX_UNSUPPORTED, "operands must be aligned to their element size");
    const ckx::QuantArgs a{p_x, static_cast<uint8_t*>(p_q), p_scale, M, K, stride_x, stride_q, stride_scale_m, stride_scale_g};
    hipError_t e = ckx::quantize_blocks_launch(a, x_type, (hipStream_t)stream);
    return e == hipSuccess ? CKX_OK : ckx::api_hip_fail(e, "quantize_blocks_f8");
}

int ckx_gemm_f8_blockscale_is_supported(int32_t M, int32_t N, int32_t K, int32_t lda, int32_t ldb, int32_t ldc,
                                        int32_t stride_sa_m, int32_t stride_sa_g, int32_t stride_sb_n, int32_t stride_sb_g,
                                        int c_type)
{
    if(M < 0 || N < 0 || K < 0)
        return api_fail(CKX_INVALID_VALUE, "negative size");
    if(!float_type(c_type))
        return api_fail(CKX_INVALID_VALUE, "C is fp32, fp16 or bf16");
    if((M > 1 && (lda < K || ldc < N)) || (N > 1 && ldb < K))
        return api_fail(CKX_UNSUPPORTED, "leading dimension smaller than the row");
    if(lda < 0 || ldb < 0 || ldc < 0 || stride_sa_m < 0 || stride_sa_g < 0 || stride_sb_n < 0 || stride_sb_g < 0)
        return api_fail(CKX_UNSUPPORTED, "negative stride");
    if(K > 1 << 30)
        return api_fail(CKX_UNSUPPORTED, "K is at most 2^30");
    if(!ckx::gemm_f8_fits(M, N))
        return api_fail(CKX_UNSUPPORTED, "more output tiles than one launch takes");
    // the rows of one tile (256 at most) are addressed through 32-bit offsets
    if((int64_t)lda * 256 > 0x7fff0000ll || (int64_t)ldb * 256 > 0x7fff0000ll)
        return api_fail(CKX_UNSUPPORTED, "256 rows of A or B span 2 GiB");
    return CKX_OK;
}

int64_t ckx_gemm_f8_blockscale_workspace_bytes(int32_t M, int32_t N, int32_t K)
{
    return M > 0 && N > 0 && K > 0 ? ckx::gemm_f8_workspace(M, N, K) : 0;
}

int ckx_gemm_f8_blockscale(const void* p_a, const void* p_b, void* p_c, const float* p_scale_a, const float* p_scale_b,
                           int32_t M, int32_t N, int32_t K, int32_t lda, int32_t ldb, int32_t ldc, int32_t stride_sa_m,
                           int32_t stride_sa_g, int32_t stride_sb_n, int32_t stride_sb_g, int c_type, void* p_workspace,
                           int64_t workspace_bytes, void* stream)
{
    int st = ckx_gemm_f8_blockscale_is_supported(M, N, K, lda, ldb, ldc, stride_sa_m, stride_sa_g, stride_sb_n, stride_sb_g,
                                                 c_type);
    if(st != CKX_OK)
        return st;
    if(M == 0 || N == 0)
        return CKX_OK;
    if(!p_c || (K > 0 && (!p_a || !p_b || !p_scale_a || !p_scale_b)))
        return api_fail(CKX_INVALID_VALUE, "null operand pointer");
    if((reinterpret_cast<uintptr_t>(p_c) & (c_type == CKX_TYPE_F32 ? 3 : 1)) || !aligned4(p_scale_a) || !aligned4(p_scale_b))
        return api_fail(CKX_UNSUPPORTED, "operands must be aligned to their element size");
    if(workspace_bytes < 0 || (p_workspace && !aligned16(p_workspace)))
        return api_fail(CKX_INVALID_VALUE, "the workspace must be 16-byte aligned");
    ckx::GemmF8Args a{};
    a.a = static_cast<const uint8_t*>(p_a), a.b = static_cast<const uint8_t*>(p_b), a.c = p_c;
    a.sa = p_scale_a, a.sb = p_scale_b, a.M = M, a.N = N, a.K = K, a.lda = lda, a.ldb = ldb, a.ldc = ldc;
    a.sa_m = stride_sa_m, a.sa_g = stride_sa_g, a.sb_n = stride_sb_n, a.sb_g = stride_sb_g;
    a.ws         = static_cast<float*>(p_workspace);
    hipError_t e = ckx::gemm_f8_launch(a, c_type, p_workspace ? workspace_bytes : 0, (hipStream_t)stream);
    return e == hipSuccess ? CKX_OK : ckx::api_hip_fail(e, "gemm_f8_blockscale");
}

int ckx_gemm_f8_blockscale_plan(int32_t M, int32_t N, int32_t K, int32_t lda, int32_t ldb, int32_t ldc, int c_type,
                                int64_t workspace_bytes, int* tile_m, int* tile_n, int* k_runs)
{
    if(!tile_m || !tile_n || !k_runs)
        return api_fail(CKX_INVALID_VALUE, "null result pointer");
    int st = ckx_gemm_f8_blockscale_is_supported(M, N, K, lda, ldb, ldc, 1, M, 1, 1, c_type);
    if(st != CKX_OK)
        return st;
    if(workspace_bytes < 0)
        return api_fail(CKX_INVALID_VALUE, "negative size");
    *tile_m = *tile_n = *k_runs = 0;
    if(M > 0 && N > 0)
        ckx::gemm_f8_plan(M, N, K, lda, ldb, c_type, workspace_bytes, tile_m, tile_n, k_runs);
    return CKX_OK;
}

int ckx_kv_cache_tables_is_supported(int32_t batch, int32_t num_free, int32_t max_blocks, int32_t stride_table,
                                     int32_t num_slots, int32_t block_size)
{
    if(batch < 0 || num_free < 0 || max_blocks < 0 || num_slots < 0)
        return api_fail(CKX_INVALID_VALUE, "negative size");
    if(block_shift(block_size) < 0)
        return api_fail(CKX_UNSUPPORTED, "block_size is 16, 32, 64 or 128");
    if(batch > ckx::kMaxTableSequences)
        return api_fail(CKX_UNSUPPORTED, "at most 8192 sequences");
    if(batch > 1 && stride_table < max_blocks)
        return api_fail(CKX_UNSUPPORTED, "table rows overlap");
    return CKX_OK;
}

int ckx_kv_cache_tables(const int32_t* p_context_lens, const int32_t* p_new_lens, const int32_t* p_free_blocks,
                        int32_t* p_block_table, int32_t* p_cu_new, int32_t* p_kv_lens, int32_t* p_slots, int32_t* p_used,
                        int32_t batch, int32_t num_free, int32_t max_blocks, int32_t stride_table, int32_t num_slots,
                        int32_t block_size, void* stream)
{
    int st = ckx_kv_cache_tables_is_supported(batch, num_free, max_blocks, stride_table, num_slots, block_size);
    if(st != CKX_OK)
        return st;
    if(!p_cu_new || !p_used || (num_slots > 0 && !p_slots) || (num_free > 0 && !p_free_blocks) ||
       (batch > 0 && (!p_context_lens || !p_new_lens || !p_kv_lens || (max_blocks > 0 && !p_block_table))))
        return api_fail(CKX_INVALID_VALUE, "null operand pointer");
    for(const void* p : {(const void*)p_context_lens, (const void*)p_new_lens, (const void*)p_free_blocks, (const void*)p_block_table,
                         (const void*)p_cu_new, (const void*)p_kv_lens, (const void*)p_slots, (const void*)p_used})
        if(!aligned4(p))
            return api_fail(CKX_UNSUPPORTED, "operands must be aligned to their element size");
    // every workgroup reads the lengths and the free list for itself, while others already write
    const struct
    {
        const int32_t* p;
        int64_t n;
    } in[]  = {{p_context_lens, batch}, {p_new_lens, batch}, {p_free_blocks, num_free}},
      out[] = {{p_block_table, batch > 0 ? (batch - 1) * (int64_t)stride_table + max_blocks : 0}, {p_cu_new, (int64_t)batch + 1},
               {p_kv_lens, batch}, {p_slots, num_slots}, {p_used, 1}};
    for(const auto& o : out)
    {
        for(const auto& i : in)
            if(i.n > 0 && o.n > 0 && i.p < o.p + o.n && o.p < i.p + i.n)
                return api_fail(CKX_INVALID_VALUE, "an output lies on an input");
        for(const auto& x : out)
            if(&x != &o && x.n > 0 && o.n > 0 && x.p < o.p + o.n && o.p < x.p + x.n)
                return api_fail(CKX_INVALID_VALUE, "two outputs overlap");
    }
    const ckx::TablesArgs a{p_context_lens, p_new_lens, p_free_blocks, p_block_table, p_cu_new, p_kv_lens, p_slots, p_used,
                            batch, num_free, max_blocks, stride_table, num_slots, block_shift(block_size)};
    hipError_t e = ckx::kv_tables_launch(a, (hipStream_t)stream);
    return e == hipSuccess ? CKX_OK : ckx::api_hip_fail(e, "kv_cache_tables");
}

int ckx_kv_cache_store8_is_supported(const ckx_kv_cache8* cache, int32_t num_tokens, int32_t stride_k_token,
                                     int32_t stride_k_head, int32_t stride_v_token, int32_t stride_v_head, int x_type)
{
    int st = check_cache(cache);
    if(st != CKX_OK)
        return st;
    if(num_tokens < 0)
        return api_fail(CKX_INVALID_VALUE, "negative size");
    if(!half_type(x_type))
        return api_fail(CKX_INVALID_VALUE, "keys and values are fp16 or bf16");
    if(!rows_apart(stride_k_token, stride_k_head, cache->num_heads, cache->head_dim) ||
       !rows_apart(stride_v_token, stride_v_head, cache->num_heads, cache->head_dim))
        return api_fail(CKX_UNSUPPORTED, "key / value strides: multiples of 8, heads at least head_dim and tokens a whole row apart");
    if(cache->num_heads > 32767)
        return api_fail(CKX_UNSUPPORTED, "at most 32767 heads");
    if(num_tokens > 1 << 29)
        return api_fail(CKX_UNSUPPORTED, "at most 2^29 tokens a call");
    return CKX_OK;
}

int ckx_kv_cache_store8(const void* p_k, const void* p_v, const int32_t* p_slots, const ckx_kv_cache8* cache,
                        int32_t num_tokens, int32_t stride_k_token, int32_t stride_k_head, int32_t stride_v_token,
                        int32_t stride_v_head, int x_type, void* stream)
{
    int st = ckx_kv_cache_store8_is_supported(cache, num_tokens, stride_k_token, stride_k_head, stride_v_token, stride_v_head,
                                              x_type);
    if(st != CKX_OK)
        return st;
    if(num_tokens == 0 || cache->num_blocks == 0 || cache->num_heads == 0)
        return CKX_OK;
    if(!p_k || !p_v || !p_slots)
        return api_fail(CKX_INVALID_VALUE, "null operand pointer");
    if((st = check_cache_pointers(cache)) != CKX_OK)
        return st;
    if(!aligned16(p_k) || !aligned16(p_v) || !aligned4(p_slots))
        return api_fail(CKX_UNSUPPORTED, "keys and values must be 16-byte aligned");
    const ckx::StoreArgs a{p_k, p_v, p_slots, *cache, num_tokens, block_shift(cache->block_size), stride_k_token, stride_k_head,
                           stride_v_token, stride_v_head};
    hipError_t e = ckx::kv_store_launch(a, x_type, (hipStream_t)stream);
    return e == hipSuccess ? CKX_OK : ckx::api_hip_fail(e, "kv_cache_store8");
}

int ckx_paged_attention8_is_supported(const ckx_kv_cache8* cache, int32_t batch, int32_t num_tokens, int32_t num_q_heads,
                                      int32_t max_kv_len, int32_t max_blocks, int32_t stride_table, int32_t stride_q_token,
                                      int32_t stride_q_head, int32_t stride_o_token, int32_t stride_o_head, float scale,
                                      int causal, int q_type)
{
    int st = check_cache(cache);
    if(st != CKX_OK)
        return st;
    if(batch < 0 || num_tokens < 0 || num_q_heads < 0 || max_kv_len < 0 || max_blocks < 0)
        return api_fail(CKX_INVALID_VALUE, "negative size");
    if(!half_type(q_type))
        return api_fail(CKX_INVALID_VALUE, "queries and outputs are fp16 or bf16");
    if(causal != 0 && causal != 1)
        return api_fail(CKX_INVALID_VALUE, "causal is 0 or 1");
    if(!std::isfinite(scale * kLog2e))
        return api_fail(CKX_INVALID_VALUE, "the score scale (times log2 e) must be finite");
    if(num_q_heads > 0 && (cache->num_heads == 0 || num_q_heads % cache->num_heads))
        return api_fail(CKX_UNSUPPORTED, "query heads are a multiple of the cache's heads");
    if(batch > 1 && stride_table < max_blocks)
        return api_fail(CKX_UNSUPPORTED, "table rows overlap");
    if((int64_t)max_blocks * cache->block_size > kMostCached)
        return api_fail(CKX_UNSUPPORTED, "a sequence has at most 2^31 - 65536 tokens");
    if(!rows_apart(stride_q_token, stride_q_head, num_q_heads, cache->head_dim) ||
       !rows_apart(stride_o_token, stride_o_head, num_q_heads, cache->head_dim))
        return api_fail(CKX_UNSUPPORTED, "query / output strides: multiples of 8, heads at least head_dim and tokens a whole row apart");
    if(batch > 0x3fffffff || (int64_t)num_tokens * num_q_heads > 0x3fffffffll ||
       (batch > 0 && num_tokens > 0 && num_q_heads > 0 &&
        !ckx::attention_fits(*cache, batch, num_tokens, num_q_heads, max_kv_len, max_blocks)))
        return api_fail(CKX_UNSUPPORTED, "more query rows than one launch takes");
    return CKX_OK;
}

int64_t ckx_paged_attention8_workspace_bytes(const ckx_kv_cache8* cache, int32_t batch, int32_t num_tokens,
                                             int32_t num_q_heads, int32_t max_kv_len, int32_t max_blocks)
{
    if(check_cache(cache) != CKX_OK || batch <= 0 || num_tokens <= 0 || num_q_heads <= 0 || max_kv_len < 0 || max_blocks < 0 ||
       cache->num_heads <= 0 || num_q_heads % cache->num_heads || batch > 0x3fffffff ||
       (int64_t)num_tokens * num_q_heads > 0x3fffffffll || (int64_t)max_blocks * cache->block_size > kMostCached)
        return 0;
    return ckx::attention_workspace(*cache, batch, num_tokens, num_q_heads, max_kv_len, max_blocks);
}

int ckx_paged_attention8(const void* p_q, void* p_o, const int32_t* p_block_table, const int32_t* p_cu_q,
                         const int32_t* p_kv_lens, const ckx_kv_cache8* cache, int32_t batch, int32_t num_tokens,
                         int32_t num_q_heads, int32_t max_kv_len, int32_t max_blocks, int32_t stride_table,
                         int32_t stride_q_token, int32_t stride_q_head, int32_t stride_o_token, int32_t stride_o_head,
                         float scale, int causal, int q_type, void* p_workspace, int64_t workspace_bytes, void* stream)
{
    int st = ckx_paged_attention8_is_supported(cache, batch, num_tokens, num_q_heads, max_kv_len, max_blocks, stride_table,
                                               stride_q_token, stride_q_head, stride_o_token, stride_o_head, scale, causal,
                                               q_type);
    if(st != CKX_OK)
        return st;
    if(batch == 0 || num_tokens == 0 || num_q_heads == 0)
        return CKX_OK;
    if(!p_q || !p_o || !p_cu_q || !p_kv_lens || (max_blocks > 0 && !p_block_table))
        return api_fail(CKX_INVALID_VALUE, "null operand pointer");
    if(cache->num_blocks > 0 && (st = check_cache_pointers(cache)) != CKX_OK)
        return st;
    if(!aligned16(p_q) || !aligned16(p_o) || !aligned4(p_block_table) || !aligned4(p_cu_q) || !aligned4(p_kv_lens))
        return api_fail(CKX_UNSUPPORTED, "queries and outputs must be 16-byte aligned");
    const int64_t need = ckx::attention_workspace(*cache, batch, num_tokens, num_q_heads, max_kv_len, max_blocks);
    if(need > 0 && (!p_workspace || workspace_bytes < need))
        return api_fail(CKX_UNSUPPORTED, "the workspace is smaller than ckx_paged_attention8_workspace_bytes");
    if(need > 0 && !aligned16(p_workspace))
        return api_fail(CKX_INVALID_VALUE, "the workspace must be 16-byte aligned");
    ckx::AttentionArgs a{};
    a.q = p_q, a.o = p_o, a.table = p_block_table, a.cu_q = p_cu_q, a.kv_lens = p_kv_lens, a.cache = *cache;
    a.batch = batch, a.tokens = num_tokens, a.heads = num_q_heads, a.group = num_q_heads / cache->num_heads;
    a.max_kv = max_kv_len, a.max_blocks = max_blocks, a.stride_table = stride_table;
    a.block_shift = block_shift(cache->block_size);
    a.sq_t = stride_q_token, a.sq_h = stride_q_head, a.so_t = stride_o_token, a.so_h = stride_o_head;
    a.scale  = scale * kLog2e; // (the kernels work in powers of two)
    a.causal = causal;
    a.ws     = static_cast<float*>(p_workspace);
    hipError_t e = ckx::attention_launch(a, q_type, (hipStream_t)stream);
    return e == hipSuccess ? CKX_OK : ckx::api_hip_fail(e, "paged_attention8");
}

} // extern "C"
