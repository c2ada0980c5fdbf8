// C ABI of the int8 linear and mixture-of-experts operators (include/ckx.h): argument checks and launch. The checks are pure host
// logic.
#include <hip/hip_runtime.h>

#include <cmath>

#include "api_error.hpp"
#include "experts.hpp"

namespace {

using ckx::api_fail;

bool float_type(int t) { return t == CKX_TYPE_F32 || t == CKX_TYPE_F16 || t == CKX_TYPE_BF16; }
bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }
int size_of(int t) { return t == CKX_TYPE_F32 ? 4 : 2; }

constexpr int kMostK    = 131071;  // 128 * 128 * K stays under 2^31
constexpr int kMostRows = 1 << 24; // of the experts' product

struct Span
{
    const void* p;
    int64_t bytes;
    bool meets(const Span& o) const
    {
        const auto a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(o.p);
        return p && o.p && bytes > 0 && o.bytes > 0 && a < b + (uintptr_t)o.bytes && b < a + (uintptr_t)bytes;
    }
};

// what the two products share
int check_product(int32_t N, int32_t K, int32_t ldb, int gated, int c_type)
{
    if(N < 0 || K < 0)
        return api_fail(CKX_INVALID_VALUE, "negative size");
    if(!float_type(c_type))
        return api_fail(CKX_INVALID_VALUE, "C is fp32, fp16 or bf16");
    if(gated != 0 && gated != 1)
        return api_fail(CKX_INVALID_VALUE, "gated is 0 or 1");
    if(K > kMostK)
        return api_fail(CKX_UNSUPPORTED, "K is at most 131071: the sums are 32-bit");
    if(gated && N > 0x3fffffff)
        return api_fail(CKX_UNSUPPORTED, "more than 2^31 - 1 rows of B");
    if((N > 1 || (gated && N > 0)) && ldb < K)
        return api_fail(CKX_UNSUPPORTED, "leading dimension smaller than the row");
    if(ldb < 0)
        return api_fail(CKX_UNSUPPORTED, "negative stride");
    return CKX_OK;
}

ckx::GemmI8Args product_of(const ckx_experts_desc& d)
{
    ckx::GemmI8Args a{};
    a.experts = d.num_experts, a.rows_a = d.num_rows_a, a.rows_per = d.rows_per, a.batch_b = d.batch_stride_b;
    a.M = d.num_rows, a.N = d.N, a.K = d.K, a.lda = d.stride_a, a.ldb = d.stride_b, a.ldc = d.stride_c, a.gated = d.gated;
    return a;
}

// what the queries answer; `name` of the kernel: empty where there is nothing to do
int plan_of_product(int32_t M, int32_t N, int32_t K, int32_t lda, int32_t ldb, int32_t ldc, int gated, int c_type, int64_t workspace_bytes, int* tile_m,
                    int* tile_n, int* k_runs, const char*& name)
{
    if(!tile_m || !tile_n || !k_runs)
        return api_fail(CKX_INVALID_VALUE, "null result pointer");
    int st = ckx_gemm_i8_tokenscale_is_supported(M, N, K, lda, ldb, ldc, gated, c_type);
    if(st != CKX_OK)
        return st;
    if(workspace_bytes < 0)
        return api_fail(CKX_INVALID_VALUE, "negative size");
    *tile_m = *tile_n = *k_runs = 0, name = "";
    ckx::GemmI8Args a{};
    a.rows_a = M, a.rows_per = 1, a.M = M, a.N = N, a.K = K, a.lda = lda, a.ldb = ldb, a.ldc = ldc, a.gated = gated;
    if(M > 0 && N > 0)
        name = ckx::gemm_i8_scaled_plan(a, workspace_bytes, tile_m, tile_n, k_runs);
    return CKX_OK;
}

int plan_of_experts(const ckx_experts_desc* d, int gathered, int* tile_m, int* tile_n, int* k_runs, const char*& name)
{
    if(!tile_m || !tile_n || !k_runs)
        return api_fail(CKX_INVALID_VALUE, "null result pointer");
    int st = ckx_experts_gemm_i8_is_supported(d);
    if(st != CKX_OK)
        return st;
    if(gathered != 0 && gathered != 1)
        return api_fail(CKX_INVALID_VALUE, "gathered is 0 or 1");
    *tile_m = *tile_n = *k_runs = 0, name = "";
    ckx::GemmI8Args a = product_of(*d);
    const int32_t none = 0; // (says that there are tables; the plan reads none)
    a.offsets = &none, a.rows = gathered ? &none : nullptr;
    if(d->num_rows > 0 && d->num_experts > 0 && d->N > 0)
        name = ckx::gemm_i8_scaled_plan(a, 0, tile_m, tile_n, k_runs);
    return CKX_OK;
}

} // namespace

extern "C" {

int ckx_route_experts_is_supported(const ckx_route_desc* d)
{
    if(!d)
        return api_fail(CKX_INVALID_VALUE, "null description");
    if(d->num_tokens < 0 || d->num_experts < 0 || d->top_k < 0 || d->num_groups < 0 || d->top_groups < 0)
        return api_fail(CKX_INVALID_VALUE, "negative size");
    if(!float_type(d->x_type))
        return api_fail(CKX_INVALID_VALUE, "logits are fp32, fp16 or bf16");
    if((d->scoring != CKX_SCORE_SOFTMAX && d->scoring != CKX_SCORE_SIGMOID) || (d->renormalise != 0 && d->renormalise != 1))
        return api_fail(CKX_INVALID_VALUE, "scoring is CKX_SCORE_SOFTMAX or _SIGMOID, renormalise 0 or 1");
    if(!std::isfinite(d->scale))
        return api_fail(CKX_INVALID_VALUE, "the scale of the weights must be finite");
    if(d->num_experts < 1 || d->num_experts > ckx::kMostExperts)
        return api_fail(CKX_UNSUPPORTED, "1 to 1024 experts");
    if(d->top_k < 1 || d->top_k > ckx::kMostTopK || d->top_k > d->num_experts)
        return api_fail(CKX_UNSUPPORTED, "top_k is 1 to 32, and at most the number of experts");
    if(d->num_groups < 1 || d->num_groups > ckx::kMostGroups || d->num_experts % d->num_groups)
        return api_fail(CKX_UNSUPPORTED, "1 to 64 groups, of as many experts each");
    if(d->top_groups < 1 || d->top_groups > d->num_groups)
        return api_fail(CKX_UNSUPPORTED, "top_groups is 1 to num_groups");
    if(d->group_best != 1 && d->group_best != 2)
        return api_fail(CKX_INVALID_VALUE, "group_best is 1 or 2");
    if((int64_t)d->num_tokens * d->top_k > kMostRows)
        return api_fail(CKX_UNSUPPORTED, "at most 2^24 pairs of token and expert");
    if(d->stride_x < 0 || (d->num_tokens > 1 && d->stride_x < d->num_experts))
        return api_fail(CKX_UNSUPPORTED, "rows of logits overlap");
    return CKX_OK;
}

int64_t ckx_route_experts_workspace_bytes(const ckx_route_desc* d)
{
    return d && ckx_route_experts_is_supported(d) == CKX_OK ? ckx::route_workspace(d->num_tokens, d->num_experts) : 0;
}

int ckx_route_experts(const void* p_logits, const float* p_bias, const int32_t* p_num_tokens, int32_t* p_ids, float* p_weights,
                      int32_t* p_offsets, int32_t* p_rows, int32_t* p_places, const ckx_route_desc* d, void* p_workspace,
                      int64_t workspace_bytes, void* stream)
{
    int st = ckx_route_experts_is_supported(d);
    if(st != CKX_OK)
        return st;
    const bool tables = p_offsets || p_rows || p_places;
    if(tables && (!p_offsets || (d->num_tokens > 0 && (!p_rows || !p_places))))
        return api_fail(CKX_INVALID_VALUE, "the tables are three: offsets, rows, places (or none)");
    if(d->num_tokens == 0 && !tables)
        return CKX_OK;
    if(d->num_tokens > 0 && (!p_logits || !p_ids || !p_weights))
        return api_fail(CKX_INVALID_VALUE, "null operand pointer");
    if(!aligned(p_logits, size_of(d->x_type)))
        return api_fail(CKX_UNSUPPORTED, "operands must be aligned to their element size");
    for(const void* p : {(const void*)p_bias, (const void*)p_num_tokens, (const void*)p_ids, (const void*)p_weights, (const void*)p_offsets,
                         (const void*)p_rows, (const void*)p_places})
        if(!aligned(p, 4))
            return api_fail(CKX_UNSUPPORTED, "operands must be aligned to their element size");
    // other workgroups still read the logits, the biases and the ids while the first already write
    const int64_t pairs = 4ll * d->num_tokens * d->top_k, rows = d->num_tokens > 0 ? d->num_tokens - 1 : 0;
    const Span in[]  = {{p_logits, d->num_tokens > 0 ? (rows * d->stride_x + d->num_experts) * size_of(d->x_type) : 0},
                        {p_bias, 4ll * d->num_experts},
                        {p_num_tokens, 4}},
               out[] = {{p_ids, pairs}, {p_weights, pairs}, {p_offsets, 4ll * d->num_experts + 4}, {p_rows, pairs}, {p_places, pairs}};
    for(const Span& o : out)
    {
        for(const Span& i : in)
            if(o.meets(i))
                return api_fail(CKX_INVALID_VALUE, "an output lies on an input");
        for(const Span& x : out)
            if(&x != &o && o.meets(x))
                return api_fail(CKX_INVALID_VALUE, "two outputs overlap");
    }
    const int64_t need = tables ? ckx::route_workspace(d->num_tokens, d->num_experts) : 0;
    if(need > 0 && (!p_workspace || workspace_bytes < need))
        return api_fail(CKX_UNSUPPORTED, "the workspace is smaller than ckx_route_experts_workspace_bytes");
    if(need > 0 && !aligned(p_workspace, 16))
        return api_fail(CKX_INVALID_VALUE, "the workspace must be 16-byte aligned");
    // (the second launch takes its counts as places, and the ids as numbers of experts)
    const Span ws{p_workspace, need};
    for(const Span& x : in)
        if(ws.meets(x))
            return api_fail(CKX_INVALID_VALUE, "the workspace lies on an input");
    for(const Span& x : out)
        if(ws.meets(x))
            return api_fail(CKX_INVALID_VALUE, "the workspace lies on an output");
    ckx::RouteArgs a{};
    a.x = p_logits, a.bias = p_bias, a.live = p_num_tokens, a.ids = p_ids, a.weights = p_weights;
    a.offsets = p_offsets, a.rows = p_rows, a.places = p_places, a.ws = p_workspace;
    a.tokens = d->num_tokens, a.experts = d->num_experts, a.top_k = d->top_k, a.groups = d->num_groups;
    a.top_groups = d->top_groups, a.group_best = d->group_best, a.stride_x = d->stride_x;
    a.sigmoid = d->scoring == CKX_SCORE_SIGMOID, a.renormalise = d->renormalise, a.scale = d->scale;
    if(a.groups == a.top_groups) // (nothing is left out)
        a.groups = a.top_groups = 1;
    hipError_t e = ckx::route_launch(a, d->x_type, (hipStream_t)stream);
    return e == hipSuccess ? CKX_OK : ckx::api_hip_fail(e, "route_experts");
}

int ckx_quantize_tokens_i8_is_supported(int32_t M, int32_t K, int32_t stride_x, int32_t stride_q, int x_type)
{
    if(M < 0 || K < 0)
        return api_fail(CKX_INVALID_VALUE, "negative size");
    if(!float_type(x_type))
        return api_fail(CKX_INVALID_VALUE, "x is fp32, fp16 or bf16");
    if(stride_x < 0 || stride_q < 0 || (M > 1 && (stride_x < K || stride_q < K)))
        return api_fail(CKX_UNSUPPORTED, "row strides are at least K");
    return CKX_OK;
}

int ckx_quantize_tokens_i8(const void* p_x, void* p_q, float* p_scale, int32_t M, int32_t K, int32_t stride_x, int32_t stride_q, int x_type,
                           void* stream)
{
    int st = ckx_quantize_tokens_i8_is_supported(M, K, stride_x, stride_q, x_type);
    if(st != CKX_OK)
        return st;
    if(M == 0)
        return CKX_OK;
    if((K > 0 && (!p_x || !p_q)) || !p_scale)
        return api_fail(CKX_INVALID_VALUE, "null operand pointer");
    if(!aligned(p_x, size_of(x_type)) || !aligned(p_scale, 4))
        return api_fail(CKX_UNSUPPORTED, "operands must be aligned to their element size");
    const ckx::TokenQuantArgs a{p_x, static_cast<int8_t*>(p_q), p_scale, M, K, stride_x, stride_q};
    hipError_t e = ckx::quantize_tokens_launch(a, x_type, (hipStream_t)stream);
    return e == hipSuccess ? CKX_OK : ckx::api_hip_fail(e, "quantize_tokens_i8");
}

int ckx_gemm_i8_tokenscale_is_supported(int32_t M, int32_t N, int32_t K, int32_t lda, int32_t ldb, int32_t ldc, int gated, int c_type)
{
    if(M < 0)
        return api_fail(CKX_INVALID_VALUE, "negative size");
    int st = check_product(N, K, ldb, gated, c_type);
    if(st != CKX_OK)
        return st;
    if(M > 1 && (lda < K || ldc < N))
        return api_fail(CKX_UNSUPPORTED, "leading dimension smaller than the row");
    if(lda < 0 || ldc < 0)
        return api_fail(CKX_UNSUPPORTED, "negative stride");
    if(!ckx::gemm_i8_scaled_fits(M, N, gated, 0))
        return api_fail(CKX_UNSUPPORTED, "more output tiles than one launch takes");
    return CKX_OK;
}

int64_t ckx_gemm_i8_tokenscale_workspace_bytes(int32_t M, int32_t N, int32_t K, int gated)
{
    return M > 0 && N > 0 && K > 0 && (gated == 0 || gated == 1) ? ckx::gemm_i8_scaled_workspace(M, N, K, gated) : 0;
}

int ckx_gemm_i8_tokenscale(const void* p_a, const void* p_b, void* p_c, const float* p_scale_a, const float* p_scale_b, const float* p_bias,
                           int32_t M, int32_t N, int32_t K, int32_t lda, int32_t ldb, int32_t ldc, int gated, int c_type, void* p_workspace,
                           int64_t workspace_bytes, void* stream)
{
    int st = ckx_gemm_i8_tokenscale_is_supported(M, N, K, lda, ldb, ldc, gated, c_type);
    if(st != CKX_OK)
        return st;
    if(M == 0 || N == 0)
        return CKX_OK;
    if(!p_c || !p_scale_a || !p_scale_b || (K > 0 && (!p_a || !p_b)))
        return api_fail(CKX_INVALID_VALUE, "null operand pointer");
    if(!aligned(p_c, size_of(c_type)) || !aligned(p_scale_a, 4) || !aligned(p_scale_b, 4) || !aligned(p_bias, 4))
        return api_fail(CKX_UNSUPPORTED, "operands must be aligned to their element size");
    if(workspace_bytes < 0 || !aligned(p_workspace, 16))
        return api_fail(CKX_INVALID_VALUE, "the workspace must be 16-byte aligned");
    ckx::GemmI8Args a{};
    a.a = static_cast<const int8_t*>(p_a), a.b = static_cast<const int8_t*>(p_b), a.c = p_c;
    a.sa = p_scale_a, a.sb = p_scale_b, a.bias = p_bias, a.rows_a = M, a.rows_per = 1;
    a.M = M, a.N = N, a.K = K, a.lda = lda, a.ldb = ldb, a.ldc = ldc, a.gated = gated, a.ws = static_cast<int*>(p_workspace);
    hipError_t e = ckx::gemm_i8_scaled_launch(a, c_type, p_workspace ? workspace_bytes : 0, (hipStream_t)stream);
    return e == hipSuccess ? CKX_OK : ckx::api_hip_fail(e, "gemm_i8_tokenscale");
}

int ckx_gemm_i8_tokenscale_plan(int32_t M, int32_t N, int32_t K, int32_t lda, int32_t ldb, int32_t ldc, int gated, int c_type,
                                int64_t workspace_bytes, int* tile_m, int* tile_n, int* k_runs)
{
    const char* name = nullptr;
    return plan_of_product(M, N, K, lda, ldb, ldc, gated, c_type, workspace_bytes, tile_m, tile_n, k_runs, name);
}

const char* ckx_gemm_i8_tokenscale_kernel_name(int32_t M, int32_t N, int32_t K, int32_t lda, int32_t ldb, int32_t ldc, int gated, int c_type,
                                               int64_t workspace_bytes)
{
    int m, n, runs;
    const char* name = nullptr;
    return plan_of_product(M, N, K, lda, ldb, ldc, gated, c_type, workspace_bytes, &m, &n, &runs, name) == CKX_OK ? name : nullptr;
}

int ckx_experts_gemm_i8_is_supported(const ckx_experts_desc* d)
{
    if(!d)
        return api_fail(CKX_INVALID_VALUE, "null description");
    if(d->num_rows < 0 || d->num_rows_a < 0 || d->num_experts < 0)
        return api_fail(CKX_INVALID_VALUE, "negative size");
    int st = check_product(d->N, d->K, d->stride_b, d->gated, d->c_type);
    if(st != CKX_OK)
        return st;
    if(d->rows_per < 1)
        return api_fail(CKX_INVALID_VALUE, "rows_per is at least 1");
    if(d->num_experts > ckx::kMostExperts || d->num_rows > kMostRows)
        return api_fail(CKX_UNSUPPORTED, "at most 1024 experts and 2^24 rows");
    if((d->num_rows_a > 1 && d->stride_a < d->K) || (d->num_rows > 1 && d->stride_c < d->N))
        return api_fail(CKX_UNSUPPORTED, "leading dimension smaller than the row");
    if(d->stride_a < 0 || d->stride_c < 0 || d->batch_stride_b < 0)
        return api_fail(CKX_UNSUPPORTED, "negative stride");
    if(!ckx::gemm_i8_scaled_fits(d->num_rows, d->N, d->gated, d->num_experts))
        return api_fail(CKX_UNSUPPORTED, "more output tiles than one launch takes");
    return CKX_OK;
}

int ckx_experts_gemm_i8(const void* p_a, const void* p_b, void* p_c, const float* p_scale_a, const float* p_scale_b, const float* p_bias,
                        const int32_t* p_offsets, const int32_t* p_rows, const ckx_experts_desc* d, void* stream)
{
    int st = ckx_experts_gemm_i8_is_supported(d);
    if(st != CKX_OK)
        return st;
    if(d->num_rows == 0 || d->num_experts == 0 || d->N == 0)
        return CKX_OK;
    if(!p_c || !p_offsets || !p_scale_b || (d->num_rows_a > 0 && !p_scale_a) || (d->K > 0 && (!p_b || (d->num_rows_a > 0 && !p_a))))
        return api_fail(CKX_INVALID_VALUE, "null operand pointer");
    if(!aligned(p_c, size_of(d->c_type)) || !aligned(p_scale_a, 4) || !aligned(p_scale_b, 4) || !aligned(p_bias, 4) || !aligned(p_offsets, 4) ||
       !aligned(p_rows, 4))
        return api_fail(CKX_UNSUPPORTED, "operands must be aligned to their element size");
    ckx::GemmI8Args a = product_of(*d);
    a.a = static_cast<const int8_t*>(p_a), a.b = static_cast<const int8_t*>(p_b), a.c = p_c;
    a.sa = p_scale_a, a.sb = p_scale_b, a.bias = p_bias, a.offsets = p_offsets, a.rows = p_rows;
    hipError_t e = ckx::gemm_i8_scaled_launch(a, d->c_type, 0, (hipStream_t)stream);
    return e == hipSuccess ? CKX_OK : ckx::api_hip_fail(e, "experts_gemm_i8");
}

int ckx_experts_gemm_i8_plan(const ckx_experts_desc* d, int gathered, int* tile_m, int* tile_n, int* k_runs)
{
    const char* name = nullptr;
    return plan_of_experts(d, gathered, tile_m, tile_n, k_runs, name);
}

const char* ckx_experts_gemm_i8_kernel_name(const ckx_experts_desc* d, int gathered)
{
    int m, n, runs;
    const char* name = nullptr;
    return plan_of_experts(d, gathered, &m, &n, &runs, name) == CKX_OK ? name : nullptr;
}

int ckx_experts_combine_is_supported(int32_t num_tokens, int32_t top_k, int32_t num_rows, int32_t N, int32_t stride_y, int32_t stride_add,
                                     int32_t stride_out, int type)
{
    if(num_tokens < 0 || top_k < 0 || num_rows < 0 || N < 0)
        return api_fail(CKX_INVALID_VALUE, "negative size");
    if(!float_type(type))
        return api_fail(CKX_INVALID_VALUE, "rows are fp32, fp16 or bf16");
    if(stride_y < 0 || stride_add < 0 || stride_out < 0 || (num_rows > 1 && stride_y < N) || (num_tokens > 1 && stride_out < N))
        return api_fail(CKX_UNSUPPORTED, "leading dimension smaller than the row");
    if((int64_t)num_tokens * top_k > kMostRows)
        return api_fail(CKX_UNSUPPORTED, "at most 2^24 pairs of token and expert");
    return CKX_OK;
}

int ckx_experts_combine(const void* p_y, const int32_t* p_places, const float* p_weights, const void* p_add, void* p_out, int32_t num_tokens,
                        int32_t top_k, int32_t num_rows, int32_t N, int32_t stride_y, int32_t stride_add, int32_t stride_out, int type,
                        void* stream)
{
    int st = ckx_experts_combine_is_supported(num_tokens, top_k, num_rows, N, stride_y, stride_add, stride_out, type);
    if(st != CKX_OK)
        return st;
    if(num_tokens == 0 || N == 0)
        return CKX_OK;
    if(!p_out || (top_k > 0 && (!p_places || !p_weights || (num_rows > 0 && !p_y))))
        return api_fail(CKX_INVALID_VALUE, "null operand pointer");
    if(!aligned(p_y, size_of(type)) || !aligned(p_add, size_of(type)) || !aligned(p_out, size_of(type)) || !aligned(p_places, 4) ||
       !aligned(p_weights, 4))
        return api_fail(CKX_UNSUPPORTED, "operands must be aligned to their element size");
    if(p_add && p_add == p_out && num_tokens > 1 && stride_add != stride_out)
        return api_fail(CKX_INVALID_VALUE, "add is out, with another stride");
    const ckx::CombineArgs a{p_y, p_places, p_weights, p_add, p_out, num_tokens, top_k, num_rows, N, stride_y, stride_add, stride_out};
    hipError_t e = ckx::combine_launch(a, type, (hipStream_t)stream);
    return e == hipSuccess ? CKX_OK : ckx::api_hip_fail(e, "experts_combine");
}

} // extern "C"
