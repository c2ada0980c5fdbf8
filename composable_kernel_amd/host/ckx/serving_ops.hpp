// C++ operators of the 8-bit serving path (include/ckx.h): block quantiser, block-scaled GEMM, cache tables, cache store and paged
// attention. Same conduct as the operators of device_ops.hpp: MakeArgument / MakeArgumentPointer, IsSupportedArgument,
// MakeInvoker()->Run. Types as template parameters: float, half_t, bhalf_t; codes are f8_t (e4m3) or int8_t.
#pragma once

#include "ckx/device_ops.hpp"

namespace ck {

struct f8_t // e4m3, as stored
{
    uint8_t bits;
};

namespace tensor_operation {
namespace device {

namespace detail {

template <typename T>
constexpr int ckx_type()
{
    if constexpr(std::is_same_v<T, float>)
        return CKX_TYPE_F32;
    else if constexpr(std::is_same_v<T, half_t>)
        return CKX_TYPE_F16;
    else if constexpr(std::is_same_v<T, bhalf_t>)
        return CKX_TYPE_BF16;
    else if constexpr(std::is_same_v<T, f8_t>)
        return CKX_TYPE_E4M3;
    else
    {
        static_assert(std::is_same_v<T, int8_t>, "type not built");
        return CKX_TYPE_I8;
    }
}

// what the operators below share: no instance list, the library chooses the kernel
template <typename Argument_, int (*Supported)(const Argument_&, int), int (*Launch)(const Argument_&, int, void*)>
struct ServingOperator : public BaseOperator
{
    using Argument = Argument_;
    using Invoker  = InvokerT<Argument, Supported, Launch>;
    Invoker MakeInvoker() const { return Invoker{CKX_INSTANCE_AUTO}; }
    bool IsSupportedArgument(const Argument& a) const { return Supported(a, CKX_INSTANCE_AUTO) == CKX_OK; }
    bool IsSupportedArgument(const BaseArgument* p) override
    {
        const auto* a = dynamic_cast<const Argument*>(p);
        return a && IsSupportedArgument(*a);
    }
    std::unique_ptr<BaseInvoker> MakeInvokerPointer() { return std::make_unique<Invoker>(CKX_INSTANCE_AUTO); }
};

struct BlockQuantizeF8Argument : public BaseArgument
{
    const void* p_x;
    void* p_q;
    float* p_scale;
    index_t M, K, StrideX, StrideQ, StrideScaleM, StrideScaleG;
    int type;
    static int Supported(const BlockQuantizeF8Argument& a, int)
    {
        return ckx_quantize_blocks_f8_is_supported(a.M, a.K, a.StrideX, a.StrideQ, a.StrideScaleM, a.StrideScaleG, a.type);
    }
    static int Launch(const BlockQuantizeF8Argument& a, int, void* stream)
    {
        return ckx_quantize_blocks_f8(a.p_x, a.p_q, a.p_scale, a.M, a.K, a.StrideX, a.StrideQ, a.StrideScaleM, a.StrideScaleG, a.type,
                                      stream);
    }
};

struct GemmBlockScaleF8Argument : public BaseArgument
{
    const void *p_a, *p_b;
    void* p_c;
    const float *p_scale_a, *p_scale_b;
    index_t M, N, K, StrideA, StrideB, StrideC, StrideScaleAM, StrideScaleAG, StrideScaleBN, StrideScaleBG;
    int type;
    static int Supported(const GemmBlockScaleF8Argument& a, int)
    {
        return ckx_gemm_f8_blockscale_is_supported(a.M, a.N, a.K, a.StrideA, a.StrideB, a.StrideC, a.StrideScaleAM, a.StrideScaleAG,
                                                   a.StrideScaleBN, a.StrideScaleBG, a.type);
    }
    static int Launch(const GemmBlockScaleF8Argument& a, int, void* stream)
    {
        return ckx_gemm_f8_blockscale(a.p_a, a.p_b, a.p_c, a.p_scale_a, a.p_scale_b, a.M, a.N, a.K, a.StrideA, a.StrideB, a.StrideC,
                                      a.StrideScaleAM, a.StrideScaleAG, a.StrideScaleBN, a.StrideScaleBG, a.type, a.p_workspace_,
                                      a.p_workspace_ ? ckx_gemm_f8_blockscale_workspace_bytes(a.M, a.N, a.K) : 0, stream);
    }
};

struct KvCacheTablesArgument : public BaseArgument
{
    const index_t *p_context_lens, *p_new_lens, *p_free_blocks;
    index_t *p_block_table, *p_cu_new, *p_kv_lens, *p_slots, *p_used;
    index_t Batch, NumFree, MaxBlocks, StrideTable, NumSlots, BlockSize;
    static int Supported(const KvCacheTablesArgument& a, int)
    {
        return ckx_kv_cache_tables_is_supported(a.Batch, a.NumFree, a.MaxBlocks, a.StrideTable, a.NumSlots, a.BlockSize);
    }
    static int Launch(const KvCacheTablesArgument& a, int, void* stream)
    {
        return ckx_kv_cache_tables(a.p_context_lens, a.p_new_lens, a.p_free_blocks, a.p_block_table, a.p_cu_new, a.p_kv_lens, a.p_slots,
                                   a.p_used, a.Batch, a.NumFree, a.MaxBlocks, a.StrideTable, a.NumSlots, a.BlockSize, stream);
    }
};

struct KvCacheStore8Argument : public BaseArgument
{
    const void *p_k, *p_v;
    const index_t* p_slots;
    ckx_kv_cache8 cache;
    index_t NumTokens, StrideKToken, StrideKHead, StrideVToken, StrideVHead;
    int type;
    static int Supported(const KvCacheStore8Argument& a, int)
    {
        return ckx_kv_cache_store8_is_supported(&a.cache, a.NumTokens, a.StrideKToken, a.StrideKHead, a.StrideVToken, a.StrideVHead,
                                                a.type);
    }
    static int Launch(const KvCacheStore8Argument& a, int, void* stream)
    {
        return ckx_kv_cache_store8(a.p_k, a.p_v, a.p_slots, &a.cache, a.NumTokens, a.StrideKToken, a.StrideKHead, a.StrideVToken,
                                   a.StrideVHead, a.type, stream);
    }
};

struct PagedAttention8Argument : public BaseArgument
{
    const void* p_q;
    void* p_o;
    const index_t *p_block_table, *p_cu_q, *p_kv_lens;
    ckx_kv_cache8 cache;
    index_t Batch, NumTokens, NumHeads, MaxKvLen, MaxBlocks, StrideTable, StrideQToken, StrideQHead, StrideOToken, StrideOHead;
    float scale;
    int causal, type;
    int64_t WorkSpaceSize() const
    {
        return ckx_paged_attention8_workspace_bytes(&cache, Batch, NumTokens, NumHeads, MaxKvLen, MaxBlocks);
    }
    static int Supported(const PagedAttention8Argument& a, int)
    {
        return ckx_paged_attention8_is_supported(&a.cache, a.Batch, a.NumTokens, a.NumHeads, a.MaxKvLen, a.MaxBlocks, a.StrideTable,
                                                 a.StrideQToken, a.StrideQHead, a.StrideOToken, a.StrideOHead, a.scale, a.causal, a.type);
    }
    static int Launch(const PagedAttention8Argument& a, int, void* stream)
    {
        return ckx_paged_attention8(a.p_q, a.p_o, a.p_block_table, a.p_cu_q, a.p_kv_lens, &a.cache, a.Batch, a.NumTokens, a.NumHeads,
                                    a.MaxKvLen, a.MaxBlocks, a.StrideTable, a.StrideQToken, a.StrideQHead, a.StrideOToken, a.StrideOHead,
                                    a.scale, a.causal, a.type, a.p_workspace_, a.p_workspace_ ? a.WorkSpaceSize() : 0, stream);
    }
};

template <typename Argument>
using ServingOperatorOf = ServingOperator<Argument, &Argument::Supported, &Argument::Launch>;

} // namespace detail

// x [M, K] -> e4m3 codes and one fp32 scale per row and group of 128 columns
template <typename XDataType>
struct DeviceBlockQuantizeF8 : public detail::ServingOperatorOf<detail::BlockQuantizeF8Argument>
{
    static Argument MakeArgument(const XDataType* p_x, f8_t* p_q, float* p_scale, index_t M, index_t K, index_t StrideX, index_t StrideQ,
                                 index_t StrideScaleM, index_t StrideScaleG)
    {
        Argument a;
        a.p_x = p_x, a.p_q = p_q, a.p_scale = p_scale, a.M = M, a.K = K, a.StrideX = StrideX, a.StrideQ = StrideQ;
        a.StrideScaleM = StrideScaleM, a.StrideScaleG = StrideScaleG, a.type = detail::ckx_type<XDataType>();
        return a;
    }
    std::string GetTypeString() const override { return "DeviceBlockQuantizeF8<auto>"; }
};

// C [M, N] = sum over groups of 128 columns of scale_a * scale_b * (A B^T): A [M, K], B [N, K] e4m3
template <typename CDataType>
struct DeviceGemmBlockScaleF8 : public detail::ServingOperatorOf<detail::GemmBlockScaleF8Argument>
{
    static Argument MakeArgument(const f8_t* p_a, const f8_t* p_b, CDataType* p_c, const float* p_scale_a, const float* p_scale_b,
                                 index_t M, index_t N, index_t K, index_t StrideA, index_t StrideB, index_t StrideC,
                                 index_t StrideScaleAM, index_t StrideScaleAG, index_t StrideScaleBN, index_t StrideScaleBG)
    {
        Argument a;
        a.p_a = p_a, a.p_b = p_b, a.p_c = p_c, a.p_scale_a = p_scale_a, a.p_scale_b = p_scale_b, a.M = M, a.N = N, a.K = K;
        a.StrideA = StrideA, a.StrideB = StrideB, a.StrideC = StrideC, a.StrideScaleAM = StrideScaleAM, a.StrideScaleAG = StrideScaleAG;
        a.StrideScaleBN = StrideScaleBN, a.StrideScaleBG = StrideScaleBG, a.type = detail::ckx_type<CDataType>();
        return a;
    }
    size_t GetWorkSpaceSize(const BaseArgument* p) const override
    {
        const auto* a = dynamic_cast<const Argument*>(p);
        return a ? (size_t)ckx_gemm_f8_blockscale_workspace_bytes(a->M, a->N, a->K) : 0;
    }
    std::string GetTypeString() const override { return "DeviceGemmBlockScaleF8<auto>"; }
};

// block tables, slots and lengths of a step from the requests' lengths
struct DeviceKvCacheTables : public detail::ServingOperatorOf<detail::KvCacheTablesArgument>
{
    static Argument MakeArgument(const index_t* p_context_lens, const index_t* p_new_lens, const index_t* p_free_blocks,
                                 index_t* p_block_table, index_t* p_cu_new, index_t* p_kv_lens, index_t* p_slots, index_t* p_used,
                                 index_t Batch, index_t NumFree, index_t MaxBlocks, index_t StrideTable, index_t NumSlots,
                                 index_t BlockSize)
    {
        Argument a;
        a.p_context_lens = p_context_lens, a.p_new_lens = p_new_lens, a.p_free_blocks = p_free_blocks, a.p_block_table = p_block_table;
        a.p_cu_new = p_cu_new, a.p_kv_lens = p_kv_lens, a.p_slots = p_slots, a.p_used = p_used, a.Batch = Batch, a.NumFree = NumFree;
        a.MaxBlocks = MaxBlocks, a.StrideTable = StrideTable, a.NumSlots = NumSlots, a.BlockSize = BlockSize;
        return a;
    }
    std::string GetTypeString() const override { return "DeviceKvCacheTables<auto>"; }
};

// new keys and values into the cache
template <typename XDataType>
struct DeviceKvCacheStore8 : public detail::ServingOperatorOf<detail::KvCacheStore8Argument>
{
    static Argument MakeArgument(const XDataType* p_k, const XDataType* p_v, const index_t* p_slots, const ckx_kv_cache8& cache,
                                 index_t NumTokens, index_t StrideKToken, index_t StrideKHead, index_t StrideVToken, index_t StrideVHead)
    {
        Argument a;
        a.p_k = p_k, a.p_v = p_v, a.p_slots = p_slots, a.cache = cache, a.NumTokens = NumTokens, a.StrideKToken = StrideKToken;
        a.StrideKHead = StrideKHead, a.StrideVToken = StrideVToken, a.StrideVHead = StrideVHead, a.type = detail::ckx_type<XDataType>();
        return a;
    }
    std::string GetTypeString() const override { return "DeviceKvCacheStore8<auto>"; }
};

// attention of query tokens over the cache
template <typename QDataType, bool Causal = true>
struct DevicePagedAttention8 : public detail::ServingOperatorOf<detail::PagedAttention8Argument>
{
    static Argument MakeArgument(const QDataType* p_q, QDataType* p_o, const index_t* p_block_table, const index_t* p_cu_q,
                                 const index_t* p_kv_lens, const ckx_kv_cache8& cache, index_t Batch, index_t NumTokens, index_t NumHeads,
                                 index_t MaxKvLen, index_t MaxBlocks, index_t StrideTable, index_t StrideQToken, index_t StrideQHead,
                                 index_t StrideOToken, index_t StrideOHead, element_wise::Scale score_element_op)
    {
        Argument a;
        a.p_q = p_q, a.p_o = p_o, a.p_block_table = p_block_table, a.p_cu_q = p_cu_q, a.p_kv_lens = p_kv_lens, a.cache = cache;
        a.Batch = Batch, a.NumTokens = NumTokens, a.NumHeads = NumHeads, a.MaxKvLen = MaxKvLen, a.MaxBlocks = MaxBlocks;
        a.StrideTable = StrideTable, a.StrideQToken = StrideQToken, a.StrideQHead = StrideQHead, a.StrideOToken = StrideOToken;
        a.StrideOHead = StrideOHead, a.scale = score_element_op.scale_, a.causal = Causal ? 1 : 0;
        a.type = detail::ckx_type<QDataType>();
        return a;
    }
    size_t GetWorkSpaceSize(const BaseArgument* p) const override
    {
        const auto* a = dynamic_cast<const Argument*>(p);
        return a ? (size_t)a->WorkSpaceSize() : 0;
    }
    std::string GetTypeString() const override { return "DevicePagedAttention8<auto>"; }
};

} // namespace device
} // namespace tensor_operation
} // namespace ck
