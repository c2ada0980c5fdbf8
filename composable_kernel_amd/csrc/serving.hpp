// Launchers of the 8-bit serving kernels (block quantiser, block-scaled GEMM, cache tables, cache store, paged attention),
// called by the C ABI once it has checked the arguments.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ckx.h"

namespace ckx {

struct QuantArgs
{
    const void* x;
    uint8_t* q;
    float* scale;
    int M, K, sx, sq, ss_m, ss_g;
};
hipError_t quantize_blocks_launch(const QuantArgs& a, int x_type, hipStream_t s);

struct GemmF8Args
{
    const uint8_t *a, *b;
    void* c;
    const float *sa, *sb;
    int M, N, K, lda, ldb, ldc;
    int sa_m, sa_g, sb_n, sb_g;
    int tiles_m, tiles_n;
    int groups, ksplit, per; // groups of 128 along K; runs they are cut into, groups a run
    float* ws;               // ksplit > 1: [ksplit][M][N] sums
};
bool gemm_f8_fits(int M, int N);
int64_t gemm_f8_workspace(int M, int N, int K);
void gemm_f8_plan(int M, int N, int K, int lda, int ldb, int c_type, int64_t workspace_bytes, int* tile_m, int* tile_n, int* k_runs);
hipError_t gemm_f8_launch(GemmF8Args a, int c_type, int64_t workspace_bytes, hipStream_t s);

struct TablesArgs
{
    const int *context, *fresh, *free;
    int *table, *cu, *kv_lens, *slots, *used;
    int batch, num_free, max_blocks, stride_table, num_slots, block_shift;
};
constexpr int kMaxTableSequences = 8192;
hipError_t kv_tables_launch(const TablesArgs& a, hipStream_t s);

struct StoreArgs
{
    const void *k, *v;
    const int* slots;
    ckx_kv_cache8 cache;
    int tokens, block_shift;
    int sk_t, sk_h, sv_t, sv_h;
};
hipError_t kv_store_launch(const StoreArgs& a, int x_type, hipStream_t s);

struct AttentionArgs
{
    const void* q;
    void* o;
    const int *table, *cu_q, *kv_lens;
    ckx_kv_cache8 cache;
    int batch, tokens, heads, group; // query heads; query heads per cache head
    int max_kv, max_blocks, stride_table, block_shift;
    int sq_t, sq_h, so_t, so_h;
    float scale; // of the scores, times log2(e)
    int causal;
    // a tile: `tile_tokens` query tokens of one sequence times `tile_heads` heads of one group; head_tiles tiles per group
    int tile_tokens, tile_heads, head_tiles, tiles;
    int splits; // shares of the cached tokens
    float* ws;
};
int64_t attention_workspace(const ckx_kv_cache8& c, int batch, int tokens, int heads, int max_kv, int max_blocks);
bool attention_fits(const ckx_kv_cache8& c, int batch, int tokens, int heads, int max_kv, int max_blocks);
hipError_t attention_launch(AttentionArgs a, int q_type, hipStream_t s);

} // namespace ckx
