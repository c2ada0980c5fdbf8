// Launchers of the int8 linear and mixture-of-experts kernels (router, token quantiser, token-scaled GEMM, the experts' GEMM and the
// weighted sum of their rows), called by the C ABI once it has checked the arguments.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ckx.h"

namespace ckx {

struct RouteArgs
{
    const void* x;
    const float* bias;
    const int* live; // tokens that are there; null: all
    int* ids;
    float* weights;
    int *offsets, *rows, *places; // null: no tables
    void* ws;                     // [chunks][experts] counts
    int tokens, experts, top_k, groups, top_groups, group_best, stride_x;
    int sigmoid, renormalise;
    float scale;
    int chunk_tokens, chunks; // tokens of a workgroup
};
constexpr int kMostExperts = 1024, kMostTopK = 32, kMostGroups = 64;
int64_t route_workspace(int tokens, int experts);
hipError_t route_launch(RouteArgs a, int x_type, hipStream_t s);

struct TokenQuantArgs
{
    const void* x;
    int8_t* q;
    float* scale;
    int M, K, sx, sq;
};
hipError_t quantize_tokens_launch(const TokenQuantArgs& a, int x_type, hipStream_t s);

struct GemmI8Args
{
    const int8_t *a, *b;
    void* c;
    const float *sa, *sb, *bias;
    // the experts' form: rows offsets[e] ... offsets[e + 1] - 1 of C belong to expert e; row i takes row rows[i] / rows_per of A
    const int *offsets, *rows;
    int experts, rows_a, rows_per;
    int64_t batch_b; // from one expert's B to the next
    int M, N, K, lda, ldb, ldc;
    int gated;
    int tiles_m, tiles_n;
    int ksteps, ksplit, per; // K tiles of 128; runs they are cut into, K tiles a run
    int* ws;                 // ksplit > 1: [ksplit][M][N or 2 N] sums
};
bool gemm_i8_scaled_fits(int M, int N, int gated, int experts);
int64_t gemm_i8_scaled_workspace(int M, int N, int K, int gated);
// the kernel's name (include/ckx.h), and what a workgroup takes
const char* gemm_i8_scaled_plan(const GemmI8Args& a, int64_t workspace_bytes, int* tile_m, int* tile_n, int* k_runs);
hipError_t gemm_i8_scaled_launch(GemmI8Args a, int c_type, int64_t workspace_bytes, hipStream_t s);

struct CombineArgs
{
    const void* y;
    const int* places;
    const float* weights;
    const void* add; // null: none
    void* out;
    int tokens, top_k, rows, N, sy, sadd, sout;
};
hipError_t combine_launch(const CombineArgs& a, int type, hipStream_t s);

} // namespace ckx
