// ckx_profiler: ckProfiler-style driver (profiler/src/profiler.cpp:48-148) for the operators of
// this library. Positional arguments follow the reference's conventions
// (profiler/src/profile_gemm.cpp:27-75, profile_convnd_fwd.cpp:81-115):
//
//   ckx_profiler gemm <dtype 1:fp16 2:bf16 3:int8> <layout 0:mk_kn 1:mk_nk 2:km_kn 3:km_nk> <verify> <init> <log> <time>
//                     M N K StrideA StrideB StrideC [epilogue 0|1|2] [scale_gemm] [scale_relu] [nrepeat]
//   ckx_profiler conv2d_fwd <dtype 1|3> <verify> <init> <log> <time>
//                     N K C Y X Hi Wi Sy Sx Dy Dx LeftPy LeftPx RightPy RightPx [epilogue sg sr] [nrepeat]
//   ckx_profiler convnd_fwd <dtype 1|3> <layout 1> <verify> <init> <log> <nrepeat> <NDim 1|2|3>
//                     N K C <filter> <input> <strides> <dilations> <left pads> <right pads>   (NDim values each)
//   ckx_profiler batched_gemm_gemm <verify> <init> <log> <time> M N K O Batch [nrepeat]
//   ckx_profiler batched_gemm_softmax_gemm <verify> <init> <log> <time> M N K O Batch [scale] [mask 0|1] [nrepeat]
//   ckx_profiler conv_fwd_bias_relu | conv_fwd_bias_relu_add <dtype 1> <verify> <init> <log> <time>
//                     N K C Y X Hi Wi Sy Sx Dy Dx LeftPy LeftPx RightPy RightPx [nrepeat]
//                     (profiler/src/profile_conv_fwd_bias_relu[_add].cpp; fp16, NHWC/KYXC/NHWK)
//   ckx_profiler gemm_splitk <dtype 1|3> <layout 1> <verify> <init> <log> <time> M N K StrideA StrideB StrideC KBatch
//                     [nrepeat]   (profiler/src/profile_gemm_splitk.cpp; PassThrough output)
//   ckx_profiler batched_gemm <dtype 1|3> <layout 1> <verify> <init> <log> <time> M N K StrideA StrideB StrideC
//                     BatchCount [nrepeat]   (profiler/src/profile_batched_gemm.cpp; dense batch strides)
//   ckx_profiler gemm_bias_relu <verify> <init> <log> <time> M N K StrideA StrideB StrideE [nrepeat]
//                     (example/03_gemm_bias_relu: E = AddRelu(half(A*B), bias row), fp16)
//   ckx_profiler gemm_bilinear <dtype 1> <layout 0..3> <verify> <init> <log> <time> M N K StrideA StrideB StrideD StrideE
//                     alpha beta [nrepeat]   (profiler/src/profile_gemm_bilinear.cpp:28-66)
//   ckx_profiler gemm_add_add_fastgelu <dtype 1> <layout 0..3> <verify> <init> <log> <time> M N K StrideA StrideB
//                     StrideD0 StrideD1 StrideE [nrepeat]   (profiler/src/profile_gemm_add_add_fastgelu.cpp:29-62)
//   ckx_profiler gemm_f8_blockscale <c type 1:fp16 2:bf16> <verify> <init> <log> <time> M N K [nrepeat]
//                     (fp16 activations through DeviceBlockQuantizeF8, then DeviceGemmBlockScaleF8; weights with 128 x 128 scales)
//   ckx_profiler paged_attention8 <cache 1:e4m3 2:int8> <verify> <init> <log> <time> Batch Context New QHeads KvHeads HeadDim
//                     BlockSize [causal 0|1] [nrepeat]   (a step of a decoder: DeviceKvCacheTables, DeviceKvCacheStore8,
//                     DevicePagedAttention8, fp16; the cached tokens are stored by a step of their own first)
//   ckx_profiler gemm_i8_tokenscale <c type 1:fp16 2:bf16> <verify> <init> <log> <time> M N K [gated 0|1] [nrepeat]
//                     (fp16 activations through DeviceTokenQuantizeI8, then DeviceGemmTokenScaleI8)
//   ckx_profiler experts_i8 <scores 1:softmax 2:sigmoid> <verify> <init> <log> <time> Tokens Experts TopK Hidden Inner [nrepeat]
//                     (a mixture of experts from its logits to its output, fp16: DeviceRouteExperts, DeviceTokenQuantizeI8, the gated
//                     DeviceExpertsGemmI8 of Inner columns, DeviceTokenQuantizeI8, DeviceExpertsGemmI8, DeviceExpertsCombine)
//
// Every instance of the family is run (DeviceOperationInstanceFactory), one "Perf:" line each
// and a final "Best Perf:" line, in the reference's format (profile_gemm_impl.hpp:176-177,
// 246-249), extended with the fraction of the MI355X roofline that binds the problem.
// verify = 1 checks that all instances agree with the first supported one (bit-exact for
// int8, rtol = atol = 1e-2 for fp16); comparison against the CPU reference is the job of the
// test-suite, which regenerates these inputs from the same seeds. The 8-bit serving operators have one kernel choice each:
// there verify = 1 compares a sample of their outputs with plain host forms in 64 bits (ckx/serving_check.hpp, experts_check.hpp), and
// init = 0 leaves inputs zero, any other fills them with decimal values. If the environment variable
// CKX_PROFILER_DUMP names a file, the best instance's output tensor is written there.
#include <cstdlib>
#include <cstring>
#include <iomanip>
#include <iostream>

#include "ckx/device_ops.hpp"
#include "ckx/experts_check.hpp"
#include "ckx/host_tensor.hpp"
#include "ckx/serving_check.hpp"
#include "ckx/serving_ops.hpp"

using namespace ck;
using namespace ck::tensor_operation;
using Row  = tensor_layout::gemm::RowMajor;
using Col  = tensor_layout::gemm::ColumnMajor;
using Pass = element_wise::PassThrough;

namespace {

constexpr double kPeakF16 = 2516.6, kPeakI8 = 5033.2, kPeakHbmGBs = 8000.0;

struct Best
{
    float ms = 0, tflops = 0, gbs = 0;
    std::string name;
    int id = -1;
};

void report(const char* tag, float ms, double flop, double bytes, const std::string& name, bool i8)
{
    const double tflops = flop / 1e9 / ms, gbs = bytes / 1e6 / ms;
    const double fm = tflops / (i8 ? kPeakI8 : kPeakF16), fh = gbs / kPeakHbmGBs;
    std::cout << tag << std::setw(10) << ms << " ms, " << tflops << " TFlops, " << gbs << " GB/s, " << name << "  ["
              << std::fixed << std::setprecision(1) << (fm >= fh ? fm : fh) * 100 << "% of "
              << (fm >= fh ? "MFMA" : "HBM") << " roofline]" << std::defaultfloat << std::setprecision(6)
              << std::endl;
}

template <typename T>
void fill(std::vector<T>& v, int init, uint64_t seed, bool conv)
{
    if constexpr(std::is_same_v<T, int8_t>)
    {
        if(init == 0)
            return;
        ckx::fill_uniform_int8(v, -5, 5, seed);
    }
    else if constexpr(std::is_same_v<T, bhalf_t>)
    {
        if(init == 0)
            return;
        if(init == 1)
        {
            std::vector<int8_t> t(v.size());
            ckx::fill_uniform_int8(t, -5, 5, seed);
            for(std::size_t i = 0; i < v.size(); ++i)
                v[i] = ckx::float_to_bf16((float)t[i]);
        }
        else
            ckx::fill_uniform_bf16(v, -1.f, 1.f, seed);
    }
    else
    {
        if(init == 0)
            return;
        if(init == 1)
        { // integer values, as the reference's init_method 1
            std::vector<int8_t> t(v.size());
            ckx::fill_uniform_int8(t, -5, 5, seed);
            for(std::size_t i = 0; i < v.size(); ++i)
                v[i] = (T)(float)t[i];
        }
        else
            ckx::fill_uniform_f16(v, conv ? -1.f : -1.f, 1.f, seed);
    }
}

template <typename T, typename Op, typename MakeArg>
int run_family(std::vector<std::unique_ptr<Op>>& ops, MakeArg make_arg, ckx::DeviceMem& out_dev, std::size_t out_elems,
               double flop, double bytes, bool verify, bool time_kernel, int nrepeat)
{
    constexpr bool i8 = std::is_same_v<T, int8_t>;
    std::cout << "found " << ops.size() << " instances" << std::endl;
    Best best;
    std::vector<T> ref, out(out_elems);
    bool pass = true;
    for(std::size_t i = 0; i < ops.size(); ++i)
    {
        auto arg = make_arg(*ops[i]);
        auto inv = ops[i]->MakeInvokerPointer();
        const std::string name = ops[i]->GetTypeString();
        if(!ops[i]->IsSupportedArgument(arg.get()))
        {
            std::cout << name << " does not support this problem" << std::endl;
            continue;
        }
        out_dev.SetZero();
        StreamConfig sc{nullptr, time_kernel, nrepeat, nrepeat >= 100 ? nrepeat / 4 : 1};
        const float ms = inv->Run(arg.get(), sc);
        ckx::hip_check(hipDeviceSynchronize());
        if(time_kernel)
        {
            report("Perf: ", ms, flop, bytes, name, i8);
            if(best.id < 0 || ms < best.ms)
                best = Best{ms, (float)(flop / 1e9 / ms), (float)(bytes / 1e6 / ms), name, (int)i};
        }
        else if(best.id < 0)
            best.id = (int)i, best.name = name;
        if(verify)
        {
            out_dev.FromDevice(out.data());
            if(ref.empty())
                ref = out;
            else
            {
                const std::size_t bad = ckx::count_errors(out, ref, 1e-2, 1e-2);
                if(bad)
                {
                    std::cout << "Error: " << name << " disagrees with the first instance on " << bad << " elements"
                              << std::endl;
                    pass = false;
                }
            }
        }
    }
    if(best.id < 0)
    {
        std::cout << "no instance supports this problem" << std::endl;
        return 1;
    }
    if(time_kernel)
        report("Best Perf: ", best.ms, flop, bytes, best.name, i8);
    if(const char* path = std::getenv("CKX_PROFILER_DUMP"))
    {
        auto arg = make_arg(*ops[best.id]);
        out_dev.SetZero();
        ops[best.id]->MakeInvokerPointer()->Run(arg.get(), StreamConfig{});
        ckx::hip_check(hipDeviceSynchronize());
        out_dev.FromDevice(out.data());
        ckx::dump_to_file(path, out);
    }
    return pass ? 0 : 1;
}

// layout codes of the reference's profiler (profiler/src/profile_gemm.cpp:13-19)
enum GemmMatrixLayout
{
    MK_KN_MN = 0,
    MK_NK_MN = 1,
    KM_KN_MN = 2,
    KM_NK_MN = 3
};

template <typename T, typename COp, typename AL, typename BL>
int profile_gemm_l(bool verify, int init, bool time_kernel, int M, int N, int K, int sa, int sb, int sc, COp cop,
                   int nrepeat)
{
    using DeviceOp = device::DeviceGemm<AL, BL, Row, T, T, T, Pass, Pass, COp>;
    auto ops       = device::instance::DeviceOperationInstanceFactory<DeviceOp>::GetInstances();
    constexpr bool a_row = std::is_same_v<AL, Row>, b_row = std::is_same_v<BL, Row>;
    sa = sa < 0 ? (a_row ? K : M) : sa, sb = sb < 0 ? (b_row ? N : K) : sb, sc = sc < 0 ? N : sc;
    std::vector<T> a((std::size_t)(a_row ? M : K) * sa), b((std::size_t)(b_row ? K : N) * sb);
    fill(a, init, 0xC0FFEE, false);
    fill(b, init, 0xC0FFEE + 1, false);
    ckx::DeviceMem da(a.size() * sizeof(T)), db(b.size() * sizeof(T)), dc((std::size_t)M * sc * sizeof(T));
    da.ToDevice(a.data());
    db.ToDevice(b.data());
    std::cout << "a_m_k: dim 2, lengths {" << M << ", " << K << "}, strides {" << (a_row ? sa : 1) << ", "
              << (a_row ? 1 : sa) << "}\n"
              << "b_k_n: dim 2, lengths {" << K << ", " << N << "}, strides {" << (b_row ? sb : 1) << ", "
              << (b_row ? 1 : sb) << "}\n"
              << "c_m_n: dim 2, lengths {" << M << ", " << N << "}, strides {" << sc << ", 1}" << std::endl;
    const double flop = 2.0 * M * N * K, bytes = sizeof(T) * ((double)M * K + (double)K * N + (double)M * N);
    return run_family<T>(
        ops,
        [&](DeviceOp& op) {
            return op.MakeArgumentPointer(da.GetDeviceBuffer(), db.GetDeviceBuffer(), dc.GetDeviceBuffer(), M, N, K,
                                          sa, sb, sc, Pass{}, Pass{}, cop);
        },
        dc, (std::size_t)M * sc, flop, bytes, verify, time_kernel, nrepeat);
}

template <typename T, typename COp>
int profile_gemm_t(int layout, bool verify, int init, bool time_kernel, int M, int N, int K, int sa, int sb, int sc,
                   COp cop, int nrepeat)
{
    switch(layout)
    {
    case MK_KN_MN: return profile_gemm_l<T, COp, Row, Row>(verify, init, time_kernel, M, N, K, sa, sb, sc, cop, nrepeat);
    case MK_NK_MN: return profile_gemm_l<T, COp, Row, Col>(verify, init, time_kernel, M, N, K, sa, sb, sc, cop, nrepeat);
    case KM_KN_MN: return profile_gemm_l<T, COp, Col, Row>(verify, init, time_kernel, M, N, K, sa, sb, sc, cop, nrepeat);
    case KM_NK_MN: return profile_gemm_l<T, COp, Col, Col>(verify, init, time_kernel, M, N, K, sa, sb, sc, cop, nrepeat);
    }
    std::cout << "this data_type & layout is not implemented" << std::endl;
    return 1;
}

int profile_gemm(int argc, char* argv[])
{
    if(argc < 14)
    {
        std::printf("arg1: tensor operation (gemm)\narg2: data type (1: fp16; 2: bf16; 3: int8)\n"
                    "arg3: matrix layout (0: A[m, k] * B[k, n] = C[m, n];\n"
                    "                     1: A[m, k] * B[n, k] = C[m, n];\n"
                    "                     2: A[k, m] * B[k, n] = C[m, n];\n"
                    "                     3: A[k, m] * B[n, k] = C[m, n])\n"
                    "arg4: verification (0: no; 1: yes)\n"
                    "arg5: initialization (0: no init; 1: integer value; 2: decimal value)\n"
                    "arg6: print tensor value (0: no; 1: yes)\narg7: time kernel (0=no, 1=yes)\n"
                    "arg8 to 13: M, N, K, StrideA, StrideB, StrideC (negative: packed)\n"
                    "arg14-16 (int8): epilogue (0 PassThrough, 1 RequantReluRequant, 2 rounded), scale_gemm, scale_relu\n"
                    "last: nrepeat\n");
        return 1;
    }
    const int dtype = std::atoi(argv[2]), layout = std::atoi(argv[3]);
    const bool verify = std::atoi(argv[4]), time_kernel = std::atoi(argv[7]);
    const int init = std::atoi(argv[5]);
    const int M = std::atoi(argv[8]), N = std::atoi(argv[9]), K = std::atoi(argv[10]);
    int sa = std::atoi(argv[11]), sb = std::atoi(argv[12]), sc = std::atoi(argv[13]);
    if(dtype == 1)
        return profile_gemm_t<half_t>(layout, verify, init, time_kernel, M, N, K, sa, sb, sc, Pass{},
                                      argc > 14 ? std::atoi(argv[14]) : 10);
    if(dtype == 2)
        return profile_gemm_t<bhalf_t>(layout, verify, init, time_kernel, M, N, K, sa, sb, sc, Pass{},
                                       argc > 14 ? std::atoi(argv[14]) : 10);
    if(dtype == 3)
    {
        const int epi  = argc > 14 ? std::atoi(argv[14]) : 0;
        const float sg = argc > 15 ? (float)std::atof(argv[15]) : 0.03f;
        const float sr = argc > 16 ? (float)std::atof(argv[16]) : 1.0f;
        const int nrep = argc > 17 ? std::atoi(argv[17]) : 10;
        if(epi == 0)
            return profile_gemm_t<int8_t>(layout, verify, init, time_kernel, M, N, K, sa, sb, sc, Pass{}, nrep);
        if(epi == 1)
            return profile_gemm_t<int8_t>(layout, verify, init, time_kernel, M, N, K, sa, sb, sc,
                                          element_wise::RequantReluRequant{sg, sr}, nrep);
        return profile_gemm_t<int8_t>(layout, verify, init, time_kernel, M, N, K, sa, sb, sc,
                                      element_wise::RequantRoundReluRequantRound{sg, sr}, nrep);
    }
    std::cout << "this data_type & layout is not implemented" << std::endl;
    return 1;
}

template <typename T, typename OutOp>
int profile_conv_t(bool verify, int init, bool time_kernel, const int* p, OutOp oop, int nrepeat)
{
    const int N = p[0], K = p[1], C = p[2], Y = p[3], X = p[4], Hi = p[5], Wi = p[6], Sy = p[7], Sx = p[8],
              Dy = p[9], Dx = p[10], LPy = p[11], LPx = p[12], RPy = p[13], RPx = p[14];
    // conv_util.cpp:103-114
    const int Ho = (Hi + LPy + RPy - ((Y - 1) * Dy + 1)) / Sy + 1, Wo = (Wi + LPx + RPx - ((X - 1) * Dx + 1)) / Sx + 1;
    auto ops     = device::instance::GetConv2dFwdInstances<T, Pass, Pass, OutOp>();
    using Op     = device::DeviceConvFwd<Pass, Pass, OutOp>;
    std::vector<T> in((std::size_t)N * Hi * Wi * C), wei((std::size_t)K * Y * X * C);
    fill(in, init, 0xC0FFEE + 2, true);
    fill(wei, init, 0xC0FFEE + 3, true);
    const std::size_t out_elems = (std::size_t)N * Ho * Wo * K;
    ckx::DeviceMem di(in.size() * sizeof(T)), dw(wei.size() * sizeof(T)), dout(out_elems * sizeof(T));
    di.ToDevice(in.data());
    dw.ToDevice(wei.data());
    std::cout << "input: N " << N << " Hi " << Hi << " Wi " << Wi << " C " << C << "; weight: K " << K << " Y " << Y
              << " X " << X << "; output: Ho " << Ho << " Wo " << Wo << std::endl;
    // conv_util.cpp:22-39 (flops) and conv_util.hpp:108-136 (bytes: whole input counted)
    const double flop  = 2.0 * N * K * Ho * Wo * C * Y * X;
    const double bytes = sizeof(T) * ((double)in.size() + (double)wei.size() + (double)out_elems);
    return run_family<T>(
        ops,
        [&](Op& op) {
            return op.MakeArgumentPointer(di.GetDeviceBuffer(), dw.GetDeviceBuffer(), dout.GetDeviceBuffer(), N, K, C,
                                          {Hi, Wi}, {Y, X}, {Ho, Wo}, {Sy, Sx}, {Dy, Dx}, {LPy, LPx}, {RPy, RPx},
                                          Pass{}, Pass{}, oop);
        },
        dout, out_elems, flop, bytes, verify, time_kernel, nrepeat);
}

int profile_conv(int argc, char* argv[])
{
    if(argc < 22)
    {
        std::printf("arg1: tensor operation (conv2d_fwd)\narg2: data type (1: fp16; 3: int8)\n"
                    "arg3: verification\narg4: initialization\narg5: print tensor value\narg6: time kernel\n"
                    "arg7 to 21: N, K, C, Y, X, Hi, Wi, Sy, Sx, Dy, Dx, LeftPy, LeftPx, RightPy, RightPx\n"
                    "arg22-24 (int8): epilogue, scale_gemm, scale_relu; last: nrepeat\n");
        return 1;
    }
    const int dtype = std::atoi(argv[2]);
    const bool verify = std::atoi(argv[3]), time_kernel = std::atoi(argv[6]);
    const int init = std::atoi(argv[4]);
    int p[15];
    for(int i = 0; i < 15; ++i)
        p[i] = std::atoi(argv[7 + i]);
    if(dtype == 1)
        return profile_conv_t<half_t>(verify, init, time_kernel, p, Pass{}, argc > 22 ? std::atoi(argv[22]) : 10);
    if(dtype == 3)
    {
        const int epi  = argc > 22 ? std::atoi(argv[22]) : 0;
        const float sg = argc > 23 ? (float)std::atof(argv[23]) : 0.03f;
        const float sr = argc > 24 ? (float)std::atof(argv[24]) : 1.0f;
        const int nrep = argc > 25 ? std::atoi(argv[25]) : 10;
        if(epi == 0)
            return profile_conv_t<int8_t>(verify, init, time_kernel, p, Pass{}, nrep);
        if(epi == 1)
            return profile_conv_t<int8_t>(verify, init, time_kernel, p, element_wise::RequantReluRequant{sg, sr}, nrep);
        return profile_conv_t<int8_t>(verify, init, time_kernel, p, element_wise::RequantRoundReluRequantRound{sg, sr},
                                      nrep);
    }
    std::cout << "this data_type is not implemented" << std::endl;
    return 1;
}

// conv forward with NDim spatial dimensions, channels-last tensors
// (profiler/src/profile_convnd_fwd.cpp:81-115: N, K, C, then filter / input / strides / dilations / left pads /
// right pads, NDim values each)
template <int NDim, typename T, typename OutOp>
int profile_convnd_t(bool verify, int init, bool time_kernel, const int* p, OutOp oop, int nrepeat)
{
    const int N = p[0], K = p[1], C = p[2];
    std::vector<index_t> filt(p + 3, p + 3 + NDim), in_len(p + 3 + NDim, p + 3 + 2 * NDim),
        st(p + 3 + 2 * NDim, p + 3 + 3 * NDim), dl(p + 3 + 3 * NDim, p + 3 + 4 * NDim),
        lp(p + 3 + 4 * NDim, p + 3 + 5 * NDim), rp(p + 3 + 5 * NDim, p + 3 + 6 * NDim), out_len(NDim);
    std::size_t in_px = N, out_px = N, taps = 1;
    for(int i = 0; i < NDim; ++i)
    {
        // conv_util.cpp:103-114
        out_len[i] = (in_len[i] + lp[i] + rp[i] - ((filt[i] - 1) * dl[i] + 1)) / st[i] + 1;
        in_px *= in_len[i], out_px *= out_len[i] > 0 ? out_len[i] : 0, taps *= filt[i];
    }
    auto ops = device::instance::GetConvNdFwdInstances<NDim, T, Pass, Pass, OutOp>();
    using Op = device::DeviceConvFwd<Pass, Pass, OutOp>;
    std::vector<T> in(in_px * C), wei((std::size_t)K * taps * C);
    fill(in, init, 0xC0FFEE + 2, true);
    fill(wei, init, 0xC0FFEE + 3, true);
    const std::size_t out_elems = out_px * K;
    ckx::DeviceMem di(in.size() * sizeof(T)), dw(wei.size() * sizeof(T)), dout(out_elems * sizeof(T));
    di.ToDevice(in.data());
    dw.ToDevice(wei.data());
    std::cout << NDim << " spatial dimensions; N " << N << " K " << K << " C " << C << "; output pixels per image "
              << out_px / (N ? N : 1) << std::endl;
    const double flop  = 2.0 * (double)out_px * K * C * (double)taps; // conv_util.cpp:22-39
    const double bytes = sizeof(T) * ((double)in.size() + (double)wei.size() + (double)out_elems);
    return run_family<T>(
        ops,
        [&](Op& op) {
            return op.MakeArgumentPointer(di.GetDeviceBuffer(), dw.GetDeviceBuffer(), dout.GetDeviceBuffer(), N, K, C,
                                          in_len, filt, out_len, st, dl, lp, rp, Pass{}, Pass{}, oop);
        },
        dout, out_elems, flop, bytes, verify, time_kernel, nrepeat);
}

template <int NDim>
int profile_convnd_dim(int dtype, bool verify, int init, bool time_kernel, const int* p, int nrepeat)
{
    if(dtype == 1)
        return profile_convnd_t<NDim, half_t>(verify, init, time_kernel, p, Pass{}, nrepeat);
    if(dtype == 3)
        return profile_convnd_t<NDim, int8_t>(verify, init, time_kernel, p, Pass{}, nrepeat);
    std::cout << "this data_type is not implemented" << std::endl;
    return 1;
}

int profile_convnd(int argc, char* argv[])
{
    const int ndim = argc > 8 ? std::atoi(argv[8]) : 0;
    if(ndim < 1 || ndim > 3 || argc != 9 + 3 + 6 * ndim)
    {
        std::printf("arg1: tensor operation (convnd_fwd)\narg2: data type (1: fp16; 3: int8)\n"
                    "arg3: data layout (1: channels last)\narg4: verification\narg5: initialization\n"
                    "arg6: print tensor value\narg7: run kernel # of times\narg8: N spatial dimensions (1, 2, 3)\n"
                    "then N, K, C, <filter>, <input>, <strides>, <dilations>, <left pads>, <right pads>\n");
        return 1;
    }
    if(std::atoi(argv[3]) != 1)
    {
        std::cout << "this data layout is not implemented" << std::endl;
        return 1;
    }
    const int dtype = std::atoi(argv[2]), init = std::atoi(argv[5]), nrep = std::atoi(argv[7]);
    const bool verify = std::atoi(argv[4]);
    int p[3 + 18];
    for(int i = 0; i < 3 + 6 * ndim; ++i)
        p[i] = std::atoi(argv[9 + i]);
    const bool time_kernel = nrep > 0;
    if(ndim == 1)
        return profile_convnd_dim<1>(dtype, verify, init, time_kernel, p, nrep > 0 ? nrep : 1);
    if(ndim == 2)
        return profile_convnd_dim<2>(dtype, verify, init, time_kernel, p, nrep > 0 ? nrep : 1);
    return profile_convnd_dim<3>(dtype, verify, init, time_kernel, p, nrep > 0 ? nrep : 1);
}

template <typename T>
int profile_gemm_splitk_t(bool verify, int init, bool time_kernel, int M, int N, int K, int sa, int sb, int sc,
                          int kbatch, int nrepeat)
{
    using DeviceOp = device::DeviceGemmSplitK<Row, Col, Row, T, T, T, Pass, Pass, Pass>;
    std::vector<std::unique_ptr<DeviceOp>> ops;
    for(int i = 0, n = ckx_num_instances(CKX_OP_GEMM_SPLITK); i < n; ++i)
        ops.push_back(std::make_unique<device::DeviceGemmSplitKMfma<Row, Col, Row, T, T, T, Pass, Pass, Pass>>(i));
    std::vector<T> a((std::size_t)M * sa), b((std::size_t)N * sb);
    fill(a, init, 0xC0FFEE, false);
    fill(b, init, 0xC0FFEE + 1, false);
    ckx::DeviceMem da(a.size() * sizeof(T)), db(b.size() * sizeof(T)), dc((std::size_t)M * sc * sizeof(T));
    const int op_code = std::is_same_v<T, int8_t> ? CKX_OP_GEMM_I8 : CKX_OP_GEMM_F16;
    ckx::DeviceMem ws((std::size_t)ckx_gemm_splitk_workspace_bytes(op_code, M, N, K, kbatch) + 16);
    da.ToDevice(a.data());
    db.ToDevice(b.data());
    const double flop = 2.0 * M * N * K, bytes = sizeof(T) * ((double)M * K + (double)K * N + (double)M * N);
    return run_family<T>(
        ops,
        [&](DeviceOp& op) {
            auto arg = op.MakeArgumentPointer(da.GetDeviceBuffer(), db.GetDeviceBuffer(), dc.GetDeviceBuffer(), M, N,
                                              K, sa, sb, sc, Pass{}, Pass{}, Pass{}, kbatch);
            op.SetWorkSpacePointer(arg.get(), ws.GetDeviceBuffer());
            return arg;
        },
        dc, (std::size_t)M * sc, flop, bytes, verify, time_kernel, nrepeat);
}

int profile_gemm_splitk(int argc, char* argv[])
{
    if(argc < 15)
    {
        std::printf("arg1: tensor operation (gemm_splitk)\narg2: data type (1: fp16; 3: int8)\n"
                    "arg3: matrix layout (1: A[m, k] * B[n, k] = C[m, n])\narg4: verification\n"
                    "arg5: initialization\narg6: print tensor value\narg7: time kernel\n"
                    "arg8 to 13: M, N, K, StrideA, StrideB, StrideC\narg14: split k into multiple batch\n");
        return 1;
    }
    const int dtype = std::atoi(argv[2]), layout = std::atoi(argv[3]);
    const bool verify = std::atoi(argv[4]), time_kernel = std::atoi(argv[7]);
    const int init = std::atoi(argv[5]);
    const int M = std::atoi(argv[8]), N = std::atoi(argv[9]), K = std::atoi(argv[10]);
    int sa = std::atoi(argv[11]), sb = std::atoi(argv[12]), sc = std::atoi(argv[13]);
    sa = sa < 0 ? K : sa, sb = sb < 0 ? K : sb, sc = sc < 0 ? N : sc;
    const int kbatch = std::atoi(argv[14]), nrep = argc > 15 ? std::atoi(argv[15]) : 10;
    if(layout != 1 || (dtype != 1 && dtype != 3))
    {
        std::cout << "this data_type & layout is not implemented" << std::endl;
        return 1;
    }
    return dtype == 1 ? profile_gemm_splitk_t<half_t>(verify, init, time_kernel, M, N, K, sa, sb, sc, kbatch, nrep)
                      : profile_gemm_splitk_t<int8_t>(verify, init, time_kernel, M, N, K, sa, sb, sc, kbatch, nrep);
}

template <typename T>
int profile_batched_gemm_t(bool verify, int init, bool time_kernel, int M, int N, int K, int sa, int sb, int sc,
                           int batch, int nrepeat)
{
    using DeviceOp = device::DeviceBatchedGemm<Row, Col, Row, T, T, T, Pass, Pass, Pass>;
    std::vector<std::unique_ptr<DeviceOp>> ops;
    for(int i = 0, n = ckx_num_instances(CKX_OP_GEMM_SPLITK); i < n; ++i) // the tile instances
        ops.push_back(std::make_unique<device::DeviceBatchedGemmMfma<Row, Col, Row, T, T, T, Pass, Pass, Pass>>(i));
    const std::size_t bsa = (std::size_t)M * sa, bsb = (std::size_t)N * sb, bsc = (std::size_t)M * sc;
    std::vector<T> a(bsa * batch), b(bsb * batch);
    fill(a, init, 0xC0FFEE, false);
    fill(b, init, 0xC0FFEE + 1, false);
    ckx::DeviceMem da(a.size() * sizeof(T)), db(b.size() * sizeof(T)), dc(bsc * batch * sizeof(T));
    da.ToDevice(a.data());
    db.ToDevice(b.data());
    const double flop  = 2.0 * M * N * K * batch;
    const double bytes = sizeof(T) * ((double)M * K + (double)K * N + (double)M * N) * batch;
    return run_family<T>(
        ops,
        [&](DeviceOp& op) {
            return op.MakeArgumentPointer(da.GetDeviceBuffer(), db.GetDeviceBuffer(), dc.GetDeviceBuffer(), M, N, K,
                                          sa, sb, sc, (index_t)bsa, (index_t)bsb, (index_t)bsc, batch, Pass{}, Pass{},
                                          Pass{});
        },
        dc, bsc * batch, flop, bytes, verify, time_kernel, nrepeat);
}

int profile_batched_gemm(int argc, char* argv[])
{
    if(argc < 15)
    {
        std::printf("arg1: tensor operation (batched_gemm)\narg2: data type (1: fp16; 3: int8)\n"
                    "arg3: matrix layout (1: A[g, m, k] * B[g, n, k] = C[g, m, n])\narg4: verification\n"
                    "arg5: initialization\narg6: print tensor value\narg7: time kernel\n"
                    "arg8 to 14: M, N, K, StrideA, StrideB, StrideC, BatchCount\n");
        return 1;
    }
    const int dtype = std::atoi(argv[2]), layout = std::atoi(argv[3]);
    const bool verify = std::atoi(argv[4]), time_kernel = std::atoi(argv[7]);
    const int init = std::atoi(argv[5]);
    const int M = std::atoi(argv[8]), N = std::atoi(argv[9]), K = std::atoi(argv[10]);
    int sa = std::atoi(argv[11]), sb = std::atoi(argv[12]), sc = std::atoi(argv[13]);
    sa = sa < 0 ? K : sa, sb = sb < 0 ? K : sb, sc = sc < 0 ? N : sc;
    const int batch = std::atoi(argv[14]), nrep = argc > 15 ? std::atoi(argv[15]) : 10;
    if(layout != 1 || (dtype != 1 && dtype != 3))
    {
        std::cout << "this data_type & layout is not implemented" << std::endl;
        return 1;
    }
    return dtype == 1 ? profile_batched_gemm_t<half_t>(verify, init, time_kernel, M, N, K, sa, sb, sc, batch, nrep)
                      : profile_batched_gemm_t<int8_t>(verify, init, time_kernel, M, N, K, sa, sb, sc, batch, nrep);
}

// conv + bias + ReLU (with_resi: + residual add), fp16
int profile_conv_bias_relu(int argc, char* argv[], bool with_resi)
{
    if(argc < 22 || std::atoi(argv[2]) != 1)
    {
        std::printf("arg1: tensor operation (conv_fwd_bias_relu[_add])\narg2: data type (1: fp16)\n"
                    "arg3: verification\narg4: initialization\narg5: print tensor value\narg6: time kernel\n"
                    "arg7 to 21: N, K, C, Y, X, Hi, Wi, Sy, Sx, Dy, Dx, LeftPy, LeftPx, RightPy, RightPx\n"
                    "arg22: nrepeat\n");
        return 1;
    }
    using T = half_t;
    const bool verify = std::atoi(argv[3]), time_kernel = std::atoi(argv[6]);
    const int init = std::atoi(argv[4]), nrepeat = argc > 22 ? std::atoi(argv[22]) : 10;
    int p[15];
    for(int i = 0; i < 15; ++i)
        p[i] = std::atoi(argv[7 + i]);
    const int N = p[0], K = p[1], C = p[2], Y = p[3], X = p[4], Hi = p[5], Wi = p[6], Sy = p[7], Sx = p[8],
              Dy = p[9], Dx = p[10], LPy = p[11], LPx = p[12], RPy = p[13], RPx = p[14];
    const int Ho = (Hi + LPy + RPy - ((Y - 1) * Dy + 1)) / Sy + 1, Wo = (Wi + LPx + RPx - ((X - 1) * Dx + 1)) / Sx + 1;
    const std::size_t out_elems = (std::size_t)N * Ho * Wo * K;
    std::vector<T> in((std::size_t)N * Hi * Wi * C), wei((std::size_t)K * Y * X * C), bias((std::size_t)K),
        resi(out_elems);
    fill(in, init, 0xC0FFEE + 2, true);
    fill(wei, init, 0xC0FFEE + 3, true);
    fill(bias, init, 0xC0FFEE + 7, true);
    fill(resi, init, 0xC0FFEE + 8, true);
    ckx::DeviceMem di(in.size() * sizeof(T)), dw(wei.size() * sizeof(T)), db(bias.size() * sizeof(T)),
        dr(resi.size() * sizeof(T)), dout(out_elems * sizeof(T));
    di.ToDevice(in.data());
    dw.ToDevice(wei.data());
    db.ToDevice(bias.data());
    dr.ToDevice(resi.data());
    std::cout << "input: N " << N << " Hi " << Hi << " Wi " << Wi << " C " << C << "; weight: K " << K << " Y " << Y
              << " X " << X << "; output: Ho " << Ho << " Wo " << Wo << std::endl;
    const double flop  = 2.0 * N * K * Ho * Wo * C * Y * X;
    const double bytes = sizeof(T) * ((double)in.size() + (double)wei.size() + (double)K +
                                      (double)out_elems * (with_resi ? 2 : 1));
    if(with_resi)
    {
        using Op = device::DeviceConvFwdBiasActivationAdd<Pass, Pass, element_wise::AddReluAdd>;
        auto ops = device::instance::DeviceOperationInstanceFactory<Op>::GetInstances();
        return run_family<T>(
            ops,
            [&](Op& op) {
                return op.MakeArgumentPointer(di.GetDeviceBuffer(), dw.GetDeviceBuffer(), dout.GetDeviceBuffer(),
                                              db.GetDeviceBuffer(), dr.GetDeviceBuffer(), N, K, C, {Hi, Wi}, {Y, X},
                                              {Ho, Wo}, {Sy, Sx}, {Dy, Dx}, {LPy, LPx}, {RPy, RPx}, Pass{}, Pass{},
                                              element_wise::AddReluAdd{});
            },
            dout, out_elems, flop, bytes, verify, time_kernel, nrepeat);
    }
    using Op = device::DeviceConvFwdBiasActivation<Pass, Pass, element_wise::AddRelu>;
    auto ops = device::instance::DeviceOperationInstanceFactory<Op>::GetInstances();
    return run_family<T>(
        ops,
        [&](Op& op) {
            return op.MakeArgumentPointer(di.GetDeviceBuffer(), dw.GetDeviceBuffer(), dout.GetDeviceBuffer(),
                                          db.GetDeviceBuffer(), N, K, C, {Hi, Wi}, {Y, X}, {Ho, Wo}, {Sy, Sx}, {Dy, Dx},
                                          {LPy, LPx}, {RPy, RPx}, Pass{}, Pass{}, element_wise::AddRelu{});
        },
        dout, out_elems, flop, bytes, verify, time_kernel, nrepeat);
}

// E = AddRelu(half(A * B), D) with D a bias row (stride 0), as example 03 sets it up
int profile_gemm_bias_relu(int argc, char* argv[])
{
    if(argc < 9)
    {
        std::printf("arg1: tensor operation (gemm_bias_relu)\narg2: verification\narg3: initialization\n"
                    "arg4: print tensor value\narg5: time kernel\narg6 to 11: M, N, K, StrideA, StrideB, StrideE\n"
                    "arg12: nrepeat\n");
        return 1;
    }
    using T = half_t;
    const bool verify = std::atoi(argv[2]), time_kernel = std::atoi(argv[5]);
    const int init = std::atoi(argv[3]);
    const int M = std::atoi(argv[6]), N = std::atoi(argv[7]), K = std::atoi(argv[8]);
    int sa = argc > 9 ? std::atoi(argv[9]) : -1, sb = argc > 10 ? std::atoi(argv[10]) : -1,
        se = argc > 11 ? std::atoi(argv[11]) : -1;
    sa = sa < 0 ? K : sa, sb = sb < 0 ? K : sb, se = se < 0 ? N : se;
    const int nrepeat = argc > 12 ? std::atoi(argv[12]) : 10;
    using Ds       = ck::Tuple<T>;
    using DeviceOp = device::DeviceGemmMultipleD<Row, Col, Row, T, T, Ds, T, Pass, Pass, element_wise::AddRelu>;
    auto ops       = device::instance::DeviceOperationInstanceFactory<DeviceOp>::GetInstances();
    std::vector<T> a((std::size_t)M * sa), b((std::size_t)N * sb), d((std::size_t)N);
    fill(a, init, 0xC0FFEE, false);
    fill(b, init, 0xC0FFEE + 1, false);
    fill(d, init, 0xC0FFEE + 9, false);
    ckx::DeviceMem da(a.size() * sizeof(T)), db(b.size() * sizeof(T)), dd(d.size() * sizeof(T)),
        de((std::size_t)M * se * sizeof(T));
    da.ToDevice(a.data());
    db.ToDevice(b.data());
    dd.ToDevice(d.data());
    const double flop = 2.0 * M * N * K, bytes = sizeof(T) * ((double)M * K + (double)K * N + (double)M * N + N);
    return run_family<T>(
        ops,
        [&](DeviceOp& op) {
            return op.MakeArgumentPointer(da.GetDeviceBuffer(), db.GetDeviceBuffer(), {dd.GetDeviceBuffer()},
                                          de.GetDeviceBuffer(), M, N, K, sa, sb, {0}, se, Pass{}, Pass{},
                                          element_wise::AddRelu{});
        },
        de, (std::size_t)M * se, flop, bytes, verify, time_kernel, nrepeat);
}

// gemm_perchannel_quant <verify> <init> <log> <time> M N K StrideA StrideB StrideE [activation: 0 PassThrough, 1 Relu] [nrepeat]
// int8 A[m,k] * B[n,k] with one fp32 requant scale per output column (the D operand) and Activation_Mul2_Clamp
template <typename Act>
int profile_gemm_perchannel_quant_t(bool verify, int init, bool time_kernel, int M, int N, int K, int sa, int sb, int se,
                                    int nrepeat)
{
    using T        = int8_t;
    using CDE      = element_wise::Activation_Mul2_Clamp<Act>;
    using DeviceOp = device::DeviceGemmMultipleD<Row, Col, Row, T, T, ck::Tuple<float>, T, Pass, Pass, CDE>;
    std::vector<std::unique_ptr<DeviceOp>> ops;
    for(int i = 0; i < ckx_num_instances(CKX_OP_GEMM_I8); ++i)
        ops.push_back(std::make_unique<device::DeviceGemmMultipleDInt8Mfma<Row, Col, Row, Act>>(i));
    std::vector<T> a((std::size_t)M * sa), b((std::size_t)N * sb);
    fill(a, init, 0xC0FFEE, false);
    fill(b, init, 0xC0FFEE + 1, false);
    std::vector<float> scale((std::size_t)N);
    for(int n = 0; n < N; ++n) // a different, exactly representable scale per column, both signs
        scale[n] = (float)((n * 37) % 61 - 20) / 256.0f;
    ckx::DeviceMem da(a.size()), db(b.size()), dd(scale.size() * sizeof(float)), de((std::size_t)M * se);
    da.ToDevice(a.data());
    db.ToDevice(b.data());
    dd.ToDevice(scale.data());
    const double flop = 2.0 * M * N * K, bytes = (double)M * K + (double)K * N + (double)M * N + 4.0 * N;
    return run_family<T>(
        ops,
        [&](DeviceOp& op) {
            return op.MakeArgumentPointer(da.GetDeviceBuffer(), db.GetDeviceBuffer(), {dd.GetDeviceBuffer()},
                                          de.GetDeviceBuffer(), M, N, K, sa, sb, {0}, se, Pass{}, Pass{}, CDE{});
        },
        de, (std::size_t)M * se, flop, bytes, verify, time_kernel, nrepeat);
}

int profile_gemm_perchannel_quant(int argc, char* argv[])
{
    if(argc < 9)
    {
        std::printf("arg1: tensor operation (gemm_perchannel_quant)\narg2: verification\narg3: initialization\n"
                    "arg4: print tensor value\narg5: time kernel\narg6 to 11: M, N, K, StrideA, StrideB, StrideE\n"
                    "arg12: activation (0: PassThrough; 1: Relu)\narg13: nrepeat\n");
        return 1;
    }
    const bool verify = std::atoi(argv[2]), time_kernel = std::atoi(argv[5]);
    const int init = std::atoi(argv[3]);
    const int M = std::atoi(argv[6]), N = std::atoi(argv[7]), K = std::atoi(argv[8]);
    int sa = argc > 9 ? std::atoi(argv[9]) : -1, sb = argc > 10 ? std::atoi(argv[10]) : -1,
        se = argc > 11 ? std::atoi(argv[11]) : -1;
    sa = sa < 0 ? K : sa, sb = sb < 0 ? K : sb, se = se < 0 ? N : se;
    const int act = argc > 12 ? std::atoi(argv[12]) : 1, nrepeat = argc > 13 ? std::atoi(argv[13]) : 10;
    return act ? profile_gemm_perchannel_quant_t<element_wise::Relu>(verify, init, time_kernel, M, N, K, sa, sb, se, nrepeat)
               : profile_gemm_perchannel_quant_t<Pass>(verify, init, time_kernel, M, N, K, sa, sb, se, nrepeat);
}

// E = cde(A * B, D0[, D1]) for the fp16 CDE operations with the reference's own profiler commands: Bilinear (one D
// tensor) and AddAddFastGelu (two). A D stride of 0 broadcasts one row; a negative stride stands for the dense default.
template <typename CDE, int NumD, typename AL, typename BL>
int profile_gemm_cde_l(bool verify, int init, bool time_kernel, int M, int N, int K, int sa, int sb, int sd0, int sd1,
                       int se, CDE cde, int nrepeat)
{
    using T        = half_t;
    using Ds       = std::conditional_t<NumD == 1, ck::Tuple<T>, ck::Tuple<T, T>>;
    using DeviceOp = device::DeviceGemmMultipleD<AL, BL, Row, T, T, Ds, T, Pass, Pass, CDE>;
    auto ops       = device::instance::DeviceOperationInstanceFactory<DeviceOp>::GetInstances();
    constexpr bool a_row = std::is_same_v<AL, Row>, b_row = std::is_same_v<BL, Row>;
    sa = sa < 0 ? (a_row ? K : M) : sa, sb = sb < 0 ? (b_row ? N : K) : sb, se = se < 0 ? N : se;
    sd0 = sd0 < 0 ? N : sd0, sd1 = sd1 < 0 ? N : sd1;
    std::vector<T> a((std::size_t)(a_row ? M : K) * sa), b((std::size_t)(b_row ? K : N) * sb);
    std::vector<T> d0(sd0 ? (std::size_t)M * sd0 : (std::size_t)N), d1(sd1 ? (std::size_t)M * sd1 : (std::size_t)N);
    fill(a, init, 0xC0FFEE, false);
    fill(b, init, 0xC0FFEE + 1, false);
    fill(d0, init, 0xC0FFEE + 9, false);
    fill(d1, init, 0xC0FFEE + 10, false);
    ckx::DeviceMem da(a.size() * sizeof(T)), db(b.size() * sizeof(T)), dd0(d0.size() * sizeof(T)),
        dd1(d1.size() * sizeof(T)), de((std::size_t)M * se * sizeof(T));
    da.ToDevice(a.data());
    db.ToDevice(b.data());
    dd0.ToDevice(d0.data());
    dd1.ToDevice(d1.data());
    const double flop  = 2.0 * M * N * K;
    const double bytes = sizeof(T) * ((double)M * K + (double)K * N + (double)M * N + (sd0 ? (double)M * N : (double)N) +
                                      (NumD > 1 ? (sd1 ? (double)M * N : (double)N) : 0.0));
    return run_family<T>(
        ops,
        [&](DeviceOp& op) {
            if constexpr(NumD == 1)
                return op.MakeArgumentPointer(da.GetDeviceBuffer(), db.GetDeviceBuffer(), {dd0.GetDeviceBuffer()},
                                              de.GetDeviceBuffer(), M, N, K, sa, sb, {sd0}, se, Pass{}, Pass{}, cde);
            else
                return op.MakeArgumentPointer(da.GetDeviceBuffer(), db.GetDeviceBuffer(),
                                              {dd0.GetDeviceBuffer(), dd1.GetDeviceBuffer()}, de.GetDeviceBuffer(), M, N,
                                              K, sa, sb, {sd0, sd1}, se, Pass{}, Pass{}, cde);
        },
        de, (std::size_t)M * se, flop, bytes, verify, time_kernel, nrepeat);
}

template <typename CDE, int NumD>
int profile_gemm_cde(int layout, bool verify, int init, bool time_kernel, int M, int N, int K, int sa, int sb, int sd0,
                     int sd1, int se, CDE cde, int nrepeat)
{
    switch(layout)
    {
    case MK_KN_MN: return profile_gemm_cde_l<CDE, NumD, Row, Row>(verify, init, time_kernel, M, N, K, sa, sb, sd0, sd1, se, cde, nrepeat);
    case MK_NK_MN: return profile_gemm_cde_l<CDE, NumD, Row, Col>(verify, init, time_kernel, M, N, K, sa, sb, sd0, sd1, se, cde, nrepeat);
    case KM_KN_MN: return profile_gemm_cde_l<CDE, NumD, Col, Row>(verify, init, time_kernel, M, N, K, sa, sb, sd0, sd1, se, cde, nrepeat);
    case KM_NK_MN: return profile_gemm_cde_l<CDE, NumD, Col, Col>(verify, init, time_kernel, M, N, K, sa, sb, sd0, sd1, se, cde, nrepeat);
    }
    std::printf("unknown matrix layout\n");
    return 1;
}

int profile_gemm_bilinear(int argc, char* argv[])
{
    if(argc < 17 || std::atoi(argv[2]) != 1)
    {
        std::printf("arg1: tensor operation (gemm_bilinear: GEMM+Bilinear)\narg2: data type (1: fp16)\n"
                    "arg3: matrix layout (0: E[m, n] = alpha * A[m, k] * B[k, n] + beta * D[m, n];\n"
                    "                     1: E[m, n] = alpha * A[m, k] * B[n, k] + beta * D[m, n];\n"
                    "                     2: E[m, n] = alpha * A[k, m] * B[k, n] + beta * D[m, n];\n"
                    "                     3: E[m, n] = alpha * A[k, m] * B[n, k] + beta * D[m, n])\n"
                    "arg4: verification (0: no; 1: yes)\narg5: initialization (0: no init; 1: integer value; 2: decimal value)\n"
                    "arg6: print tensor value (0: no; 1: yes)\narg7: time kernel (0=no, 1=yes)\n"
                    "arg8 to 14: M, N, K, StrideA, StrideB, StrideD, StrideE\narg15 to 16: alpha, beta\narg17: nrepeat\n");
        return 1;
    }
    const int layout = std::atoi(argv[3]), init = std::atoi(argv[5]);
    const bool verify = std::atoi(argv[4]), time_kernel = std::atoi(argv[7]);
    const int M = std::atoi(argv[8]), N = std::atoi(argv[9]), K = std::atoi(argv[10]);
    const int sa = std::atoi(argv[11]), sb = std::atoi(argv[12]), sd = std::atoi(argv[13]), se = std::atoi(argv[14]);
    const float alpha = (float)std::atof(argv[15]), beta = (float)std::atof(argv[16]);
    const int nrepeat = argc > 17 ? std::atoi(argv[17]) : 10;
    return profile_gemm_cde<element_wise::Bilinear, 1>(layout, verify, init, time_kernel, M, N, K, sa, sb, sd, 0, se,
                                                       element_wise::Bilinear{alpha, beta}, nrepeat);
}

int profile_gemm_add_add_fastgelu(int argc, char* argv[])
{
    if(argc < 16 || std::atoi(argv[2]) != 1)
    {
        std::printf("arg1: tensor operation (gemm_add_add_fastgelu: GEMM+Add+Add+FastGeLU)\narg2: data type (1: fp16)\n"
                    "arg3: matrix layout (0: E[m, n] = FastGeLU(A[m, k] * B[k, n] + D0[m, n] + D1[m, n]);\n"
                    "                     1: E[m, n] = FastGeLU(A[m, k] * B[n, k] + D0[m, n] + D1[m, n]);\n"
                    "                     2: E[m, n] = FastGeLU(A[k, m] * B[k, n] + D0[m, n] + D1[m, n]);\n"
                    "                     3: E[m, n] = FastGeLU(A[k, m] * B[n, k] + D0[m, n] + D1[m, n]))\n"
                    "arg4: verification (0: no; 1: yes)\narg5: initialization (0: no init; 1: integer value; 2: decimal value)\n"
                    "arg6: print tensor value (0: no; 1: yes)\narg7: time kernel (0=no, 1=yes)\n"
                    "arg8 to 15: M, N, K, StrideA, StrideB, StrideD0, StrideD1, StrideE\narg16: nrepeat\n");
        return 1;
    }
    const int layout = std::atoi(argv[3]), init = std::atoi(argv[5]);
    const bool verify = std::atoi(argv[4]), time_kernel = std::atoi(argv[7]);
    const int M = std::atoi(argv[8]), N = std::atoi(argv[9]), K = std::atoi(argv[10]);
    const int sa = std::atoi(argv[11]), sb = std::atoi(argv[12]), sd0 = std::atoi(argv[13]), sd1 = std::atoi(argv[14]),
              se = std::atoi(argv[15]);
    const int nrepeat = argc > 16 ? std::atoi(argv[16]) : 10;
    return profile_gemm_cde<element_wise::AddAddFastGelu, 2>(layout, verify, init, time_kernel, M, N, K, sa, sb, sd0,
                                                             sd1, se, element_wise::AddAddFastGelu{}, nrepeat);
}

int profile_gemm_gemm(int argc, char* argv[])
{
    if(argc < 11)
    {
        std::printf("arg1: tensor operation (batched_gemm_gemm)\narg2: verification\narg3: initialization\n"
                    "arg4: print tensor value\narg5: time kernel\narg6 to 10: M, N, K, O, Batch\nlast: nrepeat\n");
        return 1;
    }
    const bool verify = std::atoi(argv[2]), time_kernel = std::atoi(argv[5]);
    const int init = std::atoi(argv[3]);
    const int M = std::atoi(argv[6]), N = std::atoi(argv[7]), K = std::atoi(argv[8]), O = std::atoi(argv[9]),
              G = std::atoi(argv[10]);
    const int nrepeat = argc > 11 ? std::atoi(argv[11]) : 10;
    using Op = device::DeviceBatchedGemmGemm<Row, Col, Row, Row, half_t, half_t, half_t, half_t, Pass, Pass, Pass,
                                             Pass, Pass>;
    std::vector<std::unique_ptr<Op>> ops;
    for(int i = 0; i < ckx_num_instances(CKX_OP_BATCHED_GEMM_GEMM); ++i)
        ops.push_back(std::make_unique<device::DeviceBatchedGemmGemmMfma<>>(i));
    std::vector<half_t> a((std::size_t)G * M * K), b0((std::size_t)G * N * K), b1((std::size_t)G * N * O);
    if(init)
    {
        ckx::fill_uniform_f16(a, -0.5f, 0.5f, 0xC0FFEE + 4);
        ckx::fill_uniform_f16(b0, -0.5f, 0.5f, 0xC0FFEE + 5);
        ckx::fill_uniform_f16(b1, -0.5f, 0.5f, 0xC0FFEE + 6);
    }
    const std::size_t out_elems = (std::size_t)G * M * O;
    ckx::DeviceMem da(a.size() * 2), db0(b0.size() * 2), db1(b1.size() * 2), dc(out_elems * 2);
    da.ToDevice(a.data());
    db0.ToDevice(b0.data());
    db1.ToDevice(b1.data());
    const double flop  = 2.0 * G * ((double)M * N * K + (double)M * N * O);
    const double bytes = 2.0 * ((double)a.size() + b0.size() + b1.size() + out_elems);
    return run_family<half_t>(
        ops,
        [&](Op& op) {
            return op.MakeArgumentPointer(da.GetDeviceBuffer(), db0.GetDeviceBuffer(), db1.GetDeviceBuffer(),
                                          dc.GetDeviceBuffer(), M, N, K, O, G, K, K, O, O, M * K, N * K, N * O, M * O,
                                          Pass{}, Pass{}, Pass{}, Pass{}, Pass{});
        },
        dc, out_elems, flop, bytes, verify, time_kernel, nrepeat);
}

// batched_gemm_softmax_gemm <verify> <init> <log> <time> M N K O Batch [scale] [mask_out_upper_triangle] [nrepeat]
template <bool Mask>
int profile_gemm_softmax_gemm_t(bool verify, int init, bool time_kernel, int M, int N, int K, int O, int G, float scale,
                                int nrepeat)
{
    using Scale = element_wise::Scale;
    using Op = device::DeviceBatchedGemmSoftmaxGemm<Row, Col, Row, Row, half_t, half_t, half_t, half_t, Pass, Pass, Scale,
                                                    Pass, Pass, Mask>;
    std::vector<std::unique_ptr<Op>> ops;
    for(int i = 0; i < ckx_num_instances(CKX_OP_BATCHED_GEMM_SOFTMAX_GEMM); ++i)
        ops.push_back(std::make_unique<device::DeviceBatchedGemmSoftmaxGemmMfma<Scale, Mask>>(i));
    std::vector<half_t> a((std::size_t)G * M * K), b0((std::size_t)G * N * K), b1((std::size_t)G * N * O);
    if(init)
    {
        ckx::fill_uniform_f16(a, -1.0f, 1.0f, 0xC0FFEE + 7);
        ckx::fill_uniform_f16(b0, -1.0f, 1.0f, 0xC0FFEE + 8);
        ckx::fill_uniform_f16(b1, -1.0f, 1.0f, 0xC0FFEE + 9);
    }
    const std::size_t out_elems = (std::size_t)G * M * O;
    ckx::DeviceMem da(a.size() * 2), db0(b0.size() * 2), db1(b1.size() * 2), dc(out_elems * 2);
    da.ToDevice(a.data());
    db0.ToDevice(b0.data());
    db1.ToDevice(b1.data());
    const double flop  = 2.0 * G * ((double)M * N * K + (double)M * N * O);
    const double bytes = 2.0 * ((double)a.size() + b0.size() + b1.size() + out_elems);
    return run_family<half_t>(
        ops,
        [&](Op& op) {
            return op.MakeArgumentPointer(da.GetDeviceBuffer(), db0.GetDeviceBuffer(), db1.GetDeviceBuffer(),
                                          dc.GetDeviceBuffer(), M, N, K, O, G, K, K, O, O, M * K, N * K, N * O, M * O,
                                          Pass{}, Pass{}, Scale{scale}, Pass{}, Pass{});
        },
        dc, out_elems, flop, bytes, verify, time_kernel, nrepeat);
}

int profile_gemm_softmax_gemm(int argc, char* argv[])
{
    if(argc < 11)
    {
        std::printf("arg1: tensor operation (batched_gemm_softmax_gemm)\narg2: verification\narg3: initialization\n"
                    "arg4: print tensor value\narg5: time kernel\narg6 to 10: M, N, K, O, Batch\n"
                    "arg11: score scale (default 1/sqrt(K))\narg12: mask out the upper triangle (0 | 1)\nlast: nrepeat\n");
        return 1;
    }
    const bool verify = std::atoi(argv[2]), time_kernel = std::atoi(argv[5]);
    const int init = std::atoi(argv[3]);
    const int M = std::atoi(argv[6]), N = std::atoi(argv[7]), K = std::atoi(argv[8]), O = std::atoi(argv[9]),
              G = std::atoi(argv[10]);
    const float scale = argc > 11 ? (float)std::atof(argv[11]) : 1.0f / std::sqrt((float)(K > 0 ? K : 1));
    const bool mask   = argc > 12 && std::atoi(argv[12]);
    const int nrepeat = argc > 13 ? std::atoi(argv[13]) : 10;
    return mask ? profile_gemm_softmax_gemm_t<true>(verify, init, time_kernel, M, N, K, O, G, scale, nrepeat)
                : profile_gemm_softmax_gemm_t<false>(verify, init, time_kernel, M, N, K, O, G, scale, nrepeat);
}

// timed (a "Perf:" line) or untimed launch of an operator that has one kernel choice of its own
template <typename Op>
void run_one(Op& op, const typename Op::Argument& arg, const char* what, bool time_kernel, int nrepeat, double flop, double bytes, bool i8)
{
    if(!op.IsSupportedArgument(arg))
        throw std::runtime_error(std::string(what) + " is not supported: " + ckx_last_error());
    const float ms = op.MakeInvoker().Run(arg, StreamConfig{nullptr, time_kernel, nrepeat, 1});
    ckx::hip_check(hipDeviceSynchronize());
    if(time_kernel)
        report("Perf: ", ms, flop, bytes, op.GetTypeString(), i8);
}

template <typename T>
std::vector<T> from_device(const ckx::DeviceMem& m)
{
    std::vector<T> v(m.GetBufferSize() / sizeof(T));
    m.FromDevice(v.data());
    return v;
}

// reports what a check found; whether nothing was wrong
bool verified(const char* what, std::size_t bad, std::size_t checked)
{
    if(bad)
        std::cout << "Error: " << what << " differs from the plain form in " << bad << " of " << checked << " values" << std::endl;
    else
        std::cout << "verified " << what << ": " << checked << " values" << std::endl;
    return bad == 0;
}

template <typename T>
int profile_gemm_f8_t(bool verify, int init, bool time_kernel, int M, int N, int K, int nrepeat)
{
    const int groups = (K + 127) / 128, nb = (N + 127) / 128;
    std::vector<half_t> x((std::size_t)M * K);
    if(init)
        ckx::fill_uniform_f16(x, -1.f, 1.f, 0xC0FFEE + 10);
    // weights: every finite code; scales of 2^-9 ... 2^-6
    std::vector<uint8_t> w((std::size_t)N * K);
    for(std::size_t i = 0; init && i < w.size(); ++i)
    {
        w[i] = (uint8_t)(ckx::splitmix64(0xC0FFEE + 11, i) >> 56);
        w[i] = (w[i] & 127) == 127 ? 0 : w[i];
    }
    std::vector<float> sw((std::size_t)nb * groups);
    for(std::size_t i = 0; i < sw.size(); ++i)
        sw[i] = 1.0f / (float)(64 << (ckx::splitmix64(0xC0FFEE + 12, i) >> 62));
    ckx::DeviceMem dx(x.size() * 2), dq(x.size()), ds((std::size_t)M * groups * 4), dw(w.size()), dsw(sw.size() * 4),
        dc((std::size_t)M * N * sizeof(T));
    dx.ToDevice(x.data());
    dw.ToDevice(w.data());
    dsw.ToDevice(sw.data());
    device::DeviceBlockQuantizeF8<half_t> quantize;
    run_one(quantize,
            quantize.MakeArgument(static_cast<const half_t*>(dx.GetDeviceBuffer()), static_cast<f8_t*>(dq.GetDeviceBuffer()),
                                  static_cast<float*>(ds.GetDeviceBuffer()), M, K, K, K, 1, M),
            "the quantiser", time_kernel, nrepeat, 3.0 * M * K, 3.0 * M * K + 4.0 * M * groups, false);
    device::DeviceGemmBlockScaleF8<T> gemm;
    auto arg = gemm.MakeArgument(static_cast<const f8_t*>(dq.GetDeviceBuffer()), static_cast<const f8_t*>(dw.GetDeviceBuffer()),
                                 static_cast<T*>(dc.GetDeviceBuffer()), static_cast<const float*>(ds.GetDeviceBuffer()),
                                 static_cast<const float*>(dsw.GetDeviceBuffer()), M, N, K, K, K, N, 1, M, groups, 1);
    ckx::DeviceMem ws(gemm.GetWorkSpaceSize(&arg));
    if(ws.GetBufferSize() > 0)
        gemm.SetWorkSpacePointer(&arg, ws.GetDeviceBuffer());
    run_one(gemm, arg, "the product", time_kernel, nrepeat, 2.0 * M * N * K, (double)M * K + (double)N * K + 2.0 * M * N, true);
    const auto out = from_device<T>(dc);
    if(const char* path = std::getenv("CKX_PROFILER_DUMP"))
        ckx::dump_to_file(path, out);
    bool pass = true;
    if(verify)
    {
        const auto q = from_device<uint8_t>(dq);
        const auto s = from_device<float>(ds);
        std::size_t checked = 0;
        std::size_t bad = ckx::quantise_errors([&](std::size_t m, int k) { return (double)x[m * K + k]; }, q.data(), s.data(), M, K, checked);
        pass            = verified("DeviceBlockQuantizeF8", bad, checked);
        checked         = 0;
        bad             = ckx::gemm_f8_errors(
            [&](std::size_t m, std::size_t n) {
                if constexpr(std::is_same_v<T, bhalf_t>)
                    return (double)ckx::bf16_to_float(out[m * N + n]);
                else
                    return (double)out[m * N + n];
            },
            q.data(), w.data(), s.data(), sw.data(), M, N, K, std::is_same_v<T, bhalf_t> ? 0x1p-8 : 0x1p-11, checked);
        pass = verified("DeviceGemmBlockScaleF8", bad, checked) && pass;
    }
    return pass ? 0 : 1;
}

int profile_gemm_f8(int argc, char* argv[])
{
    if(argc < 10)
    {
        std::printf("arg1: tensor operation (gemm_f8_blockscale)\narg2: type of C (1: fp16, 2: bf16)\narg3: verification\n"
                    "arg4: initialization\narg5: print tensor value\narg6: time kernel\narg7 to 9: M, N, K\nlast: nrepeat\n");
        return 1;
    }
    const int M = std::atoi(argv[7]), N = std::atoi(argv[8]), K = std::atoi(argv[9]), nrepeat = argc > 10 ? std::atoi(argv[10]) : 10;
    if(M < 1 || N < 1 || K < 1)
        throw std::runtime_error("M, N and K are at least 1");
    auto* run = std::atoi(argv[2]) == 2 ? &profile_gemm_f8_t<bhalf_t> : &profile_gemm_f8_t<half_t>;
    return run(std::atoi(argv[3]) != 0, std::atoi(argv[4]), std::atoi(argv[6]) != 0, M, N, K, nrepeat);
}

template <bool Causal>
int profile_attention8_t(int type, bool verify, int init, bool time_kernel, int B, int ctx, int fresh, int heads, int kv_heads, int D, int bs, int nrepeat)
{
    const int width = (ctx + fresh + bs - 1) / bs, blocks = B * width;
    const std::size_t codes = (std::size_t)blocks * kv_heads * bs * D;
    ckx::DeviceMem dk(codes), dv(codes), dks((std::size_t)blocks * kv_heads * 4), dvs((std::size_t)blocks * kv_heads * 4);
    ckx_kv_cache8 cache{};
    cache.p_k = dk.GetDeviceBuffer(), cache.p_v = dv.GetDeviceBuffer();
    cache.p_k_scale = static_cast<float*>(dks.GetDeviceBuffer()), cache.p_v_scale = static_cast<float*>(dvs.GetDeviceBuffer());
    cache.type = type, cache.num_blocks = blocks, cache.block_size = bs, cache.num_heads = kv_heads, cache.head_dim = D;
    cache.stride_head = bs * D, cache.stride_token = D, cache.stride_scale = kv_heads, cache.stride_block = (int64_t)kv_heads * bs * D;
    // the free list: all blocks, every other one first
    std::vector<index_t> free, zero(B, 0), context(B, ctx), news(B, fresh);
    for(int i = 0; i < blocks; i += 2)
        free.push_back(i);
    for(int i = 1; i < blocks; i += 2)
        free.push_back(i);
    ckx::DeviceMem dfree(free.size() * 4), dzero(B * 4), dctx(B * 4), dnew(B * 4), dtable((std::size_t)B * width * 4), dcu((B + 1) * 4),
        dkv(B * 4), dused(4), dslots((std::size_t)B * (ctx > fresh ? ctx : fresh) * 4);
    dfree.ToDevice(free.data()), dzero.ToDevice(zero.data()), dctx.ToDevice(context.data()), dnew.ToDevice(news.data());
    auto ints = [](ckx::DeviceMem& m) { return static_cast<index_t*>(m.GetDeviceBuffer()); };
    device::DeviceKvCacheTables tables;
    device::DeviceKvCacheStore8<half_t> store;
    device::DevicePagedAttention8<half_t, Causal> attention;
    const int row = (heads + 2 * kv_heads) * D;
    index_t taken = 0;
    // a step: `n` new tokens of every sequence behind `before`; queries, keys and values as columns of one matrix
    auto step = [&](ckx::DeviceMem& dqkv, ckx::DeviceMem& before, ckx::DeviceMem& lens, int n, bool time) {
        auto targ = tables.MakeArgument(ints(before), ints(lens), ints(dfree) + taken, ints(dtable), ints(dcu), ints(dkv), ints(dslots),
                                        ints(dused), B, (index_t)free.size() - taken, width, width, B * n, bs);
        run_one(tables, targ, "the tables", time, nrepeat, (double)B * n, 4.0 * B * (4 + n), false);
        index_t used = 0;
        dused.FromDevice(&used);
        taken += used;
        const half_t* qkv = static_cast<const half_t*>(dqkv.GetDeviceBuffer());
        auto sarg = store.MakeArgument(qkv + heads * D, qkv + (heads + kv_heads) * D, ints(dslots), cache, B * n, row, D, row, D);
        run_one(store, sarg, "the store", time, nrepeat, 6.0 * B * n * kv_heads * D, 6.0 * B * n * kv_heads * D, false);
    };
    auto filled = [&](int n, uint64_t seed) {
        std::vector<half_t> v((std::size_t)B * n * row);
        if(init)
            ckx::fill_uniform_f16(v, -1.f, 1.f, seed);
        auto m = std::make_unique<ckx::DeviceMem>(v.size() * 2);
        m->ToDevice(v.data());
        return m;
    };
    if(ctx > 0)
        step(*filled(ctx, 0xC0FFEE + 13), dzero, dctx, ctx, false);
    auto dqkv = filled(fresh, 0xC0FFEE + 14);
    step(*dqkv, dctx, dnew, fresh, time_kernel);
    ckx::DeviceMem dout((std::size_t)B * fresh * heads * D * 2);
    auto arg = attention.MakeArgument(static_cast<const half_t*>(dqkv->GetDeviceBuffer()), static_cast<half_t*>(dout.GetDeviceBuffer()),
                                      ints(dtable), ints(dcu), ints(dkv), cache, B, B * fresh, heads, ctx + fresh, width, width, row, D,
                                      heads * D, D, element_wise::Scale{1.0f / std::sqrt((float)D)});
    ckx::DeviceMem ws(attention.GetWorkSpaceSize(&arg));
    if(ws.GetBufferSize() > 0)
        attention.SetWorkSpacePointer(&arg, ws.GetDeviceBuffer());
    run_one(attention, arg, "the attention", time_kernel, nrepeat, 4.0 * B * fresh * heads * D * (Causal ? ctx + (fresh + 1) / 2.0 : ctx + fresh),
            2.0 * B * (double)(ctx + fresh) * kv_heads * D + 4.0 * B * fresh * heads * D, false);
    const auto out = from_device<half_t>(dout);
    if(const char* path = std::getenv("CKX_PROFILER_DUMP"))
        ckx::dump_to_file(path, out);
    if(!verify)
        return 0;
    const auto k = from_device<uint8_t>(dk), v = from_device<uint8_t>(dv);
    const auto ks = from_device<float>(dks), vs = from_device<float>(dvs);
    const auto table = from_device<index_t>(dtable);
    const auto qkv   = from_device<half_t>(*dqkv);
    const ckx::Cache8View view{k.data(), v.data(), ks.data(), vs.data(), table.data(), blocks, kv_heads, bs, D, B, width, ctx + fresh,
                               type == CKX_TYPE_I8};
    if(!verified("DeviceKvCacheTables", view.sound() ? 0 : 1, (std::size_t)blocks))
        return 1;
    const int group = heads / kv_heads;
    auto at         = [&](int b, int i, int column) { return (double)qkv[((std::size_t)b * fresh + i) * row + column]; };
    std::size_t checked = 0;
    std::size_t bad     = ckx::store8_errors(
        [&](int b, int i, int h, int d, int value) { return at(b, i, (heads + value * kv_heads + h) * D + d); }, view, fresh, checked);
    bool pass = verified("DeviceKvCacheStore8", bad, checked);
    checked   = 0;
    bad       = ckx::attention8_errors(
        [&](int b, int i, int h, int d) { return at(b, i, h * D + d); },
        [&](int b, int i, int h, int d) { return (double)out[(((std::size_t)b * fresh + i) * heads + h) * D + d]; }, view, fresh, group,
        1.0f / std::sqrt((float)D), Causal, checked);
    pass = verified("DevicePagedAttention8", bad, checked) && pass;
    return pass ? 0 : 1;
}

int profile_attention8(int argc, char* argv[])
{
    if(argc < 14)
    {
        std::printf("arg1: tensor operation (paged_attention8)\narg2: cache (1: e4m3, 2: int8)\narg3: verification\n"
                    "arg4: initialization\narg5: print tensor value\narg6: time kernel\n"
                    "arg7 to 13: Batch, Context, New, QHeads, KvHeads, HeadDim, BlockSize\n"
                    "arg14: causal (0 | 1)\nlast: nrepeat\n");
        return 1;
    }
    int p[7];
    for(int i = 0; i < 7; ++i)
        p[i] = std::atoi(argv[7 + i]);
    if(p[0] < 1 || p[1] < 0 || p[2] < 1 || p[3] < 1 || p[4] < 1 || p[5] < 1 || p[6] < 1)
        throw std::runtime_error("sizes are at least 1, the context at least 0");
    const bool causal = argc > 14 ? std::atoi(argv[14]) != 0 : true;
    const int nrepeat = argc > 15 ? std::atoi(argv[15]) : 10, type = std::atoi(argv[2]) == 2 ? CKX_TYPE_I8 : CKX_TYPE_E4M3;
    auto* run         = causal ? &profile_attention8_t<true> : &profile_attention8_t<false>;
    return run(type, std::atoi(argv[3]) != 0, std::atoi(argv[4]), std::atoi(argv[6]) != 0, p[0], p[1], p[2], p[3], p[4], p[5], p[6], nrepeat);
}

// int8 weights: every code; scales of 2^-15 ... 2^-12
std::vector<int8_t> i8_weights(std::size_t n, int init, uint64_t seed)
{
    std::vector<int8_t> w(n);
    for(std::size_t i = 0; init && i < n; ++i)
        w[i] = (int8_t)(ckx::splitmix64(seed, i) >> 56);
    return w;
}
std::vector<float> i8_scales(std::size_t n, uint64_t seed)
{
    std::vector<float> s(n);
    for(std::size_t i = 0; i < n; ++i)
        s[i] = 1.0f / (float)(4096 << (ckx::splitmix64(seed, i) >> 62));
    return s;
}
template <typename T>
double value_of(T x)
{
    if constexpr(std::is_same_v<T, bhalf_t>)
        return (double)ckx::bf16_to_float(x);
    else
        return (double)x;
}

template <typename T, bool Gated>
int profile_gemm_i8_t(bool verify, int init, bool time_kernel, int M, int N, int K, int nrepeat)
{
    const std::size_t wide = (std::size_t)N * (Gated ? 2 : 1);
    std::vector<half_t> x((std::size_t)M * K);
    if(init)
        ckx::fill_uniform_f16(x, -1.f, 1.f, 0xC0FFEE + 15);
    const auto w  = i8_weights(wide * K, init, 0xC0FFEE + 16);
    const auto sw = i8_scales(wide, 0xC0FFEE + 17);
    ckx::DeviceMem dx(x.size() * 2), dq(x.size()), ds((std::size_t)M * 4), dw(w.size()), dsw(sw.size() * 4), dc((std::size_t)M * N * sizeof(T));
    dx.ToDevice(x.data());
    dw.ToDevice(w.data());
    dsw.ToDevice(sw.data());
    device::DeviceTokenQuantizeI8<half_t> quantize;
    run_one(quantize,
            quantize.MakeArgument(static_cast<const half_t*>(dx.GetDeviceBuffer()), static_cast<int8_t*>(dq.GetDeviceBuffer()),
                                  static_cast<float*>(ds.GetDeviceBuffer()), M, K, K, K),
            "the quantiser", time_kernel, nrepeat, 3.0 * M * K, 3.0 * M * K + 4.0 * M, false);
    device::DeviceGemmTokenScaleI8<T, Gated> gemm;
    auto arg = gemm.MakeArgument(static_cast<const int8_t*>(dq.GetDeviceBuffer()), static_cast<const int8_t*>(dw.GetDeviceBuffer()),
                                 static_cast<T*>(dc.GetDeviceBuffer()), static_cast<const float*>(ds.GetDeviceBuffer()),
                                 static_cast<const float*>(dsw.GetDeviceBuffer()), nullptr, M, N, K, K, K, N);
    ckx::DeviceMem ws(gemm.GetWorkSpaceSize(&arg));
    if(ws.GetBufferSize() > 0)
        gemm.SetWorkSpacePointer(&arg, ws.GetDeviceBuffer());
    run_one(gemm, arg, "the product", time_kernel, nrepeat, 2.0 * M * wide * K, (double)M * K + (double)wide * K + 2.0 * M * N, true);
    const auto out = from_device<T>(dc);
    if(const char* path = std::getenv("CKX_PROFILER_DUMP"))
        ckx::dump_to_file(path, out);
    if(!verify)
        return 0;
    const auto q = from_device<int8_t>(dq);
    const auto s = from_device<float>(ds);
    std::size_t checked = 0;
    std::size_t bad = ckx::token_quantise_errors([&](std::size_t m, int k) { return (double)x[m * K + k]; }, q.data(), s.data(), M, K, checked);
    bool pass       = verified("DeviceTokenQuantizeI8", bad, checked);
    checked         = 0;
    bad             = ckx::gemm_i8_errors([&](std::size_t m, std::size_t n) { return value_of(out[m * N + n]); },
                                      [](std::size_t m, std::size_t& row, std::size_t& expert) { row = m, expert = 0; },
                                      ckx::GemmI8View{q.data(), w.data(), s.data(), sw.data(), M, N, K, Gated},
                                      std::is_same_v<T, bhalf_t> ? 0x1p-8 : 0x1p-11, checked);
    pass = verified("DeviceGemmTokenScaleI8", bad, checked) && pass;
    return pass ? 0 : 1;
}

int profile_gemm_i8(int argc, char* argv[])
{
    if(argc < 10)
    {
        std::printf("arg1: tensor operation (gemm_i8_tokenscale)\narg2: type of C (1: fp16, 2: bf16)\narg3: verification\n"
                    "arg4: initialization\narg5: print tensor value\narg6: time kernel\narg7 to 9: M, N, K\narg10: gated (0 | 1)\n"
                    "last: nrepeat\n");
        return 1;
    }
    const int M = std::atoi(argv[7]), N = std::atoi(argv[8]), K = std::atoi(argv[9]), nrepeat = argc > 11 ? std::atoi(argv[11]) : 10;
    if(M < 1 || N < 1 || K < 1)
        throw std::runtime_error("M, N and K are at least 1");
    const bool gated = argc > 10 && std::atoi(argv[10]) != 0, bf16 = std::atoi(argv[2]) == 2;
    auto* run = gated ? (bf16 ? &profile_gemm_i8_t<bhalf_t, true> : &profile_gemm_i8_t<half_t, true>)
                      : (bf16 ? &profile_gemm_i8_t<bhalf_t, false> : &profile_gemm_i8_t<half_t, false>);
    return run(std::atoi(argv[3]) != 0, std::atoi(argv[4]), std::atoi(argv[6]) != 0, M, N, K, nrepeat);
}

template <device::ExpertScoring Scoring>
int profile_experts_i8_t(bool verify, int init, bool time_kernel, int T, int E, int k, int hidden, int inner, int nrepeat)
{
    const int pairs = T * k;
    std::vector<half_t> logits((std::size_t)T * E), x((std::size_t)T * hidden);
    if(init)
    {
        ckx::fill_uniform_f16(logits, -4.f, 4.f, 0xC0FFEE + 18);
        ckx::fill_uniform_f16(x, -1.f, 1.f, 0xC0FFEE + 19);
    }
    const auto up = i8_weights((std::size_t)E * 2 * inner * hidden, init, 0xC0FFEE + 20), down = i8_weights((std::size_t)E * hidden * inner, init, 0xC0FFEE + 21);
    const auto s_up = i8_scales((std::size_t)E * 2 * inner, 0xC0FFEE + 22), s_down = i8_scales((std::size_t)E * hidden, 0xC0FFEE + 23);
    auto sent = [](const auto& v) {
        auto m = std::make_unique<ckx::DeviceMem>(v.size() * sizeof(v[0]));
        m->ToDevice(v.data());
        return m;
    };
    auto dlogits = sent(logits), dx = sent(x), dup = sent(up), ddown = sent(down), dsup = sent(s_up), dsdown = sent(s_down);
    ckx::DeviceMem dids((std::size_t)pairs * 4), dweights((std::size_t)pairs * 4), doffsets((std::size_t)(E + 1) * 4), drows((std::size_t)pairs * 4),
        dplaces((std::size_t)pairs * 4), dq(x.size()), ds((std::size_t)T * 4), dh((std::size_t)pairs * inner * 2), dqh((std::size_t)pairs * inner),
        dsh((std::size_t)pairs * 4), dy((std::size_t)pairs * hidden * 2), dout(x.size() * 2);
    auto ints   = [](ckx::DeviceMem& m) { return static_cast<index_t*>(m.GetDeviceBuffer()); };
    auto floats = [](ckx::DeviceMem& m) { return static_cast<float*>(m.GetDeviceBuffer()); };
    auto halves = [](ckx::DeviceMem& m) { return static_cast<half_t*>(m.GetDeviceBuffer()); };
    auto codes  = [](ckx::DeviceMem& m) { return static_cast<int8_t*>(m.GetDeviceBuffer()); };
    device::DeviceRouteExperts<half_t, Scoring> route;
    auto rarg = route.MakeArgument(halves(*dlogits), nullptr, nullptr, ints(dids), floats(dweights), ints(doffsets), ints(drows), ints(dplaces), T, E, k, E);
    ckx::DeviceMem ws(route.GetWorkSpaceSize(&rarg));
    if(ws.GetBufferSize() > 0)
        route.SetWorkSpacePointer(&rarg, ws.GetDeviceBuffer());
    run_one(route, rarg, "the router", time_kernel, nrepeat, (double)T * E, 2.0 * T * E + 16.0 * pairs, false);
    device::DeviceTokenQuantizeI8<half_t> quantize;
    run_one(quantize, quantize.MakeArgument(halves(*dx), codes(dq), floats(ds), T, hidden, hidden, hidden), "the quantiser", time_kernel, nrepeat,
            3.0 * T * hidden, 3.0 * T * hidden, false);
    const double used = std::min(E, pairs); // experts' matrices that are read
    device::DeviceExpertsGemmI8<half_t, true> gemm_up;
    run_one(gemm_up,
            gemm_up.MakeArgument(codes(dq), codes(*dup), halves(dh), floats(ds), floats(*dsup), nullptr, ints(doffsets), ints(drows), pairs, T, E, inner,
                                 hidden, hidden, hidden, inner, (int64_t)2 * inner * hidden, k),
            "the experts' first product", time_kernel, nrepeat, 4.0 * pairs * inner * hidden,
            used * 2 * inner * hidden + (double)T * hidden + 2.0 * pairs * inner, true);
    run_one(quantize, quantize.MakeArgument(halves(dh), codes(dqh), floats(dsh), pairs, inner, inner, inner), "the quantiser", time_kernel, nrepeat,
            3.0 * pairs * inner, 3.0 * pairs * inner, false);
    device::DeviceExpertsGemmI8<half_t> gemm_down;
    run_one(gemm_down,
            gemm_down.MakeArgument(codes(dqh), codes(*ddown), halves(dy), floats(dsh), floats(*dsdown), nullptr, ints(doffsets), nullptr, pairs, pairs, E,
                                   hidden, inner, inner, inner, hidden, (int64_t)hidden * inner),
            "the experts' second product", time_kernel, nrepeat, 2.0 * pairs * hidden * inner,
            used * hidden * inner + (double)pairs * inner + 2.0 * pairs * hidden, true);
    device::DeviceExpertsCombine<half_t> combine;
    run_one(combine,
            combine.MakeArgument(halves(dy), ints(dplaces), floats(dweights), nullptr, halves(dout), T, k, pairs, hidden, hidden, 0, hidden),
            "the weighted sum", time_kernel, nrepeat, 2.0 * pairs * hidden, 2.0 * (pairs + (double)T) * hidden, false);
    const auto out = from_device<half_t>(dout);
    if(const char* path = std::getenv("CKX_PROFILER_DUMP"))
        ckx::dump_to_file(path, out);
    if(!verify)
        return 0;
    const auto ids = from_device<index_t>(dids), offsets = from_device<index_t>(doffsets), rows = from_device<index_t>(drows), places = from_device<index_t>(dplaces);
    const auto weights = from_device<float>(dweights), s = from_device<float>(ds), sh = from_device<float>(dsh);
    const auto q = from_device<int8_t>(dq), qh = from_device<int8_t>(dqh);
    const auto h = from_device<half_t>(dh), y = from_device<half_t>(dy);
    bool pass    = true;
    auto check   = [&](const char* what, auto errors) {
        std::size_t checked = 0;
        const std::size_t bad = errors(checked);
        pass                  = verified(what, bad, checked) && pass;
        return bad == 0;
    };
    if(!check("DeviceRouteExperts", [&](std::size_t& n) {
           return ckx::route_errors([&](std::size_t t, int e) { return (double)logits[t * E + e]; },
                                    ckx::RouteView{ids.data(), offsets.data(), rows.data(), places.data(), weights.data(), T, E, k,
                                                   Scoring == device::ExpertScoring::Sigmoid, true},
                                    n);
       }))
        return 1; // (the tables are indices below)
    auto expert_of = [&](std::size_t i) { return (std::size_t)ids[rows[i]]; };
    check("DeviceTokenQuantizeI8", [&](std::size_t& n) {
        return ckx::token_quantise_errors([&](std::size_t m, int j) { return (double)x[m * hidden + j]; }, q.data(), s.data(), T, hidden, n);
    });
    check("DeviceExpertsGemmI8, gated", [&](std::size_t& n) {
        return ckx::gemm_i8_errors([&](std::size_t m, std::size_t j) { return (double)h[m * inner + j]; },
                                   [&](std::size_t m, std::size_t& row, std::size_t& expert) { row = rows[m] / k, expert = expert_of(m); },
                                   ckx::GemmI8View{q.data(), up.data(), s.data(), s_up.data(), pairs, inner, hidden, true}, 0x1p-11, n);
    });
    check("DeviceTokenQuantizeI8", [&](std::size_t& n) {
        return ckx::token_quantise_errors([&](std::size_t m, int j) { return (double)h[m * inner + j]; }, qh.data(), sh.data(), pairs, inner, n);
    });
    check("DeviceExpertsGemmI8", [&](std::size_t& n) {
        return ckx::gemm_i8_errors([&](std::size_t m, std::size_t j) { return (double)y[m * hidden + j]; },
                                   [&](std::size_t m, std::size_t& row, std::size_t& expert) { row = m, expert = expert_of(m); },
                                   ckx::GemmI8View{qh.data(), down.data(), sh.data(), s_down.data(), pairs, hidden, inner, false}, 0x1p-11, n);
    });
    check("DeviceExpertsCombine", [&](std::size_t& n) {
        return ckx::combine_errors([&](std::size_t t, std::size_t j) { return (double)out[t * hidden + j]; },
                                   [&](std::size_t i, std::size_t j) { return (double)y[i * hidden + j]; }, places.data(), weights.data(), T, k, pairs, hidden,
                                   0x1p-11, n);
    });
    return pass ? 0 : 1;
}

int profile_experts_i8(int argc, char* argv[])
{
    if(argc < 12)
    {
        std::printf("arg1: tensor operation (experts_i8)\narg2: scores (1: softmax, 2: sigmoid)\narg3: verification\narg4: initialization\n"
                    "arg5: print tensor value\narg6: time kernel\narg7 to 11: Tokens, Experts, TopK, Hidden, Inner\nlast: nrepeat\n");
        return 1;
    }
    int p[5];
    for(int i = 0; i < 5; ++i)
        p[i] = std::atoi(argv[7 + i]);
    if(*std::min_element(p, p + 5) < 1 || p[2] > p[1])
        throw std::runtime_error("sizes are at least 1, TopK at most Experts");
    auto* run = std::atoi(argv[2]) == 2 ? &profile_experts_i8_t<device::ExpertScoring::Sigmoid> : &profile_experts_i8_t<device::ExpertScoring::Softmax>;
    return run(std::atoi(argv[3]) != 0, std::atoi(argv[4]), std::atoi(argv[6]) != 0, p[0], p[1], p[2], p[3], p[4], argc > 12 ? std::atoi(argv[12]) : 10);
}

} // namespace

int main(int argc, char* argv[])
{
    try
    {
        if(argc >= 2 && std::strcmp(argv[1], "gemm") == 0)
            return profile_gemm(argc, argv);
        if(argc >= 2 && (std::strcmp(argv[1], "conv2d_fwd") == 0 || std::strcmp(argv[1], "conv_fwd") == 0))
            return profile_conv(argc, argv);
        if(argc >= 2 && std::strcmp(argv[1], "batched_gemm_gemm") == 0)
            return profile_gemm_gemm(argc, argv);
        if(argc >= 2 && std::strcmp(argv[1], "batched_gemm_softmax_gemm") == 0)
            return profile_gemm_softmax_gemm(argc, argv);
        if(argc >= 2 && std::strcmp(argv[1], "convnd_fwd") == 0)
            return profile_convnd(argc, argv);
        if(argc >= 2 && std::strcmp(argv[1], "conv_fwd_bias_relu") == 0)
            return profile_conv_bias_relu(argc, argv, false);
        if(argc >= 2 && std::strcmp(argv[1], "conv_fwd_bias_relu_add") == 0)
            return profile_conv_bias_relu(argc, argv, true);
        if(argc >= 2 && std::strcmp(argv[1], "batched_gemm") == 0)
            return profile_batched_gemm(argc, argv);
        if(argc >= 2 && std::strcmp(argv[1], "gemm_splitk") == 0)
            return profile_gemm_splitk(argc, argv);
        if(argc >= 2 && std::strcmp(argv[1], "gemm_perchannel_quant") == 0)
            return profile_gemm_perchannel_quant(argc, argv);
        if(argc >= 2 && std::strcmp(argv[1], "gemm_bias_relu") == 0)
            return profile_gemm_bias_relu(argc, argv);
        if(argc >= 2 && std::strcmp(argv[1], "gemm_bilinear") == 0)
            return profile_gemm_bilinear(argc, argv);
        if(argc >= 2 && std::strcmp(argv[1], "gemm_add_add_fastgelu") == 0)
            return profile_gemm_add_add_fastgelu(argc, argv);
        if(argc >= 2 && std::strcmp(argv[1], "gemm_f8_blockscale") == 0)
            return profile_gemm_f8(argc, argv);
        if(argc >= 2 && std::strcmp(argv[1], "paged_attention8") == 0)
            return profile_attention8(argc, argv);
        if(argc >= 2 && std::strcmp(argv[1], "gemm_i8_tokenscale") == 0)
            return profile_gemm_i8(argc, argv);
        if(argc >= 2 && std::strcmp(argv[1], "experts_i8") == 0)
            return profile_experts_i8(argc, argv);
        std::printf("arg1: tensor operation (gemm: GEMM\n"
                    "                        conv2d_fwd: NHWC/KYXC/NHWK forward convolution\n"
                    "                        batched_gemm_gemm: batched fused GEMM+GEMM\n"
                    "                        batched_gemm_softmax_gemm: batched fused GEMM+Softmax+GEMM\n"
                    "                        convnd_fwd: forward convolution, 1 / 2 / 3 spatial dimensions, channels last\n"
                    "                        conv_fwd_bias_relu: ForwardConvolution+Bias+ReLU\n"
                    "                        conv_fwd_bias_relu_add: ForwardConvolution+Bias+ReLU+Add\n"
                    "                        batched_gemm: Batched GEMM\n"
                    "                        gemm_splitk: Split-K GEMM\n"
                    "                        gemm_bias_relu: GEMM+Bias+ReLU\n"
                    "                        gemm_f8_blockscale: quantiser and GEMM, e4m3 with a scale for each block of 128\n"
                    "                        paged_attention8: tables, store and attention over a cache of 8-bit blocks\n"
                    "                        gemm_i8_tokenscale: quantiser and GEMM, int8 with a scale for each token and channel\n"
                    "                        experts_i8: a mixture of experts in int8)\n");
        return 1;
    }
    catch(const std::exception& e)
    {
        std::cerr << e.what() << std::endl;
        return 2;
    }
}
