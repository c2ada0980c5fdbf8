// Launcher of the 256 x 256 tiles of the token-scaled int8 GEMM and of the experts' GEMM (gemm_i8_big.hip).
#pragma once

#include "gemm_i8_scaled.hpp"

namespace ckx {

// tiles_m: tiles of 256 rows that there are at most
hipError_t gemm_i8_big_launch(GemmI8Args& a, int c_type, int64_t tiles_m, hipStream_t s);

} // namespace ckx
