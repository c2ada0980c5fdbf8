// The calling thread's last error message (ckx_last_error()), for the entry points outside ckx_api.hip.
#pragma once

#include <hip/hip_runtime.h>

namespace ckx {

int api_fail(int code, const char* msg);                 // keeps the message, returns `code`
int api_hip_fail(hipError_t e, const char* what);        // CKX_HIP_ERROR with HIP's text

} // namespace ckx
