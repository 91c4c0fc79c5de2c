// dgnn_internal.h -- what the library's source files share and nobody else sees.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dgnn_train.h"

// Sets the calling thread's dgnn_last_error() message (printf format with one string and one number) and returns `code`.
__attribute__((visibility("hidden"))) int dgnn_fail(int code, const char* fmt, const char* a = "", long long b = 0);

#define DGNN_LAUNCHED()                                                                \
  do {                                                                                 \
    hipError_t e_ = hipGetLastError();                                                 \
    if (e_ != hipSuccess) return dgnn_fail(DGNN_E_HIP, "%s (line %lld)", hipGetErrorString(e_), __LINE__); \
  } while (0)
