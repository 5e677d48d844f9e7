// gpsr_host.hpp -- host helpers shared by the translation units of libgpsr.so (not exported).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>

#define GPSR_HIDDEN __attribute__((visibility("hidden")))

// Both keep the text for gpsr_last_error() and return the status of the entry point.
GPSR_HIDDEN int hip_fail(hipError_t e, const char* where);
GPSR_HIDDEN int arg_fail(const char* what);

#define CHECK_LAUNCH(where)                                 \
  do {                                                      \
    hipError_t e_ = hipGetLastError();                      \
    if (e_ != hipSuccess) return hip_fail(e_, where);       \
  } while (0)

static inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
