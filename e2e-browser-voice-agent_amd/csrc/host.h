// host.h -- what the library's translation units share on the host: the error message of the calling
// thread and the checks of device pointers.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>

#include "q4hip.h"

namespace q4 {

// Sets the calling thread's message (q4hip_last_error) and returns `code`.
int fail(int code, const char* fmt, ...);

// `bytes` of device memory of `device` start at p (checked before any launch, so a host pointer or
// a short buffer is an error, not a memory fault).
int check_device_span(const void* p, size_t bytes, int device, const char* what);

}  // namespace q4

#define HIPCHK(call)                                                                   \
  do {                                                                                 \
    hipError_t e_ = (call);                                                            \
    if (e_ != hipSuccess) return q4::fail(Q4HIP_EHIP, "%s: %s", #call, hipGetErrorString(e_)); \
  } while (0)
