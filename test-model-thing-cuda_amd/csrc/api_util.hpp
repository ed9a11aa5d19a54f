// api_util.hpp -- what the C ABI's source files share: the thread-local error
// message and the argument checks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/tmt_moe.h"

namespace tmt {

// Sets the calling thread's message (tmt_moe_last_error) and returns code.
int fail(int code, const char* fmt, ...);

inline bool aligned_to(const void* p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1u)) == 0; }
inline bool aligned16(const void* p) { return aligned_to(p, 16); }

}  // namespace tmt

#define HIP_TRY(call)                                                              \
    do {                                                                           \
        hipError_t err__ = (call);                                                 \
        if (err__ != hipSuccess)                                                   \
            return tmt::fail(TMT_MOE_EDEVICE, "%s failed: %s", #call, hipGetErrorString(err__)); \
    } while (0)
