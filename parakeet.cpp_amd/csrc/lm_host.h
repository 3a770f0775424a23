// lm_host.h -- what the entry points of parakeet_lm.h check and launch alike.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "last_error.h"
#include "parakeet_lm.h"

namespace pklm {

inline bool aligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
inline int log2i(int v) { return 31 - __builtin_clz((unsigned)v); }
inline bool float_type(int dtype) { return dtype == PK_DTYPE_F32 || dtype == PK_DTYPE_F16 || dtype == PK_DTYPE_BF16; }
inline int type_size(int dtype) { return dtype == PK_DTYPE_F32 ? 4 : 2; }

// A launch has fewer than 2^32 threads.
constexpr int64_t most_groups(int threads) { return UINT32_MAX / threads; }

inline int launched(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? PK_OK : pk_fail(PK_ERR_DEVICE, "%s: %s", what, hipGetErrorString(e));
}

}  // namespace pklm
