// What the files of C-ABI entry points share: the error message, status codes and checks of arguments.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bzpf.h"
#include "bzpf_kernels.h"

namespace bzpf_api {

// Sets the calling thread's message and returns the code.
int fail(int code, const char* fmt, ...);
// A launch's status as an entry point's.
int done(hipError_t e, const char* what);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool dt_ok(int dt) { return dt == BZPF_F32 || dt == BZPF_F16; }
// The training entry points: bf16 too, but not fp16 and bf16 in one call; pointers at element alignment.
inline bool dt3_ok(int dt) { return dt_ok(dt) || dt == BZPF_BF16; }
inline bool pair_ok(int a, int b) { return dt3_ok(a) && dt3_ok(b) && (a == b || a == BZPF_F32 || b == BZPF_F32); }
inline bool aligned_el(const void* p, int dt) { return (reinterpret_cast<uintptr_t>(p) & (dt == BZPF_F32 ? 3u : 1u)) == 0; }
inline hipStream_t S(void* s) { return static_cast<hipStream_t>(s); }

}  // namespace bzpf_api

#define REQUIRE(cond, ...) \
  do {                     \
    if (!(cond)) return bzpf_api::fail(BZPF_EINVAL, __VA_ARGS__); \
  } while (0)
#define REQUIRE_EL(p, dt) REQUIRE((p) != nullptr && bzpf_api::aligned_el(p, dt), "%s: %s must be non-null and aligned to its elements", __func__, #p)
#define REQUIRE_PTR(p) REQUIRE((p) != nullptr && bzpf_api::aligned16(p), "%s: %s must be a non-null 16-byte aligned pointer", __func__, #p)
