// Shared by the C ABI's sources: the thread-local message, argument checks
// and sizes.
#pragma once

#include <glm53_moe.h>
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace glm53 {

// Records the message that glm53_last_error returns and passes `code` on.
int fail(int code, const char* fmt, ...);

inline int hip_fail(hipError_t e, const char* what) {
  return fail(GLM53_DEVICE_ERROR, "%s: %s", what, hipGetErrorString(e));
}

#define HIP_TRY(expr, what)                      \
  do {                                           \
    hipError_t _e = (expr);                      \
    if (_e != hipSuccess) return hip_fail(_e, what); \
  } while (0)

#define CHECK_ARG(cond, ...)                                        \
  do {                                                              \
    if (!(cond)) return fail(GLM53_INVALID_ARGUMENT, __VA_ARGS__);  \
  } while (0)

inline hipStream_t S(void* s) { return static_cast<hipStream_t>(s); }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
inline size_t round_up(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

}  // namespace glm53
