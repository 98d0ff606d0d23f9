// Host-side pieces that the translation units of libzepp_b200.so share: the calling thread's error message and the
// driver's tensor-map encoder.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace zepp {

// records the message that zepp_last_error() returns and yields the entry points' failure code
int fail(const char* fmt, ...);

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn();

}  // namespace zepp

#define CU_OK(expr)                                                                         \
  do {                                                                                      \
    cudaError_t _e = (expr);                                                                \
    if (_e != cudaSuccess) return fail("%s failed: %s (%s:%d)", #expr, cudaGetErrorString(_e), __FILE__, __LINE__); \
  } while (0)
