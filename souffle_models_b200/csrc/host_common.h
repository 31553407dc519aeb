// What the translation units of the library share on the host: the error message, CUDA error checks, alignment, the
// driver's tensor-map encoder and the properties of the current device.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/souffle_b200.h"

namespace souffle {

// Leaves the message of souffle_last_error() (one per thread) and returns `code`.
int fail(int code, const char* fmt, ...);

#define SF_CUDA(call)                                                                          \
  do {                                                                                         \
    cudaError_t e_ = (call);                                                                   \
    if (e_ != cudaSuccess)                                                                     \
      return fail(SOUFFLE_CUDA_ERROR, "%s failed: %s (%s:%d)", #call, cudaGetErrorString(e_),  \
                  __FILE__, __LINE__);                                                         \
  } while (0)

inline bool aligned16(const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Tensor maps: the driver's entry point is fetched at run time, there is no link-time libcuda dependency.
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn();

// The number of SMs of the current device, which has to be an sm_100 one; its index, below kMaxDevices, goes to *dev_out.
constexpr int kMaxDevices = 16;
int current_sms(int* sms, int* dev_out = nullptr);

}  // namespace souffle
