// Values of the types that rows and logits come in (PG_DTYPE_*), one by one in float32
// and in vectors as memory holds them.
#pragma once

#include <hip/hip_bf16.h>

#include "pg_common.h"

namespace pg {

__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __hip_bfloat16 from_float<__hip_bfloat16>(float v) {
  return __float2bfloat16(v);
}
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }

// kVec neighbouring values, loaded and stored at once.
template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) Vec {
  T v[kVec];
};

}  // namespace pg
