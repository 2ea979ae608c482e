// Device helpers of the token operators: values in f32, bf16 and e4m3.
#pragma once

#include "device_utils.hpp"

namespace mnn {
namespace dev {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__bf16 x) { return (float)x; }
template <class T>
__device__ __forceinline__ T from_f32(float x) {
  return (T)x;  // bf16: to nearest even
}

// Maximum that keeps NaN (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
  return __builtin_elementwise_maximum(a, b);
}

// Scale of an e4m3 row from its largest magnitude: a value is kept as x * inv. No clamp is needed behind
// it: x * (448 * (1 / max)) is above 448 by three roundings at most, and all up to 464 round to 448.
constexpr float kE4m3Max = 448.f;
struct RowScale {
  float scale, inv;
};
__device__ __forceinline__ RowScale row_scale(float top) {
  top = max_nan(top, 0x1p-100f);
  return {top * (1.f / kE4m3Max), kE4m3Max * (1.f / top)};
}
// Four values to e4m3, to nearest even, the first in the lowest byte.
__device__ __forceinline__ unsigned pack_e4m3(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

}  // namespace dev
}  // namespace mnn
