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

// op of a lane's value and that of the lane 32 away.
template <class F>
__device__ __forceinline__ float other_half(float v, F op) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned x = r[0], y = r[1];  // as values: a bit cast of r[1] itself reads r[0]
  return op(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}

// c + the two bf16 values in x.
__device__ __forceinline__ float add_pair(unsigned x, float c) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x),
                                         __builtin_bit_cast(bf16x2, 0x3f803f80u), c, false);
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
