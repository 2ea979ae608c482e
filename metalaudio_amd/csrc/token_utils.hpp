// Device helpers of the token operators: values in f32, bf16 and e4m3.
#pragma once

#include "device_utils.hpp"
#include "x3.hpp"

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

// op of a lane's value and that of the lane 16 away.
template <class F>
__device__ __forceinline__ float other_row(float v, F op) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const unsigned x = r[0], y = r[1];
  return op(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}
// op over aligned groups of L lanes, the same bits in each lane of a group: neighbours, pairs, then
// mirrored halves and rows (whose parts agree by then), without LDS.
template <int L, class F>
__device__ __forceinline__ float group_reduce(float v, F op) {
  if constexpr (L > 1) v = op(v, dpp_mov<0xB1>(v));
  if constexpr (L > 2) v = op(v, dpp_mov<0x4E>(v));
  if constexpr (L > 4) v = op(v, dpp_mov<0x141>(v));
  if constexpr (L > 8) v = op(v, dpp_mov<0x140>(v));
  if constexpr (L > 16) v = other_row(v, op);
  if constexpr (L > 32) v = other_half(v, op);
  return v;
}
struct Plus {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};

// Eight consecutive values of a row as they lie in memory, 16-byte aligned.
template <class T>
struct Eight {
  typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
  static constexpr int V = (int)sizeof(T) / 2;
  uintx4 x[V];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = uintx4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = reinterpret_cast<const uintx4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < V; ++i) reinterpret_cast<uintx4*>(p)[i] = x[i];
  }
  __device__ __forceinline__ float operator[](int e) const {
    unsigned u;
    if constexpr (sizeof(T) == 4)
      u = x[e / 4][e % 4];
    else
      u = e & 1 ? x[0][e / 2] & 0xffff0000u : x[0][e / 2] << 16;
    return __builtin_bit_cast(float, u);
  }
  __device__ __forceinline__ void set(const float* v) {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 4)
          x[i][e] = __builtin_bit_cast(unsigned, v[4 * i + e]);
        else
          x[i][e] = cvt_pk_bf16(v[2 * e], v[2 * e + 1]);
      }
  }
};

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
