// Rolling caches: where a token lives, and rows of keys or values as they are kept in 8 bits.
#pragma once

#include <climits>

#include "token_utils.hpp"

namespace mnn {
namespace dev {

// Slot of token p in a cache of C slots, the first `sinks` of which stay.
__device__ __forceinline__ int kv_slot(int p, int sinks, int C) {
  return p < sinks ? p : sinks + (p - sinks) % (C - sinks);
}

// Rows of a call that are tokens of stream b, and the stream's position; 0 where it is left alone.
__device__ __forceinline__ int kv_rows(const int* pos, const int* steps, int b, int T, int& p) {
  p = pos[b];
  if (p < 0 || p > INT_MAX - T) return 0;
  return steps ? min(max(steps[b], 0), T) : T;
}

// Eight consecutive values of a head's row, whose L lanes (those behind the row hold zeros) share its scale:
// e4m3 values, and the scale.
template <int L>
__device__ __forceinline__ uint2 round_row(const float* v, float& scale) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max_nan(top, fabsf(v[e]));
  const RowScale rs = row_scale(group_reduce<L>(top, max_nan));
  scale = rs.scale;
  return make_uint2(pack_e4m3(v[0] * rs.inv, v[1] * rs.inv, v[2] * rs.inv, v[3] * rs.inv),
                    pack_e4m3(v[4] * rs.inv, v[5] * rs.inv, v[6] * rs.inv, v[7] * rs.inv));
}

// Eight e4m3 values in 32 bits.
__device__ __forceinline__ void widen_row(uint2 q, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int word = (int)(i < 2 ? q.x : q.y);
    const auto two = i & 1 ? __builtin_amdgcn_cvt_pk_f32_fp8(word, true) : __builtin_amdgcn_cvt_pk_f32_fp8(word, false);
    v[2 * i] = two[0];
    v[2 * i + 1] = two[1];
  }
}

}  // namespace dev
}  // namespace mnn
