// One query of window attention by one wave, on the vector units in fp32: the keys it sees are taken 64 at
// a time, lane j scoring key j, with a running maximum and sum; the probabilities then go round by
// shuffles while each lane gathers its output dimensions d = lane and lane + 64. Keys that the query does
// not see are not read, so what they hold cannot reach it.
#pragma once

#include "token_utils.hpp"

namespace mnn {
namespace dev {

// key_at(t) / value_at(t): row pointers of the t-th of n visible keys. Returns the outputs of dimensions
// lane and lane + 64 (HD <= 128).
template <class T, class K, class V>
__device__ __forceinline__ void window_row(const T* __restrict__ q, int hd, float scale, int64_t n,
                                           K key_at, V value_at, float& o0, float& o1) {
  const int lane = threadIdx.x & 63;
  const float qs = scale * 1.4426950408889634f;  // scores in powers of two
  float m = -INFINITY, l = 0.f;
  o0 = o1 = 0.f;
  for (int64_t t0 = 0; t0 < n; t0 += 64) {
    const int cnt = (int)(n - t0 < 64 ? n - t0 : 64);
    float s = -INFINITY;
    if (lane < cnt) {
      const T* kp = key_at(t0 + lane);
      float dot = 0.f;
      for (int d = 0; d < hd; ++d) dot = fmaf(to_f32(q[d]), to_f32(kp[d]), dot);
      s = dot * qs;
    }
    float top = s;
#pragma unroll
    for (int off = 32; off; off >>= 1) top = max_nan(top, __shfl_xor(top, off, 64));
    const float mn = max_nan(m, top);
    // all scores so far -infinity: nothing is subtracted, and the probabilities are 0 (0 / 0 in the end)
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = exp2f(m - ref);
    const float p = lane < cnt ? exp2f(s - ref) : 0.f;
    m = mn;
    float ps = p;
#pragma unroll
    for (int off = 32; off; off >>= 1) ps += __shfl_xor(ps, off, 64);
    l = l * alpha + ps;
    o0 *= alpha;
    o1 *= alpha;
    for (int j = 0; j < cnt; ++j) {
      const float pj = __shfl(p, j, 64);
      const T* vp = value_at(t0 + j);
      if (lane < hd) o0 = fmaf(pj, to_f32(vp[lane]), o0);
      if (lane + 64 < hd) o1 = fmaf(pj, to_f32(vp[lane + 64]), o1);
    }
  }
  o0 /= l;
  o1 /= l;
}

}  // namespace dev
}  // namespace mnn
