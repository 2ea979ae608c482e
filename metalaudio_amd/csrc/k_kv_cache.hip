// Rows of whole sequences into rolling caches and back: a head's row of hd values of a token by L lanes, eight
// values each, in 8 bits with a scale a row or as they are.
#include <algorithm>

#include "kv_slots.hpp"
#include "token_ops.hpp"

namespace mnn {
namespace k {

using namespace dev;

namespace {

// Of rows i of n that a stream writes, only the last of those that share a slot does: behind the sinks, the last
// C - sinks rows. So no two lanes write one place, and the result does not depend on their order.
__device__ __forceinline__ bool stays(const KVCacheArgs& a, int p, int i, int n) {
  return p < a.sinks || i >= n - (a.C - a.sinks);
}

template <class T, int L, bool HELD, bool WRITE>
__global__ __launch_bounds__(256) void kv_cache_kernel(KVCacheArgs a, int64_t units) {
  const int j = threadIdx.x % L, hd = a.hd;
  const bool on = 8 * j < hd;
  for (int64_t u = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L; u < units; u += (int64_t)gridDim.x * (256 / L)) {
    const int head = (int)(u % a.KV), i = (int)(u / a.KV % a.T), b = (int)(u / a.KV / a.T);
    int pos;
    const int n = kv_rows(a.pos, a.steps, b, a.T, pos);
    if (i >= n || (WRITE && !stays(a, pos + i, i, n))) continue;
    const int64_t slot = (int64_t)b * a.C + kv_slot(pos + i, a.sinks, a.C);
    const int64_t at = u * hd + 8 * j, to = (slot * a.KV + head) * hd + 8 * j;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      T* row = static_cast<T*>(a.rows[x]) + at;
      Eight<T> e;
      e.clear();
      if constexpr (!HELD) {
        T* cache = static_cast<T*>(a.cache[x]) + to;
        if (on) {
          e.load(WRITE ? row : cache);
          e.store(WRITE ? cache : row);
        }
      } else {
        uint2* cache = reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.cache[x]) + to);
        float* scale = a.scales[x] + slot * a.KV + head;
        float v[8];
        if constexpr (WRITE) {
          if (on) e.load(row);
#pragma unroll
          for (int d = 0; d < 8; ++d) v[d] = e[d];
          float s;
          const uint2 q = round_row<L>(v, s);
          if (on) *cache = q;
          if (j == 0) *scale = s;
        } else if (on) {
          widen_row(*cache, v);
          const float s = *scale;
#pragma unroll
          for (int d = 0; d < 8; ++d) v[d] *= s;
          e.set(v);
          e.store(row);
        }
      }
    }
  }
}

template <class T, int L, bool HELD, bool WRITE>
void launch_l(const LaunchCtx& c, const KVCacheArgs& a) {
  const int64_t units = (int64_t)a.B * a.T * a.KV;
  const dim3 grid((unsigned)std::min<int64_t>((units + 256 / L - 1) / (256 / L), 1 << 20));
  launch(c, WRITE ? "kv_cache_write" : "kv_cache_read", kv_cache_kernel<T, L, HELD, WRITE>, grid, dim3(256), 0, a, units);
}
template <class T, bool WRITE>
void launch_t(const LaunchCtx& c, const KVCacheArgs& a) {
  auto go = [&](auto held) {
    constexpr bool H = decltype(held)::value;
    if (a.hd > 64) return launch_l<T, 16, H, WRITE>(c, a);
    if (a.hd > 32) return launch_l<T, 8, H, WRITE>(c, a);
    launch_l<T, 4, H, WRITE>(c, a);
  };
  if (a.scales[0])
    go(std::true_type{});
  else
    go(std::false_type{});
}

}  // namespace

void kv_cache_write(const LaunchCtx& c, const KVCacheArgs& a) {
  a.type == MNN_F32 ? launch_t<float, true>(c, a) : launch_t<__bf16, true>(c, a);
}
void kv_cache_read(const LaunchCtx& c, const KVCacheArgs& a) {
  a.type == MNN_F32 ? launch_t<float, false>(c, a) : launch_t<__bf16, false>(c, a);
}

}  // namespace k
}  // namespace mnn
