// Rows of whole sequences into rolling caches and back: a head's row of hd values of a token by L lanes, eight
// values each, in 8 bits with a scale a row or as they are.
#include <algorithm>

#include "kv_slots.hpp"
#include "lds_dma.hpp"
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

// The row of an unrounded cache, or the rows of keys and values: all of a lane's loads go out before the first is used.
// Bound by memory and, at the sizes of a few chunks, by one trip to it: 4 x 2688 tokens' keys and values of 8 heads of 48 in f32,
// 2053 slots (32 MB read and written) 7.6 us, 4.2 TB/s; 2 x 16384 tokens of 8 heads of 64 read back to bf16 (103 MB) 17.6 us, 5.8 TB/s.
template <class T, int L, bool HELD, bool WRITE>
__global__ __launch_bounds__(256) void kv_cache_kernel(KVCacheArgs a, FastDiv by_heads) {
  constexpr int UNITS = 256 / L;  // a workgroup
  const int j = threadIdx.x % L, hd = a.hd, b = blockIdx.y;
  const bool on = 8 * j < hd;
  const int u = blockIdx.x * UNITS + threadIdx.x / L, i = by_heads(u), head = u - i * a.KV;
  if (i >= a.T) return;
  int pos;
  const int64_t at = (((int64_t)b * a.T + i) * a.KV + head) * hd + 8 * j;
  T* const rows[2] = {static_cast<T*>(a.rows[0]) + at, static_cast<T*>(a.rows[1]) + at};
  Eight<T> e[2];
  // rows that surely stay are on their way while the stream's position is
  const bool early = WRITE && a.T <= a.C - a.sinks;
  e[0].clear();
  e[1].clear();
  if (early && on) {
    e[0].load(rows[0]);
    e[1].load(rows[1]);
  }
  const int n = kv_rows(a.pos, a.steps, b, a.T, pos);
  if (i >= n || (WRITE && !stays(a, pos + i, i, n))) return;
  if (WRITE && !early && on) {
    e[0].load(rows[0]);
    e[1].load(rows[1]);
  }
  const int64_t slot = ((int64_t)b * a.C + kv_slot(pos + i, a.sinks, a.C)) * a.KV + head, to = slot * hd + 8 * j;
  if constexpr (!HELD) {
    T* const cache[2] = {static_cast<T*>(a.cache[0]) + to, static_cast<T*>(a.cache[1]) + to};
    if (!on) return;
    if (!WRITE) {
      e[0].load(cache[0]);
      e[1].load(cache[1]);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) e[x].store(WRITE ? cache[x] : rows[x]);
  } else if constexpr (WRITE) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float v[8], scale;
#pragma unroll
      for (int d = 0; d < 8; ++d) v[d] = e[x][d];
      const uint2 q = round_row<L>(v, scale);
      if (on) *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.cache[x]) + to) = q;
      if (j == 0) a.scales[x][slot] = scale;
    }
  } else if (on) {
    uint2 q[2];
    float scale[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      q[x] = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.cache[x]) + to);
      scale[x] = a.scales[x][slot];
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float v[8];
      widen_row(q[x], v);
#pragma unroll
      for (int d = 0; d < 8; ++d) v[d] *= scale[x];
      e[x].set(v);
      e[x].store(rows[x]);
    }
  }
}

template <class T, int L, bool HELD, bool WRITE>
void launch_l(const LaunchCtx& c, const KVCacheArgs& a) {
  const int64_t units = (int64_t)a.T * a.KV, wgs = (units + 256 / L - 1) / (256 / L);
  MNN_REQUIRE(units <= (1 << 30) && wgs * a.B < (1 << 24), MNN_ERR_INVALID_CONFIGURATION,  // 2^32 lanes
              "KVCache: too many tokens in one call");
  launch(c, WRITE ? "kv_cache_write" : "kv_cache_read", kv_cache_kernel<T, L, HELD, WRITE>,
         dim3((unsigned)wgs, (unsigned)a.B), dim3(256), 0, a, FastDiv(a.KV));
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
