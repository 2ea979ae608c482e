// Attention of a decoder's tokens to an encoder's states: the simplest form.
#include "kv_slots.hpp"
#include "token_ops.hpp"
#include "window_row.hpp"

namespace mnn {
namespace k {

using namespace dev;

namespace {

template <class T, class M>
__global__ __launch_bounds__(64) void memory_rows_kernel(MemoryArgs a) {
  const int lane = threadIdx.x, h = blockIdx.x % a.H, t = blockIdx.x / a.H % a.T, b = blockIdx.x / a.H / a.T;
  const int tn = a.qlen ? min(max(a.qlen[b], 0), a.T) : a.T, n = a.len ? min(max(a.len[b], 0), a.S) : a.S;
  if (t >= tn) return;
  const int head = h / (a.H / a.KV);
  auto row = [&](int64_t i, const void* x, const float* scales) {
    const int64_t at = ((int64_t)b * a.S + i) * a.KV + head;
    if constexpr (sizeof(M) == 1)
      return E4m3Row{static_cast<const uint8_t*>(x) + at * a.hd, scales[at]};
    else
      return static_cast<const T*>(x) + at * a.hd;
  };
  const int64_t at = (((int64_t)b * a.T + t) * a.H + h) * a.hd;
  float o0 = 0.f, o1 = 0.f;
  if (n > 0)
    window_row(static_cast<const T*>(a.q) + at, a.hd, a.scale, (int64_t)n, [&](int64_t i) { return row(i, a.k, a.ks); },
               [&](int64_t i) { return row(i, a.v, a.vs); }, o0, o1);
  T* o = static_cast<T*>(a.o) + at;
  if (lane < a.hd) o[lane] = from_f32<T>(o0);
  if (lane + 64 < a.hd) o[lane + 64] = from_f32<T>(o1);
}

template <class T>
void memory_t(const LaunchCtx& c, const MemoryArgs& a) {
  const int64_t rows = (int64_t)a.B * a.T * a.H;
  MNN_REQUIRE(rows < (1 << 24), MNN_ERR_INVALID_CONFIGURATION, "MemoryAttention: too many tokens in one call");
  const dim3 grid((unsigned)rows);
  if (a.ks)
    launch(c, "memory_rows", memory_rows_kernel<T, uint8_t>, grid, dim3(64), 0, a);
  else
    launch(c, "memory_rows", memory_rows_kernel<T, T>, grid, dim3(64), 0, a);
}

}  // namespace

int64_t memory_part_floats(const LaunchCtx&, const MemoryArgs&) { return 0; }
void memory_attention(const LaunchCtx& c, const MemoryArgs& a, float*) {
  a.type == MNN_F32 ? memory_t<float>(c, a) : memory_t<__bf16>(c, a);
}

}  // namespace k
}  // namespace mnn
