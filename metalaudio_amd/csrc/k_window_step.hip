// Window attention of the next tokens of each stream on rolling caches. Token p lives in slot p (p < sinks)
// or sinks + (p - sinks) % (C - sinks). A call reads the tokens before it from the cache and its own from
// its inputs, so the new rows can be written to the cache in the same launch: with C >= sinks + left + T,
// none of the slots that they take holds a token that a query of the call still sees.
#include "token_ops.hpp"
#include "window_row.hpp"

#include <climits>

namespace mnn {
namespace k {

using namespace dev;

namespace {

// Rows of this call that are tokens of stream b, and the stream's position; 0 where it is left alone.
__device__ __forceinline__ int rows_of(const WindowStepArgs& a, int b, int& pos) {
  pos = a.pos[b];
  if (pos < 0 || pos > INT_MAX - a.T) return 0;
  return a.steps ? min(max(a.steps[b], 0), a.T) : a.T;
}

__device__ __forceinline__ int slot_of(const WindowStepArgs& a, int p) {
  return p < a.sinks ? p : a.sinks + (p - a.sinks) % (a.C - a.sinks);
}

// A wave per query and head; the first head of each group writes the token's key and value.
template <class T>
__global__ __launch_bounds__(64) void window_step_any_kernel(WindowStepArgs a) {
  const int lane = threadIdx.x, h = blockIdx.x, t = blockIdx.y, b = blockIdx.z;
  int pos;
  if (t >= rows_of(a, b, pos)) return;
  const int group = a.H / a.KV, kvw = a.KV * a.hd, i = pos + t;
  const int64_t col = (int64_t)(h / group) * a.hd;
  const T* kn = static_cast<const T*>(a.k) + (int64_t)b * a.T * kvw + col;
  const T* vn = static_cast<const T*>(a.v) + (int64_t)b * a.T * kvw + col;
  T* kc = static_cast<T*>(a.kc) + (int64_t)b * a.C * kvw + col;
  T* vc = static_cast<T*>(a.vc) + (int64_t)b * a.C * kvw + col;
  const int lo = max(0, i - a.left), ns = min(a.sinks, lo);
  auto row = [&](int64_t n, const T* cache, const T* fresh) {
    const int p = (int)(n < ns ? n : lo + (n - ns));
    return p >= pos ? fresh + (int64_t)(p - pos) * kvw : cache + (int64_t)slot_of(a, p) * kvw;
  };
  const int64_t at = ((int64_t)b * a.T + t) * a.H * a.hd + (int64_t)h * a.hd;
  float o0, o1;
  window_row(static_cast<const T*>(a.q) + at, a.hd, a.scale, (int64_t)ns + (i - lo + 1),
             [&](int64_t n) { return row(n, kc, kn); }, [&](int64_t n) { return row(n, vc, vn); }, o0, o1);
  T* o = static_cast<T*>(a.o) + at;
  if (lane < a.hd) o[lane] = from_f32<T>(o0);
  if (lane + 64 < a.hd) o[lane + 64] = from_f32<T>(o1);
  if (h % group == 0) {
    const int64_t to = (int64_t)slot_of(a, i) * kvw, from = (int64_t)t * kvw;
    for (int d = lane; d < a.hd; d += 64) {
      kc[to + d] = kn[from + d];
      vc[to + d] = vn[from + d];
    }
  }
}

}  // namespace

void window_step(const LaunchCtx& c, const WindowStepArgs& a) {
  const dim3 grid(a.H, a.T, a.B);
  if (a.type == MNN_F32)
    launch(c, "window_step_any_f32", window_step_any_kernel<float>, grid, dim3(64), 0, a);
  else
    launch(c, "window_step_any_bf16", window_step_any_kernel<__bf16>, grid, dim3(64), 0, a);
}

}  // namespace k
}  // namespace mnn
