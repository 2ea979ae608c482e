// Window attention of the next tokens of each stream on rolling caches in 8 bits: the simplest form.
#include "kv_slots.hpp"
#include "token_ops.hpp"
#include "window_row.hpp"

namespace mnn {
namespace k {

using namespace dev;

namespace {

// The call's rows to the caches.
template <class T>
void write_rows(const LaunchCtx& c, const WindowStepHeldArgs& a) {
  KVCacheArgs w;
  w.rows[0] = const_cast<void*>(a.k);
  w.rows[1] = const_cast<void*>(a.v);
  w.cache[0] = a.kc;
  w.cache[1] = a.vc;
  w.scales[0] = a.ks;
  w.scales[1] = a.vs;
  w.type = a.type;
  w.pos = a.pos;
  w.steps = a.steps;
  w.B = a.B;
  w.T = a.T;
  w.C = a.C;
  w.KV = a.KV;
  w.hd = a.hd;
  w.sinks = a.sinks;
  kv_cache_write(c, w);
}

template <class T>
__global__ __launch_bounds__(64) void step_rows_kernel(WindowStepHeldArgs a) {
  const int lane = threadIdx.x, h = blockIdx.x % a.H, t = blockIdx.x / a.H % a.T, b = blockIdx.x / a.H / a.T;
  int pos;
  if (t >= kv_rows(a.pos, a.steps, b, a.T, pos)) return;
  const int i = pos + t, lo = max(0, i - a.left), ns = min(a.sinks, lo), head = h / (a.H / a.KV);
  auto row = [&](int64_t n, const void* cache, const float* scales) {
    const int p = (int)(n < ns ? n : lo + (n - ns));
    const int64_t at = ((int64_t)b * a.C + kv_slot(p, a.sinks, a.C)) * a.KV + head;
    return E4m3Row{static_cast<const uint8_t*>(cache) + at * a.hd, scales[at]};
  };
  const int64_t at = (((int64_t)b * a.T + t) * a.H + h) * a.hd;
  float o0, o1;
  window_row(static_cast<const T*>(a.q) + at, a.hd, a.scale, (int64_t)ns + (i - lo + 1),
             [&](int64_t n) { return row(n, a.kc, a.ks); }, [&](int64_t n) { return row(n, a.vc, a.vs); }, o0, o1);
  T* o = static_cast<T*>(a.o) + at;
  if (lane < a.hd) o[lane] = from_f32<T>(o0);
  if (lane + 64 < a.hd) o[lane + 64] = from_f32<T>(o1);
}

}  // namespace

int64_t window_step_e4m3_part_floats(const LaunchCtx&, const WindowStepHeldArgs&) { return 0; }

void window_step_e4m3(const LaunchCtx& c, const WindowStepHeldArgs& a, float*) {
  const int64_t rows = (int64_t)a.B * a.T * a.H;
  MNN_REQUIRE(rows < (1 << 24), MNN_ERR_INVALID_CONFIGURATION, "WindowAttention: too many streams and tokens in one step");
  if (a.type == MNN_F32) {
    write_rows<float>(c, a);
    launch(c, "step_rows_f32", step_rows_kernel<float>, dim3((unsigned)rows), dim3(64), 0, a);
  } else {
    write_rows<__bf16>(c, a);
    launch(c, "step_rows_bf16", step_rows_kernel<__bf16>, dim3((unsigned)rows), dim3(64), 0, a);
  }
}

}  // namespace k
}  // namespace mnn
