// Window attention over whole sequences: o_i = sum_j p_ij v_j, p_i = softmax of scale q_i k_j over the keys
// j <= i + right with j >= i - left or j < sinks.
#include "token_ops.hpp"
#include "window_row.hpp"

namespace mnn {
namespace k {

using namespace dev;

namespace {

template <class T>
__device__ __forceinline__ void window_query(const WindowArgs& a, int b, int h, int i, int len) {
  const int lane = threadIdx.x & 63, kvw = a.KV * a.hd;
  const int lo = max(0, i - a.left), hi = (int)min((int64_t)len - 1, (int64_t)i + a.right);
  const int ns = min(a.sinks, lo);
  const int64_t col = (int64_t)(h / (a.H / a.KV)) * a.hd;
  const T* k = static_cast<const T*>(a.k) + (int64_t)b * a.S * kvw + col;
  const T* v = static_cast<const T*>(a.v) + (int64_t)b * a.S * kvw + col;
  auto key = [&](int64_t t) { return t < ns ? t : lo + (t - ns); };
  const int64_t at = ((int64_t)b * a.S + i) * a.H * a.hd + (int64_t)h * a.hd;
  float o0, o1;
  window_row(static_cast<const T*>(a.q) + at, a.hd, a.scale, (int64_t)ns + (hi - lo + 1),
             [&](int64_t t) { return k + key(t) * kvw; }, [&](int64_t t) { return v + key(t) * kvw; }, o0,
             o1);
  T* o = static_cast<T*>(a.o) + at;
  if (lane < a.hd) o[lane] = from_f32<T>(o0);
  if (lane + 64 < a.hd) o[lane + 64] = from_f32<T>(o1);
}

// A wave per query.
template <class T>
__global__ __launch_bounds__(256) void window_any_kernel(WindowArgs a) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.S) : a.S;
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < len; i += (int64_t)gridDim.x * 4)
    window_query<T>(a, b, h, (int)i, len);
}

}  // namespace

void window_attention(const LaunchCtx& c, const WindowArgs& a) {
  const dim3 grid((unsigned)std::min<int64_t>((a.S + 3) / 4, 1 << 15), a.H, a.B);
  if (a.type == MNN_F32)
    launch(c, "window_any_f32", window_any_kernel<float>, grid, dim3(256), 0, a);
  else
    launch(c, "window_any_bf16", window_any_kernel<__bf16>, grid, dim3(256), 0, a);
}

}  // namespace k
}  // namespace mnn
