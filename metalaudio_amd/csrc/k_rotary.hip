// Rotary positions over several axes: pair (u, v) of axis a and rate f turns by the angle pos_a * f,
// (u cos - v sin, v cos + u sin). The angle is kept in turns: pos * (f / 2 pi) is one product in 64 bits,
// whose fraction is what is left of it, exact to 2^-53 of the whole (2e-7 turns at position 2^31), and the
// sine and cosine of that fraction are taken in fp32.
#include "token_ops.hpp"
#include "token_utils.hpp"

namespace mnn {
namespace k {

using namespace dev;

namespace {

__device__ __forceinline__ void turn_of(int pos, double rate, float& cs, float& sn) {
  const double t = (double)pos * rate;
  sincospif(2.f * (float)(t - rint(t)), &sn, &cs);
}

// A thread per token, tensor, head and dimension pair, or dimension behind the last axis.
template <class T>
__global__ __launch_bounds__(256) void rotary_any_kernel(RotaryArgs a) {
  const int units = a.pairs + (a.hd - 2 * a.pairs);  // of one head
  const int heads = a.heads[0] + a.heads[1];
  const int64_t total = a.B * a.S * heads * units;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int u = (int)(i % units);
    int h = (int)(i / units % heads);
    const int64_t tok = i / units / heads;
    const int which = h >= a.heads[0];
    if (which) h -= a.heads[0];
    const int64_t at = (tok * a.heads[which] + h) * a.hd;
    const T* x = static_cast<const T*>(a.x[which]) + at;
    T* y = static_cast<T*>(a.y[which]) + at;
    if (u >= a.pairs) {
      y[u + a.pairs] = x[u + a.pairs];
      continue;
    }
    int axis = 0, first = 0, j = u;  // pair j of the axis, whose dimensions begin at `first`
    while (j >= a.dims[axis] / 2) {
      j -= a.dims[axis] / 2;
      first += a.dims[axis++];
    }
    const int p0 = first + (a.interleaved ? 2 * j : j);
    const int p1 = a.interleaved ? p0 + 1 : p0 + a.dims[axis] / 2;
    float cs, sn;
    turn_of(a.pos[(a.shared ? tok % a.S : tok) * a.axes + axis], a.rate[u], cs, sn);
    const float v0 = to_f32(x[p0]), v1 = to_f32(x[p1]);
    y[p0] = from_f32<T>(v0 * cs - v1 * sn);
    y[p1] = from_f32<T>(v1 * cs + v0 * sn);
  }
}

}  // namespace

void rotary(const LaunchCtx& c, const RotaryArgs& a) {
  const int64_t total = a.B * a.S * (a.heads[0] + a.heads[1]) * (a.hd - a.pairs);
  const dim3 grid((unsigned)std::min<int64_t>((total + 255) / 256, 1 << 20));
  if (a.type == MNN_F32)
    launch(c, "rotary_any_f32", rotary_any_kernel<float>, grid, dim3(256), 0, a);
  else
    launch(c, "rotary_any_bf16", rotary_any_kernel<__bf16>, grid, dim3(256), 0, a);
}

}  // namespace k
}  // namespace mnn
