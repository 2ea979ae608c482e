// RMS norm with the residual's addition before it and an output of 32, 16 or 8 bits:
// h = x + r, y = h * rsqrt(mean(h^2) + eps) * w, and for 8 bits q = e4m3(y * (448 * (1 / max|y|))) with
// the row's scale max|y| * (1 / 448). Without weights, the rows of x are rounded to 8 bits as they are.
// h, its sum of squares and y stay in fp32; the norm is taken of h before it is rounded to the sum's type.
#include "token_ops.hpp"
#include "token_utils.hpp"

namespace mnn {
namespace k {

using namespace dev;

namespace {

// One value of a row over the whole workgroup of 256.
template <class F>
__device__ __forceinline__ float block_reduce(float v, float* sh, F op) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v = op(v, __shfl_xor(v, off, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return op(op(sh[0], sh[1]), op(sh[2], sh[3]));
}

// Any row length and alignment: a workgroup per row in three passes over memory (the row's second and
// third reads come from L2). Nothing is written before the last pass, so sum and y may be x or r.
template <class T>
__global__ __launch_bounds__(256) void rmsnorm_any_kernel(RmsNormArgs a) {
  __shared__ float sh[4];
  const T* x = static_cast<const T*>(a.x);
  const T* r = static_cast<const T*>(a.r);
  T* sum = static_cast<T*>(a.sum);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t at = row * a.F;
    auto h = [&](int i) { return to_f32(x[at + i]) + (r ? to_f32(r[at + i]) : 0.f); };
    float norm = 1.f;
    if (a.w) {
      float ss = 0.f;
      for (int i = threadIdx.x; i < a.F; i += 256) ss = fmaf(h(i), h(i), ss);
      ss = block_reduce(ss, sh, [](float p, float q) { return p + q; });
      norm = rsqrtf(ss / (float)a.F + a.eps);
    }
    auto y = [&](int i, float hv) { return a.w ? hv * norm * a.w[i] : hv; };
    RowScale rs{1.f, 1.f};
    if (a.out == MNN_E4M3) {
      float top = 0.f;
      for (int i = threadIdx.x; i < a.F; i += 256) top = max_nan(top, fabsf(y(i, h(i))));
      rs = row_scale(block_reduce(top, sh, max_nan));
    }
    __syncthreads();  // every read of the row's other passes is done
    for (int64_t i = threadIdx.x; i < a.ldy; i += 256) {
      const float hv = i < a.F ? h((int)i) : 0.f;
      const float v = i < a.F ? y((int)i, hv) : 0.f;
      if (sum && i < a.F) sum[at + i] = from_f32<T>(hv);
      const int64_t o = row * a.ldy + i;
      if (a.out == MNN_E4M3)
        static_cast<uint8_t*>(a.y)[o] = (uint8_t)pack_e4m3(v * rs.inv, 0.f, 0.f, 0.f);
      else if (a.out == MNN_BF16)
        static_cast<__bf16*>(a.y)[o] = (__bf16)v;
      else
        static_cast<float*>(a.y)[o] = v;
    }
    if (a.out == MNN_E4M3 && threadIdx.x == 0) a.scales[row] = rs.scale;
  }
}

}  // namespace

void rmsnorm(const LaunchCtx& c, const RmsNormArgs& a) {
  if (a.rows <= 0 || a.F <= 0) return;
  const dim3 grid((unsigned)std::min<int64_t>(a.rows, 1 << 20));
  if (a.in == MNN_F32)
    launch(c, "rmsnorm_any_f32", rmsnorm_any_kernel<float>, grid, dim3(256), 0, a);
  else
    launch(c, "rmsnorm_any_bf16", rmsnorm_any_kernel<__bf16>, grid, dim3(256), 0, a);
}

}  // namespace k
}  // namespace mnn
