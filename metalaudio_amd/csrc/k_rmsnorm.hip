// RMS norm with the residual's addition before it and an output of 32, 16 or 8 bits:
// h = x + r, y = h * rsqrt(mean(h^2) + eps) * w, and for 8 bits q = e4m3(y * (448 * (1 / max|y|))) with
// the row's scale max|y| * (1 / 448). Without weights, the rows of x are rounded to 8 bits as they are.
// h, its sum of squares and y stay in fp32; the norm is taken of h before it is rounded to the sum's type.
#include "token_ops.hpp"
#include "token_utils.hpp"

#include <algorithm>
#include <type_traits>

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

// Rows of up to 4096 values, a multiple of 8: a wave a row, which stays in its registers from the first read
// to the last write, lane l holding values 512 i + 8 l .. + 7; the weights too, over all of a wave's rows.
// Bound by memory (two loads and two stores a value).
template <class T, int NV, mnn_dtype OUT>
__global__ __launch_bounds__(256) void rmsnorm_wave_kernel(RmsNormArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t step = (int64_t)gridDim.x * 4;
  float w[NV][8];
  bool on[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    on[i] = 512 * i + 8 * lane < a.F;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[i][e] = a.w && on[i] ? a.w[512 * i + 8 * lane + e] : 1.f;
  }
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < a.rows; row += step) {
    const int64_t at = row * a.F + 8 * lane;
    Eight<T> x[NV], r[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i].clear();
      r[i].clear();
      if (on[i]) {
        x[i].load(static_cast<const T*>(a.x) + at + 512 * i);
        if (a.r) r[i].load(static_cast<const T*>(a.r) + at + 512 * i);
      }
    }
    float h[NV][8], ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[i][e] = a.r ? x[i][e] + r[i][e] : x[i][e];
        ss = fmaf(h[i][e], h[i][e], ss);
      }
    if (a.sum) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (on[i]) {
          Eight<T> o;
          o.set(h[i]);
          o.store(static_cast<T*>(a.sum) + at + 512 * i);
        }
    }
    float top = 0.f;
    if (a.w) {
      const float norm = rsqrtf(group_reduce<64>(ss, Plus{}) / (float)a.F + a.eps);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] = h[i][e] * norm * w[i][e];
    }
    if constexpr (OUT == MNN_E4M3) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (on[i]) top = max_nan(top, fabsf(h[i][e]));
      const RowScale rs = row_scale(group_reduce<64>(top, max_nan));
      if (lane == 0) a.scales[row] = rs.scale;
      uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.ldy + 8 * lane;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const float* v = h[i];
        if (on[i])
          *reinterpret_cast<uint2*>(y + 512 * i) =
              make_uint2(pack_e4m3(v[0] * rs.inv, v[1] * rs.inv, v[2] * rs.inv, v[3] * rs.inv),
                         pack_e4m3(v[4] * rs.inv, v[5] * rs.inv, v[6] * rs.inv, v[7] * rs.inv));
        else if (512 * i + 8 * lane < a.ldy)
          *reinterpret_cast<uint2*>(y + 512 * i) = make_uint2(0, 0);
      }
    } else {
      using O = std::conditional_t<OUT == MNN_F32, float, __bf16>;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (on[i]) {
          Eight<O> o;
          o.set(h[i]);
          o.store(static_cast<O*>(a.y) + row * a.ldy + 512 * i + 8 * lane);
        }
    }
  }
}

template <class T, int NV>
void launch_wave(const LaunchCtx& c, const RmsNormArgs& a) {
  const char* name = sizeof(T) == 4 ? "rmsnorm_wave_f32" : "rmsnorm_wave_bf16";
  // eight workgroups a compute unit keep their weights over several rows
  const dim3 grid((unsigned)std::min<int64_t>((a.rows + 3) / 4, 8 * c.dev->props.multiProcessorCount));
  if (a.out == MNN_E4M3)
    launch(c, name, rmsnorm_wave_kernel<T, NV, MNN_E4M3>, grid, dim3(256), 0, a);
  else if (a.out == MNN_BF16)
    launch(c, name, rmsnorm_wave_kernel<T, NV, MNN_BF16>, grid, dim3(256), 0, a);
  else
    launch(c, name, rmsnorm_wave_kernel<T, NV, MNN_F32>, grid, dim3(256), 0, a);
}

template <class T>
void rmsnorm_t(const LaunchCtx& c, const RmsNormArgs& a) {
  if (a.F % 8 == 0 && a.ldy % 8 == 0 && a.ldy <= 4096) {
    switch ((a.ldy + 511) / 512) {
      case 1: return launch_wave<T, 1>(c, a);
      case 2: return launch_wave<T, 2>(c, a);
      case 3: return launch_wave<T, 3>(c, a);
      case 4: return launch_wave<T, 4>(c, a);
      case 5:
      case 6: return launch_wave<T, 6>(c, a);
      default: return launch_wave<T, 8>(c, a);
    }
  }
  launch(c, sizeof(T) == 4 ? "rmsnorm_any_f32" : "rmsnorm_any_bf16", rmsnorm_any_kernel<T>,
         dim3((unsigned)std::min<int64_t>(a.rows, 1 << 20)), dim3(256), 0, a);
}

}  // namespace

void rmsnorm(const LaunchCtx& c, const RmsNormArgs& a) {
  if (a.rows <= 0 || a.F <= 0) return;
  if (a.in == MNN_F32)
    rmsnorm_t<float>(c, a);
  else
    rmsnorm_t<__bf16>(c, a);
}

}  // namespace k
}  // namespace mnn
