// RMS norm with the residual's addition before it and an output of 32, 16 or 8 bits:
// h = x + r, y = h * rsqrt(mean(h^2) + eps) * w, and for 8 bits q = e4m3(y * (448 * (1 / max|y|))) with
// the row's scale max|y| * (1 / 448), or such a maximum and scale for each block of 128 values. Without
// weights, the rows of x are rounded to 8 bits as they are.
// h, its sum of squares and y stay in fp32; the norm is taken of h before it is rounded to the sum's type.
#include "kv_slots.hpp"
#include "lds_dma.hpp"
#include "token_ops.hpp"
#include "token_utils.hpp"

#include <algorithm>
#include <type_traits>

namespace mnn {
namespace k {

using namespace dev;

namespace {

// mean(h^2) + eps is used as it came where no square that counts has left fp32's range. Otherwise (finite
// values above 1.8e19, or, with a small eps, tiny ones) the row's norm is taken of h times a power of two that
// brings the larger of max|h| and sqrt(eps) to about 1: norm(h) = norm of s h with eps s^2.
__device__ __forceinline__ bool mean_in_range(float v) { return v > 0x1p-80f && v < INFINITY; }
__device__ __forceinline__ float unit_scale(float top, float eps) {
  const int e = __builtin_amdgcn_frexp_expf(fmaxf(top, sqrtf(eps)));
  return ldexpf(1.f, min(max(-e, -126), 127));
}

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

// Any row length: a workgroup per row in three passes over memory (the row's second and third reads come
// from L2). Nothing is written before the last pass, so sum and y may be x or r.
template <class T>
__global__ __launch_bounds__(256) void rmsnorm_any_kernel(RmsNormArgs a) {
  __shared__ float sh[4];
  const T* x = static_cast<const T*>(a.x);
  const T* r = static_cast<const T*>(a.r);
  T* sum = static_cast<T*>(a.sum);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t at = row * a.F;
    auto h = [&](int i) { return to_f32(x[at + i]) + (r ? to_f32(r[at + i]) : 0.f); };
    float norm = 1.f, s = 1.f;  // s: what h is taken times, see mean_in_range
    if (a.w) {
      auto mean = [&] {
        float ss = 0.f;
        for (int i = threadIdx.x; i < a.F; i += 256) {
          const float hv = h(i) * s;
          ss = fmaf(hv, hv, ss);
        }
        return block_reduce(ss, sh, Plus{}) / (float)a.F + a.eps * s * s;
      };
      float m = mean();
      if (!mean_in_range(m)) {
        float top = 0.f;
        for (int i = threadIdx.x; i < a.F; i += 256) top = max_nan(top, fabsf(h(i)));
        top = block_reduce(top, sh, max_nan);
        if (top < INFINITY) {
          s = unit_scale(top, a.eps);
          m = mean();
        }
      }
      norm = rsqrtf(m);
    }
    auto y = [&](int i, float hv) { return a.w ? hv * s * norm * a.w[i] : hv; };
    RowScale rs{1.f, 1.f};
    if (a.out == MNN_E4M3 && !a.blocks) {
      float top = 0.f;
      for (int i = threadIdx.x; i < a.F; i += 256) top = max_nan(top, fabsf(y(i, h(i))));
      rs = row_scale(block_reduce(top, sh, max_nan));
    }
    __syncthreads();  // every read of the row's other passes is done
    if (a.blocks) {  // a wave a block, two values a lane
      const int nb = scale_blocks(a.F), lane = threadIdx.x & 63;
      for (int64_t i0 = (threadIdx.x >> 6) * kScaleBlock; i0 < a.ldy; i0 += 4 * kScaleBlock) {
        float hv[2], v[2], top = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int64_t i = i0 + lane + 64 * e;
          hv[e] = i < a.F ? h((int)i) : 0.f;
          v[e] = i < a.F ? y((int)i, hv[e]) : 0.f;
          top = max_nan(top, fabsf(v[e]));
        }
        const RowScale bs = row_scale(group_reduce<64>(top, max_nan));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int64_t i = i0 + lane + 64 * e;
          if (sum && i < a.F) sum[at + i] = from_f32<T>(hv[e]);
          if (i < a.ldy)
            static_cast<uint8_t*>(a.y)[row * a.ldy + i] = (uint8_t)pack_e4m3(v[e] * bs.inv, 0.f, 0.f, 0.f);
        }
        if (lane == 0 && i0 < a.F) a.scales[row * nb + i0 / kScaleBlock] = bs.scale;
      }
      continue;
    }
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

// Rows of whole chunks of 16 bytes that W waves hold in their registers from the first read to the last
// write: NV chunks a lane, chunk i of lane l at (64 W i + l) VE, so that a load instruction covers 1 KB in a
// row. The weights stay there too, over all the rows that a workgroup takes. Bound by memory (up to two loads
// and two stores a value): 65537 x 2048 bf16 with residual, sum and e4m3 output 175 us, 5.4 TB/s; 6436 x 2048 f32
// 32 us; 10752 x 384 bf16 9.7 us.
//
// BLK: scales of blocks, whose 128 values lie in neighbouring lanes of one chunk.
template <class T, int NV, int W, mnn_dtype OUT, bool BLK = false>
__global__ __launch_bounds__(256) void rmsnorm_rows_kernel(RmsNormArgs a) {
  constexpr int VE = 16 / (int)sizeof(T);
  typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
  __shared__ float sh[8][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = ((W == 1 ? 0 : wave * 64) + lane) * VE;
  // over the W waves of a row. `at`, 0 to 3, keeps a row's reductions apart and `parity` one row's from
  // the next one's: a wave writes a place again only behind a barrier that is behind the others' reads of it
  int parity = 0;
  auto over_row = [&](float v, int at, auto op) {
    v = group_reduce<64>(v, op);
    if constexpr (W > 1) {
      float* to = sh[4 * parity + at];
      if (lane == 0) to[wave] = v;
      __syncthreads();
      v = op(op(to[0], to[1]), op(to[2], to[3]));
    }
    return v;
  };
  auto values = [](uintx4 x, float* v) {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      unsigned u;
      if constexpr (VE == 4)
        u = x[e];
      else
        u = e & 1 ? x[e / 2] & 0xffff0000u : x[e / 2] << 16;
      v[e] = __builtin_bit_cast(float, u);
    }
  };
  bool on[NV];
  float w[NV][VE];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    on[i] = col + 64 * W * VE * i < a.F;
#pragma unroll
    for (int e = 0; e < VE; ++e) w[i][e] = a.w && on[i] ? a.w[col + 64 * W * VE * i + e] : 1.f;
  }
  const int64_t first = W == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
  for (int64_t row = first; row < a.rows; row += (int64_t)gridDim.x * (4 / W), parity ^= 1) {
    const int64_t at = row * a.F + col;
    uintx4 x[NV], r[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i] = r[i] = uintx4{0, 0, 0, 0};
      if (on[i]) {
        x[i] = *reinterpret_cast<const uintx4*>(static_cast<const T*>(a.x) + at + 64 * W * VE * i);
        if (a.r) r[i] = *reinterpret_cast<const uintx4*>(static_cast<const T*>(a.r) + at + 64 * W * VE * i);
      }
    }
    float h[NV][VE], ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float add[VE];
      values(x[i], h[i]);
      values(r[i], add);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        if (a.r) h[i][e] += add[e];
        ss = fmaf(h[i][e], h[i][e], ss);
      }
    }
    if (a.sum) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (on[i]) {
          uintx4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (VE == 4)
              o[e] = __builtin_bit_cast(unsigned, h[i][e]);
            else
              o[e] = cvt_pk_bf16(h[i][2 * e], h[i][2 * e + 1]);
          }
          *reinterpret_cast<uintx4*>(static_cast<T*>(a.sum) + at + 64 * W * VE * i) = o;
        }
    }
    if (a.w) {
      float mean = over_row(ss, 0, Plus{}) / (float)a.F + a.eps;
      if (!mean_in_range(mean)) {  // the same for every lane of the row
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < VE; ++e) top = max_nan(top, fabsf(h[i][e]));
        top = over_row(top, 2, max_nan);
        if (top < INFINITY) {
          const float s = unit_scale(top, a.eps);
          ss = 0.f;
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              h[i][e] *= s;
              ss = fmaf(h[i][e], h[i][e], ss);
            }
          mean = over_row(ss, 3, Plus{}) / (float)a.F + a.eps * s * s;
        }
      }
      const float norm = rsqrtf(mean);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) h[i][e] = h[i][e] * norm * w[i][e];
    }
    if constexpr (OUT == MNN_E4M3) {
      float inv[NV];
      if constexpr (BLK) {
        constexpr int L = kScaleBlock / VE;  // lanes a block
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float top = 0.f;
#pragma unroll
          for (int e = 0; e < VE; ++e)
            if (on[i]) top = max_nan(top, fabsf(h[i][e]));
          const RowScale rs = row_scale(group_reduce<L>(top, max_nan));
          inv[i] = rs.inv;
          const int first = col + 64 * W * VE * i;
          if (lane % L == 0 && first < a.F) a.scales[row * scale_blocks(a.F) + first / kScaleBlock] = rs.scale;
        }
      } else {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < VE; ++e)
            if (on[i]) top = max_nan(top, fabsf(h[i][e]));
        const RowScale rs = row_scale(over_row(top, 1, max_nan));
        if (lane == 0 && (W == 1 || wave == 0)) a.scales[row] = rs.scale;
#pragma unroll
        for (int i = 0; i < NV; ++i) inv[i] = rs.inv;
      }
      uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.ldy + col;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        unsigned q[VE / 4];
#pragma unroll
        for (int e = 0; e < VE / 4; ++e)
          q[e] = on[i] ? pack_e4m3(h[i][4 * e] * inv[i], h[i][4 * e + 1] * inv[i], h[i][4 * e + 2] * inv[i],
                                   h[i][4 * e + 3] * inv[i])
                       : 0u;
        if (col + 64 * W * VE * i < a.ldy) {
          if constexpr (VE == 4)
            *reinterpret_cast<unsigned*>(y + 64 * W * VE * i) = q[0];
          else
            *reinterpret_cast<uint2*>(y + 64 * W * VE * i) = make_uint2(q[0], q[1]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!on[i]) continue;
        const int64_t to = row * a.ldy + col + 64 * W * VE * i;
        if constexpr (OUT == MNN_F32) {
#pragma unroll
          for (int e = 0; e < VE; e += 4)
            *reinterpret_cast<float4*>(static_cast<float*>(a.y) + to + e) =
                make_float4(h[i][e], h[i][e + 1], h[i][e + 2], h[i][e + 3]);
        } else {
          unsigned q[VE / 2];
#pragma unroll
          for (int e = 0; e < VE / 2; ++e) q[e] = cvt_pk_bf16(h[i][2 * e], h[i][2 * e + 1]);
          if constexpr (VE == 4)
            *reinterpret_cast<uint2*>(static_cast<__bf16*>(a.y) + to) = make_uint2(q[0], q[1]);
          else
            *reinterpret_cast<uint4*>(static_cast<__bf16*>(a.y) + to) = make_uint4(q[0], q[1], q[2], q[3]);
        }
      }
    }
  }
}

// Rows of x rounded in blocks of 128, as they are: 16 lanes a block, eight values a lane, each workgroup 16 blocks and 16
// others, whose loads go out together. Bound by memory where rmsnorm_rows_kernel, made for a whole row's sums, is by its
// VALU instructions (0.83 busy): 10752 x 1536 bf16 (49.6 MB) 11.0 us in a trace, 4.5 TB/s, against 12.2.
constexpr int kUnits = 16;
template <class T>
__global__ __launch_bounds__(16 * kUnits) void round_blocks_kernel(RmsNormArgs a, FastDiv by_blocks, int units) {
  const int j = threadIdx.x % 16, nb = (int)(a.ldy / kScaleBlock);
  int u[2], col[2];
  int64_t row[2];
  Eight<T> x[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    u[i] = (2 * blockIdx.x + i) * kUnits + threadIdx.x / 16;
    const int at = by_blocks(u[i]);
    row[i] = at;
    col[i] = (u[i] - at * nb) * kScaleBlock + 8 * j;
    x[i].clear();
    if (u[i] < units && col[i] < a.F) x[i].load(static_cast<const T*>(a.x) + row[i] * a.F + col[i]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (u[i] >= units) return;
    float v[8], scale;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = x[i][e];
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.y) + row[i] * a.ldy + col[i]) = round_row<16>(v, scale);
    if (j == 0) a.scales[u[i]] = scale;
  }
}
template <class T>
void round_blocks(const LaunchCtx& c, RmsNormArgs a) {
  const int nb = scale_blocks(a.F), most = std::max(1, (1 << 27) / nb);  // rows of a launch: 2^31 lanes
  for (int64_t r0 = 0; r0 < a.rows; r0 += most) {
    RmsNormArgs s = a;
    s.rows = std::min<int64_t>(most, a.rows - r0);
    s.x = static_cast<const T*>(a.x) + r0 * a.F;
    s.y = static_cast<uint8_t*>(a.y) + r0 * a.ldy;
    s.scales = a.scales + r0 * nb;
    const int units = (int)s.rows * nb;
    launch(c, sizeof(T) == 4 ? "round_blocks_f32" : "round_blocks_bf16", round_blocks_kernel<T>,
           dim3((unsigned)((units + 2 * kUnits - 1) / (2 * kUnits))), dim3(16 * kUnits), 0, s, FastDiv(nb), units);
  }
}

template <class T, int NV, int W>
void launch_rows(const LaunchCtx& c, const RmsNormArgs& a) {
  const char* name = sizeof(T) == 4 ? "rmsnorm_rows_f32" : "rmsnorm_rows_bf16";
  // eight workgroups a compute unit keep their weights over several rows
  const int64_t wgs = W == 1 ? (a.rows + 3) / 4 : a.rows;
  const dim3 grid((unsigned)std::min<int64_t>(wgs, 8 * c.dev->props.multiProcessorCount));
  if (a.out == MNN_E4M3 && a.blocks)
    launch(c, name, rmsnorm_rows_kernel<T, NV, W, MNN_E4M3, true>, grid, dim3(256), 0, a);
  else if (a.out == MNN_E4M3)
    launch(c, name, rmsnorm_rows_kernel<T, NV, W, MNN_E4M3>, grid, dim3(256), 0, a);
  else if (a.out == MNN_BF16)
    launch(c, name, rmsnorm_rows_kernel<T, NV, W, MNN_BF16>, grid, dim3(256), 0, a);
  else
    launch(c, name, rmsnorm_rows_kernel<T, NV, W, MNN_F32>, grid, dim3(256), 0, a);
}

// Rows that are only rounded, in blocks: round_blocks_kernel. A wave a row up to four chunks a lane; a workgroup a row for longer ones, and for rows so few that a wave
// each would leave most of the GPU waiting for a handful of loads.
template <class T>
void rmsnorm_t(const LaunchCtx& c, const RmsNormArgs& a) {
  constexpr int VE = 16 / (int)sizeof(T);
  if (a.blocks && !a.w && a.F % 8 == 0 && a.ldy == (int64_t)scale_blocks(a.F) * kScaleBlock) return round_blocks<T>(c, a);
  if (a.F % VE == 0 && a.ldy % VE == 0 && a.ldy <= 8 * 256 * VE) {
    const int n = (int)((a.ldy + 64 * VE - 1) / (64 * VE));  // chunks a lane of one wave
    const bool few = a.rows < c.dev->props.multiProcessorCount;
    if (n == 1) return launch_rows<T, 1, 1>(c, a);
    if (n <= 4 && !few) {
      if (n == 2) return launch_rows<T, 2, 1>(c, a);
      if (n == 3) return launch_rows<T, 3, 1>(c, a);
      return launch_rows<T, 4, 1>(c, a);
    }
    if (n <= 4) return launch_rows<T, 1, 4>(c, a);
    if (n <= 8) return launch_rows<T, 2, 4>(c, a);
    if (n <= 16) return launch_rows<T, 4, 4>(c, a);
    return launch_rows<T, 8, 4>(c, a);
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
