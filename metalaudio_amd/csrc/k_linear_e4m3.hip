// The 8-bit linear product: y[m][n] = act(xs[m] ws[n] sum_k x[m][k] w[n][k] + bias[n]) + r[m][n], x and w
// in e4m3.
//
// Which matrix instructions: those on 8-bit operands (v_mfma_f32_*_f8f6f4, 4.2 PFLOP/s here) add the
// products of a group of lanes' bytes to about 14 bits below the largest one: a sum of 128 random
// products is 1.3e-5 off (2-norm), whichever of them is taken. bf16 output, whose rounding is a hundred
// times that (2^-9), is made with them. fp32 output is not: e4m3 values are bf16 values, so both operands
// are widened (v_cvt_scalef32_pk_bf16_fp8, two values an instruction) and multiplied by the bf16
// instructions (2.2 PFLOP/s), 9e-9 off on the same sums.
#include "token_ops.hpp"
#include "token_utils.hpp"

namespace mnn {
namespace k {

using namespace dev;

namespace {

typedef int intx8 __attribute__((ext_vector_type(8)));

// Eight e4m3 values to bf16, exactly.
__device__ __forceinline__ bf16x8 widen8(int lo, int hi) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Lane (g, r) holds 32 bytes of row r of both operands: which k they are does not matter as long as both
// sides agree. The result of (a rows, b rows): b row l % 16, a rows 4 (l / 16) + v.
template <class T>
__device__ __forceinline__ floatx4 mfma_e4m3(intx8 a, intx8 b, floatx4 c) {
  if constexpr (sizeof(T) == 2) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i += 2)
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(a[i], a[i + 1]), widen8(b[i], b[i + 1]), c, 0, 0,
                                                  0);
    return c;
  }
}

__device__ __forceinline__ intx8 load32(const uint8_t* p) {
  intx8 v;
  reinterpret_cast<int4*>(&v)[0] = reinterpret_cast<const int4*>(p)[0];
  reinterpret_cast<int4*>(&v)[1] = reinterpret_cast<const int4*>(p)[1];
  return v;
}

// Four results of one row m, columns n .. n + 3.
template <class T>
__device__ __forceinline__ void store4(const LinearE4m3Args& a, int64_t m, int n, floatx4 acc) {
  if (m >= a.M) return;
  const float xs = a.xs[m];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= a.N) return;
    float v = acc[i] * xs * a.ws[n + i] + (a.bias ? a.bias[n + i] : 0.f);
    v = apply_act(v, a.act, a.alpha);
    const int64_t at = m * a.N + n + i;
    if (a.r) v += to_f32(static_cast<const T*>(a.r)[at]);
    static_cast<T*>(a.y)[at] = from_f32<T>(v);
  }
}

// A wave per 16 x 16 results, operands straight from memory.
template <class T>
__global__ __launch_bounds__(256) void linear_e4m3_any_kernel(LinearE4m3Args a) {
  const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int64_t nt = (a.N + 15) / 16, m0 = (blockIdx.x / nt * 4 + (threadIdx.x >> 6)) * 16;
  const int n0 = (int)(blockIdx.x % nt) * 16;
  const uint8_t* x = a.x + min(m0 + r, a.M - 1) * a.K + 32 * g;
  const uint8_t* w = a.w + (int64_t)min(n0 + r, a.N - 1) * a.K + 32 * g;
  floatx4 acc{0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < a.K; k += 128) acc = mfma_e4m3<T>(load32(w + k), load32(x + k), acc);
  store4<T>(a, m0 + r, n0 + 4 * g, acc);
}

__global__ __launch_bounds__(256) void pad_rows_u8_kernel(const uint8_t* x, int64_t rows, int n,
                                                          uint8_t* y, int ld) {
  const int64_t total = rows * ld;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / ld;
    const int col = (int)(i - row * ld);
    y[i] = col < n ? x[row * n + col] : 0;
  }
}

}  // namespace

void pad_rows_u8(const LaunchCtx& c, const uint8_t* x, int64_t rows, int n, uint8_t* y, int ld) {
  const dim3 grid((unsigned)std::min<int64_t>((rows * ld + 255) / 256, 1 << 20));
  launch(c, "pad_rows_u8", pad_rows_u8_kernel, grid, dim3(256), 0, x, rows, n, y, ld);
}

void linear_e4m3(const LaunchCtx& c, const LinearE4m3Args& a) {
  const int64_t wgs = (a.M + 63) / 64 * ((a.N + 15) / 16);
  MNN_REQUIRE(wgs < (1 << 23), MNN_ERR_INVALID_CONFIGURATION, "Linear: too many rows in one call");
  if (a.out == MNN_F32)
    launch(c, "linear_e4m3_any_f32", linear_e4m3_any_kernel<float>, dim3((unsigned)wgs), dim3(256), 0, a);
  else
    launch(c, "linear_e4m3_any_bf16", linear_e4m3_any_kernel<__bf16>, dim3((unsigned)wgs), dim3(256), 0,
           a);
}

}  // namespace k
}  // namespace mnn
