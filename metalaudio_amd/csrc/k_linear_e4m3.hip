// The 8-bit linear product: y[m][n] = act(xs[m] ws[n] sum_k x[m][k] w[n][k] + bias[n]) + r[m][n], x and w
// in e4m3.
//
// Which matrix instructions: e4m3 values are bf16 values, so both operands are widened
// (v_cvt_scalef32_pk_bf16_fp8, two values an instruction) and multiplied by the bf16 instructions (2.2 PFLOP/s), whose
// sums are fp32 sums: 9e-9 off (2-norm) over 128 random products. Those on 8-bit operands (v_mfma_f32_*_f8f6f4, 4.2
// PFLOP/s here) add a group's products to about 14 bits below the largest one, 1.3e-5 off on the same sums, and lose
// whatever is smaller where large products cancel: no rounding of the result hides that.
#include "lds_dma.hpp"
#include "token_ops.hpp"
#include "token_utils.hpp"
#include "x3.hpp"

#include <type_traits>

namespace mnn {
namespace k {

using namespace dev;

namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));

// Eight e4m3 values to bf16, exactly.
__device__ __forceinline__ bf16x8 widen8(int lo, int hi) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 64 products a row: lane (g, r) holds 32 bytes of row r of both operands (which k they are does not matter
// as long as both sides agree). The result: b's row l % 32, a's rows 8 (v / 4) + 4 (l / 32) + v % 4.
struct Operand {
  bf16x8 x[4];
  __device__ __forceinline__ void set(intx4 lo, intx4 hi) {
    x[0] = widen8(lo[0], lo[1]);
    x[1] = widen8(lo[2], lo[3]);
    x[2] = widen8(hi[0], hi[1]);
    x[3] = widen8(hi[2], hi[3]);
  }
};
__device__ __forceinline__ floatx16 mul(const Operand& a, const Operand& b, floatx16 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.x[i], b.x[i], c, 0, 0, 0);
  return c;
}

// The activation of CNT values; its choice is made once for all of them (a branch an element, the same for
// every lane or not, took 32 us of a round of 256 x 256 results).
template <int CNT>
__device__ __forceinline__ void activate(float (&v)[CNT], int act, float alpha) {
  auto all = [&](auto code) {
#pragma unroll
    for (int i = 0; i < CNT; ++i) v[i] = apply_act(v[i], decltype(code)::value, alpha);
  };
  switch (act) {
    case 1: return all(std::integral_constant<int, 1>{});
    case 2: return all(std::integral_constant<int, 2>{});
    case 3: return all(std::integral_constant<int, 3>{});
    case 4: return all(std::integral_constant<int, 4>{});
    case 5: return all(std::integral_constant<int, 5>{});
    case 6: return all(std::integral_constant<int, 6>{});
    default: return;
  }
}

// Eight values of a row, or the first `cnt` of them one by one where the row is not aligned.
template <class T>
__device__ __forceinline__ void load_some(Eight<T>& x, const T* p, bool vec, int cnt) {
  if (vec) return x.load(p);
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = i < cnt ? p[i] : (T)0.f;
  __builtin_memcpy(x.x, t, sizeof(x.x));
}
template <class T>
__device__ __forceinline__ void store_some(T* p, const float* v, bool vec, int cnt) {
  if (vec) {
    Eight<T> x;
    x.set(v);
    return x.store(p);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < cnt) p[i] = from_f32<T>(v[i]);
}

// Scales and biases of CNT consecutive columns (those behind the last column: 0).
template <int CNT>
__device__ __forceinline__ void columns(const LinearE4m3Args& a, int n, float* ws, float* bias) {
#pragma unroll
  for (int i = 0; i < CNT; ++i) {
    const int c = min(n + i, a.N - 1);
    ws[i] = a.ws[c];
    bias[i] = a.bias ? a.bias[c] : 0.f;
  }
}

// BM x BN results a workgroup, WM x WN a wave, the depth 128 at a time through two slots in LDS,
// which global_load_lds fills: the rows of x, then those of w, 128 bytes each, 16-byte chunk c of row r in
// place c ^ (r / 2 % 8), so that 16 rows' reads are spread over all 64 banks (c ^ (r % 8) for rows 8 apart in the same
// ones). One barrier a step: behind it,
// the step's slot is whole and the other one free to be filled again.
//
// Rows behind the last are read as the last one; their results are not stored. The results go through LDS
// once more (the slots are done with), so that scales, residual and output are read and written row by row.
//
// Bound by the matrix instructions beside the widening and, in a grid of one or two rounds, by each round's first
// loads and results: 8192 x 4096 x 4096 to bf16 200 to 214 us (1.3 PFLOP/s), 8192 x 8192 x 8192 750 us (1.5), 10752 x
// 1536 x 384 to f32 with residual 19 us. The widening spread between the products by hand changes nothing, nor do
// waves of 128 x 128 (a third less of it, one wave a SIMD: 225 us).
template <class T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(BM / WM * (BN / WN) * 64) void linear_e4m3_kernel(LinearE4m3Args a) {
  constexpr int NW = BM / WM * (BN / WN);
  constexpr int SLOT = (BM + BN) * 128, LOADS = SLOT / 1024 / NW;
  static_assert(SLOT % (1024 * NW) == 0, "whole loads a wave");
  constexpr int FM = WM / 32, FN = WN / 32;
  constexpr int OP = WN + 4;  // floats a row of the results in LDS
  constexpr int BYTES = 2 * SLOT > NW * 32 * OP * 4 ? 2 * SLOT : NW * 32 * OP * 4;
  __shared__ __attribute__((aligned(1024))) char smem[BYTES];
  __shared__ float xs[BM];
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / (BN / WN), wn = wave % (BN / WN);
  // tiles of neighbouring rows of w beside each other on one XCD
  const int nt = (a.N + BN - 1) / BN;
  const int tile = xcd_logical_tile((int)blockIdx.x, (int)gridDim.x);
  // tiles run down GM rows of tiles, then to the next column of them: the workgroups of an XCD at one
  // time share a block of x and of w in its L2
  constexpr int GM = 8;
  const int mt = (int)((a.M + BM - 1) / BM), grp = tile / (GM * nt), in = tile - grp * GM * nt;
  const int gm = min(GM, mt - grp * GM);
  const int64_t m0 = (int64_t)(grp * GM + in % gm) * BM;
  const int n0 = in / gm * BN;

  // load i of this wave: rows 8 j .. + 7 of the slot, j = i NW + wave; the first BM rows are x's
  static_assert(NW % 2 == 0, "j is odd for odd waves");
  const int row_in = lane >> 3, chunk = (lane & 7) ^ (4 * (wave & 1) + (row_in >> 1));
  const char* src[LOADS];  // wave-uniform bases
  unsigned off[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int row = 8 * (i * NW + wave);
    const bool isx = row < BM;
    const int64_t first = isx ? m0 + row : n0 + row - BM, last = isx ? a.M - 1 : a.N - 1;
    const int64_t base = min(first, last);
    src[i] = reinterpret_cast<const char*>((isx ? a.x : a.w) + base * a.K);
    off[i] = (unsigned)min((int64_t)row_in, last - base) * (unsigned)a.K + 16u * chunk;
  }
  const unsigned lds0 = lds_address(smem);
  auto issue = [&](int k, int slot) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      lds_dma16_s(reinterpret_cast<const float*>(src[i]), off[i] + 128u * k,
                  __builtin_amdgcn_readfirstlane(lds0 + slot * SLOT + 1024u * (i * NW + wave)));
  };

  floatx16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;

  const int nk = a.K / 128;
  issue(0, 0);
  // what the results need besides: this lane's columns and the tile's row scales
  constexpr int PER_ROW = WN / 8;  // lanes
  const int cn = 8 * (lane % PER_ROW), n = n0 + wn * WN + cn;
  float ws[8], bias[8];
  columns<8>(a, n, ws, bias);
  for (int i = threadIdx.x; i < BM; i += NW * 64) xs[i] = a.xs[min(m0 + i, a.M - 1)];
  // chunk c of a row that is l32 modulo 32
  auto at = [&](int c) { return l32 * 128 + ((c ^ (l32 >> 1 & 7)) << 4); };
  const int xa = wm * WM * 128, wa = (BM + wn * WN) * 128;
  int slot = 0;
  for (int k = 0; k < nk; ++k, slot ^= 1) {
    wait_lgkmcnt0();
    wait_vmcnt<0>();
    stage_barrier();
    if (k + 1 < nk) issue(k + 1, slot ^ 1);
    const char* p = smem + slot * SLOT;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int c0 = at(4 * s + 2 * g), c1 = at(4 * s + 2 * g + 1);
      Operand x[FM], w[FN];
#pragma unroll
      for (int j = 0; j < FM; ++j)
        x[j].set(*reinterpret_cast<const intx4*>(p + xa + 4096 * j + c0),
                 *reinterpret_cast<const intx4*>(p + xa + 4096 * j + c1));
#pragma unroll
      for (int i = 0; i < FN; ++i)
        w[i].set(*reinterpret_cast<const intx4*>(p + wa + 4096 * i + c0),
                 *reinterpret_cast<const intx4*>(p + wa + 4096 * i + c1));
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = mul(w[i], x[j], acc[i][j]);
    }
  }

  // 32 rows of results at a time, through a part of LDS that is this wave's; the residual's rows are on
  // their way meanwhile (all of them are read before a row is written: they may be the output's)
  __syncthreads();
  float* out = reinterpret_cast<float*>(smem) + wave * 32 * OP;
  const bool vec = a.N % 8 == 0;
  const int cnt = a.N - n;  // columns that are there (<= 0: none)
  constexpr int PASSES = 32 * PER_ROW / 64, ROWS = 64 / PER_ROW;
#pragma unroll 1
  for (int j = 0; j < FM; ++j) {
    const int64_t mj = m0 + wm * WM + 32 * j + lane / PER_ROW;
    Eight<T> res[PASSES];
    if (a.r) {
#pragma unroll
      for (int r = 0; r < PASSES; ++r)
        if (mj + r * ROWS < a.M && cnt > 0)
          load_some(res[r], static_cast<const T*>(a.r) + (mj + r * ROWS) * a.N + n, vec, cnt);
    }
#pragma unroll
    for (int jj = 0; jj < FM; ++jj)
      if (jj == j) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<float4*>(out + l32 * OP + 32 * i + 8 * q + 4 * g) =
                make_float4(acc[i][jj][4 * q], acc[i][jj][4 * q + 1], acc[i][jj][4 * q + 2], acc[i][jj][4 * q + 3]);
      }
    wait_lgkmcnt0();
    __builtin_amdgcn_wave_barrier();
    float v[8 * PASSES];
#pragma unroll
    for (int r = 0; r < PASSES; ++r) {
      const int row = r * ROWS + lane / PER_ROW;
      const float by = xs[wm * WM + 32 * j + row];
      float* u = v + 8 * r;
      *reinterpret_cast<float4*>(u) = *reinterpret_cast<const float4*>(out + row * OP + cn);
      *reinterpret_cast<float4*>(u + 4) = *reinterpret_cast<const float4*>(out + row * OP + cn + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = fmaf(u[e] * by, ws[e], bias[e]);
    }
    activate(v, a.act, a.alpha);
#pragma unroll
    for (int r = 0; r < PASSES; ++r) {
      float* u = v + 8 * r;
      if (a.r) {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] += res[r][e];
      }
      if (mj + r * ROWS < a.M && cnt > 0)
        store_some(static_cast<T*>(a.y) + (mj + r * ROWS) * a.N + n, u, vec, cnt);
    }
    wait_lgkmcnt0();
    __builtin_amdgcn_wave_barrier();
  }
}

// Few rows (up to 32): the weights are all the traffic. A workgroup takes 32 rows of w, its eight waves an
// eighth of the depth each, operands straight from memory (a wave reads 64 bytes of 32 rows at a time, four
// such steps in flight); their sums meet in LDS. Rows of x may be of any length: what a lane would read past
// a row's end is 0.
template <class T>
__global__ __launch_bounds__(512) void linear_e4m3_few_kernel(LinearE4m3Args a) {
  __shared__ float sum[8][32][33];  // [wave][m][n]
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31, wave = threadIdx.x >> 6;
  const int n0 = blockIdx.x * 32;
  const uint8_t* x = a.x + min((int64_t)l32, a.M - 1) * a.ldx + 32 * g;
  const uint8_t* w = a.w + (int64_t)min(n0 + l32, a.N - 1) * a.K + 32 * g;
  const int steps = a.K / 64, s0 = steps * wave / 8, s1 = steps * (wave + 1) / 8;
  floatx16 acc;
#pragma unroll
  for (int v = 0; v < 16; ++v) acc[v] = 0.f;
  auto step = [&](int s, auto whole) {
    const intx4* q = reinterpret_cast<const intx4*>(w + 64 * s);
    Operand xo, wo;
    wo.set(q[0], q[1]);
    intx4 lo = 0, hi = 0;
    if (decltype(whole)::value || 64 * s + 32 * g + 32 <= a.ldx) {
      __builtin_memcpy(&lo, x + 64 * s, 16);
      __builtin_memcpy(&hi, x + 64 * s + 16, 16);
    } else {
      for (int e = 0; e < a.ldx - 64 * s - 32 * g; ++e) {
        intx4& part = e < 16 ? lo : hi;
        part[e % 16 / 4] |= (int)x[64 * s + e] << 8 * (e % 4);
      }
    }
    xo.set(lo, hi);
    acc = mul(wo, xo, acc);
  };
  const int whole = min(s1, a.ldx / 64);  // steps that end within a row
#pragma unroll 4
  for (int s = s0; s < whole; ++s) step(s, std::true_type{});
  for (int s = max(s0, whole); s < s1; ++s) step(s, std::false_type{});
#pragma unroll
  for (int v = 0; v < 16; ++v) sum[wave][l32][8 * (v / 4) + 4 * g + v % 4] = acc[v];
  __syncthreads();
  for (int e = threadIdx.x; e < 32 * a.M; e += 512) {
    const int m = e / 32, n = n0 + e % 32;
    if (n >= a.N) continue;
    float v[1] = {0.f}, ws, bias;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[0] += sum[i][m][e % 32];
    columns<1>(a, n, &ws, &bias);
    v[0] = fmaf(v[0] * a.xs[m], ws, bias);
    activate(v, a.act, a.alpha);
    const int64_t at = (int64_t)m * a.N + n;
    if (a.r) v[0] += to_f32(static_cast<const T*>(a.r)[at]);
    static_cast<T*>(a.y)[at] = from_f32<T>(v[0]);
  }
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

namespace {
template <class T, int BM, int BN, int WM, int WN>
void launch_tile(const LaunchCtx& c, const LinearE4m3Args& a, const char* name) {
  const int64_t tiles = (a.M + BM - 1) / BM * ((a.N + BN - 1) / BN);
  MNN_REQUIRE(tiles < (1 << 22), MNN_ERR_INVALID_CONFIGURATION, "Linear: too many rows in one call");
  constexpr int threads = BM / WM * (BN / WN) * 64;
  launch(c, name, linear_e4m3_kernel<T, BM, BN, WM, WN>, dim3((unsigned)tiles), dim3(threads), 0, a);
}

template <class T>
void linear_e4m3_t(const LaunchCtx& c, const LinearE4m3Args& a) {
  constexpr bool F32 = sizeof(T) == 4;
  MNN_REQUIRE(a.K % 128 == 0 && (a.ldx == a.K || a.M <= kLinearFew), MNN_ERR_INVALID_ARGUMENT,
              "linear_e4m3: rows of x are not padded");
  if (a.M <= kLinearFew)
    return launch(c, F32 ? "linear_e4m3_few_f32" : "linear_e4m3_few_bf16", linear_e4m3_few_kernel<T>,
                  dim3((unsigned)((a.N + 31) / 32)), dim3(512), 0, a);
  // 256 square where the rounds of one tile a compute unit are 7/8 full: a third less widening a product, but one
  // workgroup a compute unit, whose last round costs a whole one. us at (M, K, N), 256 / 128 / 64 square: 8192 x 4096 x
  // 4096 bf16 203 / 227 / 281, f32 215 / 235 / 285; 10752 x 384 x 1536 bf16 (252 tiles) 19.2 / 20.2 / 23.6; 8192 x
  // 1024 x 1536 bf16 (192 tiles) 32 / 29 / 35; 12800 x 1024 x 1536 bf16 (300 tiles) 58 / 44 / 52.
  const int64_t cus = c.dev->props.multiProcessorCount;
  auto tiles = [&](int b) { return (a.M + b - 1) / b * ((a.N + b - 1) / b); };
  if (7 * ((tiles(256) + cus - 1) / cus * cus) <= 8 * tiles(256))
    return launch_tile<T, 256, 256, 128, 64>(c, a, F32 ? "linear_e4m3_256_f32" : "linear_e4m3_256_bf16");
  // 128 square from three quarters of the compute units on, 128 / 64 square: 10752 x 1536 x 384 (252 tiles) f32 19.3 /
  // 19.5, bf16 17.1 / 19.2; 2688 x 384 x 1152 bf16 (189) 7.8 / 7.8; 5376 x 1536 x 384 f32 (126) 16.3 / 12.9
  if (4 * tiles(128) >= 3 * cus)
    return launch_tile<T, 128, 128, 64, 32>(c, a, F32 ? "linear_e4m3_128_f32" : "linear_e4m3_128_bf16");
  launch_tile<T, 64, 64, 32, 32>(c, a, F32 ? "linear_e4m3_64_f32" : "linear_e4m3_64_bf16");
}
}  // namespace

void linear_e4m3(const LaunchCtx& c, const LinearE4m3Args& a) {
  if (a.M <= 0) return;
  if (a.out == MNN_F32)
    linear_e4m3_t<float>(c, a);
  else
    linear_e4m3_t<__bf16>(c, a);
}

}  // namespace k
}  // namespace mnn
