// Window attention over whole sequences: o_i = sum_j p_ij v_j, p_i = softmax of scale q_i k_j over the keys
// j <= i + right with j >= i - left or j < sinks.
#include "lds_dma.hpp"
#include "token_ops.hpp"
#include "window_row.hpp"
#include "x3.hpp"

#include <algorithm>
#include <type_traits>

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

// A workgroup takes the keys that BQ queries of one head see, in blocks that lie in LDS, by NW waves: NW / KW
// groups of 32 queries by KW groups of keys, which take every KW-th block and whose results are joined at the
// end (KW > 1 for grids that would leave most of the GPU idle: then each of a few waves a compute unit waits for
// its next block for longer than it computes). Each wave computes the TRANSPOSED scores S^T = K Q^T on
// v_mfma_f32_32x32x16_bf16: the accumulator (lane (g, q): keys 8 (v / 4) + 4 g + v % 4 of query q) is the B operand
// that O^T += V^T P^T needs when its k slots take those keys, so P goes from the softmax straight into the second
// product. K and V lie in LDS row by row as
// they come; V^T's fragments (4 keys of one dimension a lane) are transposed on the way out by
// ds_read_b64_tr_b16. f32 values are three bf16 parts each and six partial products are kept (x3.hpp); the
// workgroup splits a block of K and V as it stores it.
//
// Only the blocks that a query of the workgroup sees are visited, and of those a wave computes the ones
// that its own queries see; the mask is applied where a block is not wholly visible to all 32. While one
// block is computed the next one's rows are on their way to registers.
//
// Bound by the vector units' issue beside the matrix instructions: 16384 tokens, 1023 back, 8 / 2 heads of 64 in bf16
// 52 us (0.6 PFLOP/s); f32, 2 x 1345 ragged tokens, 168 both ways, 8 heads of 48 20.4 us (split of K, V and P).
//
// Softmax: p = exp2(c s - ref) with a reference that moves only when a block's maximum exceeds it by 2^8.
//
// A key that a query does not see has probability 0, but 0 times a value that is not finite is NaN, and
// parts of tiny or overflowing f32 values are off; and in bf16 c ref, rounded, of scores past 2^31 is so far from c times
// the largest score that all probabilities may come out as 0 (their sum is about 1 or more otherwise). Queries whose
// result is not finite, whose sum is small or, in f32, whose result is below 2^-109 are computed again by window_query.
template <class T, int KS, int KW, int NW>
struct WindowCfg {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int PARTS = F32 ? 3 : 1;
  static constexpr int BKV = F32 ? 32 : 64;   // keys per block
  static constexpr int NT = BKV / 32;
  static constexpr int DT = (KS + 1) / 2;     // 32-row tiles of O^T
  // bytes from one key's row to the next in LDS: 8 rows of 16-byte reads on distinct banks
  static constexpr int PITCH = KS * 32 + (KS % 2 ? 0 : 16);
  static constexpr int PLANE = BKV * PITCH;
  static constexpr int CHUNKS = BKV * KS * 2;  // of 8 values, in a block of K or V
  static constexpr int THREADS = 64 * NW, BQ = 32 * NW / KW;
  static constexpr int PER = (KW * CHUNKS + THREADS - 1) / THREADS;
  // K planes, then V planes, of KW blocks; V's fragments of the last 32 dimensions may reach 32 bytes past
  // its rows. At the end, the other key groups' results: maximum, sum and O^T of each lane
  static constexpr int SLOT = 2 * PARTS * PLANE;
  static constexpr int JOIN = (KW - 1) * (NW / KW) * (16 * DT + 2) * 256;
  static constexpr int LDS = KW * SLOT + 64 > JOIN ? KW * SLOT + 64 : JOIN;
  // workgroups a CU, as the registers allow without spilling
  static constexpr int OCC = KW > 1 ? 1
                             : F32  ? (KS > 6 ? 1 : KS > 4 ? 2 : 3)
                                    : (KS > 6 ? 2 : KS > 4 ? 3 : 4);
};

template <class T, int KS, int KW, int NW>
__global__ __launch_bounds__((WindowCfg<T, KS, KW, NW>::THREADS), (WindowCfg<T, KS, KW, NW>::OCC)) void window_kernel(WindowArgs a) {
  using Cfg = WindowCfg<T, KS, KW, NW>;
  constexpr int PARTS = Cfg::PARTS, BKV = Cfg::BKV, NT = Cfg::NT, DT = Cfg::DT, PITCH = Cfg::PITCH;
  constexpr int PLANE = Cfg::PLANE, PER = Cfg::PER, SLOT = Cfg::SLOT, BQ = Cfg::BQ;
  constexpr int THREADS = Cfg::THREADS;
  constexpr bool F32 = Cfg::F32;
  __shared__ __attribute__((aligned(16))) char smem[Cfg::LDS];

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), qg = wave / KW, kg = wave % KW;
  // consecutive units, the heads that share K and V first, run on one XCD and share its L2
  const int nq = (a.S + BQ - 1) / BQ, G = a.H / a.KV;
  int unit = xcd_logical_tile((int)blockIdx.x, (int)gridDim.x);
  const int gi = unit % G;
  unit /= G;
  const int q0 = unit % nq * BQ;
  unit /= nq;
  const int kvh = unit % a.KV, b = unit / a.KV, h = kvh * G + gi;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.S) : a.S;
  if (q0 >= len) return;
  const int qw = q0 + 32 * qg;                // this wave's first query
  const int qn = min(qw + 31, len - 1);       // and last
  const int qi = qw + l32;                    // the lane's
  const int kvw = a.KV * a.hd, qrow = a.H * a.hd;
  const T* kb = static_cast<const T*>(a.k) + (int64_t)b * a.S * kvw + kvh * a.hd;
  const T* vb = static_cast<const T*>(a.v) + (int64_t)b * a.S * kvw + kvh * a.hd;

  // last key that query i sees
  auto behind = [&](int i) { return (int)min((unsigned)i + (unsigned)a.right, (unsigned)len - 1); };

  // blocks: those of the sinks before the window's first, then the window's
  const int last = min(q0 + BQ - 1, len - 1);
  const int first_blk = max(0, q0 - a.left) / BKV;
  const int last_blk = behind(last) / BKV;
  const int sink_blks = (int)min((int64_t)first_blk, ((int64_t)a.sinks + BKV - 1) / BKV);
  const int n = sink_blks + last_blk - first_blk + 1;
  auto block_of = [&](int t) { return t < sink_blks ? t : first_blk + t - sink_blks; };

  // KW blocks of K and V on their way: 8 values a chunk
  typedef float floatx8 __attribute__((ext_vector_type(8)));
  typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
  using Chunk = std::conditional_t<F32, floatx8, uintx4>;
  Chunk ck[PER], cv[PER];
  auto each = [&](auto f) {  // f(i, block of the KW, row, chunk) for each chunk of the thread's
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = tid + THREADS * i, j = KW == 1 ? 0 : e / Cfg::CHUNKS;
      const int row = (KW == 1 ? e : e % Cfg::CHUNKS) / (2 * KS), c = e % (2 * KS);
      if (e < KW * Cfg::CHUNKS && 8 * c < a.hd) f(i, j, row, c);
    }
  };
  // blocks past the last and rows past the last key: the last ones again (the former are not computed, the
  // latter's scores masked). One block is read from a scalar base at 32-bit offsets (64-bit addresses of each
  // row: 54.6 -> 53.2 us at 16384 tokens)
  const unsigned row_bytes = (unsigned)(kvw * sizeof(T));  // BKV of them: below 2^31
  auto fetch = [&](int t) {
    const int blk0 = block_of(t * KW);
    const unsigned end = min(BKV, len - 1 - blk0 * BKV) * row_bytes;  // of KW = 1: where the last row begins
    const char* kt = reinterpret_cast<const char*>(kb + (int64_t)blk0 * BKV * kvw);
    const char* vt = reinterpret_cast<const char*>(vb + (int64_t)blk0 * BKV * kvw);
    each([&](int i, int j, int row, int c) {
      if constexpr (KW == 1) {
        const unsigned col = 8 * sizeof(T) * c, at = min(row * row_bytes, end) + col;
        ck[i] = *reinterpret_cast<const Chunk*>(kt + at);
        cv[i] = *reinterpret_cast<const Chunk*>(vt + at);
      } else {
        const int blk = block_of(min(t * KW + j, n - 1));
        const int64_t at = (int64_t)min(blk * BKV + row, len - 1) * kvw + 8 * c;
        ck[i] = *reinterpret_cast<const Chunk*>(kb + at);
        cv[i] = *reinterpret_cast<const Chunk*>(vb + at);
      }
    });
  };
  auto parts_of = [&](Chunk x, float by) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[e] * by;
    return split8(y);
  };
  auto put = [&](Chunk x, char* to) {
    if constexpr (F32) {
      const Split8 s = parts_of(x, 1.f);
      *reinterpret_cast<bf16x8*>(to) = s.h;
      *reinterpret_cast<bf16x8*>(to + PLANE) = s.m;
      *reinterpret_cast<bf16x8*>(to + 2 * PLANE) = s.l;
    } else {
      *reinterpret_cast<Chunk*>(to) = x;
    }
  };
  auto store = [&] {
    each([&](int i, int j, int row, int c) {
      char* at = smem + j * SLOT + row * PITCH + 16 * c;
      put(ck[i], at);
      put(cv[i], at + PARTS * PLANE);
    });
  };
  if (a.hd < 16 * KS) {  // columns behind the head's last stay zero
    for (int e = tid; e < KW * 2 * PARTS * BKV; e += THREADS)
      for (int c = a.hd / 8; c < 2 * KS; ++c)
        *reinterpret_cast<float4*>(smem + e * PITCH + 16 * c) = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  fetch(0);

  // Q: B operand, query l32, dimensions 16 s + 8 g .. + 7. f32: times the scale in powers of two; bf16: as
  // it is, up to the scale's sign, the scale in the exponent instead.
  const float qs = a.scale * 1.4426950408889634f;
  const float cs = F32 ? 1.f : fabsf(qs);
  bf16x8 qf[KS][PARTS];
  {
    const T* p = static_cast<const T*>(a.q) + ((int64_t)b * a.S + min(qi, len - 1)) * qrow + h * a.hd + 8 * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      Chunk x = 0;
      if (16 * s + 8 * g < a.hd) x = *reinterpret_cast<const Chunk*>(p + 16 * s);
      if constexpr (F32) {
        const Split8 sp = parts_of(x, qs);
        qf[s][0] = sp.h;
        qf[s][1] = sp.m;
        qf[s][2] = sp.l;
      } else {
        qf[s][0] = __builtin_bit_cast(bf16x8, x ^ (qs < 0.f ? 0x80008000u : 0u));
      }
    }
  }

  floatx16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[t][v] = 0.f;
  float ref = 0.f, lsum = 0.f;  // ref: in the scores' units
  bool begun = false;           // whether the query has seen a key

  const char* kf0 = smem + kg * SLOT + l32 * PITCH + 16 * g;
  const char* vf0 = smem + kg * SLOT + PARTS * PLANE + (4 * g + ((lane & 15) >> 2)) * PITCH + 32 * ((lane >> 4) & 1) +
                    8 * (lane & 3);
  auto vfrag = [&](int part, int t, int ks) {  // dimensions 32 t + l32, keys 16 ks + 4 g + {0..3, 8..11}
    typedef short short4v __attribute__((ext_vector_type(4)));
    const char* p = vf0 + part * PLANE + 16 * ks * PITCH + 64 * t;
    union {
      short4v s[2];
      bf16x8 f;
    } u;
    u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)p);
    u.s[1] =
        __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(p + 8 * PITCH));
    return u.f;
  };

  const int last_n = behind(qn), last_w = behind(qw);  // of the wave's last and first query
  store();
  for (int t = 0; t * KW < n; ++t) {
    lds_barrier();
    const int k0 = block_of(t * KW + kg) * BKV, k1 = k0 + BKV - 1;
    if ((t + 1) * KW < n) fetch(t + 1);
    // seen by any query of the wave?
    const bool any = qw <= qn && t * KW + kg < n && k0 <= last_n && (k1 >= qw - a.left || k0 < a.sinks);
    if (any) {
      floatx16 st[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) st[j][v] = 0.f;
      if constexpr (F32) {
        floatx16 low;  // the five smaller products, in an accumulator of their own (x3.hpp)
#pragma unroll
        for (int v = 0; v < 16; ++v) low[v] = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          Split8 kx, qx{qf[s][0], qf[s][1], qf[s][2]};
          kx.h = *reinterpret_cast<const bf16x8*>(kf0 + 32 * s);
          kx.m = *reinterpret_cast<const bf16x8*>(kf0 + PLANE + 32 * s);
          kx.l = *reinterpret_cast<const bf16x8*>(kf0 + 2 * PLANE + 32 * s);
#pragma unroll
          for (int p = 0; p < 5; ++p) low = mfma_x3(kx, qx, low, p);
          st[0] = mfma_x3(kx, qx, st[0], 5);
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) st[0][v] += low[v];
      } else {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int j = 0; j < NT; ++j)
            st[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                *reinterpret_cast<const bf16x8*>(kf0 + 32 * j * PITCH + 32 * s), qf[s][0], st[j], 0, 0, 0);
      }
      const bool whole = (k0 >= qn - a.left || k1 < a.sinks) && k1 <= last_w;
      if (!whole) {
        // a bit a key: keys below hi, and not below lo or below the sinks' end; then two instructions a score
        // that need no lane masks (three comparisons a score: 55.5 -> 54 us; 16384 keys)
        const int first = k0 + 4 * g;  // the lane's: key c below is first + c
        const int hi = behind(qi) + 1 - first;
        const int lo = qi - a.left - first, sk = a.sinks - first;
        auto below = [](int n) { return (unsigned)((1ull << min(max(n, 0), 32)) - 1); };  // the first n of 32
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int seen = (int)(below(hi - 32 * j) & (~below(lo - 32 * j) | below(sk - 32 * j)));
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const unsigned m = (unsigned)__builtin_amdgcn_sbfe(seen, 8 * (v / 4) + v % 4, 1);
            const float x = st[j][v];
            st[j][v] = __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, x) & m) | (0xff800000u & ~m));
          }
        }
      }
      // maximum keeps NaN, which costs no canonical forms; a NaN neither moves the reference nor passes
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int v = 0; v < 16; v += 2) mx = max_nan(max_nan(mx, st[j][v]), st[j][v + 1]);
      const auto far = [&] { return begun ? (mx - ref) * cs > 8.f : mx > -INFINITY; };
      if (__any(far())) {
        mx = other_half(mx, max_nan);  // the query's other keys
        const bool move = far();
        // the first visible key has nothing to rescale
        const float alpha = !move ? 1.f : begun ? __builtin_amdgcn_exp2f((ref - mx) * cs) : 0.f;
        lsum *= alpha;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] *= alpha;
        ref = move ? mx : ref;
        begun |= move;
      }
      // ahead of the waves that are at their scores: this part feeds both pipes (57.4 -> 55.5 us at 16384 keys)
      __builtin_amdgcn_s_setprio(1);
      const float off = ref * cs;
      // the block's probabilities are added up by themselves before they join the running sum
      float ps = 0.f;
#pragma unroll
      for (int ks = 0; ks < 2 * NT; ++ks) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = __builtin_amdgcn_exp2f(fmaf(st[ks >> 1][8 * (ks & 1) + e], cs, -off));
          if (F32) ps += p[e];
        }
        if constexpr (F32) {
          const Split8 px = split8(p);
#pragma unroll
          for (int i = 0; i < DT; ++i) {
            const Split8 vx{vfrag(0, i, ks), vfrag(1, i, ks), vfrag(2, i, ks)};
#pragma unroll
            for (int m = 0; m < 6; ++m) o[i] = mfma_x3(vx, px, o[i], m);
          }
        } else {
          // probabilities to bf16, to nearest (each is off by 2^-9 of itself at most), and the sum of
          // those, two an instruction
          const uintx4 pb{cvt_pk_bf16(p[0], p[1]), cvt_pk_bf16(p[2], p[3]), cvt_pk_bf16(p[4], p[5]),
                          cvt_pk_bf16(p[6], p[7])};
          const bf16x8 px = __builtin_bit_cast(bf16x8, pb);
#pragma unroll
          for (int e = 0; e < 4; ++e) ps = add_pair(pb[e], ps);
#pragma unroll
          for (int i = 0; i < DT; ++i)
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vfrag(0, i, ks), px, o[i], 0, 0, 0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
      lsum += ps;
    }
    lds_barrier();
    if ((t + 1) * KW < n) store();
  }

  if constexpr (KW > 1) {  // the other key groups' results to the first's waves
    constexpr int PER_WAVE = (16 * DT + 2) * 64;
    float* sh = reinterpret_cast<float*>(smem) + lane;
    if (kg) {
      float* to = sh + (qg * (KW - 1) + kg - 1) * PER_WAVE;
      to[0] = begun ? ref : lsum == 0.f ? -INFINITY : 0.f;  // NaN scores leave ref at 0 and a sum of NaN
      to[64] = lsum;
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) to[64 * (2 + 16 * i + v)] = o[i][v];
    }
    __syncthreads();
    if (kg) return;
#pragma unroll 1
    for (int j = 0; j < KW - 1; ++j) {
      const float* from = sh + (qg * (KW - 1) + j) * PER_WAVE;
      const float r = from[0];
      if (r == -INFINITY) continue;  // it saw nothing of this query's
      const float top = begun ? max_nan(ref, r) : r;
      const float by0 = begun ? __builtin_amdgcn_exp2f((ref - top) * cs) : 0.f;
      const float by1 = __builtin_amdgcn_exp2f((r - top) * cs);
      lsum = lsum * by0 + from[64] * by1;
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[i][v] = o[i][v] * by0 + from[64 * (2 + 16 * i + v)] * by1;
      ref = top;
      begun = true;
    }
  }

  const float l = other_half(lsum, [](float x, float y) { return x + y; });
  const float inv = 1.f / l;
  float chk = l * 0.f;
  bool bad = !F32 && l < 0x1p-60f;
#pragma unroll
  for (int c = 0; c < 2 * KS; ++c)  // dimensions 8 c + 4 g .. + 3
    if (8 * c < a.hd) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = o[c / 4][4 * (c % 4) + e];
        chk = fmaf(x, 0.f, chk);
        if (F32) bad |= (x != 0.f) & (fabsf(x) < l * 0x1p-109f);
      }
    }
  unsigned long long again = __ballot(qi < len && (bad || !(chk == 0.f)));
  again = (again | (again >> 32)) & 0xffffffffull;
  if (qi < len && !((again >> l32) & 1)) {
    T* out = static_cast<T*>(a.o) + ((int64_t)b * a.S + qi) * qrow + h * a.hd + 4 * g;
#pragma unroll
    for (int c = 0; c < 2 * KS; ++c)
      if (8 * c < a.hd) {
        const floatx16& ot = o[c / 4];
        const int v = 4 * (c % 4);
        if constexpr (F32)
          *reinterpret_cast<float4*>(out + 8 * c) =
              make_float4(ot[v] * inv, ot[v + 1] * inv, ot[v + 2] * inv, ot[v + 3] * inv);
        else
          *reinterpret_cast<uint2*>(out + 8 * c) =
              make_uint2(cvt_pk_bf16(ot[v] * inv, ot[v + 1] * inv),
                         cvt_pk_bf16(ot[v + 2] * inv, ot[v + 3] * inv));
      }
  }
  while (again) {
    const int j = __builtin_ctzll(again);
    again &= again - 1;
    window_query<T>(a, b, h, qw + j, len);
  }
}

template <class T, int KS, int KW, int NW>
void launch_window_kw(const LaunchCtx& c, const WindowArgs& a) {
  using Cfg = WindowCfg<T, KS, KW, NW>;
  const int64_t units = (int64_t)cdiv(a.S, Cfg::BQ) * a.H * a.B;
  MNN_REQUIRE(units < (1 << 24), MNN_ERR_INVALID_CONFIGURATION,
              "WindowAttention: too many tokens in one call");
  launch(c, sizeof(T) == 4 ? "window_f32" : "window_bf16", window_kernel<T, KS, KW, NW>, dim3((unsigned)units),
         dim3(Cfg::THREADS), 0, a);
}

template <class T, int KS>
void launch_window(const LaunchCtx& c, const WindowArgs& a) {
  // Key groups by how much of the GPU 128 queries a workgroup would fill. us for KW = 1 / 2 / 4, 8 heads:
  // f32 hd 48 1344 tokens, 168 both ways (88 workgroups): 33 / 27 / 18; 2 x 1344, 511 both ways (176): 62 / 50 /
  // 48; 4096, 2047 back (256): 111 / 88 / 98; 4 x 1344 (352): 45 / 49 / 50. bf16 hd 64 the same: 17 / 14 / 10,
  // 26 / 21 / 25, 42 / 33 / 41, 21 / 20 / 27; 16384, 1023 back (1024): 58 / 61 / 116. f32 hd 128 has registers
  // for one wave a SIMD with KW = 1: 16384, 1023 back 534 / 430.
  // Where workgroups of 96 queries, 4 key groups, 12 waves fit the compute units at once, each has a quarter less to do and a
  // third wave a SIMD: 2 x 1344, 168 both ways, f32 hd 48 24.7 -> 20.8, hd 64 28.2 -> 24.5; 3008, 2047 back, f32 hd 64
  // 88 -> 70, bf16 31.6 -> 25.5 (2 x 1344, 168 both ways 13.0 -> 13.1); in two rounds they lose (bf16 hd 64, 4 x 1344 17 -> 25).
  const int64_t wgs = (int64_t)cdiv(a.S, 128) * a.H * a.B, cus = c.dev->props.multiProcessorCount;
  const int64_t keys = std::min<int64_t>(a.S, (int64_t)128 + a.left + a.right + a.sinks);
  constexpr bool F32 = sizeof(T) == 4, FOUR = KS <= 5 || !F32;  // four blocks fit in LDS
  if (keys > 2 * WindowCfg<T, KS, 1, 4>::BKV) {
    if constexpr (FOUR)
      if (2 * wgs < cus) return launch_window_kw<T, KS, 4, 8>(c, a);
    if constexpr (KS <= 4)
      if ((int64_t)cdiv(a.S, 96) * a.H * a.B <= cus) return launch_window_kw<T, KS, 4, 12>(c, a);
    if (4 * wgs < 5 * cus || (F32 && KS > 6)) return launch_window_kw<T, KS, 2, 8>(c, a);
  }
  launch_window_kw<T, KS, 1, 4>(c, a);
}

template <class T>
void launch_window_t(const LaunchCtx& c, const WindowArgs& a) {
  switch ((a.hd + 15) / 16) {
    case 1:
    case 2: return launch_window<T, 2>(c, a);
    case 3: return launch_window<T, 3>(c, a);
    case 4: return launch_window<T, 4>(c, a);
    case 5: return launch_window<T, 5>(c, a);
    case 6: return launch_window<T, 6>(c, a);
    default: return launch_window<T, 8>(c, a);
  }
}

}  // namespace

void window_attention(const LaunchCtx& c, const WindowArgs& a) {
  if (a.type == MNN_F32)
    launch_window_t<float>(c, a);
  else
    launch_window_t<__bf16>(c, a);
}

}  // namespace k
}  // namespace mnn
