// Softmax attention of a wave's queries to blocks of 32 keys on the bf16 matrix cores, for keys and values in f32, bf16 or
// e4m3: 32 queries to keys in LDS that other waves use as well (AttendMany), or 16 to keys of the wave's own (AttendFew).
//
// The scores are computed TRANSPOSED, S^T = K Q^T: a lane's accumulators hold 4 or 16 keys of one query, and are the B
// operand that O^T += V^T P^T needs when its k slots take those keys, so P goes from the softmax straight into the second
// product. V lies in LDS row by row, in bf16; V^T's fragments (4 keys of one dimension a lane) are transposed on the way
// out by ds_read_b64_tr_b16.
//
// f32 operands are three bf16 parts each and six partial products are kept (x3.hpp). e4m3 values are bf16 values, so
// they take one part, and three products with f32 queries and probabilities; their rows' scales multiply the scores,
// and the probabilities before these are rounded or split.
//
// Softmax: p = exp2(s - ref), s in powers of two, with a reference that moves only when a block's maximum exceeds
// it by 2^8. AttendMany takes bf16 scores as the products give them and p as exp2(c s - c ref) in one fused step: c ref is
// rounded, by the same amount for all keys of a reference, but of scores past 2^31 all probabilities may come out as 0
// then (their sum is about 1 or more otherwise): such rows are computed again, too.
//
// Results that are not finite (a value of 2^120 or more times p <= 2^8, or parts of values that are not finite) or,
// in f32, so small that parts of them have left bf16's range are computed again by attend_row.
#pragma once

#include "kv_slots.hpp"
#include "token_utils.hpp"
#include "x3.hpp"

namespace mnn {
namespace dev {

struct E4m3 {
  uint8_t x;
};

// Eight values of a row as they come: split in three for f32, else one part.
template <class M>
struct Parts {
  static constexpr int N = sizeof(M) == 4 ? 3 : 1;
  bf16x8 p[N];
};
template <class M>
__device__ __forceinline__ Parts<M> parts_of(const Eight<M>& x) {
  Parts<M> r;
  if constexpr (sizeof(M) == 4) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = x[e];
    const Split8 s = split8(v);
    r.p[0] = s.h;
    r.p[1] = s.m;
    r.p[2] = s.l;
  } else {
    r.p[0] = __builtin_bit_cast(bf16x8, x.x[0]);
  }
  return r;
}
template <>
struct Eight<E4m3> {
  uint2 x;
  __device__ __forceinline__ void clear() { x = make_uint2(0, 0); }
  __device__ __forceinline__ void load(const E4m3* p) { x = *reinterpret_cast<const uint2*>(p); }
};
__device__ __forceinline__ Parts<E4m3> parts_of(const Eight<E4m3>& x) {
  Parts<E4m3> r;
  r.p[0] = widen8((int)x.x.x, (int)x.x.y);
  return r;
}

// What both have in common. T: of queries and output, M: of keys and values.
template <class T, class M>
struct AttendTypes {
  static constexpr bool F32 = sizeof(T) == 4, HELD = sizeof(M) == 1;
  static constexpr int PQ = F32 ? 3 : 1, PM = Parts<M>::N;
  // a result below this may miss bits of its operands' parts (x3.hpp): those below 2^-110 of f32 values, or of
  // probabilities times a scale, with values up to 448 of them
  static constexpr float TINY_RESULT = HELD ? 0x1p-96f : 0x1p-109f;
  // Whether a result has to be computed again.
  static __device__ __forceinline__ bool doubtful(float x) {
    return !(x * 0.f == 0.f) || (F32 && x != 0.f && fabsf(x) < TINY_RESULT);
  }
  // Q as B operand; f32 times the scale in powers of two, bf16 as it is, up to the scale's sign.
  static __device__ __forceinline__ void take_q(const Eight<T>& x, float qs, bf16x8 (&q)[PQ]) {
    if constexpr (F32) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = x[e] * qs;
      const Split8 sp = split8(v);
      q[0] = sp.h;
      q[1] = sp.m;
      q[2] = sp.l;
    } else {
      q[0] = __builtin_bit_cast(bf16x8, x.x[0] ^ (qs < 0.f ? 0x80008000u : 0u));
    }
  }
  // Products of keys and queries; `low`: the smaller ones of parts, in an accumulator of their own (x3.hpp).
  template <class Acc, class Mfma>
  static __device__ __forceinline__ void products(const Parts<M>& k, const bf16x8 (&q)[PQ], Acc& st, Acc& low, Mfma mfma) {
    if constexpr (PM == 3) {
      low = mfma(k.p[2], q[0], low);
      low = mfma(k.p[0], q[2], low);
      low = mfma(k.p[1], q[1], low);
      low = mfma(k.p[1], q[0], low);
      low = mfma(k.p[0], q[1], low);
    } else if constexpr (PQ == 3) {
      low = mfma(k.p[0], q[2], low);
      low = mfma(k.p[0], q[1], low);
    }
    st = mfma(k.p[0], q[0], st);
  }
  // Eight probabilities (e4m3: times their values' scales) to the second product; v(part, tile): fragments of V^T.
  // PP: the bf16 parts that a probability beside bf16 values is taken in, one (off by 2^-8 of itself at most) or two
  // (2^-16); v_exp_f32 and the sums are fp32's. Returns the sum of the rounded ones, of one part, without scales; else 0.
  template <int PP, int TILES, class Acc, class V, class Mfma>
  static __device__ __forceinline__ float values(const float (&p)[8], V v, Acc (&o)[TILES], Mfma mfma) {
    typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
    float ps = 0.f;
    if constexpr (F32) {
      const Split8 px = split8(p);
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        const bf16x8 h = v(0, i);
        if constexpr (PM == 3) {
          const bf16x8 m = v(1, i), l = v(2, i);
          o[i] = mfma(l, px.h, o[i]);
          o[i] = mfma(h, px.l, o[i]);
          o[i] = mfma(m, px.m, o[i]);
          o[i] = mfma(m, px.h, o[i]);
        } else {
          o[i] = mfma(h, px.l, o[i]);
        }
        o[i] = mfma(h, px.m, o[i]);
        o[i] = mfma(h, px.h, o[i]);
      }
    } else {
      const uintx4 pb{cvt_pk_bf16(p[0], p[1]), cvt_pk_bf16(p[2], p[3]), cvt_pk_bf16(p[4], p[5]), cvt_pk_bf16(p[6], p[7])};
      const bf16x8 px = __builtin_bit_cast(bf16x8, pb);
      if constexpr (PP == 2) {
        uintx4 rb;
#pragma unroll
        for (int e = 0; e < 4; ++e) rb[e] = cvt_pk_bf16(p[2 * e] - bf16_lo(pb[e]), p[2 * e + 1] - bf16_hi(pb[e]));
        const bf16x8 rx = __builtin_bit_cast(bf16x8, rb);
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
          const bf16x8 f = v(0, i);
          o[i] = mfma(f, rx, o[i]);
          o[i] = mfma(f, px, o[i]);
        }
      } else {
        if (!HELD) {  // two an instruction
#pragma unroll
          for (int e = 0; e < 4; ++e) ps = add_pair(pb[e], ps);
        }
#pragma unroll
        for (int i = 0; i < TILES; ++i) o[i] = mfma(v(0, i), px, o[i]);
      }
    }
    return ps;
  }
};

// Four keys of one dimension a lane, eight of them in two reads.
__device__ __forceinline__ bf16x8 read_transposed(const char* p, int to_next) {
  typedef short short4v __attribute__((ext_vector_type(4)));
  union {
    short4v s[2];
    bf16x8 f;
  } u;
  u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)p);
  u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(p + to_next));
  return u.f;
}
// The first n of 32 keys, as bits.
__device__ __forceinline__ unsigned keys_below(int n) { return (unsigned)((1ull << min(max(n, 0), 32)) - 1); }
// A score, or -infinity where bit `key` is 0: two instructions that need no lane masks.
__device__ __forceinline__ float masked_score(float x, int seen, int key) {
  const unsigned m = (unsigned)__builtin_amdgcn_sbfe(seen, key, 1);
  return __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, x) & m) | (0xff800000u & ~m));
}

// 32 queries a wave on v_mfma_f32_32x32x16_bf16, heads of up to 16 KS dimensions: lane (g, q) holds the scores of keys
// 8 (v / 4) + 4 g + v % 4 of query q.
template <class T, class M, int KS>
struct AttendMany : AttendTypes<T, M> {
  using A = AttendTypes<T, M>;
  using A::F32;
  using A::HELD;
  using A::PM;
  using A::PQ;
  static constexpr bool RAW = !F32 && !HELD;  // scores are multiplied by cs in the exponent
  static constexpr int DT = (KS + 1) / 2;     // 32-row tiles of O^T
  // bytes from one key's row to the next in LDS: 8 rows of 16-byte reads on distinct banks
  static constexpr int PITCH = KS * 32 + (KS % 2 ? 0 : 16);

  bf16x8 q[KS][PQ];
  floatx16 o[DT];
  float ref, sum;  // the query's; the sum of the lane's keys
  bool begun;      // whether the query has a score above -infinity
  float cs;        // what is left to multiply scores by

  static __device__ __forceinline__ floatx16 mfma(bf16x8 a, bf16x8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[t][v] = 0.f;
    ref = 0.f;
    sum = 0.f;
    begun = false;
  }
  __device__ __forceinline__ void load_q(const T* p, bool on, int hd, float scale) {
    const int g = (threadIdx.x & 63) >> 5;
    const float qs = scale * 1.4426950408889634f;
    cs = F32 ? 1.f : fabsf(qs);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      Eight<T> x;
      x.clear();
      if (on && 16 * s + 8 * g < hd) x.load(p + 16 * s + 8 * g);
      A::take_q(x, qs, q[s]);
    }
  }
  // Scores of 32 keys, k(s): dimensions 16 s + 8 g .. + 7 of key l32.
  template <class K>
  __device__ __forceinline__ floatx16 scores(K k) const {
    floatx16 st, low;
#pragma unroll
    for (int v = 0; v < 16; ++v) st[v] = low[v] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) A::products(k(s), q[s], st, low, mfma);
    if constexpr (F32) {
#pragma unroll
      for (int v = 0; v < 16; ++v) st[v] += low[v];
    }
    return st;
  }
  // seen: bit i for the lane's key i + 4 g
  static __device__ __forceinline__ void mask(floatx16& st, int seen) {
#pragma unroll
    for (int v = 0; v < 16; ++v) st[v] = masked_score(st[v], seen, 8 * (v / 4) + v % 4);
  }
  // The larger of mx and scores st; keeps NaN, which neither moves the reference nor passes.
  static __device__ __forceinline__ float largest(const floatx16& st, float mx) {
#pragma unroll
    for (int v = 0; v < 16; v += 2) mx = max_nan(max_nan(mx, st[v]), st[v + 1]);
    return mx;
  }
  // Moves the reference for scores up to mx where it has to.
  __device__ __forceinline__ void refer(float mx) {
    const float unit = RAW ? cs : 1.f;
    const auto far = [&] { return begun ? (mx - ref) * unit > 8.f : mx > -INFINITY; };
    if (__any(far())) {
      mx = other_half(mx, max_nan);  // the query's other keys
      const bool move = far();
      // the first visible key has nothing to rescale
      const float alpha = !move ? 1.f : begun ? __builtin_amdgcn_exp2f((ref - mx) * unit) : 0.f;
      sum *= alpha;
#pragma unroll
      for (int i = 0; i < DT; ++i) o[i] *= alpha;
      ref = move ? mx : ref;
      begun |= move;
    }
  }
  // Probabilities of 32 keys and the second product; v(part, t, ks): dimensions 32 t + l32, keys 16 ks + 4 g + {0..3,
  // 8..11}; vs(i): the scale (e4m3) of the value of the lane's i-th key.
  template <class V, class S>
  __device__ __forceinline__ void add(const floatx16& st, V v, S vs) {
    float ps = 0.f;  // added up by themselves before they join the running sum
    const float off = ref * cs;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float s = st[8 * ks + e];
        p[e] = __builtin_amdgcn_exp2f(RAW ? fmaf(s, cs, -off) : s - ref);
        if (!RAW) ps += p[e];
        if (HELD) p[e] *= vs(8 * ks + e);
      }
      // one part: results of 1.8e-3 (2-norm, e4m3 2.4e-3) where two give 1.66e-3, for 319 us against 437 (8192 tokens on
      // 16384 states; e4m3 364 against 537), since the instructions beside the exponentials bound these calls
      ps += A::template values<1>(p, [&](int part, int t) { return v(part, t, ks); }, o, mfma);
    }
    sum += ps;
  }
  // Where the lane's fragments of V^T begin in a block of V in LDS.
  static __device__ __forceinline__ const char* v_first(const char* block) {
    const int lane = threadIdx.x & 63, g = lane >> 5;
    return block + (4 * g + ((lane & 15) >> 2)) * PITCH + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
  }
  static __device__ __forceinline__ bf16x8 v_frag(const char* first, int plane, int part, int t, int ks) {
    return read_transposed(first + part * plane + 16 * ks * PITCH + 64 * t, 8 * PITCH);
  }
};

// 16 queries a wave on v_mfma_f32_16x16x32_bf16, heads of up to 32 KS dimensions, 32 keys in two tiles of 16: lane (g, q),
// g of 4, holds the scores of keys 16 j + 4 g + v of query q.
template <class T, class M, int KS>
struct AttendFew : AttendTypes<T, M> {
  using A = AttendTypes<T, M>;
  using A::F32;
  using A::HELD;
  using A::PM;
  using A::PQ;
  static constexpr int OT = 2 * KS;  // 16-row tiles of O^T
  // bytes from one key's row of V to the next in LDS: 8 rows of 32-byte reads on all banks
  static constexpr int PITCH = 64 * KS + 32;
  static constexpr int PLANE = 32 * PITCH;

  bf16x8 q[KS][PQ];
  floatx4 o[OT];
  float ref, sum;  // the query's; the sum of the lane's keys
  bool begun;      // whether the query has a score above -infinity
  float cs;        // what is left to multiply scores by

  static __device__ __forceinline__ floatx4 mfma(bf16x8 a, bf16x8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  // The dimensions of chunk s of lane group g: 8 of them. Rows of e4m3 are read 16 bytes a lane, two chunks.
  static __device__ __forceinline__ int dim_of(int s, int g) {
    if (HELD && !(KS % 2 && s == KS - 1)) return 64 * (s / 2) + 16 * g + 8 * (s % 2);
    return 32 * s + 8 * g;
  }
  // Whether a chunk may lie behind a head's last dimension: heads have more than 32 (KS - 1) of them.
  static constexpr bool may_end(int s) { return HELD && KS % 2 == 0 ? s >= KS - 2 : s == KS - 1; }

  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int t = 0; t < OT; ++t) o[t] = floatx4{0.f, 0.f, 0.f, 0.f};
    ref = 0.f;
    sum = 0.f;
    begun = false;
  }
  // The queries in two steps, their loads and what is made of them, with others between them.
  static __device__ __forceinline__ void fetch_q(const T* p, bool on, int hd, Eight<T> (&x)[KS]) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = dim_of(s, g);
      x[s].clear();
      if (on && d < hd) x[s].load(p + d);
    }
  }
  __device__ __forceinline__ void take_q(const Eight<T> (&x)[KS], float scale) {
    const float qs = scale * 1.4426950408889634f;
    cs = F32 ? 1.f : fabsf(qs);
#pragma unroll
    for (int s = 0; s < KS; ++s) A::take_q(x[s], qs, q[s]);
  }
  // Scores of 16 keys, k(s): chunk s of the lane's key.
  template <class K>
  __device__ __forceinline__ floatx4 scores(K k) const {
    floatx4 st{0.f, 0.f, 0.f, 0.f}, low{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s) A::products(k(s), q[s], st, low, mfma);
    if constexpr (F32) st += low;
    return st;
  }
  // Moves the reference for scores up to mx where it has to.
  __device__ __forceinline__ void refer(float mx) {
    const auto far = [&] { return begun ? mx - ref > 8.f : mx > -INFINITY; };
    if (__any(far())) {
      mx = other_half(other_row(mx, max_nan), max_nan);  // the query's other keys
      const bool move = far();
      // the first visible key has nothing to rescale
      const float alpha = !move ? 1.f : begun ? __builtin_amdgcn_exp2f(ref - mx) : 0.f;
      sum *= alpha;
#pragma unroll
      for (int i = 0; i < OT; ++i) o[i] *= alpha;
      ref = move ? mx : ref;
      begun |= move;
    }
  }
  // Probabilities of 32 keys and the second product; v(part, t): dimensions 16 t + lane % 16, keys 4 g + {0..3, 16..19};
  // vs: the scales (e4m3) of the values of the lane's keys.
  template <class V>
  __device__ __forceinline__ void add(const floatx4 (&st)[2], V v, const float (&vs)[8]) {
    float p[8], ps = 0.f;  // added up by themselves before they join the running sum
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = __builtin_amdgcn_exp2f(st[e / 4][e % 4] - ref);
      ps += p[e];
      if (HELD) p[e] *= vs[e];
    }
    // bf16 calls: two parts, so that their results keep a rounding's distance, as the step on unrounded caches does (2-norm
    // 1.7e-3 against 2.4e-3 with one part), where memory or one block's chain bounds the call
    A::template values<2>(p, v, o, mfma);
    sum += ps;
  }
  // Where the lane's fragments of V^T begin in a block of V in LDS.
  static __device__ __forceinline__ const char* v_first(const char* block) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
    return block + (4 * g + ((lane & 15) >> 2)) * PITCH + 8 * (lane & 3);
  }
  static __device__ __forceinline__ bf16x8 v_frag(const char* first, int part, int t) {
    return read_transposed(first + part * PLANE + 32 * t, 16 * PITCH);
  }
};

// Results that workgroups pass to each other within a launch. Stores and loads go to where all XCDs agree (agent scope:
// no L2 keeps such a store to itself, none answers such a load from an older copy), so that no L2 has to be written back
// or emptied around them (a release and an acquire fence a workgroup took 12 us for 512 of them).
__device__ __forceinline__ void put_shared(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get_shared(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether the calling workgroup is the last of n that share out the keys of one unit, whose count (0 before and after)
// they pass on their way out: what the others have put_shared is then there for get_shared. Uniform over the workgroup.
__device__ __forceinline__ bool last_of(int* count, int n, int* shared) {
  // every wave's stores have arrived before the workgroup counts
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const int before = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *shared = before == n - 1;
    if (before == n - 1) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return *shared != 0;
}

// One query by one wave, on the vector units in fp32, in two passes: the scores' maximum and their sum, then the
// outputs of dimensions lane and lane + 64, each value times its own probability. The keys that the query sees are
// taken 64 at a time, lane j scoring key j; others are not read. key_at(t) / value_at(t): rows of the t-th of n
// visible keys.
template <class T, class K, class V>
__device__ __forceinline__ void attend_row(const T* __restrict__ q, int hd, float scale, int64_t n, K key_at, V value_at,
                                           float& o0, float& o1) {
  const int lane = threadIdx.x & 63;
  const float qs = scale * 1.4426950408889634f;
  auto score = [&](int64_t t) {
    if (t >= n) return -INFINITY;
    const auto kp = key_at(t);
    float dot = 0.f;
    for (int d = 0; d < hd; ++d) dot = fmaf(to_f32(q[d]) * qs, to_f32(kp[d]), dot);
    return dot;
  };
  float m = -INFINITY, l = 0.f;
  for (int64_t t0 = 0; t0 < n; t0 += 64) {
    const float s = score(t0 + lane), mn = max_nan(m, group_reduce<64>(s, max_nan));
    const float ref = mn == -INFINITY ? 0.f : mn;
    l = l * __builtin_amdgcn_exp2f(m - ref) + group_reduce<64>(t0 + lane < n ? __builtin_amdgcn_exp2f(s - ref) : 0.f, Plus{});
    m = mn;
  }
  const float ref = m == -INFINITY ? 0.f : m, inv = 1.f / l;
  o0 = o1 = 0.f;
  for (int64_t t0 = 0; t0 < n; t0 += 64) {
    const int cnt = (int)(n - t0 < 64 ? n - t0 : 64);
    const float p = lane < cnt ? __builtin_amdgcn_exp2f(score(t0 + lane) - ref) * inv : 0.f;
    for (int j = 0; j < cnt; ++j) {
      const float pj = __shfl(p, j, 64);
      const auto vp = value_at(t0 + j);
      if (lane < hd) o0 = fmaf(pj, to_f32(vp[lane]), o0);
      if (lane + 64 < hd) o1 = fmaf(pj, to_f32(vp[lane + 64]), o1);
    }
  }
}

// A row of 8-bit values and its scale, or a row that is still to be rounded to them, read as what they stand for.
template <class T>
struct HeldRow {
  const uint8_t* p;
  const T* fresh;  // not null: the row as it came
  float scale, inv;
  __device__ __forceinline__ float operator[](int d) const {
    const int q = fresh ? (int)pack_e4m3(to_f32(fresh[d]) * inv, 0.f, 0.f, 0.f) : (int)p[d];
    return __builtin_amdgcn_cvt_f32_fp8(q, 0) * scale;
  }
  static __device__ __forceinline__ HeldRow rounding(const T* x, int hd) {
    float top = 0.f;
    for (int d = 0; d < hd; ++d) top = max_nan(top, fabsf(to_f32(x[d])));
    const RowScale rs = row_scale(top);
    return {nullptr, x, rs.scale, rs.inv};
  }
};

}  // namespace dev
}  // namespace mnn
