// Attention of a decoder's tokens to an encoder's states, whole sequences of both: o_i = sum_j p_ij v_j, p_i = softmax
// of scale q_i k_j over the states j of the sequence.
//
// A workgroup takes 32 NW rows (row = token * G + head of the group: all heads that read one key/value head share its
// states) and the keys of a sequence, or a range of them, in blocks that lie in LDS in bf16 parts, two slots, so that
// one barrier a block is enough: behind it the next block's rows are fetched to registers, this one is computed
// (attend.hpp), and the next one is split or widened and stored to the other slot. Of workgroups that share out the keys
// of the same rows the last one to finish joins the results of all of them.
//
// Bound by the vector units' issue beside the matrix instructions in bf16 (0.69 and 0.45 of the time; of the issue for 32 x 32
// scores 256 of some 470 clocks are exponentials): 8192 tokens on 16384 states, 8 / 2 heads of 64 300 to 320 us, 0.9 PFLOP/s, on
// e4m3 states 343 to 363. In f32 by the six products' matrix instructions beside the split of P (0.52 and 0.51): 4 x 1344
// tokens on 2688 ragged states, 8 heads of 48, 91 to 97 us.
#include <algorithm>
#include <type_traits>

#include "attend.hpp"
#include "lds_dma.hpp"
#include "rows_attention.hpp"

namespace mnn {
namespace k {

using namespace dev;

namespace {

template <class T, class M, int KS, int NW>
struct MemoryCfg {
  using A = AttendMany<T, M, KS>;
  static constexpr int BKV = sizeof(M) == 4 ? 32 : 64, NT = BKV / 32;
  static constexpr int THREADS = 64 * NW, BQ = 32 * NW;
  static constexpr int PLANE = BKV * A::PITCH;
  static constexpr int CHUNKS = BKV * KS * 2;  // of 8 values, in a block of K or V
  static constexpr int PER = (CHUNKS + THREADS - 1) / THREADS;
  // K planes, V planes, scales; V's fragments of the last 32 dimensions may reach 32 bytes past its rows
  static constexpr int SLOT = 2 * A::PM * PLANE + 64 + (A::HELD ? 2 * BKV * 4 : 0);
  static constexpr int LDS = 2 * SLOT;
  // waves a SIMD, as the registers allow without spilling
  static constexpr int OCC = A::F32    ? (A::PM == 3 ? (KS > 6 ? 1 : 2) : (KS > 4 ? 1 : 2))
                             : A::HELD ? (KS > 4 ? 2 : KS > 2 ? 3 : 4)
                                       : (KS > 5 ? 2 : KS > 4 ? 3 : 4);
};

struct Unit {
  int b, kvh, tile, row0, rows, n, sp;  // rows: of the sequence's, n: its states
};
// The tiles of a head that share a range of keys are a set.
__device__ __forceinline__ bool unit_of(const MemoryArgs& a, const XcdGroups& sets, int nsplit, int bq, Unit& u) {
  const int set = sets.set_of((int)blockIdx.x, u.tile), head = set / nsplit;
  u.sp = set - head * nsplit;
  u.b = head / a.KV;
  u.kvh = head - u.b * a.KV;
  if (u.b >= a.B || u.tile < 0) return false;
  u.row0 = u.tile * bq;
  u.rows = (a.qlen ? min(max(a.qlen[u.b], 0), a.T) : a.T) * (a.H / a.KV);
  u.n = a.len ? min(max(a.len[u.b], 0), a.S) : a.S;
  return u.row0 < u.rows;
}
// Where row r of a sequence's head group lies in q and o.
__device__ __forceinline__ int64_t row_at(const MemoryArgs& a, const Unit& u, int r) {
  const int G = a.H / a.KV, t = r / G;
  return (((int64_t)u.b * a.T + t) * a.H + u.kvh * G + (r - t * G)) * a.hd;
}

// Row r once more, by one wave.
template <class T, class M>
__device__ __forceinline__ void memory_row_again(const MemoryArgs& a, const Unit& u, int r) {
  const int lane = threadIdx.x & 63;
  auto row = [&](int64_t i, const void* x, const float* scales) {
    const int64_t at = ((int64_t)u.b * a.S + i) * a.KV + u.kvh;
    if constexpr (sizeof(M) == 1)
      return HeldRow<T>{static_cast<const uint8_t*>(x) + at * a.hd, nullptr, scales[at], 0.f};
    else
      return static_cast<const M*>(x) + at * a.hd;
  };
  const int64_t at = row_at(a, u, r);
  float o0, o1;
  attend_row(static_cast<const T*>(a.q) + at, a.hd, a.scale, (int64_t)u.n, [&](int64_t i) { return row(i, a.k, a.ks); },
             [&](int64_t i) { return row(i, a.v, a.vs); }, o0, o1);
  T* o = static_cast<T*>(a.o) + at;
  if (lane < a.hd) o[lane] = from_f32<T>(o0);
  if (lane + 64 < a.hd) o[lane + 64] = from_f32<T>(o1);
}

template <class T, class M, int KS, int NW>
__global__ __launch_bounds__((MemoryCfg<T, M, KS, NW>::THREADS), (MemoryCfg<T, M, KS, NW>::OCC)) void memory_kernel(
    MemoryArgs a, XcdGroups sets, int nsplit, float* part, int* counts) {
  using Cfg = MemoryCfg<T, M, KS, NW>;
  using A = typename Cfg::A;
  constexpr int BKV = Cfg::BKV, NT = Cfg::NT, PM = A::PM, PLANE = Cfg::PLANE, SLOT = Cfg::SLOT, PER = Cfg::PER;
  constexpr int THREADS = Cfg::THREADS, PITCH = A::PITCH;
  constexpr bool HELD = A::HELD;
  __shared__ __attribute__((aligned(16))) char smem[Cfg::LDS];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Unit u;
  if (!unit_of(a, sets, nsplit, Cfg::BQ, u)) return;
  const int nb = (u.n + BKV - 1) / BKV;
  const int b0 = (int)((int64_t)nb * u.sp / nsplit), b1 = (int)((int64_t)nb * (u.sp + 1) / nsplit);
  const int hd = a.hd, kvw = a.KV * hd;
  const M* kb = static_cast<const M*>(a.k) + (int64_t)u.b * a.S * kvw + u.kvh * hd;
  const M* vb = static_cast<const M*>(a.v) + (int64_t)u.b * a.S * kvw + u.kvh * hd;

  // a block of K and V on its way, 8 values a chunk; rows behind the last key: that one again (their scores are masked;
  // a value of it that is not finite makes the results not finite, which computes them again)
  Eight<M> ck[PER], cv[PER];
  float sc = 0.f;
  auto each = [&](auto f) {  // f(i, row, chunk) for each chunk of the thread's
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = tid + THREADS * i, row = e / (2 * KS), c = e % (2 * KS);
      if (e < Cfg::CHUNKS && 8 * c < hd) f(i, row, c);
    }
  };
  const unsigned row_bytes = (unsigned)(kvw * sizeof(M));  // 64 of them: below 2^31
  auto fetch = [&](int blk) {
    const unsigned end = (unsigned)min(BKV - 1, u.n - 1 - blk * BKV) * row_bytes;  // where the last row begins
    const char* kt = reinterpret_cast<const char*>(kb + (int64_t)blk * BKV * kvw);
    const char* vt = reinterpret_cast<const char*>(vb + (int64_t)blk * BKV * kvw);
    each([&](int i, int row, int c) {
      const unsigned at = min((unsigned)row * row_bytes, end) + 8 * sizeof(M) * c;
      ck[i].load(reinterpret_cast<const M*>(kt + at));
      cv[i].load(reinterpret_cast<const M*>(vt + at));
    });
    if constexpr (HELD)
      if (tid < 2 * BKV)
        sc = (tid < BKV ? a.ks : a.vs)[((int64_t)u.b * a.S + min(blk * BKV + tid % BKV, u.n - 1)) * a.KV + u.kvh];
  };
  A at;
  auto store = [&](int slot) {
    char* s = smem + slot * SLOT;
    each([&](int i, int row, int c) {
      const Parts<M> k = parts_of(ck[i]), v = parts_of(cv[i]);
      char* to = s + row * PITCH + 16 * c;
#pragma unroll
      for (int p = 0; p < PM; ++p) {
        *reinterpret_cast<bf16x8*>(to + p * PLANE) = k.p[p];
        *reinterpret_cast<bf16x8*>(to + (PM + p) * PLANE) = v.p[p];
      }
    });
    if constexpr (HELD)
      if (tid < 2 * BKV)
        reinterpret_cast<float*>(s + 2 * PM * PLANE + 64)[tid] = tid < BKV ? sc * at.cs : sc;
  };
  if (hd < 16 * KS)  // columns behind the head's last stay zero
    for (int e = tid; e < 2 * 2 * PM * BKV; e += THREADS) {
      const int slot = e / (2 * PM * BKV), row = e % (2 * PM * BKV);
      for (int c = hd / 8; c < 2 * KS; ++c)
        *reinterpret_cast<float4*>(smem + slot * SLOT + row * PITCH + 16 * c) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  if (b0 < b1) fetch(b0);

  const int row = u.row0 + 32 * wave + l32;
  const bool mine = row < u.rows;
  at.begin();
  at.load_q(static_cast<const T*>(a.q) + row_at(a, u, min(row, u.rows - 1)), mine, hd, a.scale);
  const bool any = u.row0 + 32 * wave < u.rows;  // of the wave's rows

  if (b0 < b1) store(0);
  for (int blk = b0; blk < b1; ++blk) {
    const int slot = (blk - b0) & 1;
    lds_barrier();
    if (blk + 1 < b1) fetch(blk + 1);
    if (any) {
      const char* s = smem + slot * SLOT;
      const char* kf = s + l32 * PITCH + 16 * g;
      const float* scl = reinterpret_cast<const float*>(s + 2 * PM * PLANE + 64);
      floatx16 st[NT];
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        st[j] = at.scores([&](int c) {
          Parts<M> x;
#pragma unroll
          for (int p = 0; p < PM; ++p) x.p[p] = *reinterpret_cast<const bf16x8*>(kf + p * PLANE + 32 * j * PITCH + 32 * c);
          return x;
        });
        if constexpr (HELD) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 f = *reinterpret_cast<const float4*>(scl + 32 * j + 8 * i + 4 * g);
            st[j][4 * i] *= f.x;
            st[j][4 * i + 1] *= f.y;
            st[j][4 * i + 2] *= f.z;
            st[j][4 * i + 3] *= f.w;
          }
        }
      }
      const int left = u.n - blk * BKV;
      if (left < BKV) {
#pragma unroll
        for (int j = 0; j < NT; ++j) A::mask(st[j], (int)keys_below(left - 32 * j - 4 * g));
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) mx = A::largest(st[j], mx);
      at.refer(mx);
      // ahead of the waves that are at their scores: this part feeds both pipes
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const char* v0 = A::v_first(s + PM * PLANE + 32 * j * PITCH);
        float4 f[4];
        if constexpr (HELD) {
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] = *reinterpret_cast<const float4*>(scl + BKV + 32 * j + 8 * i + 4 * g);
        }
        at.add(st[j], [&](int p, int t, int ks) { return A::v_frag(v0, PLANE, p, t, ks); },
               [&](int v) { return v % 4 == 0 ? f[v / 4].x : v % 4 == 1 ? f[v / 4].y : v % 4 == 2 ? f[v / 4].z : f[v / 4].w; });
      }
      __builtin_amdgcn_s_setprio(0);
    }
    if (blk + 1 < b1) store(slot ^ 1);
  }

  float l = other_half(at.sum, Plus{});
  if (nsplit > 1) {
    // O^T, reference and sum to the workspace, a register of all lanes beside each other; the last of the unit's
    // workgroups joins them, in the keys' order
    constexpr int REGS = 16 * A::DT + 2;
    const int64_t step = (int64_t)NW * REGS * 64;  // from one range to the next
    const int unit = (u.b * a.KV + u.kvh) * sets.size + u.tile;
    float* first = part + ((int64_t)unit * nsplit * NW + wave) * REGS * 64 + lane;
    float* to = first + u.sp * step;
    if (any) {
#pragma unroll
      for (int i = 0; i < A::DT; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) put_shared(to + 64 * (16 * i + v), at.o[i][v]);
      // the reference in powers of two; NaN scores leave it at 0 and a sum of NaN
      put_shared(to + 64 * (REGS - 2), at.begun || !(l == 0.f) ? at.ref * (A::RAW ? at.cs : 1.f) : -INFINITY);
      put_shared(to + 64 * (REGS - 1), l);
    }
    if (!last_of(counts + unit, nsplit, reinterpret_cast<int*>(smem)) || !any) return;
    float top = -INFINITY;
    for (int s = 0; s < nsplit; ++s) top = max_nan(top, get_shared(first + s * step + 64 * (REGS - 2)));
    const float ref = top == -INFINITY ? 0.f : top;
    l = 0.f;
    at.begin();
    for (int s = 0; s < nsplit; ++s) {
      const float* p = first + s * step;
      const float by = __builtin_amdgcn_exp2f(get_shared(p + 64 * (REGS - 2)) - ref);
      l = fmaf(get_shared(p + 64 * (REGS - 1)), by, l);
#pragma unroll
      for (int i = 0; i < A::DT; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) at.o[i][v] = fmaf(get_shared(p + 64 * (16 * i + v)), by, at.o[i][v]);
    }
  }
  if (!any) return;
  const float inv = u.n ? 1.f / l : 0.f;
  bool bad = A::RAW && l < 0x1p-60f && u.n;
#pragma unroll
  for (int c = 0; c < 2 * KS; ++c)  // dimensions 8 c + 4 g .. + 3
    if (8 * c < hd) {
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= A::doubtful(at.o[c / 4][4 * (c % 4) + e] * inv);
    }
  unsigned long long again = __ballot(mine && bad);
  again = (again | (again >> 32)) & 0xffffffffull;
  if (mine && !((again >> l32) & 1)) {
    T* out = static_cast<T*>(a.o) + row_at(a, u, row) + 4 * g;
#pragma unroll
    for (int c = 0; c < 2 * KS; ++c)
      if (8 * c < hd) {
        const floatx16& ot = at.o[c / 4];
        const int v = 4 * (c % 4);
        if constexpr (A::F32)
          *reinterpret_cast<float4*>(out + 8 * c) =
              make_float4(ot[v] * inv, ot[v + 1] * inv, ot[v + 2] * inv, ot[v + 3] * inv);
        else
          *reinterpret_cast<uint2*>(out + 8 * c) =
              make_uint2(cvt_pk_bf16(ot[v] * inv, ot[v + 1] * inv), cvt_pk_bf16(ot[v + 2] * inv, ot[v + 3] * inv));
      }
  }
  while (again) {
    const int j = __builtin_ctzll(again);
    again &= again - 1;
    memory_row_again<T, M>(a, u, u.row0 + 32 * wave + j);
  }
}

constexpr int kMaxSplits = 16;
struct Plan {
  bool few;  // rows so few that the other kernel takes them
  int waves, tiles, nsplit;
  int64_t units;
};
Plan plan_of(const MemoryArgs& a, int cus) {
  Plan p;
  const int64_t rows = (int64_t)a.T * (a.H / a.KV), heads = (int64_t)a.B * a.KV;
  // Tiles of 16 rows (k_rows.hip) up to a workgroup for four compute units, or where one holds all rows of a head: their
  // workgroups share out the keys in finer ranges, but each reads all of them for its 16 rows. us there / here, 4 heads of
  // 64, bf16: one sequence of 128 rows on 16384 states 26 / 33, on 1344 13.4 / 15.2 (f32 15.5 / 25.9), of 512 rows on
  // 16384 39 / 35, on 4096 17 / 24; 16 sequences of 32 rows on 1344 17 / 15, of 16 rows 12 / 15.
  p.few = rows <= 16 || heads * cdiv(rows, 16) <= cus / 4;
  // bf16: 256 rows by 8 waves where that leaves a workgroup for each compute unit (blocks are staged for twice the rows):
  // us at 128 / 256 rows, 8 / 2 heads of 64: 8192 tokens on 16384 states 345 / 320, in 8 bits 571 / 369; 4 x 1344 on
  // 2688, 8 heads of 48 51 / 57. f32 there 150 / 170
  p.waves = a.type == MNN_BF16 && heads * cdiv(rows, 256) >= cus ? 8 : 4;
  p.tiles = (int)cdiv(rows, 32 * p.waves);
  p.units = heads * p.tiles;
  // ranges of 256 keys and more, while all workgroups run at once, 12 or 16 waves a compute unit
  p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({a.S / 256, (p.waves == 8 ? 2 : 3) * cus / p.units, kMaxSplits}));
  if (p.units > kJoinCounts) p.nsplit = 1;
  return p;
}

template <class T, class M, int KS, int NW>
void launch_nw(const LaunchCtx& c, const MemoryArgs& a, const Plan& p, const Join& join) {
  const int64_t n = (int64_t)a.B * a.KV * p.nsplit;
  const XcdGroups sets(n, p.tiles);
  MNN_REQUIRE(sets.grid(n) * 64 * NW < ((int64_t)1 << 32), MNN_ERR_INVALID_CONFIGURATION,
              "MemoryAttention: too many tokens in one call");
  launch(c, NW == 8 ? "memory_256" : "memory_128", memory_kernel<T, M, KS, NW>, dim3((unsigned)sets.grid(n)), dim3(64 * NW),
         0, a, sets, p.nsplit, join.part, join.counts);
}
template <class T, class M, int KS>
void launch_ks(const LaunchCtx& c, const MemoryArgs& a, const Plan& p, const Join& join) {
  if constexpr (sizeof(T) == 2)
    if (p.waves == 8) return launch_nw<T, M, KS, 8>(c, a, p, join);
  launch_nw<T, M, KS, 4>(c, a, p, join);
}
template <class T, class M>
void memory_tm(const LaunchCtx& c, const MemoryArgs& a, const Plan& p, const Join& join) {
  MNN_REQUIRE(p.units * p.nsplit < (1 << 23) && (int64_t)a.T * (a.H / a.KV) <= (1 << 30), MNN_ERR_INVALID_CONFIGURATION,
              "MemoryAttention: too many tokens in one call");
  MNN_REQUIRE(p.nsplit == 1 || (join.part && join.counts && p.units <= kJoinCounts), MNN_ERR_INVALID_ARGUMENT,
              "memory attention: split keys need a workspace");
  switch ((a.hd + 15) / 16) {
    case 1:
    case 2: launch_ks<T, M, 2>(c, a, p, join); break;
    case 3: launch_ks<T, M, 3>(c, a, p, join); break;
    case 4: launch_ks<T, M, 4>(c, a, p, join); break;
    case 5: launch_ks<T, M, 5>(c, a, p, join); break;
    case 6: launch_ks<T, M, 6>(c, a, p, join); break;
    default: launch_ks<T, M, 8>(c, a, p, join);
  }
}

}  // namespace

JoinSize memory_join(const LaunchCtx& c, const MemoryArgs& a) {
  const Plan p = plan_of(a, c.dev->props.multiProcessorCount);
  if (p.few) return memory_rows_join(c, a);
  if (p.nsplit == 1) return {};
  const int dt = a.hd > 96 ? 4 : (a.hd + 31) / 32;  // 32-row tiles of O^T, as AttendMany has them
  return {p.units * p.nsplit * p.waves * (16 * dt + 2) * 64, (int)p.units};
}
void memory_attention(const LaunchCtx& c, const MemoryArgs& a, const Join& join) {
  const Plan p = plan_of(a, c.dev->props.multiProcessorCount);
  if (p.few) return memory_rows(c, a, join);
  if (a.type == MNN_F32)
    a.ks ? memory_tm<float, E4m3>(c, a, p, join) : memory_tm<float, float>(c, a, p, join);
  else
    a.ks ? memory_tm<__bf16, E4m3>(c, a, p, join) : memory_tm<__bf16, __bf16>(c, a, p, join);
}

}  // namespace k
}  // namespace mnn
