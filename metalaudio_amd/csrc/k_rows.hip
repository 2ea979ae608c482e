// Attention of a few rows of each sequence to many keys (rows_attention.hpp), and the window attention's step on
// rolling caches in 8 bits.
//
// The rows that read one key/value head, tokens x heads of its group, are taken 16 at a time by a workgroup, or by
// several that share out the keys. Each wave computes its own blocks of 32 keys for all 16 rows on the matrix cores
// (attend.hpp): K goes from memory to registers as the A operand, V through a part of LDS that is the wave's, so that
// no wave waits for another one before the end, where their results are joined. The next block is on its way while
// one is computed. Of workgroups that share out the keys of the same rows the last one to finish joins the results of
// all of them, in the order of their keys.
//
// The matrix cores and the softmax run at 16 rows whatever there are (32 rows: twice the softmax, and registers for two
// waves a SIMD instead of four); rows on the vector units, eight lanes a key, cost as much for each.
//
// Bound by the loads where there are many streams, each lane group reading short rows: 64 streams on 4096 keys in 8 bits, 16 / 4 heads
// of 64, bf16 (142 MB) 28.8 us with the 256 MB cache warm, 4.9 TB/s, 35 us from memory; on 2688 ragged states (70 MB) 18 to 20 us.
// Lines touched a block or two ahead lose (36 and 41 us), as do loads around the caches. By the length of this form
// (V through LDS, two joins) and its code's first fetch where there are few: one stream on 516 keys in 8 bits, 8 heads of 48, f32 8.7 us, one token on 1344 states
// 11.7 (bf16 8.1), 8 streams' 16 tokens on 1043 keys 12 us; one stream on 516 f32 keys by k_window_step.hip, its row on the vector units, 7 to 8.
#include <algorithm>
#include <type_traits>

#include "attend.hpp"
#include "lds_dma.hpp"
#include "rows_attention.hpp"

namespace mnn {
namespace k {

using namespace dev;

namespace {

struct RowsArgs {
  const void* q;
  void* o;
  void *k, *v;          // [B][S][KV][hd], only written by a step
  float *ks, *vs;       // [B][S][KV] of e4m3
  const void *kn, *vn;  // a step's own rows [B][T][KV][hd]
  const int *c0, *c1;   // [B]: tokens and keys (or null) of each sequence; a step: positions and tokens (or null)
  int B, T, S, H, KV, hd;
  int left, sinks;      // of a step
  float scale;
};
// How the launch is cut.
struct RowsCut {
  XcdGroups sets;          // heads of a sequence's tile and key range
  int G, tiles, nsplit, slots;
  FastDiv by_G, by_tiles, by_split, by_hd;
  float* part;
  int* counts;
};

// What a workgroup answers: rows row0 .. row0 + 15 (row = token * G + head of the group) of sequence b, and the keys
// that any of them sees, numbered from 0. A step's: the sinks before the window's first token, then the window;
// so a key is a sink if its number is below `sinks`, whichever the window's first token is.
struct Rows {
  int b, kvh, row0, rows;      // rows: of the tile's 16
  int n;                       // keys
  int pos, nt, t0, t1, lo, ns, ring, wrapped;  // of a step; wrapped: place in the ring of token max(lo, sinks)
};
template <bool STEP>
__device__ __forceinline__ bool rows_of(const RowsArgs& a, const RowsCut& c, Rows& w) {
  if constexpr (STEP)
    w.nt = kv_rows(a.c0, a.c1, w.b, a.T, w.pos);
  else
    w.nt = a.c0 ? min(max(a.c0[w.b], 0), a.T) : a.T;
  w.rows = min(16, w.nt * c.G - w.row0);
  if (w.rows <= 0) return false;
  if constexpr (STEP) {
    w.t0 = c.by_G(w.row0);
    w.t1 = c.by_G(w.row0 + w.rows - 1);
    w.lo = max(0, w.pos + w.t0 - a.left);
    w.ns = min(a.sinks, w.lo);
    w.n = w.ns + (w.pos + w.t0 - w.lo) + (w.t1 - w.t0) + 1;
    w.ring = a.S - a.sinks;
    w.wrapped = (int)((unsigned)(max(w.lo, a.sinks) - a.sinks) % (unsigned)w.ring);
  } else {
    w.n = a.c1 ? min(max(a.c1[w.b], 0), a.S) : a.S;
  }
  return true;
}
// Token of key `idx` of a step, and its slot.
__device__ __forceinline__ int token_of(const Rows& w, int idx) { return idx < w.ns ? idx : w.lo + (idx - w.ns); }
__device__ __forceinline__ int slot_of(const RowsArgs& a, const Rows& w, int p) {
  if (p < a.sinks) return p;
  const int at = w.wrapped + (p - max(w.lo, a.sinks));  // below twice the ring: at most C - sinks tokens are seen
  return a.sinks + (at >= w.ring ? at - w.ring : at);
}

// Row r of the tile once more, by one wave, on the keys that it sees alone.
template <class T, class M, bool STEP>
__device__ void row_again(const RowsArgs& a, const Rows& w, int r) {
  const int lane = threadIdx.x & 63, G = a.H / a.KV, t = (w.row0 + r) / G, h = w.kvh * G + (w.row0 + r) % G;
  const int64_t at = (((int64_t)w.b * a.T + t) * a.H + h) * a.hd;
  const T* q = static_cast<const T*>(a.q) + at;
  auto held = [&](const void* x, const float* scales, int64_t slot) {
    const int64_t i = ((int64_t)w.b * a.S + slot) * a.KV + w.kvh;
    if constexpr (sizeof(M) == 1)
      return HeldRow<T>{static_cast<const uint8_t*>(x) + i * a.hd, nullptr, scales[i], 0.f};
    else
      return static_cast<const M*>(x) + i * a.hd;
  };
  float o0, o1;
  if constexpr (STEP) {
    const int i = w.pos + t, lo = max(0, i - a.left), ns = min(a.sinks, lo);
    auto row = [&](int64_t n, const void* x, const float* scales, const void* fresh) {
      const int p = (int)(n < ns ? n : lo + (n - ns));
      if (p >= w.pos)
        return HeldRow<T>::rounding(static_cast<const T*>(fresh) + (((int64_t)w.b * a.T + p - w.pos) * a.KV + w.kvh) * a.hd,
                                    a.hd);
      return held(x, scales, kv_slot(p, a.sinks, a.S));
    };
    attend_row(q, a.hd, a.scale, (int64_t)ns + (i - lo + 1), [&](int64_t n) { return row(n, a.k, a.ks, a.kn); },
               [&](int64_t n) { return row(n, a.v, a.vs, a.vn); }, o0, o1);
  } else {
    attend_row(q, a.hd, a.scale, (int64_t)w.n, [&](int64_t n) { return held(a.k, a.ks, n); },
               [&](int64_t n) { return held(a.v, a.vs, n); }, o0, o1);
  }
  T* o = static_cast<T*>(a.o) + at;
  if (lane < a.hd) o[lane] = from_f32<T>(o0);
  if (lane + 64 < a.hd) o[lane + 64] = from_f32<T>(o1);
}

// W: waves of a workgroup.
template <class T, class M, int KS, int W>
struct RowsCfg {
  using A = AttendFew<T, M, KS>;
  static constexpr int WAVE = A::PM * A::PLANE + (A::HELD ? 256 : 0);  // V's block, and the scales
  // waves a SIMD, as the registers allow
  static constexpr int OCC = W == 16 || KS == 1 ? 4
                             : A::PM == 3       ? (KS == 2 ? 2 : 1)
                             : A::F32           ? (KS == 2 ? 3 : 2)
                             : KS == 4          ? 2
                             : KS == 3          ? 3
                                                : 4;
  // bytes: the waves' blocks, or at the end their references and sums and results (lanes of rows that there are)
  static int lds(int slots) { return std::max(W * WAVE, 4 * (W * 32 + 16 + 64 + W * 4 * A::OT * 4 * slots)); }
};

template <class T, class M, int KS, int W, bool STEP>
__global__ __launch_bounds__((W * 64), (RowsCfg<T, M, KS, W>::OCC)) void rows_kernel(
    RowsArgs a, RowsCut c) {
  using Cfg = RowsCfg<T, M, KS, W>;
  using A = typename Cfg::A;
  constexpr int PM = A::PM, PLANE = A::PLANE;
  constexpr bool HELD = A::HELD;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // the heads of a sequence, whose rows share cache lines, are a set; sets: key ranges, tiles, sequences
  const int hd = a.hd;
  Rows w;
  int set = c.sets.set_of((int)blockIdx.x, w.kvh), rest = c.by_split(set);
  const int sp = set - rest * c.nsplit, G = c.G, slots = c.slots;
  w.b = c.by_tiles(rest);
  if (w.b >= a.B || w.kvh < 0) return;
  const int tile = rest - w.b * c.tiles;
  w.row0 = 16 * tile;
  // the queries' loads go out before the sequence's lengths have come; rows that are no tokens are not used
  const int row = w.row0 + l16, t = c.by_G(row);
  Eight<T> q[KS];
  A::fetch_q(static_cast<const T*>(a.q) + (((int64_t)w.b * a.T + t) * a.H + w.kvh * G + (row - t * G)) * hd, t < a.T, hd, q);
  if (!rows_of<STEP>(a, c, w)) return;

  A at;
  at.begin();
  // the query's keys by number: below hi, and not below first or below the sinks' end
  int hi = w.n, first = 0, first_last = 0, hi_least = w.n;
  if constexpr (STEP) {
    const int i = w.pos + min(t, w.t1);
    hi = w.ns + (i - w.lo) + 1;
    first = w.ns + (max(0, i - a.left) - w.lo);
    hi_least = w.ns + (w.pos + w.t0 - w.lo) + 1;
    first_last = w.ns + (max(0, w.pos + w.t1 - a.left) - w.lo);
  }

  const int nb = (w.n + 31) / 32, each = c.by_split(nb + c.nsplit - 1), b0 = sp * each, b1 = min(nb, b0 + each);
  struct Block {
    Eight<M> k[2][KS], v[2][KS];  // of keys l16 and 16 + l16
    float scale;                  // of lanes below 32: the scale of key lane, of the others: of value lane - 32
  };
  const int64_t seq = (int64_t)w.b * a.S * a.KV + w.kvh;
  const M* kb = static_cast<const M*>(a.k) + seq * hd;
  const M* vb = static_cast<const M*>(a.v) + seq * hd;
  const float* sb = HELD ? (lane < 32 ? a.ks : a.vs) + seq : nullptr;
  const bool wide = hd % 16 == 0;
  auto load = [&](const M* row, Eight<M>(&x)[KS]) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = A::dim_of(s, g);
      if constexpr (HELD) {
        if (s % 2 == 0 && s + 1 < KS && wide) {  // two chunks at once
          const uint4 two = *reinterpret_cast<const uint4*>(row + (A::may_end(s) ? min(d, hd - 16) : d));
          x[s].x = make_uint2(two.x, two.y);
          x[s + 1].x = make_uint2(two.z, two.w);
          continue;
        }
        if (s % 2 == 1 && wide) continue;
      }
      x[s].load(row + (A::may_end(s) ? min(d, hd - 8) : d));
    }
  };
  // a step's own keys and values, rounded as the cache will hold them: lanes of other keys read the call's first row
  // and leave it
  auto own_rows = [&](const int (&idx)[2], Block& x) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int p = token_of(w, idx[j]) - w.pos;
      const bool mine = p >= 0;
      if (!__any(mine)) continue;
      const int64_t from = (((int64_t)w.b * a.T + max(p, 0)) * a.KV + w.kvh) * hd;
      Eight<T> e[2][KS];
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const int d = A::dim_of(s, g);
          e[kv][s].load(static_cast<const T*>(kv ? a.vn : a.kn) + from + (A::may_end(s) ? min(d, hd - 8) : d));
        }
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        float top = 0.f;  // of the row; a chunk behind its end is one of it again
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(e[kv][s][i]));
        const RowScale rs = row_scale(other_half(other_row(top, max_nan), max_nan));
        if constexpr (HELD) {
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const Eight<T>& t = e[kv][s];
            const uint2 r = make_uint2(pack_e4m3(t[0] * rs.inv, t[1] * rs.inv, t[2] * rs.inv, t[3] * rs.inv),
                                       pack_e4m3(t[4] * rs.inv, t[5] * rs.inv, t[6] * rs.inv, t[7] * rs.inv));
            uint2& to = (kv ? x.v[j][s] : x.k[j][s]).x;
            to.x = mine ? r.x : to.x;
            to.y = mine ? r.y : to.y;
          }
          x.scale = mine && g == 2 * kv + j ? rs.scale : x.scale;
        }
      }
    }
  };
  // keys behind the last: the last one again (their scores are masked, their values cleared); a step's own keys,
  // which the cache does not hold yet: the slot that they will have first, then the rows themselves
  const int kvw = a.KV * hd;
  auto fetch = [&](int blk, Block& x) {
    int idx[2], slot[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      idx[j] = min(blk * 32 + 16 * j + l16, w.n - 1);
      slot[j] = STEP ? slot_of(a, w, token_of(w, idx[j])) : idx[j];
      const int64_t at = (int64_t)slot[j] * kvw;
      load(kb + at, x.k[j]);
      load(vb + at, x.v[j]);
    }
    if constexpr (HELD) x.scale = sb[(int64_t)(g & 1 ? slot[1] : slot[0]) * a.KV];
    if constexpr (STEP)
      if (token_of(w, min(blk * 32 + 31, w.n - 1)) >= w.pos) own_rows(idx, x);
  };

  char* mem = smem + wave * Cfg::WAVE;
  float* scl = reinterpret_cast<float*>(mem + PM * PLANE);
  const char* v0 = A::v_first(mem);
  auto compute = [&](int blk, Block& x) {
    const int k0 = blk * 32;
    if (k0 + 32 > w.n) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (k0 + 16 * j + l16 >= w.n) {
#pragma unroll
          for (int s = 0; s < KS; ++s) x.v[j][s].clear();
          if ((g & 1) == j) x.scale = 0.f;
        }
    }
    if constexpr (HELD) scl[lane] = lane < 32 ? x.scale * at.cs : x.scale;
    floatx4 st[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      st[j] = at.scores([&](int s) {
        if (A::may_end(s) && A::dim_of(s, g) >= hd) x.k[j][s].clear();
        return parts_of(x.k[j][s]);
      });
    // V to the wave's LDS: its reads below wait for these writes, and the next block's writes come behind them
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const Parts<M> p = parts_of(x.v[j][s]);
#pragma unroll
        for (int i = 0; i < PM; ++i)
          *reinterpret_cast<bf16x8*>(mem + i * PLANE + (16 * j + l16) * A::PITCH + 2 * A::dim_of(s, g)) = p.p[i];
      }
    __builtin_amdgcn_wave_barrier();
    float vs[8];
    if constexpr (HELD) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 f = *reinterpret_cast<const float4*>(scl + 16 * j + 4 * g);
        const float4 h = *reinterpret_cast<const float4*>(scl + 32 + 16 * j + 4 * g);
        st[j] *= floatx4{f.x, f.y, f.z, f.w};
        vs[4 * j] = h.x;
        vs[4 * j + 1] = h.y;
        vs[4 * j + 2] = h.z;
        vs[4 * j + 3] = h.w;
      }
    } else if constexpr (!A::F32) {
#pragma unroll
      for (int j = 0; j < 2; ++j) st[j] *= at.cs;
    }
    const bool whole = k0 + 32 <= hi_least && (k0 >= first_last || k0 + 32 <= a.sinks);
    if (!whole) {
      const int c = k0 + 4 * g;  // the lane's: key i below is c + i
      const int seen = (int)(keys_below(hi - c) & (STEP ? ~keys_below(first - c) | keys_below(a.sinks - c) : ~0u));
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) st[j][v] = masked_score(st[j][v], seen, 16 * j + v);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j) mx = max_nan(max_nan(max_nan(mx, st[j][0]), st[j][1]), max_nan(st[j][2], st[j][3]));
    at.refer(mx);
    at.add(st, [&](int part, int t) { return A::v_frag(v0, part, t); }, vs);
    __builtin_amdgcn_wave_barrier();
  };

  // one copy of the code: a launch fetches all that it executes once, some 100 ns for 64 bytes, which is most of a short
  // call's time (two copies, for blocks that alternate: 17 keys a wave more 1.9 us more)
  at.take_q(q, a.scale);
  Block x, next;
  const int mine0 = b0 + wave;
#pragma unroll 1
  for (int blk = mine0;; blk += W) {
    if (blk < b1) fetch(blk, next);
    if (blk != mine0) compute(blk - W, x);
    if (blk >= b1) break;
    x = next;
  }

  // the step's own rows to their slots: no key that is still seen lies there
  if constexpr (STEP && HELD) {
    if (w.row0 == 0 && sp == 0) {
      const int j = tid % 16;
      for (int i = tid / 16; i < w.nt; i += W * 4) {
        const int64_t slot = seq + (int64_t)kv_slot(w.pos + i, a.sinks, a.S) * a.KV;
        const int64_t from = (((int64_t)w.b * a.T + i) * a.KV + w.kvh) * hd + 8 * j;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          Eight<T> e;
          e.clear();
          if (8 * j < hd) e.load(static_cast<const T*>(kv ? a.vn : a.kn) + from);
          float v[8], scale;
#pragma unroll
          for (int d = 0; d < 8; ++d) v[d] = e[d];
          const uint2 q = round_row<16>(v, scale);
          if (8 * j < hd) *reinterpret_cast<uint2*>(static_cast<uint8_t*>(kv ? a.v : a.k) + slot * hd + 8 * j) = q;
          if (j == 0) (kv ? a.vs : a.ks)[slot] = scale;
        }
      }
    }
  }

  // the waves' references, then their results times what these make of them, through LDS, only the rows' lanes
  const int nr = w.rows;
  constexpr int N = 4 * A::OT;
  float* refs = reinterpret_cast<float*>(smem);  // [W][16]
  float* sums = refs + W * 16;                   // [W][16]
  float* tops = sums + W * 16;                   // [16]
  int* again = reinterpret_cast<int*>(tops + 16);  // [16], and one for last_of
  float* res = tops + 64;                        // [W][N][4][slots]
  // NaN scores leave no reference and a sum of NaN, which stays one times 0
  const float ref = at.begun ? at.ref : -INFINITY, l = other_half(other_row(at.sum, Plus{}), Plus{});
  __syncthreads();
  if (lane < 16) refs[wave * 16 + lane] = ref;
  if (tid < 16) again[tid] = 0;
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < W; ++i) top = max_nan(top, refs[i * 16 + l16]);
  const float by = __builtin_amdgcn_exp2f(ref - (top == -INFINITY ? 0.f : top));
  if (lane < 16) {
    sums[wave * 16 + lane] = l * by;
    tops[lane] = top;  // the same from every wave
  }
  if (l16 < nr) {
    float* to = res + (wave * N * 4 + g) * slots + l16;
#pragma unroll
    for (int i = 0; i < A::OT; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) to[(4 * i + v) * 4 * slots] = at.o[i][v] * by;
  }
  __syncthreads();
  auto finish = [&](int r, int d, float y, float l) {
    y = w.n ? y / l : 0.f;
    const int rr = w.row0 + r, t = c.by_G(rr);
    static_cast<T*>(a.o)[(((int64_t)w.b * a.T + t) * a.H + w.kvh * G + (rr - t * G)) * hd + d] = from_f32<T>(y);
    if (A::doubtful(y)) again[r] = 1;
  };
  const int ld = hd + 2, unit = (w.b * a.KV + w.kvh) * c.tiles + tile;
  float* mine = c.part + ((int64_t)unit * c.nsplit + sp) * slots * ld;
  for (int e = tid; e < nr * hd; e += W * 64) {
    const int r = c.by_hd(e), d = e - r * hd;
    const float* f = res + ((4 * (d / 16) + d % 4) * 4 + d % 16 / 4) * slots + r;  // register, lane group
    float l = 0.f, y = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      l += sums[i * 16 + r];
      y += f[i * N * 4 * slots];
    }
    if (c.nsplit > 1) {
      put_shared(mine + r * ld + d, y);
      if (d == 0) {
        put_shared(mine + r * ld + hd, tops[r]);
        put_shared(mine + r * ld + hd + 1, l);
      }
    } else {
      finish(r, d, y, l);
    }
  }
  if (c.nsplit > 1) {
    if (!last_of(c.counts + unit, c.nsplit, again + 16)) return;
    const float* all = c.part + (int64_t)unit * c.nsplit * slots * ld;
    for (int e = tid; e < nr * hd; e += W * 64) {
      const int r = c.by_hd(e), d = e - r * hd;
      const float* f = all + r * ld;
      float top = -INFINITY, l = 0.f, y = 0.f;
      // four ranges at a time, their loads at once; a later, larger reference takes the sums so far down
      for (int s0 = 0; s0 < c.nsplit; s0 += 4) {
        float ref[4], sum[4], val[4], m = top;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float* p = f + (int64_t)min(s0 + i, c.nsplit - 1) * slots * ld;
          ref[i] = get_shared(p + hd);
          sum[i] = get_shared(p + hd + 1);
          val[i] = get_shared(p + d);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max_nan(m, ref[i]);
        const float from = m == -INFINITY ? 0.f : m, down = __builtin_amdgcn_exp2f(top - from);
        l *= down;
        y *= down;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float by = s0 + i < c.nsplit ? __builtin_amdgcn_exp2f(ref[i] - from) : 0.f;
          l = fmaf(sum[i], by, l);
          y = fmaf(val[i], by, y);
        }
        top = m;
      }
      finish(r, d, y, l);
    }
  }
  __syncthreads();
  for (int r = wave; r < nr; r += W)
    if (again[r]) row_again<T, M, STEP>(a, w, r);
}

// How a call is cut: tiles of 16 rows, the waves of a workgroup, and how many workgroups share a tile's keys.
constexpr int kMaxSplits = 64;
struct Plan {
  int tiles, waves, nsplit;
  int64_t units;
};
Plan plan_of(const RowsArgs& a, mnn_dtype type, int64_t keys, int cus) {
  Plan p;
  p.tiles = (int)cdiv((int64_t)a.T * (a.H / a.KV), 16);
  p.units = (int64_t)a.B * a.KV * p.tiles;
  // 16 waves where 8-bit keys come to that many blocks a compute unit (and the registers allow four waves a SIMD): us with 8 /
  // 16, 16 / 4 heads of 64: 64 streams on 4096 keys 37 / 28, on 2688 states 24 / 19; 8 heads, 16 streams on 2048 17 / 15; 8 / 2
  // heads, 8 streams' 16 tokens on 1024 13.5 / 15.2. Keys of 16 bits are bound by memory (33 / 33). 4 where f32 keys of
  // more than 64 dimensions take a SIMD's registers for one wave
  const bool held = a.ks != nullptr, fits = a.hd <= (type == MNN_BF16 ? 64 : 32);
  p.waves = held && fits && p.units * keys >= (int64_t)16 * 32 * cus ? 16 : !held && type == MNN_F32 && a.hd > 64 ? 4 : 8;
  // a block for each wave, while that leaves no more workgroups than compute units: one that waits for others costs 2 us
  p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({cdiv(keys, 32 * p.waves), cus / p.units, kMaxSplits}));
  return p;
}
int slots_of(const RowsArgs& a) { return (int)std::min<int64_t>(16, (int64_t)a.T * (a.H / a.KV)); }
JoinSize join_of(const RowsArgs& a, const Plan& p) {
  if (p.nsplit == 1) return {};
  return {p.units * p.nsplit * slots_of(a) * (a.hd + 2), (int)p.units};
}

template <class T, class M, int KS, int W, bool STEP>
void launch_w(const LaunchCtx& c, const RowsArgs& a, const Plan& p, const Join& join) {
  const int64_t n = (int64_t)a.B * p.tiles * p.nsplit;
  const XcdGroups sets(n, a.KV);
  const int G = a.H / a.KV;
  const RowsCut cut{sets,          G,          p.tiles, p.nsplit, slots_of(a), FastDiv(G), FastDiv(p.tiles), FastDiv(p.nsplit),
                    FastDiv(a.hd), join.part, join.counts};
  launch(c, STEP ? "rows_step" : "rows_memory", rows_kernel<T, M, KS, W, STEP>, dim3((unsigned)sets.grid(n)), dim3(64 * W),
         (size_t)RowsCfg<T, M, KS, W>::lds(slots_of(a)), a, cut);
}
template <class T, class M, int KS, bool STEP>
void launch_ks(const LaunchCtx& c, const RowsArgs& a, const Plan& p, const Join& join) {
  if constexpr (sizeof(M) == 1 && KS <= (sizeof(T) == 2 ? 2 : 1))
    if (p.waves == 16) return launch_w<T, M, KS, 16, STEP>(c, a, p, join);
  launch_w<T, M, KS, (sizeof(M) == 4 && KS > 2 ? 4 : 8), STEP>(c, a, p, join);
}
template <class T, class M, bool STEP>
void launch_rows(const LaunchCtx& c, const RowsArgs& a, const Plan& p, const Join& join) {
  // rows are numbered by ints, up to the last tile's end; a grid of 2^32 lanes
  MNN_REQUIRE((int64_t)a.T * (a.H / a.KV) < (1 << 24) && p.units * p.nsplit < (1 << 20), MNN_ERR_INVALID_CONFIGURATION,
              (STEP ? "WindowAttention" : "MemoryAttention") << ": too many sequences and tokens in one call");
  MNN_REQUIRE(p.nsplit == 1 || (join.part && join.counts && p.units <= kJoinCounts), MNN_ERR_INVALID_ARGUMENT,
              "rows of attention: split keys need a workspace");
  switch ((a.hd + 31) / 32) {
    case 1: return launch_ks<T, M, 1, STEP>(c, a, p, join);
    case 2: return launch_ks<T, M, 2, STEP>(c, a, p, join);
    case 3: return launch_ks<T, M, 3, STEP>(c, a, p, join);
    default: return launch_ks<T, M, 4, STEP>(c, a, p, join);
  }
}

RowsArgs step_args(const WindowStepHeldArgs& s) {
  RowsArgs a{};
  a.q = s.q;
  a.o = s.o;
  a.k = s.kc;
  a.v = s.vc;
  a.ks = s.ks;
  a.vs = s.vs;
  a.kn = s.k;
  a.vn = s.v;
  a.c0 = s.pos;
  a.c1 = s.steps;
  a.B = s.B;
  a.T = s.T;
  a.S = s.C;
  a.H = s.H;
  a.KV = s.KV;
  a.hd = s.hd;
  a.left = s.left;
  a.sinks = s.sinks;
  a.scale = s.scale;
  return a;
}
int64_t step_keys(const WindowStepHeldArgs& a) {
  return std::min<int64_t>((int64_t)a.left + a.sinks + std::min(a.T, 16), a.C);
}
RowsArgs memory_args(const MemoryArgs& m) {
  RowsArgs a{};
  a.q = m.q;
  a.o = m.o;
  a.k = const_cast<void*>(m.k);
  a.v = const_cast<void*>(m.v);
  a.ks = const_cast<float*>(m.ks);
  a.vs = const_cast<float*>(m.vs);
  a.c0 = m.qlen;
  a.c1 = m.len;
  a.B = m.B;
  a.T = m.T;
  a.S = m.S;
  a.H = m.H;
  a.KV = m.KV;
  a.hd = m.hd;
  a.scale = m.scale;
  return a;
}

}  // namespace

JoinSize window_step_e4m3_join(const LaunchCtx& c, const WindowStepHeldArgs& s) {
  const RowsArgs a = step_args(s);
  return join_of(a, plan_of(a, s.type, step_keys(s), c.dev->props.multiProcessorCount));
}
void window_step_e4m3(const LaunchCtx& c, const WindowStepHeldArgs& s, const Join& part) {
  const RowsArgs a = step_args(s);
  const Plan p = plan_of(a, s.type, step_keys(s), c.dev->props.multiProcessorCount);
  if (s.type == MNN_F32)
    launch_rows<float, E4m3, true>(c, a, p, part);
  else
    launch_rows<__bf16, E4m3, true>(c, a, p, part);
}

JoinSize memory_rows_join(const LaunchCtx& c, const MemoryArgs& m) {
  const RowsArgs a = memory_args(m);
  return join_of(a, plan_of(a, m.type, m.S, c.dev->props.multiProcessorCount));
}
void memory_rows(const LaunchCtx& c, const MemoryArgs& m, const Join& part) {
  const RowsArgs a = memory_args(m);
  const Plan p = plan_of(a, m.type, m.S, c.dev->props.multiProcessorCount);
  if (m.type == MNN_F32)
    m.ks ? launch_rows<float, E4m3, false>(c, a, p, part) : launch_rows<float, float, false>(c, a, p, part);
  else
    m.ks ? launch_rows<__bf16, E4m3, false>(c, a, p, part) : launch_rows<__bf16, __bf16, false>(c, a, p, part);
}

}  // namespace k
}  // namespace mnn
