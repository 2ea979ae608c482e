// Attention of a few rows of each sequence to many keys (rows_attention.hpp), and the window attention's step on
// rolling caches in 8 bits.
//
// The rows that read one key/value head, tokens x heads of its group, are taken 32 at a time by a workgroup, or by
// several that share out the keys. Each wave computes its own blocks of 32 keys for all 32 rows on the matrix cores
// (attend.hpp): K goes from memory to registers as the A operand, V through a part of LDS that is the wave's, so that
// no wave waits for another one before the end, where their results are joined. The next block is on its way while
// one is computed.
//
// The matrix cores and the softmax run at 32 rows whatever there are: a block of 32 keys, 4 KB of e4m3 at heads of 64,
// takes a SIMD some 700 cycles, 14 TB/s over the GPU; rows on the vector units, eight lanes a key, cost those as much
// for each row.
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

// What a workgroup answers: rows row0 .. row0 + 31 (row = token * G + head of the group) of sequence b, and the keys
// that any of them sees, numbered from 0. A step's: the sinks before the window's first token, then the window;
// so a key is a sink if its number is below `sinks`, whichever the window's first token is.
struct Rows {
  int b, kvh, row0, rows;      // rows: of the tile's 32
  int n;                       // keys
  int pos, nt, t0, lo, ns, ring, wrapped;  // of a step; wrapped: place in the ring of token max(lo, sinks)
};
template <bool STEP>
__device__ __forceinline__ bool rows_of(const RowsArgs& a, int unit, int tiles, Rows& w) {
  const int G = a.H / a.KV;
  w.row0 = unit % tiles * 32;
  w.kvh = unit / tiles % a.KV;
  w.b = unit / tiles / a.KV;
  if constexpr (STEP)
    w.nt = kv_rows(a.c0, a.c1, w.b, a.T, w.pos);
  else
    w.nt = a.c0 ? min(max(a.c0[w.b], 0), a.T) : a.T;
  w.rows = min(32, w.nt * G - w.row0);
  if (w.rows <= 0) return false;
  if constexpr (STEP) {
    w.t0 = w.row0 / G;
    const int t1 = (w.row0 + w.rows - 1) / G;
    w.lo = max(0, w.pos + w.t0 - a.left);
    w.ns = min(a.sinks, w.lo);
    w.n = w.ns + (w.pos + w.t0 - w.lo) + (t1 - w.t0) + 1;
    w.ring = a.S - a.sinks;
    w.wrapped = (max(w.lo, a.sinks) - a.sinks) % w.ring;
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

template <class T, class M, int KS>
struct RowsCfg {
  using A = Attend<T, M, KS, false>;
  // waves: 4 where their registers do not fit in two waves a SIMD
  static constexpr int W = KS > (sizeof(M) == 4 ? 3 : A::F32 ? 4 : 6) ? 4 : 8;
  static constexpr int WAVE = A::PM * A::PLANE + 64 + (A::HELD ? 256 : 0);  // V's block, and the scales
  static constexpr int REGS = 16 * A::DT + 1;
  // bytes: the waves' blocks, or at the end their results (lanes of rows that there are), references and sums
  static int lds(int rows) { return std::max(W * WAVE, W * 4 * (REGS * 2 * rows + rows)) + 4 * 32; }
};

template <class T, class M, int KS, bool STEP>
__global__ __launch_bounds__((RowsCfg<T, M, KS>::W * 64)) void rows_kernel(RowsArgs a, int tiles, int nsplit,
                                                                           int slots, float* part) {
  using Cfg = RowsCfg<T, M, KS>;
  using A = Attend<T, M, KS, false>;
  constexpr int W = Cfg::W, PM = A::PM, PLANE = A::PLANE;
  constexpr bool HELD = A::HELD;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // consecutive units, the tiles and key ranges of one head first, run on one XCD and share its L2
  const int id = xcd_logical_tile((int)blockIdx.x, (int)gridDim.x);
  const int unit = id / nsplit, sp = id % nsplit, G = a.H / a.KV, hd = a.hd;
  Rows w;
  if (!rows_of<STEP>(a, unit, tiles, w)) return;

  A at;
  at.begin();
  const int row = w.row0 + l32, t = row / G;
  at.load_q(static_cast<const T*>(a.q) + (((int64_t)w.b * a.T + t) * a.H + w.kvh * G + row % G) * hd, l32 < w.rows, hd,
            a.scale);
  // the query's keys by number: below hi, and not below first or below the sinks' end
  int hi = w.n, first = 0, first_last = 0, hi_least = w.n;
  if constexpr (STEP) {
    const int i = w.pos + min(t, (w.row0 + w.rows - 1) / G);
    hi = w.ns + (i - w.lo) + 1;
    first = w.ns + (max(0, i - a.left) - w.lo);
    hi_least = w.ns + (w.pos + w.t0 - w.lo) + 1;
    first_last = w.ns + (max(0, w.pos + (w.row0 + w.rows - 1) / G - a.left) - w.lo);
  }

  const int nb = (w.n + 31) / 32, b0 = (int)((int64_t)nb * sp / nsplit), b1 = (int)((int64_t)nb * (sp + 1) / nsplit);
  struct Block {
    Eight<M> k[KS], v[KS];
    float scale;  // of lane half 0: the key's, of half 1: the value's
  };
  const int64_t seq = (int64_t)w.b * a.S * a.KV + w.kvh;
  const M* kb = static_cast<const M*>(a.k) + seq * hd;
  const M* vb = static_cast<const M*>(a.v) + seq * hd;
  const float* sb = HELD ? (g ? a.vs : a.ks) + seq : nullptr;
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
        if (s % 2 == 1 && wide && s < KS) continue;
      }
      x[s].load(row + (A::may_end(s) ? min(d, hd - 8) : d));
    }
  };
  // keys behind the last: the last one again (their scores are masked, their values cleared); a step's own keys,
  // which the cache does not hold yet: the slot that they will have
  auto fetch = [&](int blk, Block& x) {
    const int idx = min(blk * 32 + l32, w.n - 1);
    const int64_t slot = STEP ? slot_of(a, w, token_of(w, idx)) : idx;
    load(kb + slot * a.KV * hd, x.k);
    load(vb + slot * a.KV * hd, x.v);
    if constexpr (HELD) x.scale = sb[slot * a.KV];
  };
  // a step's own keys and values, rounded as the cache will hold them
  auto own_rows = [&](int idx, Block& x) {
    const int p = token_of(w, min(idx, w.n - 1));
    const bool mine = p >= w.pos;
    const int64_t from = (((int64_t)w.b * a.T + (mine ? p - w.pos : 0)) * a.KV + w.kvh) * hd;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const T* src = static_cast<const T*>(kv ? a.vn : a.kn) + from;
      Eight<T> e[KS];
      float top = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = A::dim_of(s, g);
        e[s].clear();
        if (mine && d < hd) e[s].load(src + d);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(e[s][i]));
      }
      const RowScale rs = row_scale(other_half(top, max_nan));
      if constexpr (HELD) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const uint2 q = make_uint2(
              pack_e4m3(e[s][0] * rs.inv, e[s][1] * rs.inv, e[s][2] * rs.inv, e[s][3] * rs.inv),
              pack_e4m3(e[s][4] * rs.inv, e[s][5] * rs.inv, e[s][6] * rs.inv, e[s][7] * rs.inv));
          if (mine) (kv ? x.v[s] : x.k[s]).x = q;
        }
        if (mine && g == kv) x.scale = rs.scale;
      }
    }
  };

  char* mem = smem + wave * Cfg::WAVE;
  float* scl = reinterpret_cast<float*>(mem + PM * PLANE + 64);
  const char* v0 = A::v_first(mem);
  auto compute = [&](int blk, Block& x) {
    const int k0 = blk * 32;
    if constexpr (STEP)
      if (token_of(w, min(k0 + 31, w.n - 1)) >= w.pos) own_rows(k0 + l32, x);
    if (k0 + 32 > w.n) {
      const bool there = k0 + l32 < w.n;
#pragma unroll
      for (int s = 0; s < KS; ++s)
        if (!there) x.v[s].clear();
      if (!there) x.scale = 0.f;
    }
    // V to the wave's LDS: its reads below wait for these writes, and the next block's writes come behind them
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const Parts<M> p = parts_of(x.v[s]);
#pragma unroll
      for (int i = 0; i < PM; ++i)
        *reinterpret_cast<bf16x8*>(mem + i * PLANE + l32 * A::PITCH + 2 * A::dim_of(s, g)) = p.p[i];
    }
    if constexpr (HELD) scl[lane] = g ? x.scale : x.scale * at.cs;
    __builtin_amdgcn_wave_barrier();
    floatx16 st = at.scores([&](int s) {
      if (A::may_end(s) && A::dim_of(s, g) >= hd) x.k[s].clear();
      return parts_of(x.k[s]);
    });
    if constexpr (HELD) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 f = *reinterpret_cast<const float4*>(scl + 8 * j + 4 * g);
        st[4 * j] *= f.x;
        st[4 * j + 1] *= f.y;
        st[4 * j + 2] *= f.z;
        st[4 * j + 3] *= f.w;
      }
    } else if constexpr (!A::F32) {
#pragma unroll
      for (int v = 0; v < 16; ++v) st[v] *= at.cs;
    }
    const bool whole = k0 + 32 <= hi_least && (k0 >= first_last || k0 + 32 <= a.sinks);
    if (!whole) {
      const int c = k0 + 4 * g;  // the lane's: key i below is c + i
      A::mask(st, (int)(A::below(hi - c) & (STEP ? ~A::below(first - c) | A::below(a.sinks - c) : ~0u)));
    }
    at.refer(A::largest(st, -INFINITY));
    float4 f[4];
    if constexpr (HELD) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = *reinterpret_cast<const float4*>(scl + 32 + 8 * j + 4 * g);
    }
    at.add(st, [&](int part, int t, int ks) { return A::v_frag(v0, PLANE, part, t, ks); },
           [&](int v) { return v % 4 == 0 ? f[v / 4].x : v % 4 == 1 ? f[v / 4].y : v % 4 == 2 ? f[v / 4].z : f[v / 4].w; });
    __builtin_amdgcn_wave_barrier();
  };

  Block x[2];
  int blk = b0 + wave;
  if (blk < b1) fetch(blk, x[0]);
  for (; blk < b1; blk += 2 * W) {
    if (blk + W < b1) fetch(blk + W, x[1]);
    compute(blk, x[0]);
    if (blk + W >= b1) break;
    if (blk + 2 * W < b1) fetch(blk + 2 * W, x[0]);
    compute(blk + W, x[1]);
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

  // the waves' results through LDS, only the rows' lanes
  const int nr = w.rows;
  constexpr int REGS = Cfg::REGS;
  float* res = reinterpret_cast<float*>(smem);              // [W][REGS][2][slots]
  float* refs = res + W * REGS * 2 * slots;                 // [W][slots]
  int* again = reinterpret_cast<int*>(refs + W * slots);    // [32]
  __syncthreads();
  if (l32 < nr) {
    float* to = res + wave * REGS * 2 * slots + g * slots + l32;
#pragma unroll
    for (int i = 0; i < A::DT; ++i)
#pragma unroll
      for (int v = 0; v < 16; ++v) to[(16 * i + v) * 2 * slots] = at.o[i][v];
    to[16 * A::DT * 2 * slots] = at.sum;
    // NaN scores leave the reference at 0 and a sum of NaN
    if (g == 0) refs[wave * slots + l32] = at.begun || !(at.sum == 0.f) ? at.ref : -INFINITY;
  }
  if (tid < 32) again[tid] = 0;
  __syncthreads();
  const int ld = hd + 2;
  for (int e = tid; e < nr * hd; e += W * 64) {
    const int r = e / hd, d = e % hd;
    const int reg = 16 * (d / 32) + 4 * (d % 32 / 8) + d % 4, half = d / 4 & 1;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < W; ++i) top = max_nan(top, refs[i * slots + r]);
    const float from = top == -INFINITY ? 0.f : top;
    float l = 0.f, y = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float by = __builtin_amdgcn_exp2f(refs[i * slots + r] - from);
      const float* f = res + i * REGS * 2 * slots + r;
      l = fmaf(f[16 * A::DT * 2 * slots] + f[16 * A::DT * 2 * slots + slots], by, l);
      y = fmaf(f[(reg * 2 + half) * slots], by, y);
    }
    if (nsplit > 1) {
      float* f = part + ((int64_t)id * 32 + r) * ld;
      f[d] = y;
      if (d == 0) {
        f[hd] = top;
        f[hd + 1] = l;
      }
    } else {
      y = w.n ? y / l : 0.f;
      const int rr = w.row0 + r;
      static_cast<T*>(a.o)[(((int64_t)w.b * a.T + rr / G) * a.H + w.kvh * G + rr % G) * hd + d] = from_f32<T>(y);
      if (A::doubtful(y)) again[r] = 1;
    }
  }
  if (nsplit > 1) return;
  __syncthreads();
  for (int r = wave; r < nr; r += W)
    if (again[r]) row_again<T, M, STEP>(a, w, r);
}

// Joins the key ranges of split rows: a workgroup per unit. The ranges' references and sums come first, all at once,
// and become factors; the outputs are then read eight ranges at a time.
constexpr int kMaxSplits = 64;
template <class T, class M, bool STEP>
__global__ __launch_bounds__(256) void rows_join_kernel(RowsArgs a, int tiles, int nsplit, const float* part) {
  __shared__ float by[32][kMaxSplits], inv[32];
  __shared__ int again[32];
  const int G = a.H / a.KV, hd = a.hd, ld = hd + 2, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Rows w;
  if (!rows_of<STEP>(a, blockIdx.x, tiles, w)) return;
  const float* unit0 = part + (int64_t)blockIdx.x * nsplit * 32 * ld;
  for (int r = wave; r < w.rows; r += 4) {  // lane s: range s
    float top = -INFINITY, l = 0.f;
    if (lane < nsplit) {
      top = unit0[((int64_t)lane * 32 + r) * ld + hd];
      l = unit0[((int64_t)lane * 32 + r) * ld + hd + 1];
    }
    const float all = group_reduce<64>(top, max_nan), ref = all == -INFINITY ? 0.f : all;
    const float f = __builtin_amdgcn_exp2f(top - ref);
    const float sum = group_reduce<64>(l * f, Plus{});
    if (lane < nsplit) by[r][lane] = f;
    if (lane == 0) {
      inv[r] = 1.f / sum;
      again[r] = 0;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < w.rows * hd; e += 256) {
    const int r = e / hd, d = e % hd;
    float y = 0.f;
    for (int s0 = 0; s0 < nsplit; s0 += 8) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = unit0[((int64_t)min(s0 + i, nsplit - 1) * 32 + r) * ld + d];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (s0 + i < nsplit) y = fmaf(v[i], by[r][s0 + i], y);
    }
    y = w.n ? y * inv[r] : 0.f;
    const int rr = w.row0 + r;
    static_cast<T*>(a.o)[(((int64_t)w.b * a.T + rr / G) * a.H + w.kvh * G + rr % G) * hd + d] = from_f32<T>(y);
    if (Attend<T, M, 8, false>::doubtful(y)) again[r] = 1;
  }
  __syncthreads();
  for (int r = wave; r < w.rows; r += 4)
    if (again[r]) row_again<T, M, STEP>(a, w, r);
}

// How a call is cut: tiles of 32 rows, and how many workgroups share a tile's keys.
struct Plan {
  int tiles, nsplit;
  int64_t units;
};
Plan plan_of(const RowsArgs& a, int64_t keys, int cus) {
  Plan p;
  p.tiles = (int)cdiv((int64_t)a.T * (a.H / a.KV), 32);
  p.units = (int64_t)a.B * a.KV * p.tiles;
  p.nsplit = keys < 640 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>({keys / 256, cus / p.units, kMaxSplits}));
  return p;
}
int64_t part_floats(const RowsArgs& a, const Plan& p) {
  return p.nsplit == 1 ? 0 : p.units * p.nsplit * 32 * (a.hd + 2);
}

template <class T, class M, int KS, bool STEP>
void launch_ks(const LaunchCtx& c, const RowsArgs& a, const Plan& p, float* part) {
  using Cfg = RowsCfg<T, M, KS>;
  const int slots = (int)std::min<int64_t>(32, (int64_t)a.T * (a.H / a.KV));
  launch(c, STEP ? "rows_step" : "rows_memory", rows_kernel<T, M, KS, STEP>, dim3((unsigned)(p.units * p.nsplit)),
         dim3(64 * Cfg::W), (size_t)Cfg::lds(slots), a, p.tiles, p.nsplit, slots, part);
}
template <class T, class M, bool STEP>
void launch_rows(const LaunchCtx& c, const RowsArgs& a, const Plan& p, float* part) {
  MNN_REQUIRE(p.units * p.nsplit < (1 << 22), MNN_ERR_INVALID_CONFIGURATION,
              (STEP ? "WindowAttention" : "MemoryAttention") << ": too many sequences and tokens in one call");
  MNN_REQUIRE(p.nsplit == 1 || part, MNN_ERR_INVALID_ARGUMENT, "rows of attention: split keys need a workspace");
  switch ((a.hd + 15) / 16) {
    case 1:
    case 2: launch_ks<T, M, 2, STEP>(c, a, p, part); break;
    case 3: launch_ks<T, M, 3, STEP>(c, a, p, part); break;
    case 4: launch_ks<T, M, 4, STEP>(c, a, p, part); break;
    case 5: launch_ks<T, M, 5, STEP>(c, a, p, part); break;
    case 6: launch_ks<T, M, 6, STEP>(c, a, p, part); break;
    default: launch_ks<T, M, 8, STEP>(c, a, p, part);
  }
  if (p.nsplit > 1)
    launch(c, "rows_join", rows_join_kernel<T, M, STEP>, dim3((unsigned)p.units), dim3(256), 0, a, p.tiles, p.nsplit,
           (const float*)part);
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
  return std::min<int64_t>((int64_t)a.left + a.sinks + std::min(a.T, 32), a.C);
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

int64_t window_step_e4m3_part_floats(const LaunchCtx& c, const WindowStepHeldArgs& s) {
  const RowsArgs a = step_args(s);
  return part_floats(a, plan_of(a, step_keys(s), c.dev->props.multiProcessorCount));
}
void window_step_e4m3(const LaunchCtx& c, const WindowStepHeldArgs& s, float* part) {
  const RowsArgs a = step_args(s);
  const Plan p = plan_of(a, step_keys(s), c.dev->props.multiProcessorCount);
  if (s.type == MNN_F32)
    launch_rows<float, E4m3, true>(c, a, p, part);
  else
    launch_rows<__bf16, E4m3, true>(c, a, p, part);
}

int64_t memory_rows_part_floats(const LaunchCtx& c, const MemoryArgs& m) {
  const RowsArgs a = memory_args(m);
  return part_floats(a, plan_of(a, m.S, c.dev->props.multiProcessorCount));
}
void memory_rows(const LaunchCtx& c, const MemoryArgs& m, float* part) {
  const RowsArgs a = memory_args(m);
  const Plan p = plan_of(a, m.S, c.dev->props.multiProcessorCount);
  if (m.type == MNN_F32)
    m.ks ? launch_rows<float, E4m3, false>(c, a, p, part) : launch_rows<float, float, false>(c, a, p, part);
  else
    m.ks ? launch_rows<__bf16, E4m3, false>(c, a, p, part) : launch_rows<__bf16, __bf16, false>(c, a, p, part);
}

}  // namespace k
}  // namespace mnn
