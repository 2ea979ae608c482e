// Window attention of the next tokens of each stream on rolling caches. Token p lives in slot p (p < sinks)
// or sinks + (p - sinks) % (C - sinks). A call reads the tokens before it from the cache and its own from
// its inputs, so the new rows can be written to the cache in the same launch: with C >= sinks + left + T,
// none of the slots that they take holds a token that a query of the call still sees.
#include "token_ops.hpp"
#include "window_row.hpp"

#include <algorithm>
#include <climits>

namespace mnn {
namespace k {

using namespace dev;

namespace {

// Rows of this call that are tokens of stream b, and the stream's position; 0 where it is left alone.
__device__ __forceinline__ int rows_of(const WindowStepArgs& a, int b, int& pos) {
  pos = a.pos[b];
  if (pos < 0 || pos > INT_MAX - a.T) return 0;
  return a.steps ? min(max(a.steps[b], 0), a.T) : a.T;
}

__device__ __forceinline__ int slot_of(const WindowStepArgs& a, int p) {
  return p < a.sinks ? p : a.sinks + (p - a.sinks) % (a.C - a.sinks);
}

// Keys that tokens pos + t0 .. pos + t1 see, and the position of key `idx` of them: ns sinks, then the tokens from
// lo on. Positions reach 2^31 - 1, so no sum on the way may pass them: as constant expressions, one that did would
// not compile.
constexpr int keys_of(int ns, int pos, int t0, int t1, int lo) { return ns + (pos + t0 - lo) + (t1 - t0) + 1; }
constexpr int key_at(int ns, int lo, int idx) { return idx < ns ? idx : lo + (idx - ns); }
static_assert(keys_of(33, INT_MAX - 16, 0, 15, INT_MAX - 616) == 33 + 600 + 16 &&
                  key_at(33, INT_MAX - 616, 33 + 600 + 15) == INT_MAX - 1,
              "the farthest call of 16 tokens, 600 back, 33 sinks");

// The rows of a call that one workgroup answers: R of the T * G queries (token t, head g of the group) that
// read key/value head kvh of stream b, and the keys that any of them sees, numbered from 0: the sinks before
// the window's first token, then the window.
struct Rows {
  int b, kvh, row0, pos, nt;  // nt: tokens of the stream in this call
  int t0, t1;                 // first and last token among the rows
  int lo, ns, n;              // the window's first token, sinks before it, keys in all
  int ring, wrapped;          // wrapped: place in the ring of token max(lo, sinks)
};
template <int R>
__device__ __forceinline__ bool rows_setup(const WindowStepArgs& a, int unit, int tiles, Rows& w) {
  const int rt = unit % tiles, G = a.H / a.KV;
  w.kvh = unit / tiles % a.KV;
  w.b = unit / tiles / a.KV;
  w.row0 = rt * R;
  w.nt = rows_of(a, w.b, w.pos);
  w.t0 = w.row0 / G;
  if (w.t0 >= w.nt) return false;
  w.t1 = min(w.nt - 1, (w.row0 + R - 1) / G);
  w.lo = max(0, w.pos + w.t0 - a.left);
  w.ns = min(a.sinks, w.lo);
  w.n = keys_of(w.ns, w.pos, w.t0, w.t1, w.lo);
  w.ring = a.C - a.sinks;
  w.wrapped = (max(w.lo, a.sinks) - a.sinks) % w.ring;
  return true;
}

// Query (t, h) of stream b by one wave, without the keys that it does not see.
template <class T>
__device__ __forceinline__ void step_query(const WindowStepArgs& a, int b, int h, int t, int pos) {
  const int lane = threadIdx.x & 63, group = a.H / a.KV, kvw = a.KV * a.hd, i = pos + t;
  const int64_t col = (int64_t)(h / group) * a.hd;
  const T* kn = static_cast<const T*>(a.k) + (int64_t)b * a.T * kvw + col;
  const T* vn = static_cast<const T*>(a.v) + (int64_t)b * a.T * kvw + col;
  const T* kc = static_cast<const T*>(a.kc) + (int64_t)b * a.C * kvw + col;
  const T* vc = static_cast<const T*>(a.vc) + (int64_t)b * a.C * kvw + col;
  const int lo = max(0, i - a.left), ns = min(a.sinks, lo);
  auto row = [&](int64_t n, const T* cache, const T* fresh) {
    const int p = (int)(n < ns ? n : lo + (n - ns));
    return p >= pos ? fresh + (int64_t)(p - pos) * kvw : cache + (int64_t)slot_of(a, p) * kvw;
  };
  const int64_t at = ((int64_t)b * a.T + t) * a.H * a.hd + (int64_t)h * a.hd;
  float o0, o1;
  window_row(static_cast<const T*>(a.q) + at, a.hd, a.scale, (int64_t)ns + (i - lo + 1),
             [&](int64_t n) { return row(n, kc, kn); }, [&](int64_t n) { return row(n, vc, vn); }, o0, o1);
  T* o = static_cast<T*>(a.o) + at;
  if (lane < a.hd) o[lane] = from_f32<T>(o0);
  if (lane + 64 < a.hd) o[lane + 64] = from_f32<T>(o1);
}

// bf16: pairs of products an instruction, exact and added in fp32
__device__ __forceinline__ float dot8(const Eight<__bf16>& x, const Eight<__bf16>& y) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned u = x.x[0][i], v = y.x[0][i];
    s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, u), __builtin_bit_cast(bf16x2, v), s,
                                        false);
  }
  return s;
}
__device__ __forceinline__ float dot8(const Eight<float>& x, const Eight<float>& y) {
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) s = fmaf(x[e], y[e], s);
  return s;
}

// Sum over the lanes that hold the same dimensions: groups of L lanes (4, 8 or 16), 64 / L of them.
template <int L>
__device__ __forceinline__ float across_groups(float v) {
  if constexpr (L <= 4) v += __shfl_xor(v, 4, 64);
  if constexpr (L <= 8) v += dpp_mov<0x128>(v);  // row_ror:8
  return other_half(other_row(v, Plus{}), Plus{});
}

// W waves answer R rows. L lanes take a key, eight dimensions each (head dims that are no power of two leave
// some idle), so a wave holds 64 / L keys at a time, U of those computed while the next U are on their way;
// every group of L lanes keeps running maxima, sums and outputs of its own, which are joined at the end, first
// in the wave, then in LDS, then, if the keys are split over workgroups, by window_join_kernel. On the vector
// units: a key's row feeds R dot products only, 4 bytes of cache an instruction at R = 1, and the matrix units
// would stand idle for the loads just the same. One row of f32 at 64 streams, 8 heads of 128, 1024 keys runs
// at 5.7 TB/s; four rows of bf16 (64 streams, 16 / 4 heads of 64, 2048 keys) at 3.7 TB/s, bound by the vector
// units. Waves: 8, or 12 with half the keys in flight where four rows of bf16 leave them no more registers
// (us at 16 without / 8 with / 12 with the next keys in flight: the latter case 30.6 / 31.9 / 30.1, one stream of
// 8 heads of 48 in f32 6.9 / 6.5 / -).
template <class T, int L, int R, int W>
__global__ __launch_bounds__(W * 64) void window_step_kernel(WindowStepArgs a, int tiles, int nsplit,
                                                             float* part) {
  constexpr int KPW = 64 / L, U = sizeof(T) == 4 ? 2 : R > 2 ? 2 : 4;
  extern __shared__ float sh[];  // [W][R][hd + 2], [R]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane % L, grp = lane / L;
  const int sp = blockIdx.x % nsplit, unit = blockIdx.x / nsplit;
  const int G = a.H / a.KV, kvw = a.KV * a.hd, hd = a.hd;
  const bool on = 8 * j < hd;
  // the queries, before the stream's position has come: rows that are no tokens are not used
  Eight<T> q[R];
  {
    const int row0 = unit % tiles * R, kvh = unit / tiles % a.KV, b = unit / tiles / a.KV;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int t = (row0 + r) / G, h = kvh * G + (row0 + r) % G;
      q[r].clear();
      if (on && t < a.T)
        q[r].load(static_cast<const T*>(a.q) + ((int64_t)b * a.T + t) * a.H * hd + (int64_t)h * hd + 8 * j);
    }
  }
  Rows w;
  if (!rows_setup<R>(a, unit, tiles, w)) return;
  const int64_t col = (int64_t)w.kvh * hd + (on ? 8 * j : 0);
  const T* kn = static_cast<const T*>(a.k) + (int64_t)w.b * a.T * kvw + col;
  const T* vn = static_cast<const T*>(a.v) + (int64_t)w.b * a.T * kvw + col;
  T* kc = static_cast<T*>(a.kc) + (int64_t)w.b * a.C * kvw + col;
  T* vc = static_cast<T*>(a.vc) + (int64_t)w.b * a.C * kvw + col;

  const float qs = a.scale * 1.4426950408889634f;
  float m[R], l[R], o[R][8];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[r][e] = 0.f;
  }
  const int begin = (int)((int64_t)w.n * sp / nsplit), end = (int)((int64_t)w.n * (sp + 1) / nsplit);
  const bool mixed = w.t0 != w.t1;  // rows of several tokens, which see different keys
  // U keys a group at a time; the next ones are on their way while these are computed
  struct Keys {
    Eight<T> k[U], v[U];
    int p[U];  // the lane's keys as positions, -1: none
  };
  auto fetch = [&](int i, Keys& x) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int idx = i + u * KPW + grp;
      x.p[u] = idx >= end ? -1 : key_at(w.ns, w.lo, idx);
      x.k[u].clear();
      x.v[u].clear();
      if (on && idx < end) {
        int slot = x.p[u];
        if (slot >= a.sinks) {
          slot = w.wrapped + (slot - max(w.lo, a.sinks));
          slot = a.sinks + (slot >= w.ring ? slot - w.ring : slot);
        }
        const bool fresh = x.p[u] >= w.pos;
        const int64_t at = (int64_t)(fresh ? x.p[u] - w.pos : slot) * kvw;
        x.k[u].load((fresh ? kn : kc) + at);
        x.v[u].load((fresh ? vn : vc) + at);
      }
    }
  };
  auto compute = [&](const Keys& x) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float s[U], top = m[r];
      const int mine = (int)((unsigned)w.pos + (unsigned)((w.row0 + r) / G));  // rows past the call's last wrap, unused
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u] = group_reduce<L>(dot8(x.k[u], q[r]), Plus{}) * qs;
        const int p = x.p[u];
        // without short circuits, which become branches (16 tokens, 8 heads of 48: 13.3 -> 12.0 us)
        const bool seen = (p >= 0) & (!mixed | ((p <= mine) & ((p >= mine - a.left) | (p < a.sinks))));
        s[u] = seen ? s[u] : -INFINITY;
        top = max_nan(top, s[u]);
      }
      const float ref = top == -INFINITY ? 0.f : top;
      const float alpha = __builtin_amdgcn_exp2f(m[r] - ref);
      m[r] = top;
      l[r] *= alpha;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[r][e] *= alpha;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float pu = __builtin_amdgcn_exp2f(s[u] - ref);
        l[r] += pu;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[r][e] = fmaf(pu, x.v[u][e], o[r][e]);
      }
    }
  };
  constexpr int STEP = W * KPW * U;
  Keys x[2];
  int i = begin + wave * KPW * U;
  if (i < end) fetch(i, x[0]);
  for (; i < end; i += 2 * STEP) {
    if (i + STEP < end) fetch(i + STEP, x[1]);
    compute(x[0]);
    if (i + STEP >= end) break;
    if (i + 2 * STEP < end) fetch(i + 2 * STEP, x[0]);
    compute(x[1]);
  }

  // the new tokens' keys and values to their slots
  if (w.row0 == 0 && sp == 0 && on) {
    for (int t = threadIdx.x / L; t < w.nt; t += W * KPW) {
      const int64_t to = (int64_t)slot_of(a, w.pos + t) * kvw, from = (int64_t)t * kvw;
      Eight<T> x;
      x.load(kn + from);
      x.store(kc + to);
      x.load(vn + from);
      x.store(vc + to);
    }
  }

  // the wave's groups, then the waves
  const int ld = hd + 2;
  float* again = sh + W * R * ld;  // rows to compute again
  if (threadIdx.x < R) again[threadIdx.x] = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float top = m[r];
#pragma unroll
    for (int off = L; off < 64; off <<= 1) top = max_nan(top, __shfl_xor(top, off, 64));
    const float ref = top == -INFINITY ? 0.f : top;
    const float by = __builtin_amdgcn_exp2f(m[r] - ref);
    const float lr = across_groups<L>(l[r] * by);
    float* to = sh + (wave * R + r) * ld;
    if (lane == 0) {
      to[hd] = top;
      to[hd + 1] = lr;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = across_groups<L>(o[r][e] * by);
      if (grp == 0 && on) to[8 * j + e] = x;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < R * hd; e += W * 64) {
    const int r = e / hd, d = e % hd, row = w.row0 + r, t = row / G;
    if (t >= w.nt) continue;
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < W; ++v) top = max_nan(top, sh[(v * R + r) * ld + hd]);
    const float ref = top == -INFINITY ? 0.f : top;
    float lr = 0.f, x = 0.f;
#pragma unroll
    for (int v = 0; v < W; ++v) {
      const float* f = sh + (v * R + r) * ld;
      const float by = __builtin_amdgcn_exp2f(f[hd] - ref);
      lr = fmaf(f[hd + 1], by, lr);
      x = fmaf(f[d], by, x);
    }
    if (nsplit > 1) {
      float* f = part + ((int64_t)blockIdx.x * R + r) * ld;
      f[d] = x;
      if (d == 0) {
        f[hd] = top;
        f[hd + 1] = lr;
      }
    } else {
      x /= lr;
      static_cast<T*>(a.o)[((int64_t)w.b * a.T + t) * a.H * hd + (int64_t)(w.kvh * G + row % G) * hd + d] =
          from_f32<T>(x);
      // a key that this row does not see had weight 0 times a value that is not finite, perhaps
      if (mixed && !(x * 0.f == 0.f)) again[r] = 1.f;
    }
  }
  if (nsplit > 1 || !mixed) return;
  __syncthreads();
  for (int r = wave; r < R; r += W) {
    const int row = w.row0 + r;
    if (row / G < w.nt && again[r] == 1.f)
      step_query<T>(a, w.b, w.kvh * G + row % G, row / G, w.pos);
  }
}

// Joins the key ranges of split rows: a workgroup per unit, thread (row, dimension). The ranges' maxima and
// sums come first, all at once, and become factors; the outputs are then read eight ranges at a time (one
// after another, a range cost half a microsecond).
constexpr int kMaxSplits = 32;
template <class T, int R>
__global__ __launch_bounds__(256) void window_join_kernel(WindowStepArgs a, int tiles, int nsplit,
                                                          const float* part) {
  __shared__ float by[R][kMaxSplits], inv[R];
  __shared__ int again[R];
  const int G = a.H / a.KV, hd = a.hd, ld = hd + 2;
  const float* unit0 = part + (int64_t)blockIdx.x * nsplit * R * ld;
  Rows w;
  if (!rows_setup<R>(a, blockIdx.x, tiles, w)) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (wave < R) {  // a wave a row, lane s the range s
    const int r = wave;
    float top = -INFINITY, l = 0.f;
    if (lane < nsplit) {
      top = unit0[((int64_t)lane * R + r) * ld + hd];
      l = unit0[((int64_t)lane * R + r) * ld + hd + 1];
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
  for (int e = threadIdx.x; e < R * hd; e += 256) {
    const int r = e / hd, d = e % hd, row = w.row0 + r, t = row / G;
    if (t >= w.nt) continue;
    float x = 0.f;
    for (int s0 = 0; s0 < nsplit; s0 += 8) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = unit0[((int64_t)min(s0 + i, nsplit - 1) * R + r) * ld + d];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (s0 + i < nsplit) x = fmaf(v[i], by[r][s0 + i], x);
    }
    x *= inv[r];
    static_cast<T*>(a.o)[((int64_t)w.b * a.T + t) * a.H * hd + (int64_t)(w.kvh * G + row % G) * hd + d] =
        from_f32<T>(x);
    if (!(x * 0.f == 0.f)) again[r] = 1;
  }
  if (w.t0 == w.t1) return;
  __syncthreads();
  for (int r = wave; r < R; r += 4) {
    const int row = w.row0 + r;
    if (row / G < w.nt && again[r]) step_query<T>(a, w.b, w.kvh * G + row % G, row / G, w.pos);
  }
}

// How a call is cut: rows a workgroup, its waves, and how many workgroups share a unit's keys.
struct Plan {
  int R, nsplit;
  int64_t tiles;
};
template <class T, int R>
constexpr int kWaves = sizeof(T) == 2 && R == 4 ? 12 : 8;
Plan plan_of(const WindowStepArgs& a, int cus) {
  Plan p;
  const int64_t rows = (int64_t)a.T * (a.H / a.KV);
  p.R = rows >= 4 ? 4 : rows >= 2 ? 2 : 1;
  p.tiles = (rows + p.R - 1) / p.R;
  const int64_t units = (int64_t)a.B * a.KV * p.tiles;
  const int64_t keys = std::min<int64_t>((int64_t)a.left + a.sinks + a.T, a.C);
  // A second launch costs about 2 us: keys are split only from 640 on, into ranges of 256, and while that
  // leaves no more workgroups than compute units. us in one, ranges of 512 / 256 / 128: one stream, 4096 keys,
  // 8 / 2 heads of 64, f32 - / 16.8 / 15.1 / 15.3; 8 heads of 128, bf16 - / 12.1 / 10.9 / 12.0; 8 streams, 1024
  // keys, 8 heads of 64, f32 12.0 / 11.9 / 10.5 / 10.5; one stream, 516 keys, 8 heads of 48, f32 6.8 / - / 9.0 / 8.5.
  p.nsplit = keys < 640 ? 1
                        : (int)std::max<int64_t>(1, std::min<int64_t>({keys / 256, cus / std::max<int64_t>(units, 1),
                                                                       kMaxSplits}));
  return p;
}

template <class T, int L, int R>
void launch_step(const LaunchCtx& c, const WindowStepArgs& a, const Plan& p, float* part) {
  constexpr int W = kWaves<T, R>;
  const int64_t units = (int64_t)a.B * a.KV * p.tiles;
  MNN_REQUIRE(units * p.nsplit < (1 << 22), MNN_ERR_INVALID_CONFIGURATION,
              "WindowAttention: too many streams and tokens in one step");
  const size_t lds = sizeof(float) * (W * R * (a.hd + 2) + R);
  launch(c, sizeof(T) == 4 ? "window_step_f32" : "window_step_bf16", window_step_kernel<T, L, R, W>,
         dim3((unsigned)(units * p.nsplit)), dim3(64 * W), lds, a, (int)p.tiles, p.nsplit, part);
  if (p.nsplit > 1)
    launch(c, sizeof(T) == 4 ? "window_join_f32" : "window_join_bf16", window_join_kernel<T, R>,
           dim3((unsigned)units), dim3(256), 0, a, (int)p.tiles, p.nsplit, (const float*)part);
}
template <class T, int L>
void launch_step_r(const LaunchCtx& c, const WindowStepArgs& a, const Plan& p, float* part) {
  if (p.R == 4) return launch_step<T, L, 4>(c, a, p, part);
  if (p.R == 2) return launch_step<T, L, 2>(c, a, p, part);
  launch_step<T, L, 1>(c, a, p, part);
}
template <class T>
void launch_step_t(const LaunchCtx& c, const WindowStepArgs& a, const Plan& p, float* part) {
  if (a.hd > 64) return launch_step_r<T, 16>(c, a, p, part);
  if (a.hd > 32) return launch_step_r<T, 8>(c, a, p, part);
  launch_step_r<T, 4>(c, a, p, part);
}

}  // namespace

int64_t window_step_part_floats(const LaunchCtx& c, const WindowStepArgs& a) {
  const Plan p = plan_of(a, c.dev->props.multiProcessorCount);
  return p.nsplit == 1 ? 0 : (int64_t)a.B * a.KV * p.tiles * p.nsplit * p.R * (a.hd + 2);
}

void window_step(const LaunchCtx& c, const WindowStepArgs& a, float* part) {
  const Plan p = plan_of(a, c.dev->props.multiProcessorCount);
  MNN_REQUIRE(p.nsplit == 1 || part, MNN_ERR_INVALID_ARGUMENT, "window step: split keys need a workspace");
  if (a.type == MNN_F32)
    launch_step_t<float>(c, a, p, part);
  else
    launch_step_t<__bf16>(c, a, p, part);
}

}  // namespace k
}  // namespace mnn
