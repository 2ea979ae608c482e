// Rotary positions over several axes: pair (u, v) of axis a and rate f turns by the angle pos_a * f,
// (u cos - v sin, v cos + u sin). The angle is kept in turns: pos * (f / 2 pi) is one product in 64 bits,
// whose fraction is what is left of it, exact to 2^-53 of the whole (2e-7 turns at position 2^31). The sine and
// cosine are taken in fp32 of the fraction rounded to fp32; what that rounding left out (up to 9e-8 of an angle,
// more than the rounding of the results) is turned by as well, to first order.
#include "token_ops.hpp"
#include "token_utils.hpp"

#include <algorithm>

namespace mnn {
namespace k {

using namespace dev;

namespace {

__device__ __forceinline__ void turn_of(int pos, double rate, float& cs, float& sn) {
  const double t = (double)pos * rate, f = t - rint(t);
  const float h = (float)f, rest = (float)(f - (double)h) * 6.2831853f;
  float c, s;
  sincospif(2.f * h, &s, &c);
  cs = fmaf(-s, rest, c);
  sn = fmaf(c, rest, s);
}

// i / d with by = floor(2^32 / d): the high product is the quotient or one less, for any i below 2^32.
struct Divisor {
  unsigned d, by;
};
__device__ __forceinline__ int quotient(int i, Divisor v) {
  const unsigned q = __umulhi((unsigned)i, v.by);
  return (int)(q + ((unsigned)i - q * v.d >= v.d));
}

// A workgroup takes `toks` tokens: first their sines and cosines, once for all heads of both tensors, into
// LDS, then the rows. A thread's unit is VE pairs: VE values and their VE partners half an axis away, or 2 VE
// values in a row where pairs are interleaved; 2 VE values (one, for VE = 1) behind the last axis pass. VE = 8
// or 4 makes them 16-byte accesses of f32 and 16 or 8 of bf16, where every axis is a whole number of units.
// Both partners are read before either is written, so the output may be the input. Bound by memory: 4 x 2688 tokens
// of 8 + 8 heads of 48 in bf16 (33 MB) 8.3 us (9.4 with divisions in place of quotient(), 20 with the sines taken again for
// each head; four units a thread read ahead of the sines are no faster).
template <class T, int VE, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a, int toks, Divisor tok_units,
                                                     Divisor head_units, Divisor tok_pairs) {
  extern __shared__ float2 turns[];  // [toks][pairs]
  constexpr int RU = VE == 1 ? 1 : 2 * VE;
  typedef T Part __attribute__((ext_vector_type(VE)));
  const int turning = a.pairs / VE, units = (int)head_units.d, per_tok = (int)tok_units.d;  // of a head, a token
  const int64_t total = a.B * a.S;
  for (int64_t tok0 = (int64_t)blockIdx.x * toks; tok0 < total; tok0 += (int64_t)gridDim.x * toks) {
    const int n = (int)min((int64_t)toks, total - tok0);
    for (int i = threadIdx.x; i < n * a.pairs; i += 256) {
      const int ti = quotient(i, tok_pairs), u = i - ti * a.pairs;
      const int64_t tok = tok0 + ti;
      int axis = 0, j = u;
      while (j >= a.dims[axis] / 2) j -= a.dims[axis++] / 2;  // ends: u is one of the axes' pairs
      float2 t;
      turn_of(a.pos[(a.shared ? tok % a.S : tok) * a.axes + axis], a.rate[u], t.x, t.y);
      turns[i] = t;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * per_tok; i += 256) {
      const int ti = quotient(i, tok_units), rest = i - ti * per_tok;
      int h = quotient(rest, head_units);
      const int u = rest - h * units, which = h >= a.heads[0];
      if (which) h -= a.heads[0];
      const int64_t at = ((tok0 + ti) * (which ? a.heads[1] : a.heads[0]) + h) * a.hd;
      const T* x = static_cast<const T*>(which ? a.x[1] : a.x[0]) + at;
      T* y = static_cast<T*>(which ? a.y[1] : a.y[0]) + at;
      if (u >= turning) {
        const int d = 2 * a.pairs + (u - turning) * RU;
        if constexpr (VE == 1) {
          y[d] = x[d];
        } else {
          const Part p = *reinterpret_cast<const Part*>(x + d), q = *reinterpret_cast<const Part*>(x + d + VE);
          *reinterpret_cast<Part*>(y + d) = p;
          *reinterpret_cast<Part*>(y + d + VE) = q;
        }
        continue;
      }
      int j = u * VE, first = 0;  // pair j of the axis, whose dimensions begin at `first`
      int half = a.dims[0] / 2;
      if constexpr (!INTER) {
#pragma unroll
        for (int axis = 0; axis < 3; ++axis)
          if (j >= half) {  // only while the axes before were passed too
            j -= half;
            first += 2 * half;
            half = a.dims[axis + 1] / 2;
          } else {
            break;
          }
      }
      const int d0 = INTER ? 2 * j : first + j, d1 = INTER ? d0 + VE : d0 + half;
      const Part p = *reinterpret_cast<const Part*>(x + d0), q = *reinterpret_cast<const Part*>(x + d1);
      float in[2 * VE], out[2 * VE];  // p then q
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        in[e] = to_f32((T)p[e]);
        in[VE + e] = to_f32((T)q[e]);
      }
      const float2* t = turns + ti * a.pairs + u * VE;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float2 c = t[e];
        if (INTER) {
          out[2 * e] = in[2 * e] * c.x - in[2 * e + 1] * c.y;
          out[2 * e + 1] = in[2 * e + 1] * c.x + in[2 * e] * c.y;
        } else {
          out[e] = in[e] * c.x - in[VE + e] * c.y;
          out[VE + e] = in[VE + e] * c.x + in[e] * c.y;
        }
      }
      Part po, qo;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        po[e] = from_f32<T>(out[e]);
        qo[e] = from_f32<T>(out[VE + e]);
      }
      *reinterpret_cast<Part*>(y + d0) = po;
      *reinterpret_cast<Part*>(y + d1) = qo;
    }
    __syncthreads();
  }
}

// Whether units of VE pairs fill every axis, and what is behind them.
bool whole_units(const RotaryArgs& a, int VE) {
  bool ok = a.hd % VE == 0 && (a.hd - 2 * a.pairs) % (2 * VE) == 0 && a.pairs % VE == 0;
  for (int i = 0; i < a.axes && !a.interleaved; ++i) ok = ok && a.dims[i] / 2 % VE == 0;
  return ok;
}

template <class T, int VE>
void launch_rotary(const LaunchCtx& c, const RotaryArgs& a) {
  const int heads = a.heads[0] + a.heads[1], of_head = a.pairs / VE + (a.hd - 2 * a.pairs) / (VE == 1 ? 1 : 2 * VE);
  const int64_t units = (int64_t)heads * of_head;
  // tokens a workgroup: four units a thread, as few as the compute units still have work for, and as the
  // table of turns has room for (16 KB)
  const int64_t tokens = a.B * a.S, cus = c.dev->props.multiProcessorCount;
  int64_t toks = std::max<int64_t>(1, 1024 / units);
  toks = std::min({toks, std::max<int64_t>(1, tokens / (2 * cus)), std::max<int64_t>(1, 2048 / a.pairs)});
  const dim3 grid((unsigned)std::min<int64_t>((tokens + toks - 1) / toks, 1 << 20));
  const char* name = sizeof(T) == 4 ? "rotary_f32" : "rotary_bf16";
  const size_t lds = sizeof(float2) * toks * a.pairs;
  auto by = [](int64_t d) { return Divisor{(unsigned)d, d == 1 ? ~0u : (unsigned)((1ull << 32) / d)}; };
  if (a.interleaved)
    launch(c, name, rotary_kernel<T, VE, true>, grid, dim3(256), lds, a, (int)toks, by(units), by(of_head), by(a.pairs));
  else
    launch(c, name, rotary_kernel<T, VE, false>, grid, dim3(256), lds, a, (int)toks, by(units), by(of_head), by(a.pairs));
}
template <class T>
void rotary_t(const LaunchCtx& c, const RotaryArgs& a) {
  if constexpr (sizeof(T) == 2)
    if (whole_units(a, 8)) return launch_rotary<T, 8>(c, a);
  if (whole_units(a, 4)) return launch_rotary<T, 4>(c, a);
  launch_rotary<T, 1>(c, a);
}

}  // namespace

void rotary(const LaunchCtx& c, const RotaryArgs& a) {
  if (a.type == MNN_F32)
    rotary_t<float>(c, a);
  else
    rotary_t<__bf16>(c, a);
}

}  // namespace k
}  // namespace mnn
