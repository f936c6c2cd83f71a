// Rotary positions with several axes: channel pair i of a token at position pos_a (a: the pair's axis) is turned by
//   angle = pos_a * theta^(-2 i / n),   (a, b) -> (a cos - b sin, b cos + a sin)
// i counts within the axis and n is the axis' channels, or (joint) i counts over all pairs and n over all rotated
// channels. Pairs are (i, i + half) or (interleaved) (2 i, 2 i + 1); channels behind the rotated ones are copied. The
// backward pass is the same turn by the negative angle.
// Memory bound: x is read once, y written once (2 x 16,368 tokens x 20 heads x 128 channels bf16: 65 to 72 us = 5.1 to
// 4.7 TB/s; a copy of 4 GB: 4.7; 256 tokens x 16 heads x 32: 4.7 us, half of it the launch). An angle is computed once per
// token and pair and used for all heads a thread walks. It is formed in revolutions in 64 bits (a position of 2^30 leaves
// 22 bits behind the point, fp32 would leave none), reduced to an eighth of a turn there, and only the rest is rounded to
// fp32.
#include <algorithm>

#include "common.h"
#include "launch.h"

namespace {

template <int TYPE>
struct RElem;
template <>
struct RElem<0> {
  typedef float type;
  static CFL_DEVICE float get(float v) { return v; }
  static CFL_DEVICE float put(float v) { return v; }
};
template <>
struct RElem<1> {
  typedef bf16_t type;
  static CFL_DEVICE float get(bf16_t v) { return bf2f(v); }
  static CFL_DEVICE bf16_t put(float v) { return f2bf(v); }
};
template <>
struct RElem<2> {
  typedef _Float16 type;
  static CFL_DEVICE float get(_Float16 v) { return (float)v; }
  static CFL_DEVICE _Float16 put(float v) { return (_Float16)v; }
};

// cos and sin of `rev` revolutions: the nearest quarter turn taken off in 64 bits, then their Taylor series on the rest,
// |x| <= pi / 4 (the terms left out are below x^11 / 11! = 1.8e-9 and x^12 / 12! = 1.2e-10). The math library's
// sinpif and cospif were two thirds of a small call: each thread forms 8 angles before its first store.
CFL_DEVICE void turn(double rev, float& c, float& s) {
  const double f = rev - floor(rev);
  const double q = rint(4.0 * f);                         // quarter turns, 0..4
  const float x = (float)((f - 0.25 * q) * 6.283185307179586);
  const float x2 = x * x;
  const float s0 = fmaf(x * x2, fmaf(x2, fmaf(x2, fmaf(x2, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
  const float c0 = fmaf(
      x2, fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const int k = (int)q;
  const float a = k & 1 ? s0 : c0, b = k & 1 ? c0 : s0;
  c = k == 1 || k == 2 ? -a : a;
  s = k & 2 ? -b : b;
}

struct RotaryGrid {
  FastDiv div_u, div_h, div_s;
  int units, chunks, hpt;          // vector units of a token, head groups, heads per group
  int64_t total;
};

constexpr int MAX_HALF = 2048;

CFL_DEVICE int axis_of(const RotaryParams& p, int i) { return (i >= p.end[0]) + (i >= p.end[1]) + (i >= p.end[2]); }

// V elements per memory access. A unit of a token is V rotated pairs (half-split: two vectors; interleaved: V / 2 pairs
// in one vector), or a vector of the copied channels.
template <int TYPE, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p, const RotaryGrid g) {
  typedef typename RElem<TYPE>::type E;
  struct alignas(V * sizeof(E)) Vec { E e[V]; };
  extern __shared__ double rate[];                          // revolutions per position of each pair
  for (int i = threadIdx.x; i < p.half; i += 256) {
    // the axis of a pair by comparisons: an index into the parameters would be a load for each step
    const int a = axis_of(p, i), first = a == 0 ? 0 : a == 1 ? p.end[0] : a == 2 ? p.end[1] : p.end[2];
    const int last = a == 0 ? p.end[0] : a == 1 ? p.end[1] : a == 2 ? p.end[2] : p.end[3];
    const int n = p.joint ? p.half : last - first, k = p.joint ? i : i - first;
    rate[i] = exp2(-p.log2_theta * (double)k / (double)n) * 0.15915494309189533577;     // 2 k / (2 n); 1 / (2 pi)
  }
  __syncthreads();
  constexpr int P = INTER && V > 1 ? V / 2 : V;             // pairs per unit
  const int pu = p.half / P;                                // units that hold pairs
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < g.total; id += (int64_t)gridDim.x * 256) {
    const int x = (int)id, t0 = fdiv32(x, g.div_u), u = x - t0 * g.units;
    const int tok = fdiv32(t0, g.div_h), h0 = (t0 - tok * g.chunks) * g.hpt, h1 = imin(h0 + g.hpt, p.H);
    const int b = fdiv32(tok, g.div_s), s = tok - b * p.S;
    const E* src = reinterpret_cast<const E*>(p.x) + b * p.x_sb + s * p.x_ss;
    E* dst = reinterpret_cast<E*>(p.y) + b * p.y_sb + s * p.y_ss;
    if (u >= pu) {                                          // copied channels
      const int d = 2 * p.half + (u - pu) * V;
      for (int h = h0; h < h1; ++h)
        *reinterpret_cast<Vec*>(dst + h * p.y_sh + d) = *reinterpret_cast<const Vec*>(src + h * p.x_sh + d);
      continue;
    }
    float c[P], sn[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int i = u * P + j;
      const int64_t at = axis_of(p, i) * p.p_sa + b * p.p_sb + s * p.p_ss;
      const double pos = p.pos_type == 0   ? (double)reinterpret_cast<const int32_t*>(p.pos)[at]
                         : p.pos_type == 1 ? (double)reinterpret_cast<const int64_t*>(p.pos)[at]
                                           : (double)reinterpret_cast<const float*>(p.pos)[at];
      turn(pos * rate[i], c[j], sn[j]);
      if (p.inverse) sn[j] = -sn[j];
    }
#pragma unroll 4
    for (int h = h0; h < h1; ++h) {
      const E* xs = src + h * p.x_sh;
      E* ys = dst + h * p.y_sh;
      if constexpr (INTER && V > 1) {
        const Vec v = *reinterpret_cast<const Vec*>(xs + u * V);
        Vec o;
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const float a = RElem<TYPE>::get(v.e[2 * j]), bb = RElem<TYPE>::get(v.e[2 * j + 1]);
          o.e[2 * j] = RElem<TYPE>::put(a * c[j] - bb * sn[j]);
          o.e[2 * j + 1] = RElem<TYPE>::put(bb * c[j] + a * sn[j]);
        }
        *reinterpret_cast<Vec*>(ys + u * V) = o;
      } else {
        const int i0 = INTER ? 2 * u : u * V, i1 = INTER ? 2 * u + 1 : u * V + p.half;
        const Vec v = *reinterpret_cast<const Vec*>(xs + i0), w = *reinterpret_cast<const Vec*>(xs + i1);
        Vec o0, o1;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float a = RElem<TYPE>::get(v.e[j]), bb = RElem<TYPE>::get(w.e[j]);
          o0.e[j] = RElem<TYPE>::put(a * c[j] - bb * sn[j]);
          o1.e[j] = RElem<TYPE>::put(bb * c[j] + a * sn[j]);
        }
        *reinterpret_cast<Vec*>(ys + i0) = o0;
        *reinterpret_cast<Vec*>(ys + i1) = o1;
      }
    }
  }
}

template <int TYPE, int V>
int go(const RotaryParams& p, hipStream_t st) {
  RotaryGrid g;
  const int P = p.interleaved && V > 1 ? V / 2 : V;
  g.units = p.half / P + (p.D - 2 * p.half) / V;
  const int64_t tokens = (int64_t)p.B * p.S;
  // heads per thread: as many as leave 2^17 threads, so that a few tokens still fill the card
  g.hpt = (int)std::max<int64_t>(1, std::min<int64_t>(p.H, tokens * g.units * p.H >> 17));
  g.chunks = (p.H + g.hpt - 1) / g.hpt;
  g.total = tokens * g.units * g.chunks;
  if (g.total > 0x7fffffff) return 2;
  g.div_u = fast_div(g.units);
  g.div_h = fast_div(g.chunks);
  g.div_s = fast_div(p.S);
  const unsigned n = (unsigned)std::min<int64_t>((g.total + 255) / 256, 4096);
  if (p.interleaved) rotary_kernel<TYPE, V, true><<<n, 256, p.half * 8, st>>>(p, g);
  else rotary_kernel<TYPE, V, false><<<n, 256, p.half * 8, st>>>(p, g);
  return hipGetLastError() == hipSuccess ? 0 : 3;
}

template <int TYPE>
int run(const RotaryParams& p, hipStream_t st) {
  constexpr int V = 16 / sizeof(typename RElem<TYPE>::type);
  const int64_t all = p.x_sb | p.x_ss | p.x_sh | p.y_sb | p.y_ss | p.y_sh | p.D |
                      (p.interleaved ? 2 * p.half : p.half);
  const bool vec = all % V == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && reinterpret_cast<uintptr_t>(p.y) % 16 == 0;
  return vec ? go<TYPE, V>(p, st) : go<TYPE, 1>(p, st);
}

}  // namespace

int rotary_apply(const RotaryParams& p, hipStream_t st) {
  if (p.half < 1 || p.half > MAX_HALF || 2 * p.half > p.D || p.end[3] != p.half) return 1;
  if ((int64_t)p.B * p.S * p.H == 0) return 0;
  switch (p.type) {
    case 0: return run<0>(p, st);
    case 1: return run<1>(p, st);
    case 2: return run<2>(p, st);
    default: return 1;
  }
}
