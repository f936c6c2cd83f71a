// Layer norm over the last axis, forward and backward.
//   mu = mean(x)   r = 1 / sqrt(mean((x - mu)^2) + eps)   xh = (x - mu) r   y = xh w + b
//   g = dy w   dx = r (g - mean(g) - xh mean(g xh))   dw = sum_rows dy xh   db = sum_rows dy
// Memory bound: x (and dy) is read once, y (dx) written once. A row is held in registers by LPR lanes (a group of a
// wave, a wave, or a block), so the variance is the two-pass one - sums of squares of x - mu, exact where the mean is
// large - at no extra read. The backward pass computes mu and r again from the row it holds anyway instead of reading
// 8 saved bytes per row (a quarter of a 32-channel bf16 row).
// dw / db: a lane owns the same columns in every row of its block, adds them up in fp32 registers, the block joins its
// lanes through LDS and writes one partial row; a second launch adds the partial rows in order. No atomics: results
// do not depend on the order in which blocks run.
#include <algorithm>

#include "common.h"
#include "launch.h"

namespace {

template <int TYPE>
struct Elem;
template <>
struct Elem<0> {
  typedef float type;
  static constexpr int V = 4;
  static CFL_DEVICE float get(float v) { return v; }
  static CFL_DEVICE float put(float v) { return v; }
};
template <>
struct Elem<1> {
  typedef bf16_t type;
  static constexpr int V = 8;
  static CFL_DEVICE float get(bf16_t v) { return bf2f(v); }
  static CFL_DEVICE bf16_t put(float v) { return f2bf(v); }
};
template <>
struct Elem<2> {
  typedef _Float16 type;
  static constexpr int V = 8;
  static CFL_DEVICE float get(_Float16 v) { return (float)v; }
  static CFL_DEVICE _Float16 put(float v) { return (_Float16)v; }
};

// V consecutive elements as floats (V = 1, or a 16-byte vector)
template <int TYPE, int V>
CFL_DEVICE void load_v(const typename Elem<TYPE>::type* p, float* f) {
  typedef typename Elem<TYPE>::type E;
  if constexpr (V == 1) {
    f[0] = Elem<TYPE>::get(*p);
  } else {
    struct alignas(16) Vec { E e[V]; };
    const Vec v = *reinterpret_cast<const Vec*>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = Elem<TYPE>::get(v.e[j]);
  }
}
template <int TYPE, int V>
CFL_DEVICE void store_v(typename Elem<TYPE>::type* p, const float* f) {
  typedef typename Elem<TYPE>::type E;
  if constexpr (V == 1) {
    *p = Elem<TYPE>::put(f[0]);
  } else {
    struct alignas(16) Vec { E e[V]; };
    Vec v;
#pragma unroll
    for (int j = 0; j < V; ++j) v.e[j] = Elem<TYPE>::put(f[j]);
    *reinterpret_cast<Vec*>(p) = v;
  }
}

// NSUM sums over the LPR lanes of a row, the result in each of them. Groups inside a wave exchange lanes; a block-wide
// row (LPR > 64) goes through LDS: `red` holds NSUM * LPR / 64 floats, one barrier pair per call.
template <int LPR, int NSUM>
CFL_DEVICE void row_sum(float* v, float* red) {
#pragma unroll
  for (int n = 0; n < NSUM; ++n)
#pragma unroll
    for (int o = 1; o < (LPR < 64 ? LPR : 64); o <<= 1) v[n] = xor_add(v[n], o);
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int n = 0; n < NSUM; ++n) red[n * W + (threadIdx.x >> 6)] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NSUM; ++n) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) t += red[n * W + w];
      v[n] = t;
    }
    __syncthreads();
  }
}

// mu and r of the row held in x; masked elements (columns past C) hold 0 on entry and on return x - mu is 0 there
template <int LPR, int NV, int V>
CFL_DEVICE float center(float (*x)[V], const int* col, int C, float eps, float* red) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) s += x[k][j];
  row_sum<LPR, 1>(&s, red);
  const float mu = s / (float)C;
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      x[k][j] = col[k] < C ? x[k][j] - mu : 0.f;
      q = fmaf(x[k][j], x[k][j], q);
    }
  row_sum<LPR, 1>(&q, red);
  return 1.f / sqrtf(q / (float)C + eps);
}

template <int LPR>
constexpr int threads() { return LPR > 256 ? LPR : 256; }

// rows go to row groups (LPR lanes) in turn; NV vectors of V elements a lane: vector k of lane q starts at column
// (k LPR + q) V
template <int TYPE, int V, int LPR, int NV>
__global__ __launch_bounds__(threads<LPR>()) void ln_fwd_kernel(const LayerNormParams p) {
  typedef typename Elem<TYPE>::type E;
  constexpr int NT = threads<LPR>(), RPB = NT / LPR;
  __shared__ float red[LPR > 64 ? LPR / 64 : 1];
  const int q = threadIdx.x % LPR;
  int col[NV];
  float w[NV][V], b[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    col[k] = (k * LPR + q) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool in = col[k] < p.C;
      w[k][j] = in && p.w ? p.w[col[k] + j] : 1.f;
      b[k][j] = in && p.b ? p.b[col[k] + j] : 0.f;
    }
  }
  for (int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR; r - threadIdx.x / LPR < p.rows;
       r += (int64_t)gridDim.x * RPB) {
    const bool ok = r < p.rows;
    const E* xr = reinterpret_cast<const E*>(p.x) + r * p.x_stride;
    float x[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[k][j] = 0.f;
      if (ok && col[k] < p.C) load_v<TYPE, V>(xr + col[k], x[k]);
    }
    const float rs = center<LPR, NV, V>(x, col, p.C, p.eps, red);
    E* yr = reinterpret_cast<E*>(p.y) + r * p.C;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[k][j] = fmaf(x[k][j] * rs, w[k][j], b[k][j]);
      if (ok && col[k] < p.C) store_v<TYPE, V>(yr + col[k], x[k]);
    }
  }
}

template <int TYPE, int V, int LPR, int NV>
__global__ __launch_bounds__(threads<LPR>()) void ln_bwd_kernel(const LayerNormParams p) {
  typedef typename Elem<TYPE>::type E;
  constexpr int NT = threads<LPR>(), RPB = NT / LPR;
  __shared__ float red[LPR > 64 ? 2 * (LPR / 64) : 1];
  const int q = threadIdx.x % LPR;
  int col[NV];
  float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    col[k] = (k * LPR + q) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[k][j] = col[k] < p.C && p.w ? p.w[col[k] + j] : 1.f;
      dw[k][j] = db[k][j] = 0.f;
    }
  }
  for (int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR; r - threadIdx.x / LPR < p.rows;
       r += (int64_t)gridDim.x * RPB) {
    const bool ok = r < p.rows;
    const E* xr = reinterpret_cast<const E*>(p.x) + r * p.x_stride;
    const E* gr = reinterpret_cast<const E*>(p.gy) + r * p.gy_stride;
    float x[NV][V], g[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[k][j] = g[k][j] = 0.f;
      if (ok && col[k] < p.C) {
        load_v<TYPE, V>(xr + col[k], x[k]);
        load_v<TYPE, V>(gr + col[k], g[k]);
      }
    }
    const float rs = center<LPR, NV, V>(x, col, p.C, p.eps, red);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[k][j] *= rs;
        dw[k][j] = fmaf(g[k][j], x[k][j], dw[k][j]);
        db[k][j] += g[k][j];
        g[k][j] *= w[k][j];
        s[0] += g[k][j];
        s[1] = fmaf(g[k][j], x[k][j], s[1]);
      }
    if (p.y == nullptr) continue;
    row_sum<LPR, 2>(s, red);
    const float m0 = s[0] / (float)p.C, m1 = s[1] / (float)p.C;
    E* yr = reinterpret_cast<E*>(p.y) + r * p.C;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[k][j] = rs * (g[k][j] - m0 - x[k][j] * m1);
      if (ok && col[k] < p.C) store_v<TYPE, V>(yr + col[k], x[k]);
    }
  }
  if (p.ws == nullptr) return;
  // join the row groups that own the same columns, one vector at a time: lanes of a wave, then the block's waves
  constexpr int W = RPB > 1 ? (LPR < 64 ? NT / 64 : RPB) : 1, G = LPR < 64 ? LPR : 64;
  __shared__ float part[W > 1 ? W * G * 2 * V : 1];
  float* out = p.ws + (int64_t)blockIdx.x * 2 * p.C;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int o = G; o < 64; o <<= 1) {
        dw[k][j] = xor_add(dw[k][j], o);
        db[k][j] = xor_add(db[k][j], o);
      }
    if constexpr (W > 1) {
      const int wv = threadIdx.x >> 6, l = threadIdx.x & 63;
      if (k > 0) __syncthreads();
      if (l < G)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          part[((wv * 2) * V + j) * G + l] = dw[k][j];
          part[((wv * 2 + 1) * V + j) * G + l] = db[k][j];
        }
      __syncthreads();
      if (threadIdx.x < G)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float a = 0.f, b = 0.f;
#pragma unroll
          for (int u = 0; u < W; ++u) {
            a += part[((u * 2) * V + j) * G + l];
            b += part[((u * 2 + 1) * V + j) * G + l];
          }
          dw[k][j] = a;
          db[k][j] = b;
        }
    }
    if (threadIdx.x < LPR && col[k] < p.C)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        out[col[k] + j] = dw[k][j];
        out[p.C + col[k] + j] = db[k][j];
      }
  }
}

// dw / db = sums of the partial rows: a block owns 32 columns of one of the two, 8 threads a column
__global__ __launch_bounds__(256) void ln_bwd_join_kernel(const LayerNormParams p) {
  __shared__ float s[8][33];
  const int cl = threadIdx.x & 31, g = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
  float* out = blockIdx.y ? p.db : p.dw;
  if (out == nullptr) return;
  float a = 0.f;
  if (c < p.C) {
    const float* src = p.ws + (int64_t)blockIdx.y * p.C + c;
#pragma unroll 4
    for (int b = g; b < p.blocks; b += 8) a += src[(int64_t)b * 2 * p.C];
  }
  s[g][cl] = a;
  __syncthreads();
  if (g == 0 && c < p.C) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += s[k][cl];
    out[c] = t;
  }
}

template <int TYPE, int V, int LPR, int NV>
void go(const LayerNormParams& p, bool bwd, hipStream_t st) {
  constexpr int NT = threads<LPR>(), RPB = NT / LPR;
  if (bwd) {
    ln_bwd_kernel<TYPE, V, LPR, NV><<<p.blocks, NT, 0, st>>>(p);
  } else {
    const int64_t n = (p.rows + RPB - 1) / RPB;
    ln_fwd_kernel<TYPE, V, LPR, NV><<<(unsigned)std::min<int64_t>(n, 4096), NT, 0, st>>>(p);
  }
}

// lanes per row by the row's vectors: the smallest group that holds it
template <int TYPE, int V>
int pick(const LayerNormParams& p, bool bwd, hipStream_t st) {
  const int n = (p.C + V - 1) / V;
  if (n <= 4) go<TYPE, V, 4, 1>(p, bwd, st);
  else if (n <= 8) go<TYPE, V, 8, 1>(p, bwd, st);
  else if (n <= 16) go<TYPE, V, 16, 1>(p, bwd, st);
  else if (n <= 32) go<TYPE, V, 32, 1>(p, bwd, st);
  else if (n <= 64) go<TYPE, V, 64, 1>(p, bwd, st);
  else if (n <= 128) go<TYPE, V, 64, 2>(p, bwd, st);
  else if (n <= 256) go<TYPE, V, 64, 4>(p, bwd, st);
  else if constexpr (V == 1) {
    if (n <= 512) go<TYPE, V, 64, 8>(p, bwd, st);
    else if (n <= 2048) go<TYPE, V, 256, 8>(p, bwd, st);
    else if (n <= 8192) go<TYPE, V, 1024, 8>(p, bwd, st);
    else go<TYPE, V, 1024, 16>(p, bwd, st);
  } else {
    if (n <= 512) go<TYPE, V, 256, 2>(p, bwd, st);
    else if (n <= 1024) go<TYPE, V, 256, 4>(p, bwd, st);
    else go<TYPE, V, 1024, 16 / V>(p, bwd, st);
  }
  return hipGetLastError() == hipSuccess ? 0 : 3;
}

bool aligned(const void* p, int64_t stride, int C, int V, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % V == 0 && C % V == 0 && size * V == 16;
}

template <int TYPE>
int run(const LayerNormParams& p, bool bwd, hipStream_t st) {
  constexpr int V = Elem<TYPE>::V, size = sizeof(typename Elem<TYPE>::type);
  const bool vec = aligned(p.x, p.x_stride, p.C, V, size) && (!bwd || aligned(p.gy, p.gy_stride, p.C, V, size));
  return vec ? pick<TYPE, V>(p, bwd, st) : pick<TYPE, 1>(p, bwd, st);
}

int run_type(const LayerNormParams& p, bool bwd, hipStream_t st) {
  if (p.C < 1 || p.rows < 1 || p.C > LAYER_NORM_MAX_C) return 1;
  switch (p.type) {
    case 0: return run<0>(p, bwd, st);
    case 1: return run<1>(p, bwd, st);
    case 2: return run<2>(p, bwd, st);
    default: return 1;
  }
}

}  // namespace

int layer_norm_fwd(const LayerNormParams& p, hipStream_t st) { return run_type(p, false, st); }

// blocks of the backward pass = partial rows of dw / db
int layer_norm_bwd_blocks(int64_t rows, int C) {
  const int64_t per = C <= 64 ? 32 : 4;            // rows a block holds at a time, at least
  return (int)std::max<int64_t>(1, std::min<int64_t>(512, (rows + per - 1) / per));
}

int layer_norm_bwd(const LayerNormParams& p, hipStream_t st) {
  const int rc = run_type(p, true, st);
  if (rc || p.ws == nullptr) return rc;
  ln_bwd_join_kernel<<<dim3((p.C + 31) / 32, 2), 256, 0, st>>>(p);
  return hipGetLastError() == hipSuccess ? 0 : 3;
}
