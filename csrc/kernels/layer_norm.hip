// Layer norm over the last axis, forward and backward.
//   mu = mean(x)   r = 1 / sqrt(mean((x - mu)^2) + eps)   xh = (x - mu) r   y = xh w + b
//   g = dy w   dx = r (g - mean(g) - xh mean(g xh))   dw = sum_rows dy xh   db = sum_rows dy
// Memory bound: x (and dy) is read once, y (dx) written once. A row is held in registers by LPR lanes (a group of a
// wave, a wave, or a block), so the variance is the two-pass one - sums of squares of x - mu, exact where the mean is
// large - at no extra read. The backward pass computes mu and r again from the row it holds anyway instead of reading
// 8 saved bytes per row (a quarter of a 32-channel bf16 row).
// 16,384 x 4,096 fp16: forward 47 us = 5.7 TB/s, backward 95 + 5 us = 4.0 TB/s (a copy of 4 GB: 4.7; part of these
// tensors stays in the last-level cache); 262,144 x 32 bf16: 8.0 us and 13.6 + 3.8 us = 4.2 and 2.9 TB/s.
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

// V consecutive elements (V = 1, or a 16-byte vector), as they lie in memory
template <int TYPE, int V>
struct alignas(V * sizeof(typename Elem<TYPE>::type)) Vec {
  typename Elem<TYPE>::type e[V];
};

// the vectors of this lane's columns of a row; columns past C read as 0
template <int TYPE, int V, int NV>
CFL_DEVICE void load_row(const typename Elem<TYPE>::type* row, const int* col, int C, bool ok, Vec<TYPE, V>* v) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    Vec<TYPE, V> t = {};
    if (ok && col[k] < C) t = *reinterpret_cast<const Vec<TYPE, V>*>(row + col[k]);
    v[k] = t;
  }
}
template <int TYPE, int V>
CFL_DEVICE void store_v(typename Elem<TYPE>::type* p, const float* f) {
  Vec<TYPE, V> v;
#pragma unroll
  for (int j = 0; j < V; ++j) v.e[j] = Elem<TYPE>::put(f[j]);
  *reinterpret_cast<Vec<TYPE, V>*>(p) = v;
}

// a sum over the row's lanes of one wave (all of them where LPR <= 64)
template <int LPR>
CFL_DEVICE float lane_sum(float v) {
#pragma unroll
  for (int o = 1; o < (LPR < 64 ? LPR : 64); o <<= 1) v = xor_add(v, o);
  return v;
}

// sum / n by the reciprocal, corrected once: where the sum of equal values is exact, their mean is that value
CFL_DEVICE float mean_of(float sum, float n, float inv) {
  const float m = sum * inv;
  return fmaf(fmaf(-m, n, sum), inv, m);
}

// What the statistics need that is the same for every row: 1 / C and, for a row of several waves, the columns of this
// wave and of each.
template <int LPR>
struct RowShape {
  static constexpr int W = LPR > 64 ? LPR / 64 : 1;
  float inv, own, n;             // 1 / C; 1 / columns of this wave (0: none); those columns
  float part[W];                 // columns of each wave
};
template <int LPR, int NV, int V>
CFL_DEVICE RowShape<LPR> row_shape(int C) {
  RowShape<LPR> s;
  s.inv = 1.f / (float)C;
  s.own = s.inv;
  s.n = (float)C;
  if constexpr (LPR > 64) {
#pragma unroll
    for (int u = 0; u < LPR / 64; ++u) {
      int n = 0;
#pragma unroll
      for (int k = 0; k < NV; ++k) n += imax(0, imin(C - (k * LPR + 64 * u) * V, 64 * V));
      s.part[u] = (float)n;
      if (u == (int)(threadIdx.x % LPR) >> 6) {
        s.own = n > 0 ? 1.f / (float)n : 0.f;
        s.n = (float)n;
      }
    }
  }
  return s;
}

// x -> x less the mean of this wave's columns (0 in the columns past C); returns r, and in `d` what has to be added to
// the columns of vector k for x - mu. A row of several waves joins the waves' own means and sums of squares:
// M2 = sum M2_w + n_w (mu_w - mu)^2, with one exchange through LDS. `red` alternates between two buffers from row to row,
// so one barrier per exchange is enough: a buffer is written again only after a barrier that every wave reaches behind
// its reads.
template <int LPR, int NV, int V>
CFL_DEVICE float center(float (*x)[V], const int* col, int C, float eps, const RowShape<LPR>& sh, float2* red,
                        float* d) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) s += x[k][j];
  const float mw = mean_of(lane_sum<LPR>(s), sh.n, sh.own);
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const float mk = col[k] < C ? mw : 0.f;                // the columns past C hold 0 and stay 0
#pragma unroll
    for (int j = 0; j < V; ++j) {
      x[k][j] -= mk;
      q = fmaf(x[k][j], x[k][j], q);
    }
    d[k] = 0.f;
  }
  q = lane_sum<LPR>(q);
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    if ((threadIdx.x & 63) == 0) red[(threadIdx.x % LPR) >> 6] = make_float2(mw, q);
    __syncthreads();
    float2 w[W];
    float mu = 0.f;
#pragma unroll
    for (int u = 0; u < W; ++u) {
      w[u] = red[u];
      mu = fmaf(w[u].x, sh.part[u], mu);
    }
    mu = mean_of(mu, (float)C, sh.inv);
    q = 0.f;
#pragma unroll
    for (int u = 0; u < W; ++u) q += fmaf(sh.part[u] * (w[u].x - mu), w[u].x - mu, w[u].y);
#pragma unroll
    for (int k = 0; k < NV; ++k) d[k] = col[k] < C ? mw - mu : 0.f;
  }
  return rsqrtf(fmaf(q, sh.inv, eps));
}

// a lane's columns of a fp32 weight (`dflt` where there is none, or past C)
template <int NV, int V>
CFL_DEVICE void load_weight(const float* p, const int* col, int C, float dflt, float (*w)[V]) {
  const bool vec = V >= 4 && p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
#pragma unroll
    for (int j = 0; j < V; ++j) w[k][j] = dflt;
    if (p == nullptr || col[k] >= C) continue;
    if (vec) {
#pragma unroll
      for (int j = 0; j + 3 < V; j += 4) {
        const float4 t = *reinterpret_cast<const float4*>(p + col[k] + j);
        w[k][j] = t.x; w[k][j + 1] = t.y; w[k][j + 2] = t.z; w[k][j + 3] = t.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) w[k][j] = p[col[k] + j];
    }
  }
}

// rows go to row groups (LPR lanes) in turn; NV vectors of V elements a lane: vector k of lane q starts at column
// (k LPR + q) V. The next row's loads are under way while a row is worked on.
template <int TYPE, int V, int LPR, int NV, int NT>
__global__ __launch_bounds__(NT) void ln_fwd_kernel(const LayerNormParams p) {
  typedef typename Elem<TYPE>::type E;
  constexpr int RPB = NT / LPR;
  __shared__ float2 red[2][RPB][LPR > 64 ? LPR / 64 : 1];
  const int q = threadIdx.x % LPR, g = threadIdx.x / LPR;
  int col[NV];
  float w[NV][V], b[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    col[k] = (k * LPR + q) * V;
  }
  load_weight<NV, V>(p.w, col, p.C, 1.f, w);
  load_weight<NV, V>(p.b, col, p.C, 0.f, b);
  const RowShape<LPR> sh = row_shape<LPR, NV, V>(p.C);
  const E* xb = reinterpret_cast<const E*>(p.x);
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t r = (int64_t)blockIdx.x * RPB + g;
  Vec<TYPE, V> xn[NV];
  load_row<TYPE, V, NV>(xb + r * p.x_stride, col, p.C, r < p.rows, xn);
  for (int par = 0; r - g < p.rows; r += step, par ^= 1) {
    const bool ok = r < p.rows;
    float x[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) x[k][j] = Elem<TYPE>::get(xn[k].e[j]);
    load_row<TYPE, V, NV>(xb + (r + step) * p.x_stride, col, p.C, r + step < p.rows, xn);
    float d[NV];
    const float rs = center<LPR, NV, V>(x, col, p.C, p.eps, sh, red[par][g], d);
    E* yr = reinterpret_cast<E*>(p.y) + r * p.C;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[k][j] = fmaf(fmaf(x[k][j], rs, d[k] * rs), w[k][j], b[k][j]);
      if (ok && col[k] < p.C) store_v<TYPE, V>(yr + col[k], x[k]);
    }
  }
}

template <int TYPE, int V, int LPR, int NV, int NT>
__global__ __launch_bounds__(NT) void ln_bwd_kernel(const LayerNormParams p) {
  typedef typename Elem<TYPE>::type E;
  constexpr int RPB = NT / LPR;
  __shared__ float2 red[2][RPB][LPR > 64 ? LPR / 64 : 1], red2[2][RPB][LPR > 64 ? LPR / 64 : 1];
  const int q = threadIdx.x % LPR, gr = threadIdx.x / LPR;
  int col[NV];
  float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    col[k] = (k * LPR + q) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) dw[k][j] = db[k][j] = 0.f;
  }
  load_weight<NV, V>(p.w, col, p.C, 1.f, w);
  const RowShape<LPR> sh = row_shape<LPR, NV, V>(p.C);
  const E *xb = reinterpret_cast<const E*>(p.x), *gb = reinterpret_cast<const E*>(p.gy);
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t r = (int64_t)blockIdx.x * RPB + gr;
  Vec<TYPE, V> xn[NV], gn[NV];
  load_row<TYPE, V, NV>(xb + r * p.x_stride, col, p.C, r < p.rows, xn);
  load_row<TYPE, V, NV>(gb + r * p.gy_stride, col, p.C, r < p.rows, gn);
  for (int par = 0; r - gr < p.rows; r += step, par ^= 1) {
    const bool ok = r < p.rows;
    float x[NV][V], g[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[k][j] = Elem<TYPE>::get(xn[k].e[j]);
        g[k][j] = Elem<TYPE>::get(gn[k].e[j]);
      }
    load_row<TYPE, V, NV>(xb + (r + step) * p.x_stride, col, p.C, r + step < p.rows, xn);
    load_row<TYPE, V, NV>(gb + (r + step) * p.gy_stride, col, p.C, r + step < p.rows, gn);
    float d[NV];
    float rs = center<LPR, NV, V>(x, col, p.C, p.eps, sh, red[par][gr], d);
    rs = ok ? rs : 0.f;                                    // no row: 1 / sqrt(eps) may be infinite, and 0 times it NaN
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[k][j] = fmaf(x[k][j], rs, d[k] * rs);
        dw[k][j] = fmaf(g[k][j], x[k][j], dw[k][j]);
        db[k][j] += g[k][j];
        g[k][j] *= w[k][j];
        s0 += g[k][j];
        s1 = fmaf(g[k][j], x[k][j], s1);
      }
    if (p.y == nullptr) continue;
    s0 = lane_sum<LPR>(s0);
    s1 = lane_sum<LPR>(s1);
    if constexpr (LPR > 64) {
      if ((threadIdx.x & 63) == 0) red2[par][gr][q >> 6] = make_float2(s0, s1);
      __syncthreads();
      s0 = s1 = 0.f;
#pragma unroll
      for (int u = 0; u < LPR / 64; ++u) {
        s0 += red2[par][gr][u].x;
        s1 += red2[par][gr][u].y;
      }
    }
    // the mean taken from dy w before anything is scaled: a row of one column gives 0 and not the rounding of a product
    // (equal values in several columns leave the rounding of their sum and of 1 / C)
    const float m0 = s0 * sh.inv, m1 = s1 * sh.inv;
    E* yr = reinterpret_cast<E*>(p.y) + r * p.C;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[k][j] = rs * fmaf(x[k][j], -m1, g[k][j] - m0);
      if (ok && col[k] < p.C) store_v<TYPE, V>(yr + col[k], x[k]);
    }
  }
  if (p.dw == nullptr && p.db == nullptr) return;
  // join the row groups that own the same columns: lanes of a wave, then the block's waves, one element of every lane at
  // a time through LDS. J waves hold a wave-wide set of columns each.
  constexpr int J = LPR > 64 ? RPB : NT / 64, G = LPR < 64 ? LPR : 64;
  __shared__ float2 part[J > 1 ? NT / 64 * G : 1];
  // one block: its sums are the result
  float* odw = gridDim.x == 1 ? p.dw : p.ws + (int64_t)blockIdx.x * 2 * p.C;
  float* odb = gridDim.x == 1 ? p.db : p.ws + (int64_t)blockIdx.x * 2 * p.C + p.C;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float2 t = make_float2(dw[k][j], db[k][j]);
#pragma unroll
      for (int o = G; o < 64; o <<= 1) {
        t.x = xor_add(t.x, o);
        t.y = xor_add(t.y, o);
      }
      if constexpr (J > 1) {
        constexpr int SETS = LPR > 64 ? LPR / 64 : 1;      // waves of one row
        const int wv = threadIdx.x >> 6, l = threadIdx.x & 63;
        if (k + j > 0) __syncthreads();
        if (l < G) part[wv * G + l] = t;
        __syncthreads();
        if (wv < SETS && l < G) {
          t = make_float2(0.f, 0.f);
#pragma unroll
          for (int u = 0; u < J; ++u) {
            const float2 v = part[(u * SETS + wv) * G + l];
            t.x += v.x;
            t.y += v.y;
          }
        }
      }
      if (threadIdx.x < LPR && col[k] < p.C) {
        if (odw) odw[col[k] + j] = t.x;
        if (odb) odb[col[k] + j] = t.y;
      }
    }
}

// dw / db = sums of the partial rows: a block owns 32 columns of one of the two, 32 threads a column
__global__ __launch_bounds__(1024) void ln_bwd_join_kernel(const LayerNormParams p) {
  __shared__ float s[32][33];
  const int cl = threadIdx.x & 31, g = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
  float* out = blockIdx.y ? p.db : p.dw;
  if (out == nullptr) return;
  float a = 0.f;
  if (c < p.C) {
    const float* src = p.ws + (int64_t)blockIdx.y * p.C + c;
#pragma unroll 8
    for (int b = g; b < p.blocks; b += 32) a += src[(int64_t)b * 2 * p.C];
  }
  s[g][cl] = a;
  __syncthreads();
  if (g == 0 && c < p.C) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += s[k][cl];
    out[c] = t;
  }
}

// Backward: 512 threads (256 registers each: 16 elements of x, dy, w, dw, db and the next row's vectors) and up to 512
// blocks. Fewer blocks leave memory idle, more cost partial rows of dw and db: 16,384 x 4,096 fp16 121 / 106 / 111 us
// and 32,768 x 1,024 bf16 48 / 41 / 45 us for 256 / 512 / 1,024 blocks; 1,024 threads 114 and 48 us for 512 blocks.
// Forward: 256 threads; more than 2,048 blocks load w and b too often (32,768 x 1,024: 65 us for 8,192, 22 for 2,048).
constexpr int bwd_threads = 512;

template <int TYPE, int V, int LPR, int NV>
int go(const LayerNormParams& p, bool bwd, bool count, hipStream_t st) {
  constexpr int NT = bwd_threads, RPB = NT / LPR, NTF = LPR > 256 ? LPR : 256, RPBF = NTF / LPR;
  static_assert(LPR <= NT, "a row fits the block");
  // up to four rows a row group: one block, whose sums need no join
  if (count) return p.rows <= 4 * RPB ? 1 : (int)std::min<int64_t>(512, (p.rows + RPB - 1) / RPB);
  if (bwd)
    ln_bwd_kernel<TYPE, V, LPR, NV, NT><<<p.blocks, NT, 0, st>>>(p);
  else
    ln_fwd_kernel<TYPE, V, LPR, NV, NTF>
        <<<(unsigned)std::min<int64_t>(2048, (p.rows + RPBF - 1) / RPBF), NTF, 0, st>>>(p);
  return hipGetLastError() == hipSuccess ? 0 : 3;
}

// lanes per row by the row's vectors: the smallest group that holds it
template <int TYPE, int V>
int pick(const LayerNormParams& p, bool bwd, bool count, hipStream_t st) {
  const int n = (p.C + V - 1) / V;
  if (n <= 4) return go<TYPE, V, 4, 1>(p, bwd, count, st);
  if (n <= 8) return go<TYPE, V, 8, 1>(p, bwd, count, st);
  if (n <= 16) return go<TYPE, V, 16, 1>(p, bwd, count, st);
  if (n <= 32) return go<TYPE, V, 32, 1>(p, bwd, count, st);
  if (n <= 64) return go<TYPE, V, 64, 1>(p, bwd, count, st);
  if constexpr (V == 8) {
    if (n <= 128) return go<TYPE, V, 128, 1>(p, bwd, count, st);
    if (n <= 256) return go<TYPE, V, 256, 1>(p, bwd, count, st);
    if (n <= 512) return go<TYPE, V, 512, 1>(p, bwd, count, st);
    return go<TYPE, V, 512, 2>(p, bwd, count, st);
  } else if constexpr (V == 4) {
    if (n <= 128) return go<TYPE, V, 64, 2>(p, bwd, count, st);
    if (n <= 256) return go<TYPE, V, 128, 2>(p, bwd, count, st);
    if (n <= 512) return go<TYPE, V, 256, 2>(p, bwd, count, st);
    if (n <= 1024) return go<TYPE, V, 512, 2>(p, bwd, count, st);
    return go<TYPE, V, 512, 4>(p, bwd, count, st);
  } else {
    if (n <= 128) return go<TYPE, V, 64, 2>(p, bwd, count, st);
    if (n <= 256) return go<TYPE, V, 64, 4>(p, bwd, count, st);
    if (n <= 512) return go<TYPE, V, 64, 8>(p, bwd, count, st);
    if (n <= 1024) return go<TYPE, V, 128, 8>(p, bwd, count, st);
    if (n <= 2048) return go<TYPE, V, 256, 8>(p, bwd, count, st);
    if (n <= 4096) return go<TYPE, V, 512, 8>(p, bwd, count, st);
    return go<TYPE, V, 512, 16>(p, bwd, count, st);
  }
}

bool aligned(const void* p, int64_t stride, int C, int V, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % V == 0 && C % V == 0 && size * V == 16;
}

template <int TYPE>
int run(const LayerNormParams& p, bool bwd, bool count, hipStream_t st) {
  constexpr int V = Elem<TYPE>::V, size = sizeof(typename Elem<TYPE>::type);
  const bool vec = aligned(p.x, p.x_stride, p.C, V, size) && (!bwd || aligned(p.gy, p.gy_stride, p.C, V, size));
  return vec ? pick<TYPE, V>(p, bwd, count, st) : pick<TYPE, 1>(p, bwd, count, st);
}

int run_type(const LayerNormParams& p, bool bwd, bool count, hipStream_t st) {
  switch (p.type) {
    case 0: return run<0>(p, bwd, count, st);
    case 1: return run<1>(p, bwd, count, st);
    default: return run<2>(p, bwd, count, st);
  }
}

bool valid(const LayerNormParams& p) {
  return p.C >= 1 && p.C <= LAYER_NORM_MAX_C && p.rows >= 1 && p.type >= 0 && p.type <= 2;
}

}  // namespace

int layer_norm_fwd(const LayerNormParams& p, hipStream_t st) { return valid(p) ? run_type(p, false, false, st) : 1; }

// blocks of the backward pass = partial rows of dw / db
int layer_norm_bwd_blocks(const LayerNormParams& p) { return valid(p) ? run_type(p, true, true, nullptr) : 0; }

int layer_norm_bwd(const LayerNormParams& p, hipStream_t st) {
  if (!valid(p) || p.blocks < 1) return 1;
  const int rc = run_type(p, true, false, st);
  if (rc || p.blocks == 1 || (p.dw == nullptr && p.db == nullptr)) return rc;
  ln_bwd_join_kernel<<<dim3((p.C + 31) / 32, 2), 1024, 0, st>>>(p);
  return hipGetLastError() == hipSuccess ? 0 : 3;
}
