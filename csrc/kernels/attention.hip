// Attention, forward:  o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j - lse_i) over the keys j that row i may attend.
//
// One pass over the keys with the running maximum and sum of the softmax. S^T = K Q^T is computed instead of Q K^T, so a
// lane holds 16 keys of ONE row (attention.h): the row's maximum and sum are sums within the lane plus one exchange with
// the lane 32 away, the rescaling factor is the lane's own scalar, and exp(S^T) rounded to 16 bits is the B operand of
// O^T = V^T P^T as it stands. K and V tiles go from memory to LDS by LDS-DMA loads, one tile ahead.
//
// Rounding: scores, maximum, sum and output accumulate in fp32. P enters the second product in two parts of the inputs'
// type (attn_fine), the output is rounded once.
// Split. Four waves own 32 rows each and share the tiles (64 keys); up to 32 rows in all, the waves split a tile's keys
// instead and join through LDS. Few row blocks: blocks share a walk (attn_splits) and a second launch joins the parts.
// 256 registers, two waves a SIMD or more: at 512 the compiler puts the first product's result into accumulation
// registers and copies every score (16 heads x 4,096 tokens x 128 channels, weights in one part: 479 us against 294).
// Bound. Up to 64 channels by the vector unit (80 % busy, the matrix cores 52 %), at 128 channels by the matrix cores
// (58 %) and it (49 %); no LDS bank conflicts. 2 images x 16 heads x 4,096 tokens of 128 channels 376 us = 1,097 TFLOP/s
// over the three products that two-part weights make of two; 4 images, 64 channels 420 us = 982 (a library product of
// 8,192^3 reaches 1,213). One query of 64 (image, head)s over 4,096 keys of 32 channels: 9.0 us + 2.5 us to join = 2.9 TB/s.
// Rows that may attend nothing are those without a maximum: 0, and their saved lse2 is +inf (exp2(s - inf) = 0 in the
// backward pass).
#include <algorithm>
#include <cfloat>

#include "attention.h"

namespace {

using namespace attn;

// row maxima may lag the running maximum by 2^SLACK: P then reaches 2^SLACK (times 2^UP: in both types' range, the
// relative precision is the same) and most tiles rescale nothing
constexpr float SLACK = 8.f;

// up to this many rows the four waves of a block split the keys of a tile, beyond it the rows
constexpr int FEW_ROWS = 32;

// whether the mask bits of a tile's KW keys allow one of the first `left`
template <int KW>
CFL_DEVICE bool attended(unsigned long long bits, int left) {
  const unsigned long long m = left >= 64 ? ~0ull : (1ull << imax(left, 0)) - 1;
  return (bits & m & (KW == 64 ? ~0ull : (1ull << (KW & 63)) - 1)) != 0;
}

// QT: 32-row tiles per wave; WR x WK: waves along the rows and along the keys of a tile; KW keys per wave and tile
template <class T, int DP, int QT, int WR, int WK, int KW, int MINW, int KIND, bool FINE>
__global__ __launch_bounds__(64 * WR * WK, MINW) void attn_fwd_kernel(const AttnParams p) {
  constexpr int NT = 64 * WR * WK, KT = KW * WK, TILE = KT * DP, CPR = DP / 8, CH = KT * CPR / NT;
  constexpr int NK = KW / 32, NKK = DP / 16, ND = DP / 32;
  constexpr bool MASK = KIND == ATTN_MASK;
  const bool causal = KIND == ATTN_CAUSAL || (MASK && p.causal);
  static_assert(KT * CPR % NT == 0, "whole DMA instructions");
  __shared__ __attribute__((aligned(1024))) bf16_t smem[4 * TILE];

  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5, wr = wid / WK, wk = wid % WK;
  constexpr int BR = 32 * QT * WR;
  const int nrb = (p.M + BR - 1) / BR, bhn = p.B * p.Hkv;
  int rb0, bh, sp;
  locate(p, nrb, bhn, p.splits, rb0, bh, sp);
  const int rb = causal ? nrb - 1 - rb0 : rb0;          // causal: long rows first
  const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const int len = p.lengths ? imin(imax(p.lengths[b], 0), p.Sk) : p.Sk;
  const int off = causal ? p.Sk - p.Sq : 0;
  const int r_end = imin(rb * BR + BR, p.M);

  // this lane's rows: their queries as B operands, and the first key each may not attend
  s8v qf[QT][NKK];
  int lim[QT], ri[QT], rg[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = rb * BR + (wr * QT + t) * 32 + c;
    const bool ok = r < p.M;
    const int rr = ok ? r : p.M - 1, i = fdiv(rr, p.div_g), g = rr - i * p.G;
    ri[t] = i;
    rg[t] = g;
    lim[t] = !ok ? 0 : causal ? imin(imax(i + off + 1, 0), len) : len;
    const bf16_t* q = reinterpret_cast<const bf16_t*>(p.q.p) + b * p.q.sb + i * p.q.ss + (hk * p.G + g) * p.q.sh;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      const int d = 16 * kk + 8 * h;
      u4v w = {0, 0, 0, 0};
      if (ok && d < p.D) w = *reinterpret_cast<const u4v*>(q + d);
      qf[t][kk] = __builtin_bit_cast(s8v, w);
    }
  }
  // first key past every row of the block / of this wave (rows are in query order)
  const int i_last = fdiv(r_end - 1, p.div_g);
  const int kend = causal ? imin(imax(i_last + off + 1, 0), len) : len;
  const int wr0 = rb * BR + wr * QT * 32;
  const int wi0 = fdiv(imin(wr0, p.M - 1), p.div_g), wi1 = fdiv(imin(wr0 + QT * 32, p.M) - 1, p.div_g);
  const int wlast = wr0 >= p.M ? 0 : causal ? imin(imax(wi1 + off + 1, 0), len) : len;
  const int wfull = causal ? imin(imax(wi0 + off + 1, 0), len) : len;   // keys below it: allowed for every row

  const int tiles = (p.Sk + KT - 1) / KT, tps = (tiles + p.splits - 1) / p.splits;
  const int t0 = sp * tps, t1 = imin(imin(t0 + tps, tiles), (kend + KT - 1) / KT);

  // the block's part of a tile: CH 16-byte chunks per thread and tensor, the swizzle in the source address
  uint32_t vk[CH], vv[CH];
  int vrow[CH];
#pragma unroll
  for (int n = 0; n < CH; ++n) {
    const int id = tid + NT * n, row = id / CPR, d = ((id % CPR) ^ swz<DP>(row)) * 8;
    vrow[n] = d < p.D ? row : 0x7fffffff;
    vk[n] = (uint32_t)(row * (int)p.k.ss + d) * 2;
    vv[n] = (uint32_t)(row * (int)p.v.ss + d) * 2;
  }
  const bf16_t* kb = reinterpret_cast<const bf16_t*>(p.k.p) + b * p.k.sb + hk * p.k.sh;
  const bf16_t* vb = reinterpret_cast<const bf16_t*>(p.v.p) + b * p.v.sb + hk * p.v.sh;
  auto issue = [&](int t, int buf) {
    const int rem = len - t * KT;
    const u4v rk = rsrc(kb + (int64_t)t * KT * p.k.ss), rv = rsrc(vb + (int64_t)t * KT * p.v.ss);
    const bf16_t* dst = smem + buf * 2 * TILE + wid * 512;
#pragma unroll
    for (int n = 0; n < CH; ++n) {
      dma16(rk, vrow[n] < rem ? vk[n] : CFL_OOB, dst + NT * 8 * n);
      dma16(rv, vrow[n] < rem ? vv[n] : CFL_OOB, dst + TILE + NT * 8 * n);
    }
  };

  // boolean mask: this lane's rows' words
  const unsigned long long* mrow[QT];
  unsigned long long word[QT];
  if (MASK) {
#pragma unroll
    for (int t = 0; t < QT; ++t)
      mrow[t] = p.mask.bits + (b * p.mask.sb + (hk * p.G + rg[t]) * p.mask.sh + (p.mask.rows > 1 ? ri[t] : 0)) *
                                  (int64_t)p.mask.words;
  }
  __shared__ uint8_t classes[MASK ? MASK_TILES + 64 : 1];
  TileMask tm;
  if (MASK)
    tm.fill(p, b, hk, classes, tiles, [&](int t, int& i0, int& i1, int& w0, int& w1) {
      i0 = fdiv(rb * BR, p.div_g);
      i1 = i_last;
      w0 = t * KT / 64;
      w1 = imin((t * KT + KT - 1) / 64, p.mask.words - 1);
    });
  auto next = [&](int t) { return MASK ? tm.next(t, t1) : t; };
  auto words = [&](int t) {
    const int w = imin((t * KT + wk * KW) >> 6, p.mask.words - 1);
#pragma unroll
    for (int u = 0; u < QT; ++u) word[u] = mrow[u][w];
  };

  f16v acc[ND][QT];
  float m[QT], l[QT];
  const float sc = p.scale * LOG2E;
  const int fo = lds_at<DP>(c, h);
  const TransAt<DP> ta(lane);
  auto walk = [&](auto safe) {
    constexpr bool SAFE = decltype(safe)::value;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      m[t] = -INFINITY;
      l[t] = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][t][e] = 0.f;
    }

    int t = next(t0);
    if (t < t1) {
      if (MASK) words(t);
      issue(t, 0);
    }
    wait_vm();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // the tile in buffer B. Taking turns with a constant buffer leaves all LDS offsets to the instructions.
    auto step = [&](auto B) {
      const int buf = B;
      const bool part = MASK && tm.part;
      const int tn = next(t + 1);
      unsigned long long cur[QT];
      const int key0 = t * KT + wk * KW;
      if (MASK) {
#pragma unroll
        for (int u = 0; u < QT; ++u) cur[u] = word[u] >> (key0 & 32);
        if (tn < t1) words(tn);
      }
      if (tn < t1) issue(tn, buf ^ 1);

      if (key0 < wlast) {
        const bf16_t* sk = smem + buf * 2 * TILE + wk * KW * DP;
        const bf16_t* sv = sk + TILE;
        // a wave in its products goes first, those in their softmax fill in (2 % here, nothing in the backward kernels)
        __builtin_amdgcn_s_setprio(1);
        f16v s[NK][QT];
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
          for (int u = 0; u < QT; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[k][u][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk)
#pragma unroll
          for (int k = 0; k < NK; ++k) {
            const s8v a = frag_x<DP>(sk + 32 * k * DP, fo, kk);
#pragma unroll
            for (int u = 0; u < QT; ++u) s[k][u] = T::mma(a, qf[u][kk], s[k][u]);
          }
        if (MASK && part) {
#pragma unroll
          for (int u = 0; u < QT; ++u)
#pragma unroll
            for (int k = 0; k < NK; ++k) {
              const uint32_t w = (uint32_t)(cur[u] >> (32 * k)) >> (4 * h);
#pragma unroll
              for (int e = 0; e < 16; ++e)
                s[k][u][e] = (w >> ((e & 3) + 8 * (e >> 2))) & 1 ? s[k][u][e] : -INFINITY;
            }
        }
        if (key0 + KW > wfull) {
#pragma unroll
          for (int u = 0; u < QT; ++u)
#pragma unroll
            for (int k = 0; k < NK; ++k) {
              const int left = lim[u] - key0 - 32 * k - 4 * h;
#pragma unroll
              for (int e = 0; e < 16; ++e) s[k][u][e] = (e & 3) + 8 * (e >> 2) < left ? s[k][u][e] : -INFINITY;
            }
        }
        __builtin_amdgcn_s_setprio(0);
        Packed<T, FINE> pb[QT][2 * NK];
        uint32_t seen[QT][NK];
#pragma unroll
        for (int u = 0; u < QT; ++u) {
          float mx = s[0][u][0];
#pragma unroll
          for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[k][u][e]);
          mx = max_halves(mx) * sc;
          // a row with a key that it may attend has a maximum, if all of its scores are -inf or NaN: its sum is then not
          // that of an empty row
          const int left = lim[u] - key0;
          const bool some = KIND == ATTN_PLAIN || (MASK && part ? attended<KW>(cur[u], left) : left > 0);
          mx = fmaxf(mx, some ? -FLT_MAX : -INFINITY);
          if (__any(mx > m[u] + SLACK)) {
            // only the rows that need it: what a row rounds does not depend on the rows next to it
            const bool up = mx > m[u] + SLACK;
            const float al = up ? exp2_(m[u] - mx) : 1.f;
            m[u] = up ? mx : m[u];
            l[u] *= al;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
              for (int e = 0; e < 16; ++e) acc[d][u][e] *= al;
          }
          const float ms = (m[u] == -INFINITY ? 0.f : m[u]) - T::UP;
          float sum = 0.f;
#pragma unroll
          for (int k = 0; k < NK; ++k) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              s[k][u][e] = exp2_(fmaf(s[k][u][e], sc, -ms));
              sum += s[k][u][e];
            }
            if constexpr (SAFE) seen[u][k] = weighed(s[k][u]);
            pb[u][2 * k].set(s[k][u], 0);
            pb[u][2 * k + 1].set(s[k][u], 1);
          }
          l[u] += sum;
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ks = 0; ks < 2 * NK; ++ks)
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            s8v a = frag_t<DP>(sv + 16 * ks * DP, ta, d);
            if constexpr (SAFE) {
              s8v pos, neg;
              __builtin_amdgcn_sched_barrier(0);           // few registers matter here, not speed
              a = clean<T>(a, pos, neg);
#pragma unroll
              for (int u = 0; u < QT; ++u) poison<T>(acc[d][u], pos, neg, seen[u][ks >> 1] >> 8 * (ks & 1));
            }
#pragma unroll
            for (int u = 0; u < QT; ++u) acc[d][u] = pb[u][ks].mma(a, acc[d][u]);
          }
      }
      __builtin_amdgcn_s_setprio(0);
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      t = tn;
    };
    while (t < t1) {
      step(std::integral_constant<int, 0>{});
      if (t >= t1) break;
      step(std::integral_constant<int, 1>{});
    }

  };
  walk(std::false_type{});
  if constexpr (KIND != ATTN_PLAIN) {
    float z = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int u = 0; u < QT; ++u) z += finite_sum(acc[d][u]);
    if (__syncthreads_or(z != 0.f)) walk(std::true_type{});
  }

#pragma unroll
  for (int u = 0; u < QT; ++u) l[u] += other_half(l[u]);

  if constexpr (WK > 1) {
    // join the waves that share rows: the first one collects the others' (m, l) and accumulators through LDS
    static_assert(QT == 1 && WR == 1, "key-split waves hold one row tile");
    constexpr int SEG = ND * 1024 + 64;                     // floats per wave
    static_assert((WK - 1) * SEG * 4 <= (int)sizeof(smem), "LDS of the join");
    float* sf = reinterpret_cast<float*>(smem);
    if (wk > 0) {
      float* mine = sf + (wk - 1) * SEG;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) mine[(d * 16 + e) * 64 + lane] = acc[d][0][e];
      if (h == 0) {
        mine[ND * 1024 + 2 * c] = m[0];
        mine[ND * 1024 + 2 * c + 1] = l[0];
      }
    }
    __syncthreads();
    if (wk > 0) return;
    float mn = m[0], f[WK];
#pragma unroll
    for (int w = 1; w < WK; ++w) mn = fmaxf(mn, sf[(w - 1) * SEG + ND * 1024 + 2 * c]);
    const float ms = mn == -INFINITY ? 0.f : mn;
    f[0] = exp2_(m[0] - ms);
    l[0] *= f[0];
#pragma unroll
    for (int w = 1; w < WK; ++w) {
      f[w] = exp2_(sf[(w - 1) * SEG + ND * 1024 + 2 * c] - ms);
      l[0] = fmaf(sf[(w - 1) * SEG + ND * 1024 + 2 * c + 1], f[w], l[0]);
    }
    m[0] = mn;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float x = acc[d][0][e] * f[0];
#pragma unroll
        for (int w = 1; w < WK; ++w) x = fmaf(sf[(w - 1) * SEG + (d * 16 + e) * 64 + lane], f[w], x);
        acc[d][0][e] = x;
      }
  }

#pragma unroll
  for (int u = 0; u < QT; ++u) {
    const int r = rb * BR + (wr * QT + u) * 32 + c;
    const bool ok = r < p.M;
    const int64_t row = (int64_t)bh * p.M + r;
    if (p.splits > 1) {
      const int64_t part = (int64_t)sp * bhn * p.M + row;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        store_part<DP>(p.ws_o + part * DP, acc[d][u], 1.f, d, h, ok);
      }
      if (ok && h == 0) {
        p.ws_ml[part * 2] = m[u];
        p.ws_ml[part * 2 + 1] = l[u];
      }
      continue;
    }
    const bool none = m[u] == -INFINITY;                   // l may be 0 elsewhere too: every score -inf, 0 / 0
    const float inv = none ? 0.f : 1.f / l[u];
    const int64_t at = b * p.o.sb + ri[u] * p.o.ss + (hk * p.G + rg[u]) * p.o.sh;
    bf16_t *o = reinterpret_cast<bf16_t*>(p.o.p) + at, *rest = p.o_rest ? p.o_rest + at : nullptr;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      store_row<T>(o, acc[d][u], inv, d, p.D, h, ok, rest);
    }
    if (ok && h == 0 && p.lse2)
      p.lse2[row] = none ? INFINITY : m[u] + __builtin_amdgcn_logf(l[u]) - (T::UP + T::P_UP);
  }
}

// joins the key splits of a row: one thread per 4 channels
template <class T, int DP>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnParams p) {
  constexpr int TPR = DP / 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)p.B * p.Hkv * p.M;
  const int64_t row = id / TPR;
  const int d = (int)(id % TPR) * 4;
  if (row >= rows) return;
  // parts in order, eight at a time so that their loads are under way together
  float mn = -INFINITY, l = 0.f, a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
  for (int s0 = 0; s0 < p.splits; s0 += 8) {
    float2 ml[8];
    float4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t at = imin(s0 + j, p.splits - 1) * rows + row;
      ml[j] = *reinterpret_cast<const float2*>(p.ws_ml + at * 2);
      v[j] = *reinterpret_cast<const float4*>(p.ws_o + at * DP + d);
    }
    float top = mn;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, s0 + j < p.splits ? ml[j].x : -INFINITY);
    const float ms = top == -INFINITY ? 0.f : top, f0 = exp2_(mn - ms);
    mn = top;
    l *= f0; a0 *= f0; a1 *= f0; a2 *= f0; a3 *= f0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (s0 + j < p.splits) {
        const float f = exp2_(ml[j].x - ms);
        l = fmaf(ml[j].y, f, l);
        a0 = fmaf(v[j].x, f, a0);
        a1 = fmaf(v[j].y, f, a1);
        a2 = fmaf(v[j].z, f, a2);
        a3 = fmaf(v[j].w, f, a3);
      }
  }
  const int bh = (int)(row / p.M), r = (int)(row - (int64_t)bh * p.M), b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const int i = fdiv(r, p.div_g), g = r - i * p.G;
  const bool none = mn == -INFINITY;
  const float inv = none ? 0.f : 1.f / l;
  if (d < p.D) {
    const int64_t at = b * p.o.sb + i * p.o.ss + (hk * p.G + g) * p.o.sh + d;
    a0 *= inv; a1 *= inv; a2 *= inv; a3 *= inv;
    const uint2 w = make_uint2(T::pack2(a0, a1), T::pack2(a2, a3));
    *reinterpret_cast<uint2*>(reinterpret_cast<bf16_t*>(p.o.p) + at) = w;
    if (p.o_rest)
      *reinterpret_cast<uint2*>(p.o_rest + at) =
          make_uint2(T::pack2((a0 - T::lo(w.x)) * T::REST, (a1 - T::hi(w.x)) * T::REST),
                     T::pack2((a2 - T::lo(w.y)) * T::REST, (a3 - T::hi(w.y)) * T::REST));
  }
  if (d == 0 && p.lse2) p.lse2[row] = none ? INFINITY : mn + __builtin_amdgcn_logf(l) - (T::UP + T::P_UP);
}

// mask bytes -> words: one wave per (32 mask rows, 64 keys), all of its loads under way together
__global__ __launch_bounds__(256) void attn_mask_kernel(const AttnMaskArgs a) {
  const int nib = (a.Im + 31) >> 5, lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), per = (int64_t)nib * a.words;
  if (unit >= per * a.Bm * a.Hm) return;
  const int64_t lead = unit / per;
  const int ib = (int)((unit - lead * per) / a.words), w = (int)(unit % a.words);
  const int b = (int)(lead / a.Hm), h = (int)(lead % a.Hm), key = 64 * w + lane;
  const uint8_t* src = a.src + b * a.sb + h * a.sh + (int64_t)imin(key, a.Sk - 1) * a.sk;
  const int n = imin(32, a.Im - 32 * ib);
  uint8_t v[32];
#pragma unroll
  for (int k = 0; k < 32; ++k) v[k] = src[(int64_t)(32 * ib + imin(k, n - 1)) * a.si];
  unsigned long long any = 0, all = ~0ull, mine = 0;
#pragma unroll
  for (int k = 0; k < 32; ++k) {
    const unsigned long long bits = __ballot(key < a.Sk && v[k] != 0);   // rows past the last repeat it
    any |= bits;
    all &= bits;
    mine = lane == k ? bits : mine;
  }
  if (lane < n) a.bits[(lead * a.Im + 32 * ib + lane) * a.words + w] = mine;
  if (lane == 0) a.cls[unit] = any == 0 ? 0 : all == ~0ull ? 2 : 1;
}

template <class T, int DP, int QT, int WR, int WK, int KW, int MINW, bool FINE>
void launch(const AttnParams& p, hipStream_t st) {
  const int64_t n = (int64_t)((p.M + 32 * QT * WR - 1) / (32 * QT * WR)) * p.B * p.Hkv * p.splits;
  if (p.mask.bits)
    attn_fwd_kernel<T, DP, QT, WR, WK, KW, MINW, ATTN_MASK, FINE><<<(unsigned)n, 64 * WR * WK, 0, st>>>(p);
  else if (p.causal)
    attn_fwd_kernel<T, DP, QT, WR, WK, KW, MINW, ATTN_CAUSAL, FINE><<<(unsigned)n, 64 * WR * WK, 0, st>>>(p);
  else
    attn_fwd_kernel<T, DP, QT, WR, WK, KW, MINW, ATTN_PLAIN, FINE><<<(unsigned)n, 64 * WR * WK, 0, st>>>(p);
}

template <class T, int DP>
void fwd(const AttnParams& p, hipStream_t st) {
  if (p.M <= FEW_ROWS) launch<T, DP, 1, 1, 4, 32, 1, true>(p, st);       // bound by memory
  else if (attn_fine()) launch<T, DP, 1, 4, 1, 64, 2, true>(p, st);
  else launch<T, DP, 1, 4, 1, 64, 2, false>(p, st);
  if (p.splits > 1) {
    const int64_t n = (int64_t)p.B * p.Hkv * p.M * (DP / 4);
    attn_join_kernel<T, DP><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(p);
  }
}

template <class T>
void fwd_d(const AttnParams& p, hipStream_t st) {
  if (p.D <= 32) fwd<T, 32>(p, st);
  else if (p.D <= 64) fwd<T, 64>(p, st);
  else if (p.D <= 96) fwd<T, 96>(p, st);
  else fwd<T, 128>(p, st);
}

}  // namespace

int attn_mask_bits(const AttnMaskArgs& a, hipStream_t st) {
  const int64_t units = (int64_t)a.Bm * a.Hm * ((a.Im + 31) / 32) * a.words;
  if (units == 0) return 0;
  if ((units + 3) / 4 > ATTN_MAX_BLOCKS) return 2;
  attn_mask_kernel<<<(unsigned)((units + 3) / 4), 256, 0, st>>>(a);
  return hipGetLastError() == hipSuccess ? 0 : 3;
}

// P and dS are operands of 16 bits in the second products. Rounded to one part they cost as much as the rounding of the
// results does: the errors of dq, dk, dv and the output are 1.37 to 1.48 times those of rounding nothing but the results.
// With what that rounding took away as a second operand (attention.h Packed) they are 1.00 to 1.02, at any size of call,
// so two parts are the rule and one part is the tuning key's. The price is a second set of second products (us, one
// part -> two, forward and backward): 16 images x 8 heads x 1,024 tokens of 64 channels 48 -> 63 and 144 -> 189, 2 x 16
// heads x 4,096 tokens of 128 channels 278 -> 372 and 874 -> 1,128.
bool attn_fine() { return cfl_tune(TUNE_ATTN_FINE) != 1; }

// Blocks that share the keys of a row block: enough for two blocks a CU where there are few row blocks, at least four
// tiles each. (Blocks of 64 rows with two waves along the keys instead, for such grids, were slower: 4 images x 8 heads
// x 1,600 tokens of 64 channels 43 us against 40, weights in one part.)
int attn_splits(int B, int Hkv, int M, int Sk) {
  const int64_t blocks = (int64_t)((M + 127) / 128) * B * Hkv;
  const int tile = M <= FEW_ROWS ? 128 : 64;
  return (int)std::max<int64_t>(1, std::min<int64_t>(512 / blocks, (Sk + tile - 1) / tile / 4));
}

int attn_fwd(const AttnParams& p, hipStream_t st) {
  if (p.D < 8 || p.D > 128 || p.D % 8 || p.M < 1 || p.Sk < 0 || p.splits < 1) return 1;
  const int rows = p.M <= FEW_ROWS ? FEW_ROWS : 128;
  const int64_t grid = ((int64_t)p.M + rows - 1) / rows * p.B * p.Hkv * p.splits;
  if (grid > ATTN_MAX_BLOCKS) return 2;
  if (p.fp16) fwd_d<FP16>(p, st);
  else fwd_d<BF16>(p, st);
  return hipGetLastError() == hipSuccess ? 0 : 3;
}
