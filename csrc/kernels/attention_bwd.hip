// Attention, backward. With p_ij = exp2(scale log2(e) q_i.k_j - lse2_i) computed again from the saved row sums:
//   delta_i = do_i.o_i     dp_ij = do_i.v_j     ds_ij = p_ij (dp_ij - delta_i)
//   dv_j = sum_i p_ij do_i     dk_j = scale sum_i ds_ij q_i     dq_i = scale sum_j ds_ij k_j
// Two kernels: one owns rows and walks the keys (delta, dq), one owns keys and walks the rows (dk, dv; the rows of every
// head that shares the key head, so their sum needs no join). The scores and dp are computed in both, and no gradient is
// summed by atomics in exchange: results do not depend on the order in which blocks run, and nothing but the gradients is
// written.
// Bound: the matrix cores and the vector unit (4 images x 16 heads x 4,096 tokens of 64 channels: 65 % and 69 % busy in dq,
// 54 % and 60 % in dk and dv; at 128 channels 65 % and 47 %, 69 % and 50 %); the LDS carries a fragment per product, 8 of 32
// cycles, without conflicts. Two images of 128 channels: 457 + 657 us = 1,233 TFLOP/s over the 10 products that two-part
// operands make of 7 (a library product of 8,192^3: 1,213). 64 keys a wave halve the LDS traffic but leave one wave a
// SIMD: slower at every width but 32 (128 channels, one part: 1,045 us against 953 then).
// delta is taken from the output before its rounding (o + what that took away): with few keys dp - delta cancels, and a
// rounded o would leave its whole step there.
// Rounding: P and dS enter the second products in two parts of the inputs' type (attn_fine), in fp16 times powers of two
// that keep them in its range (attention.h FP16, Fit); everything else is fp32 until the gradients are rounded once.
#include <algorithm>

#include "attention.h"

namespace {

using namespace attn;

// dq: QT 32-row tiles per wave, 4 waves along the rows, tiles of KT keys
template <class T, int DP, int QT, int KIND, bool FINE>
__global__ __launch_bounds__(256, 2) void attn_dq_kernel(const AttnParams p) {
  constexpr int NT = 256, KT = 64, TILE = KT * DP, CPR = DP / 8, CH = KT * CPR / NT;
  static_assert(KT * CPR % NT == 0, "whole DMA instructions");
  constexpr int NK = KT / 32, NKK = DP / 16, ND = DP / 32, BR = 128 * QT;
  constexpr bool MASK = KIND == ATTN_MASK;
  const bool causal = KIND == ATTN_CAUSAL || (MASK && p.causal);
  __shared__ __attribute__((aligned(1024))) bf16_t smem[4 * TILE];

  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  const int nrb = (p.M + BR - 1) / BR, bhn = p.B * p.Hkv;
  int rb0, bh, sp;
  locate(p, nrb, bhn, p.splits, rb0, bh, sp);
  const int rb = causal ? nrb - 1 - rb0 : rb0;
  const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const int len = p.lengths ? imin(imax(p.lengths[b], 0), p.Sk) : p.Sk;
  const int off = causal ? p.Sk - p.Sq : 0;

  s8v qf[QT][NKK], gf[QT][NKK];
  int lim[QT], ri[QT], rg[QT];
  float lse[QT], delta[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = rb * BR + (wid * QT + t) * 32 + c;
    const bool ok = r < p.M;
    const int rr = ok ? r : p.M - 1, i = fdiv(rr, p.div_g), g = rr - i * p.G;
    ri[t] = i;
    rg[t] = g;
    lse[t] = p.lse2[(int64_t)bh * p.M + rr];
    const bool use = ok && lse[t] != INFINITY;            // an empty row takes part in nothing, whatever it holds
    lim[t] = !use ? 0 : causal ? imin(imax(i + off + 1, 0), len) : len;
    const bf16_t* q = reinterpret_cast<const bf16_t*>(p.q.p) + b * p.q.sb + i * p.q.ss + (hk * p.G + g) * p.q.sh;
    const bf16_t* go = reinterpret_cast<const bf16_t*>(p.go.p) + b * p.go.sb + i * p.go.ss + (hk * p.G + g) * p.go.sh;
    const int64_t at = b * p.o.sb + i * p.o.ss + (hk * p.G + g) * p.o.sh;
    const bf16_t *o = reinterpret_cast<const bf16_t*>(p.o.p) + at, *rest = p.o_rest + at;
    float dl = 0.f;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      const int d = 16 * kk + 8 * h;
      u4v wq = {0, 0, 0, 0}, wg = wq, wo = wq, wr = wq;
      if (use && d < p.D) {
        wq = *reinterpret_cast<const u4v*>(q + d);
        wg = *reinterpret_cast<const u4v*>(go + d);
        wo = *reinterpret_cast<const u4v*>(o + d);
        wr = *reinterpret_cast<const u4v*>(rest + d);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x)
        dl = fmaf(T::lo(wg[x]), fmaf(T::lo(wr[x]), 1.f / T::REST, T::lo(wo[x])),
                  fmaf(T::hi(wg[x]), fmaf(T::hi(wr[x]), 1.f / T::REST, T::hi(wo[x])), dl));
      qf[t][kk] = __builtin_bit_cast(s8v, wq);
      gf[t][kk] = __builtin_bit_cast(s8v, wg);
    }
    delta[t] = dl + other_half(dl);
    if (ok && h == 0 && sp == 0) p.delta[(int64_t)bh * p.M + r] = -delta[t];
  }
  if (p.dq.p == nullptr) return;

  const int r_end = imin(rb * BR + BR, p.M), i_last = fdiv(r_end - 1, p.div_g);
  const int kend = causal ? imin(imax(i_last + off + 1, 0), len) : len;
  const int wr0 = rb * BR + wid * QT * 32;
  const int wi0 = fdiv(imin(wr0, p.M - 1), p.div_g), wi1 = fdiv(imin(wr0 + QT * 32, p.M) - 1, p.div_g);
  const int wlast = wr0 >= p.M ? 0 : causal ? imin(imax(wi1 + off + 1, 0), len) : len;
  const int wfull = causal ? imin(imax(wi0 + off + 1, 0), len) : len;
  const int tiles = (p.Sk + KT - 1) / KT, tps = (tiles + p.splits - 1) / p.splits;
  const int t0 = sp * tps, t1 = imin(imin(t0 + tps, tiles), (kend + KT - 1) / KT);

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
      w0 = w1 = t;
    });
  auto next = [&](int t) { return MASK ? tm.next(t, t1) : t; };
  auto words = [&](int t) {
#pragma unroll
    for (int u = 0; u < QT; ++u) word[u] = mrow[u][imin(t, p.mask.words - 1)];
  };

  f16v acc[ND][QT];
  Fit<T> fit[QT];
  const float sc = p.scale * LOG2E;
  const TransAt<DP> ta(lane);
  auto walk = [&](auto safe) {
    constexpr bool SAFE = decltype(safe)::value;
#pragma unroll
    for (int t = 0; t < QT; ++t) fit[t].start();
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][t][e] = 0.f;

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
      const int key0 = t * KT;
      const bool part = MASK && tm.part;
      const int tn = next(t + 1);
      unsigned long long cur[QT];
      if (MASK) {
#pragma unroll
        for (int u = 0; u < QT; ++u) cur[u] = word[u];
        if (tn < t1) words(tn);
      }
      if (tn < t1) issue(tn, buf ^ 1);
      if (key0 < wlast) {
        const bf16_t* sk = smem + buf * 2 * TILE;
        const bf16_t* sv = sk + TILE;
        const bool edge = key0 + KT > wfull;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
          f16v s[QT], dp[QT];
          // 128 channels: fragment addresses are formed at each read from one offset that the compiler must not see
          // through, or it keeps all of them in registers that are not there
          int fo = lds_at<DP>(c, h);
          if (DP == 128) asm volatile("" : "+v"(fo));
          float nd[QT];
#pragma unroll
          for (int u = 0; u < QT; ++u) {
            nd[u] = -delta[u];
            if (DP == 128) asm volatile("" : "+v"(nd[u])); // or 16 copies of it stay in registers
          }
#pragma unroll
          for (int u = 0; u < QT; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              s[u][e] = 0.f;
              dp[u][e] = nd[u];                            // the product sums dp - delta
            }
#pragma unroll
          for (int kk = 0; kk < NKK; ++kk) {
            const s8v a = frag_x<DP>(sk + 32 * k * DP, fo, kk);
#pragma unroll
            for (int u = 0; u < QT; ++u) s[u] = T::mma(a, qf[u][kk], s[u]);
          }
#pragma unroll
          for (int kk = 0; kk < NKK; ++kk) {
            const s8v a = frag_x<DP>(sv + 32 * k * DP, fo, kk);
#pragma unroll
            for (int u = 0; u < QT; ++u) dp[u] = T::mma(a, gf[u][kk], dp[u]);
          }
          Packed<T, FINE> db[QT][2];
          if (DP == 128) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int u = 0; u < QT; ++u) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[u][e] = exp2_(fmaf(s[u][e], sc, fit[u].ef - lse[u]));   // f p: it is only in dS
            if (MASK && part) {
              const uint32_t w = (uint32_t)(cur[u] >> (32 * k)) >> (4 * h);
#pragma unroll
              for (int e = 0; e < 16; ++e) s[u][e] = (w >> ((e & 3) + 8 * (e >> 2))) & 1 ? s[u][e] : 0.f;
            }
            if (edge) {
              const int left = lim[u] - key0 - 32 * k - 4 * h;
#pragma unroll
              for (int e = 0; e < 16; ++e) s[u][e] = (e & 3) + 8 * (e >> 2) < left ? s[u][e] : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float ds = s[u][e] * dp[u][e];
              s[u][e] = SAFE && s[u][e] == 0.f ? 0.f : ds;
            }
            fit[u].pack(s[u], db[u], [&](float g) {
#pragma unroll
              for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[d][u][e] *= g;
            });
          }
          if (DP == 128) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int d = 0; d < ND; ++d) {
              s8v a = frag_t<DP>(sk + (32 * k + 16 * ks) * DP, ta, d);
              if constexpr (SAFE) {                          // an allowed key that is not finite shows in its scores
                s8v pos, neg;
                __builtin_amdgcn_sched_barrier(0);         // few registers matter here, not speed
                a = clean<T>(a, pos, neg);
              }
#pragma unroll
              for (int u = 0; u < QT; ++u) acc[d][u] = db[u][ks].mma(a, acc[d][u]);
            }
        }
      }
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
  for (int u = 0; u < QT; ++u) {
    const bool ok = rb * BR + (wid * QT + u) * 32 + c < p.M;
    if (p.splits > 1) {
      const int64_t part = ((int64_t)sp * bhn + bh) * p.M + rb * BR + (wid * QT + u) * 32 + c;
#pragma unroll
      for (int d = 0; d < ND; ++d) store_part<DP>(p.ws_o + part * DP, acc[d][u], fit[u].undo(p.grad_scale), d, h, ok);
      continue;
    }
    bf16_t* o = reinterpret_cast<bf16_t*>(p.dq.p) + b * p.dq.sb + ri[u] * p.dq.ss + (hk * p.G + rg[u]) * p.dq.sh;
#pragma unroll
    for (int d = 0; d < ND; ++d) store_row<T>(o, acc[d][u], fit[u].undo(p.grad_scale), d, p.D, h, ok);
  }
}

// dk, dv: KQ 32-key tiles per wave, 4 waves along the keys, tiles of RT rows. The wave's keys are B operands in registers
// for the whole walk, its values too, or (VL: from 96 channels, where dk and dv take half of the 256 registers that let
// two waves share a SIMD) in LDS.
template <class T, int DP, int KQ, int RT, bool VL, int KIND, bool FINE>
__global__ __launch_bounds__(256, 2) void attn_dkv_kernel(const AttnParams p) {
  constexpr int NT = 256, TILE = RT * DP, CPR = DP / 8, CH = RT * CPR / NT, VTILE = VL ? 128 * KQ * DP : 0;
  static_assert(RT * CPR % NT == 0 && VTILE / 8 % NT == 0, "whole DMA instructions");
  constexpr int NR = RT / 32, NKK = DP / 16, ND = DP / 32, BK = 128 * KQ;
  constexpr bool MASK = KIND == ATTN_MASK;
  const bool causal = KIND == ATTN_CAUSAL || (MASK && p.causal);
  __shared__ __attribute__((aligned(1024))) bf16_t smem[4 * TILE + VTILE];
  __shared__ __attribute__((aligned(256))) float sstat[2][2][64];      // [buffer][lse2, -delta][row]

  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  const int nkb = (p.Sk + BK - 1) / BK, bhn = p.B * p.Hkv;
  int kb, bh, sp;
  locate(p, nkb, bhn, p.kv_splits, kb, bh, sp);             // causal: the first keys have the most rows
  const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const int len = p.lengths ? imin(imax(p.lengths[b], 0), p.Sk) : p.Sk;
  const int off = causal ? p.Sk - p.Sq : 0;
  const int wkey0 = kb * BK + wid * KQ * 32;

  // B operands of the wave's own keys or values
  auto own_frag = [&](const AttnTensor& x, int key, int kk) {
    const int d = 16 * kk + 8 * h;
    u4v w = {0, 0, 0, 0};
    if (key < len && d < p.D)
      w = *reinterpret_cast<const u4v*>(reinterpret_cast<const bf16_t*>(x.p) + b * x.sb + key * x.ss + hk * x.sh + d);
    return __builtin_bit_cast(s8v, w);
  };
  s8v kf[KQ][NKK], vf[KQ][VL ? 1 : NKK];
  int rmin[KQ];                                              // first row that may attend this lane's key
#pragma unroll
  for (int t = 0; t < KQ; ++t) {
    const int key = wkey0 + 32 * t + c;
    rmin[t] = causal ? imin(imax(key - off, 0), p.Sq) * p.G : 0;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      kf[t][kk] = own_frag(p.k, key, kk);
      if (!VL) vf[t][VL ? 0 : kk] = own_frag(p.v, key, kk);
    }
  }
  const bf16_t* svals = smem + 4 * TILE + wid * KQ * 32 * DP;
  if (VL) {
    const u4v rv = rsrc(reinterpret_cast<const bf16_t*>(p.v.p) + b * p.v.sb + (int64_t)kb * BK * p.v.ss + hk * p.v.sh);
#pragma unroll
    for (int n = 0; n < VTILE / 8 / NT; ++n) {
      const int id = tid + NT * n, row = id / CPR, d = ((id % CPR) ^ swz<DP>(row)) * 8;
      dma16(rv, kb * BK + row < len && d < p.D ? (uint32_t)(row * (int)p.v.ss + d) * 2 : CFL_OOB,
            smem + 4 * TILE + wid * 512 + NT * 8 * n);
    }
  }
  const int klast = imin(kb * BK + BK, p.Sk) - 1;
  const int tiles = (p.M + RT - 1) / RT;
  const int tfirst = causal ? imin(imax(kb * BK - off, 0), p.Sq) * p.G / RT : 0;
  const int tps = (tiles - tfirst + p.kv_splits - 1) / p.kv_splits;      // the walk's own tiles in even parts
  const int t0 = tfirst + sp * tps, t1 = kb * BK < len ? imin(t0 + tps, tiles) : 0;
  // rows below wfirst attend no key of this wave, rows from wfull on every one
  const int wfirst = causal ? imin(imax(wkey0 - off, 0), p.Sq) * p.G : 0;
  const int wfull = causal ? imin(imax(imin(wkey0 + 32 * KQ, p.Sk) - 1 - off, 0), p.Sq) * p.G : 0;

  int vrow[CH], vd[CH];
#pragma unroll
  for (int n = 0; n < CH; ++n) {
    const int id = tid + NT * n, row = id / CPR;
    vrow[n] = row;
    vd[n] = ((id % CPR) ^ swz<DP>(row)) * 8;
  }
  const bf16_t* qb = reinterpret_cast<const bf16_t*>(p.q.p) + b * p.q.sb + hk * p.G * p.q.sh;
  const bf16_t* gb = reinterpret_cast<const bf16_t*>(p.go.p) + b * p.go.sb + hk * p.G * p.go.sh;
  auto issue = [&](int t, int buf) {
    const int r0 = t * RT, i0 = fdiv(r0, p.div_g), rem = p.M - r0;
    const u4v rq = rsrc(qb + (int64_t)i0 * p.q.ss), rg = rsrc(gb + (int64_t)i0 * p.go.ss);
    const bf16_t* dst = smem + buf * 2 * TILE + wid * 512;
#pragma unroll
    for (int n = 0; n < CH; ++n) {
      const int r = imin(r0 + vrow[n], p.M - 1), i = fdiv(r, p.div_g), g = r - i * p.G;
      const bool in = vd[n] < p.D;
      const uint32_t oq = (uint32_t)((i - i0) * (int)p.q.ss + g * (int)p.q.sh + vd[n]) * 2;
      const uint32_t og = (uint32_t)((i - i0) * (int)p.go.ss + g * (int)p.go.sh + vd[n]) * 2;
      dma16(rq, in ? oq : CFL_OOB, dst + NT * 8 * n);
      dma16(rg, in && vrow[n] < rem ? og : CFL_OOB, dst + TILE + NT * 8 * n);
    }
    // rows past the last: the last row's query and lse2 (0 times a key that is not finite would be NaN), do = delta = 0
    if (wid < 2) {
      const u4v rs = rsrc((wid ? p.delta : p.lse2) + (int64_t)bh * p.M + r0);
      dma4(rs, wid == 0 ? 4u * imin(lane, rem - 1) : lane < rem ? 4u * lane : CFL_OOB, &sstat[buf][wid][0]);
    }
  };

  __shared__ uint8_t classes[MASK ? MASK_TILES + 64 : 1];
  TileMask tm;
  if (MASK)
    tm.fill(p, b, hk, classes, tiles, [&](int t, int& i0, int& i1, int& w0, int& w1) {
      i0 = fdiv(t * RT, p.div_g);
      i1 = fdiv(imin(t * RT + RT, p.M) - 1, p.div_g);
      w0 = kb * BK >> 6;
      w1 = klast >> 6;
    });
  auto next = [&](int t) { return MASK ? tm.next(t, t1) : t; };
  // mask bits of row 32 * n + c of the tile against the wave's keys
  uint32_t bits[NR][KQ], cur[NR][KQ];
  auto words = [&](int t) {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int r = imin(t * RT + 32 * n + c, p.M - 1), i = fdiv(r, p.div_g), g = r - i * p.G;
      const unsigned long long* m =
          p.mask.bits +
          (b * p.mask.sb + (hk * p.G + g) * p.mask.sh + (p.mask.rows > 1 ? i : 0)) * (int64_t)p.mask.words;
#pragma unroll
      for (int u = 0; u < KQ; ++u) {
        const int k0 = imin(wkey0 + 32 * u, p.Sk - 1);
        bits[n][u] = (uint32_t)(m[k0 >> 6] >> (k0 & 32));
      }
    }
  };

  f16v dk[ND][KQ], dv[ND][KQ];
  Fit<T> fit[KQ];
  const float sc = p.scale * LOG2E;
  const TransAt<DP> ta(lane);
  auto walk = [&](auto safe) {
    constexpr bool SAFE = decltype(safe)::value;
#pragma unroll
    for (int u = 0; u < KQ; ++u) fit[u].start();
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int u = 0; u < KQ; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[d][u][e] = dv[d][u][e] = 0.f;

    int t = t1 > t0 ? next(t0) : t0;
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
      if (MASK) {
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int u = 0; u < KQ; ++u) cur[n][u] = bits[n][u];
        if (tn < t1) words(tn);
      }
      if (tn < t1) issue(tn, buf ^ 1);
      const bf16_t* sq = smem + buf * 2 * TILE;
      const bf16_t* sg = sq + TILE;
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const int r0 = t * RT + 32 * n;
        if (r0 + 32 <= wfirst || r0 >= p.M || wkey0 >= len) continue;
        const bool edge = r0 < wfull;
        // VL: addresses from one offset, as in attn_dq_kernel
        int fo = lds_at<DP>(c, h);
        if (VL) asm volatile("" : "+v"(fo));
        f16v s[KQ], dp[KQ];
        if (VL) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < KQ; ++u)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f4v y = *reinterpret_cast<const f4v*>(&sstat[buf][1][32 * n + 8 * q + 4 * h]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              s[u][4 * q + j] = 0.f;
              dp[u][4 * q + j] = y[j];                     // the product sums dp - delta
            }
          }
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
          const s8v a = frag_x<DP>(sq + 32 * n * DP, fo, kk);
#pragma unroll
          for (int u = 0; u < KQ; ++u)
            // the second walk reads its keys each time: it needs their registers, not speed
            s[u] = T::mma(a, VL && SAFE ? own_frag(p.k, wkey0 + 32 * u + c, kk) : kf[u][kk], s[u]);
          if (VL && kk % 8 == 7) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
          const s8v a = frag_x<DP>(sg + 32 * n * DP, fo, kk);
#pragma unroll
          for (int u = 0; u < KQ; ++u)
            dp[u] = T::mma(a, VL ? frag_x<DP>(svals + 32 * u * DP, fo, kk) : vf[u][VL ? 0 : kk], dp[u]);
          if (VL && kk % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
        Packed<T, FINE> pb[KQ][2], db[KQ][2];
        uint32_t seen[KQ];
        if (VL) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < KQ; ++u) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f4v x = *reinterpret_cast<const f4v*>(&sstat[buf][0][32 * n + 8 * q + 4 * h]);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[u][4 * q + j] = exp2_(fmaf(s[u][4 * q + j], sc, -x[j]));
          }
          if (MASK && part) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int row = (e & 3) + 8 * (e >> 2);
              const uint32_t lo = __builtin_amdgcn_readlane(cur[n][u], row);
              const uint32_t hi = __builtin_amdgcn_readlane(cur[n][u], row + 4);
              s[u][e] = __builtin_amdgcn_inverse_ballot_w64(((unsigned long long)hi << 32) | lo) ? s[u][e] : 0.f;
            }
          }
          if (edge) {
            const int from = rmin[u] - r0 - 4 * h;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[u][e] = (e & 3) + 8 * (e >> 2) >= from ? s[u][e] : 0.f;
          }
          if constexpr (SAFE) seen[u] = weighed(s[u]);
          pb[u][0].set(s[u], 0);
          pb[u][1].set(s[u], 1);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            dp[u][e] *= s[u][e];
            if constexpr (T::NARROW) dp[u][e] *= fit[u].f;
            if constexpr (SAFE) dp[u][e] = s[u][e] == 0.f ? 0.f : dp[u][e];
          }
          fit[u].pack(dp[u], db[u], [&](float g) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
              for (int e = 0; e < 16; ++e) dk[d][u][e] *= g;
          });
        }
        if (VL) __builtin_amdgcn_sched_barrier(0);
        auto add_dv = [&]() {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int d = 0; d < ND; ++d) {
              const bf16_t* rows = sg + (32 * n + 16 * ks) * DP;
              s8v a = SAFE ? frag_t2<DP>(rows, ta, d) : frag_t<DP>(rows, ta, d);
              if constexpr (SAFE) {
                s8v pos, neg;
                __builtin_amdgcn_sched_barrier(0);           // few registers matter here, not speed
                a = clean<T>(a, pos, neg);
#pragma unroll
                for (int u = 0; u < KQ; ++u) poison<T>(dv[d][u], pos, neg, seen[u] >> 8 * ks);
              }
#pragma unroll
              for (int u = 0; u < KQ; ++u) dv[d][u] = pb[u][ks].mma(a, dv[d][u]);
            }
        };
        auto add_dk = [&]() {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int d = 0; d < ND; ++d) {
              const bf16_t* rows = sq + (32 * n + 16 * ks) * DP;
              s8v a = SAFE ? frag_t2<DP>(rows, ta, d) : frag_t<DP>(rows, ta, d);
              if constexpr (SAFE) {                            // an allowed query that is not finite shows in its scores
                s8v pos, neg;
                __builtin_amdgcn_sched_barrier(0);           // few registers matter here, not speed
                a = clean<T>(a, pos, neg);
              }
#pragma unroll
              for (int u = 0; u < KQ; ++u) dk[d][u] = db[u][ks].mma(a, dk[d][u]);
            }
        };
        if (!SAFE) add_dv();                                 // clean and poison need the registers of db
        add_dk();
        if (SAFE) add_dv();
      }
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
      for (int u = 0; u < KQ; ++u) z += finite_sum(dk[d][u]) + finite_sum(dv[d][u]);
    if (__syncthreads_or(z != 0.f)) walk(std::true_type{});
  }
#pragma unroll
  for (int u = 0; u < KQ; ++u) {
    const int key = wkey0 + 32 * u + c;
    bf16_t* ko = reinterpret_cast<bf16_t*>(p.dk.p) + b * p.dk.sb + key * p.dk.ss + hk * p.dk.sh;
    bf16_t* vo = reinterpret_cast<bf16_t*>(p.dv.p) + b * p.dv.sb + key * p.dv.ss + hk * p.dv.sh;
    if (p.kv_splits > 1) {
      const int64_t part = ((int64_t)sp * bhn + bh) * p.Sk + key, half = (int64_t)p.kv_splits * bhn * p.Sk;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        store_part<DP>(p.ws_kv + part * DP, dk[d][u], fit[u].undo(p.grad_scale), d, h, key < len);
        store_part<DP>(p.ws_kv + (half + part) * DP, dv[d][u], p_undo<T>(), d, h, key < len);
      }
      continue;
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      if (p.dk.p) store_row<T>(ko, dk[d][u], fit[u].undo(p.grad_scale), d, p.D, h, key < p.Sk, nullptr, key >= len);
      if (p.dv.p) store_row<T>(vo, dv[d][u], p_undo<T>(), d, p.D, h, key < p.Sk, nullptr, key >= len);
    }
  }
}

// gradients of a token tensor from the parts of `splits` blocks: one thread per 4 channels, parts in order
template <class T, int DP>
__global__ __launch_bounds__(256) void attn_sum_kernel(const float* ws, int splits, AttnTensor out, int B, int H, int G,
                                                       int rows, int D, FastDiv div_g, const int* lengths) {
  constexpr int TPR = DP / 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)B * H * rows, row = id / TPR;
  const int d = (int)(id % TPR) * 4;
  if (row >= all || d >= D) return;
  const int bh = (int)(row / rows), r = (int)(row - (int64_t)bh * rows), b = bh / H, hk = bh - b * H;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  const int n = lengths && r >= lengths[b] ? 0 : splits;    // keys behind the image's: nothing was written
  for (int s = 0; s < n; ++s) {
    const float4 v = *reinterpret_cast<const float4*>(ws + (s * all + row) * DP + d);
    a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
  }
  const int i = fdiv(r, div_g), g = r - i * G;
  bf16_t* o = reinterpret_cast<bf16_t*>(out.p) + b * out.sb + i * out.ss + (hk * G + g) * out.sh + d;
  *reinterpret_cast<uint2*>(o) = make_uint2(T::pack2(a.x, a.y), T::pack2(a.z, a.w));
}

template <class T, int DP, int KIND, bool FINE>
void bwd(const AttnParams& p, hipStream_t st) {
  const int64_t bhn = (int64_t)p.B * p.Hkv;
  attn_dq_kernel<T, DP, 1, KIND, FINE><<<(unsigned)((p.M + 127) / 128 * bhn * p.splits), 256, 0, st>>>(p);
  if (p.splits > 1 && p.dq.p)
    attn_sum_kernel<T, DP><<<(unsigned)((bhn * p.M * (DP / 4) + 255) / 256), 256, 0, st>>>(
        p.ws_o, p.splits, p.dq, p.B, p.Hkv, p.G, p.M, p.D, p.div_g, nullptr);
  if ((p.dk.p == nullptr && p.dv.p == nullptr) || p.Sk == 0) return;
  attn_dkv_kernel<T, DP, 1, DP == 128 ? 32 : 64, DP >= 96, KIND, FINE>
      <<<(unsigned)((p.Sk + 127) / 128 * bhn * p.kv_splits), 256, 0, st>>>(p);
  if (p.kv_splits > 1) {
    const int64_t n = bhn * p.Sk;
    const unsigned grid = (unsigned)((n * (DP / 4) + 255) / 256);
    const FastDiv one = fast_div(1);
    if (p.dk.p)
      attn_sum_kernel<T, DP><<<grid, 256, 0, st>>>(p.ws_kv, p.kv_splits, p.dk, p.B, p.Hkv, 1, p.Sk, p.D, one, p.lengths);
    if (p.dv.p)
      attn_sum_kernel<T, DP><<<grid, 256, 0, st>>>(p.ws_kv + p.kv_splits * n * DP, p.kv_splits, p.dv, p.B, p.Hkv, 1,
                                                   p.Sk, p.D, one, p.lengths);
  }
}

template <class T, int KIND>
void bwd_d(const AttnParams& p, hipStream_t st) {
  if (p.D <= 32) attn_fine() ? bwd<T, 32, KIND, true>(p, st) : bwd<T, 32, KIND, false>(p, st);
  else if (p.D <= 64) attn_fine() ? bwd<T, 64, KIND, true>(p, st) : bwd<T, 64, KIND, false>(p, st);
  else if (p.D <= 96) attn_fine() ? bwd<T, 96, KIND, true>(p, st) : bwd<T, 96, KIND, false>(p, st);
  else attn_fine() ? bwd<T, 128, KIND, true>(p, st) : bwd<T, 128, KIND, false>(p, st);
}

}  // namespace

// Blocks that share a row block's keys (dq) and a key block's rows (dk, dv): as attn_splits, up to two blocks a CU, or
// four for causal dk, dv, whose blocks are as unequal as their keys (2 images, 16 heads that share 2, 8,192 tokens, 128
// channels: 2,862 / 2,041 / 2,053 us for 512 / 1,024 / 2,048 blocks); at least four tiles each. Lengths make blocks
// empty, not unequal: more than one round of them only costs parts (6 images of 1,531 keys, all full: 122 us for 512, 131
// for 1,024; 60 % full: 110 and 106). These with operands in one part.
void attn_bwd_splits(int B, int Hkv, int M, int Sk, bool causal, int& splits, int& kv_splits) {
  const int64_t bhn = (int64_t)B * Hkv, qb = (M + 127) / 128 * bhn, kb = std::max<int64_t>(1, (Sk + 127) / 128 * bhn);
  splits = (int)std::max<int64_t>(1, std::min<int64_t>(512 / qb, (Sk + 63) / 64 / 4));
  kv_splits = (int)std::max<int64_t>(1, std::min<int64_t>((causal ? 1024 : 512) / kb, (M + 63) / 64 / 4));
}

int attn_bwd(const AttnParams& p, hipStream_t st) {
  if (p.D < 8 || p.D > 128 || p.D % 8 || p.M < 1 || p.Sk < 0 || p.splits < 1 || p.kv_splits < 1) return 1;
  if ((p.M + 127) / 128 * (int64_t)p.B * p.Hkv * p.splits > ATTN_MAX_BLOCKS ||
      (p.Sk + 127) / 128 * (int64_t)p.B * p.Hkv * p.kv_splits > ATTN_MAX_BLOCKS)
    return 2;
  const int kind = p.mask.bits ? ATTN_MASK : p.causal ? ATTN_CAUSAL : ATTN_PLAIN;
  if (kind == ATTN_MASK) p.fp16 ? bwd_d<FP16, ATTN_MASK>(p, st) : bwd_d<BF16, ATTN_MASK>(p, st);
  else if (kind == ATTN_CAUSAL) p.fp16 ? bwd_d<FP16, ATTN_CAUSAL>(p, st) : bwd_d<BF16, ATTN_CAUSAL>(p, st);
  else p.fp16 ? bwd_d<FP16, ATTN_PLAIN>(p, st) : bwd_d<BF16, ATTN_PLAIN>(p, st);
  return hipGetLastError() == hipSuccess ? 0 : 3;
}
