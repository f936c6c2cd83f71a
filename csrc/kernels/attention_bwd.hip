// Attention, backward. With p_ij = exp2(scale log2(e) q_i.k_j - lse2_i) computed again from the saved row sums:
//   delta_i = do_i.o_i     dp_ij = do_i.v_j     ds_ij = p_ij (dp_ij - delta_i)
//   dv_j = sum_i p_ij do_i     dk_j = scale sum_i ds_ij q_i     dq_i = scale sum_j ds_ij k_j
// Two kernels: one owns rows and walks the keys (delta, dq), one owns keys and walks the rows (dk, dv; the rows of every
// head that shares the key head, so their sum needs no join). The scores and dp are computed in both: 7 products
// instead of the 5 of a single pass, and in exchange no gradient is summed by atomics: results do not depend on the
// order in which blocks run, and nothing but the gradients is written.
// Rounding: P and dS are rounded to the inputs' type as operands of the second products; everything else is fp32 until
// the gradients are rounded once.
#include "attention.h"

namespace {

using namespace attn;

// dq: QT 32-row tiles per wave, 4 waves along the rows, tiles of KT keys
template <class T, int DP, int QT, bool MASK>
__global__ __launch_bounds__(256) void attn_dq_kernel(const AttnParams p) {
  constexpr int NT = 256, KT = 64, TILE = KT * DP, CPR = DP / 8, CH = KT * CPR / NT;
  constexpr int NK = KT / 32, NKK = DP / 16, ND = DP / 32, BR = 128 * QT;
  __shared__ __attribute__((aligned(1024))) bf16_t smem[4 * TILE];

  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  const int nrb = (p.M + BR - 1) / BR;
  const int lin = xcd_swizzle(blockIdx.x, gridDim.x);
  const int bh = lin / nrb, rb0 = lin - bh * nrb;
  const int rb = p.causal ? nrb - 1 - rb0 : rb0;
  const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const int len = p.lengths ? imin(imax(p.lengths[b], 0), p.Sk) : p.Sk;
  const int off = p.causal ? p.Sk - p.Sq : 0;

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
    lim[t] = !use ? 0 : p.causal ? imin(imax(i + off + 1, 0), len) : len;
    const bf16_t* q = reinterpret_cast<const bf16_t*>(p.q.p) + b * p.q.sb + i * p.q.ss + (hk * p.G + g) * p.q.sh;
    const bf16_t* go = reinterpret_cast<const bf16_t*>(p.go.p) + b * p.go.sb + i * p.go.ss + (hk * p.G + g) * p.go.sh;
    const bf16_t* o = reinterpret_cast<const bf16_t*>(p.o.p) + b * p.o.sb + i * p.o.ss + (hk * p.G + g) * p.o.sh;
    float dl = 0.f;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      const int d = 16 * kk + 8 * h;
      u4v wq = {0, 0, 0, 0}, wg = wq, wo = wq;
      if (use && d < p.D) {
        wq = *reinterpret_cast<const u4v*>(q + d);
        wg = *reinterpret_cast<const u4v*>(go + d);
        wo = *reinterpret_cast<const u4v*>(o + d);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) dl = fmaf(T::lo(wg[x]), T::lo(wo[x]), fmaf(T::hi(wg[x]), T::hi(wo[x]), dl));
      qf[t][kk] = __builtin_bit_cast(s8v, wq);
      gf[t][kk] = __builtin_bit_cast(s8v, wg);
    }
    delta[t] = dl + other_half(dl);
    if (ok && h == 0) p.delta[(int64_t)bh * p.M + r] = delta[t];
  }
  if (p.dq.p == nullptr) return;

  const int r_end = imin(rb * BR + BR, p.M), i_last = fdiv(r_end - 1, p.div_g);
  const int kend = p.causal ? imin(imax(i_last + off + 1, 0), len) : len;
  const int wr0 = rb * BR + wid * QT * 32;
  const int wi0 = fdiv(imin(wr0, p.M - 1), p.div_g), wi1 = fdiv(imin(wr0 + QT * 32, p.M) - 1, p.div_g);
  const int wlast = wr0 >= p.M ? 0 : p.causal ? imin(imax(wi1 + off + 1, 0), len) : len;
  const int wfull = p.causal ? imin(imax(wi0 + off + 1, 0), len) : len;
  const int tiles = (p.Sk + KT - 1) / KT, t1 = (kend + KT - 1) / KT;

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
  TileMask tm;
  if (MASK) tm.init(p, b, hk);
  const int ib0 = fdiv(rb * BR, p.div_g), ib1 = i_last;
  auto next = [&](int t) {
    if (!MASK) return t;
    return tm.next(t, t1, [&](int u) { return tm.cls(p, ib0, ib1, u, u, u < tiles); });
  };
  auto words = [&](int t) {
#pragma unroll
    for (int u = 0; u < QT; ++u) word[u] = mrow[u][imin(t, p.mask.words - 1)];
  };

  f16v acc[ND][QT];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[d][t][e] = 0.f;
  const float sc = p.scale * LOG2E;

  int t = next(0), buf = 0;
  if (t < t1) {
    if (MASK) words(t);
    issue(t, 0);
  }
  wait_vm();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  while (t < t1) {
    const int key0 = t * KT;
    const bool part = MASK && !tm.is_whole(t);
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
#pragma unroll
        for (int u = 0; u < QT; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[u][e] = dp[u][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
          const s8v a = frag<DP>(sk, 32 * k + c, 2 * kk + h);
#pragma unroll
          for (int u = 0; u < QT; ++u) s[u] = T::mma(a, qf[u][kk], s[u]);
        }
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
          const s8v a = frag<DP>(sv, 32 * k + c, 2 * kk + h);
#pragma unroll
          for (int u = 0; u < QT; ++u) dp[u] = T::mma(a, gf[u][kk], dp[u]);
        }
        s8v db[QT][2];
#pragma unroll
        for (int u = 0; u < QT; ++u) {
#pragma unroll
          for (int e = 0; e < 16; ++e) s[u][e] = exp2_(fmaf(s[u][e], sc, -lse[u])) * (dp[u][e] - delta[u]);
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
          db[u][0] = pack_b<T>(s[u], 0);
          db[u][1] = pack_b<T>(s[u], 1);
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const s8v a = frag_t<DP>(sk, 32 * k + 16 * ks, d, lane);
#pragma unroll
            for (int u = 0; u < QT; ++u) acc[d][u] = T::mma(a, db[u][ks], acc[d][u]);
          }
      }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    buf ^= 1;
    t = tn;
  }
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    const bool ok = rb * BR + (wid * QT + u) * 32 + c < p.M;
    bf16_t* o = reinterpret_cast<bf16_t*>(p.dq.p) + b * p.dq.sb + ri[u] * p.dq.ss + (hk * p.G + rg[u]) * p.dq.sh;
#pragma unroll
    for (int d = 0; d < ND; ++d) store_row<T>(o, acc[d][u], p.scale, d, p.D, h, ok);
  }
}

// dk, dv: KQ 32-key tiles per wave, 4 waves along the keys, tiles of RT rows
template <class T, int DP, int KQ, bool MASK>
__global__ __launch_bounds__(256) void attn_dkv_kernel(const AttnParams p) {
  constexpr int NT = 256, RT = 64, TILE = RT * DP, CPR = DP / 8, CH = RT * CPR / NT;
  constexpr int NR = RT / 32, NKK = DP / 16, ND = DP / 32, BK = 128 * KQ;
  __shared__ __attribute__((aligned(1024))) bf16_t smem[4 * TILE];
  __shared__ __attribute__((aligned(256))) float sstat[2][2][RT];      // [buffer][lse2, delta][row]

  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  const int nkb = (p.Sk + BK - 1) / BK;
  const int lin = xcd_swizzle(blockIdx.x, gridDim.x);
  const int bh = lin / nkb, kb = lin - bh * nkb;            // causal: the first keys have the most rows
  const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const int len = p.lengths ? imin(imax(p.lengths[b], 0), p.Sk) : p.Sk;
  const int off = p.causal ? p.Sk - p.Sq : 0;
  const int wkey0 = kb * BK + wid * KQ * 32;

  s8v kf[KQ][NKK], vf[KQ][NKK];
  int rmin[KQ];                                              // first row that may attend this lane's key
#pragma unroll
  for (int t = 0; t < KQ; ++t) {
    const int key = wkey0 + 32 * t + c;
    rmin[t] = p.causal ? imin(imax(key - off, 0), p.Sq) * p.G : 0;
    const bf16_t* k = reinterpret_cast<const bf16_t*>(p.k.p) + b * p.k.sb + key * p.k.ss + hk * p.k.sh;
    const bf16_t* v = reinterpret_cast<const bf16_t*>(p.v.p) + b * p.v.sb + key * p.v.ss + hk * p.v.sh;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      const int d = 16 * kk + 8 * h;
      u4v wk = {0, 0, 0, 0}, wv = wk;
      if (key < len && d < p.D) {
        wk = *reinterpret_cast<const u4v*>(k + d);
        wv = *reinterpret_cast<const u4v*>(v + d);
      }
      kf[t][kk] = __builtin_bit_cast(s8v, wk);
      vf[t][kk] = __builtin_bit_cast(s8v, wv);
    }
  }
  const int klast = imin(kb * BK + BK, p.Sk) - 1;
  const int tiles = (p.M + RT - 1) / RT;
  const int t0 = p.causal ? imin(imax(kb * BK - off, 0), p.Sq) * p.G / RT : 0;
  const int t1 = kb * BK < len ? tiles : 0;
  // rows below wfirst attend no key of this wave, rows from wfull on every one
  const int wfirst = p.causal ? imin(imax(wkey0 - off, 0), p.Sq) * p.G : 0;
  const int wfull = p.causal ? imin(imax(imin(wkey0 + 32 * KQ, p.Sk) - 1 - off, 0), p.Sq) * p.G : 0;

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
      const int r = r0 + vrow[n], i = fdiv(r, p.div_g), g = r - i * p.G;
      const bool in = vrow[n] < rem && vd[n] < p.D;
      const uint32_t oq = (uint32_t)((i - i0) * (int)p.q.ss + g * (int)p.q.sh + vd[n]) * 2;
      const uint32_t og = (uint32_t)((i - i0) * (int)p.go.ss + g * (int)p.go.sh + vd[n]) * 2;
      dma16(rq, in ? oq : CFL_OOB, dst + NT * 8 * n);
      dma16(rg, in ? og : CFL_OOB, dst + TILE + NT * 8 * n);
    }
    // rows past the last read 0 everywhere: p = 1, do = 0, ds = 0
    if (wid < 2) {
      const u4v rs = rsrc((wid ? p.delta : p.lse2) + (int64_t)bh * p.M + r0);
      dma4(rs, lane < rem ? 4u * lane : CFL_OOB, &sstat[buf][wid][0]);
    }
  };

  TileMask tm;
  if (MASK) tm.init(p, b, hk);
  auto next = [&](int t) {
    if (!MASK) return t;
    return tm.next(t, t1, [&](int u) {
      const int last = imin(u * RT + RT, p.M) - 1;
      return tm.cls(p, fdiv(imin(u * RT, p.M - 1), p.div_g), fdiv(imax(last, 0), p.div_g), kb * BK >> 6, klast >> 6,
                    u < tiles);
    });
  };
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
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int u = 0; u < KQ; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) dk[d][u][e] = dv[d][u][e] = 0.f;
  const float sc = p.scale * LOG2E;

  int t = t1 > t0 ? next(t0) : t0, buf = 0;
  if (t < t1) {
    if (MASK) words(t);
    issue(t, 0);
  }
  wait_vm();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  while (t < t1) {
    const bool part = MASK && !tm.is_whole(t);
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
      f16v s[KQ], dp[KQ];
#pragma unroll
      for (int u = 0; u < KQ; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[u][e] = dp[u][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) {
        const s8v a = frag<DP>(sq, 32 * n + c, 2 * kk + h);
#pragma unroll
        for (int u = 0; u < KQ; ++u) s[u] = T::mma(a, kf[u][kk], s[u]);
      }
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) {
        const s8v a = frag<DP>(sg, 32 * n + c, 2 * kk + h);
#pragma unroll
        for (int u = 0; u < KQ; ++u) dp[u] = T::mma(a, vf[u][kk], dp[u]);
      }
      float lse[16], dl[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 x = *reinterpret_cast<const float4*>(&sstat[buf][0][32 * n + 8 * q + 4 * h]);
        const float4 y = *reinterpret_cast<const float4*>(&sstat[buf][1][32 * n + 8 * q + 4 * h]);
        lse[4 * q] = x.x; lse[4 * q + 1] = x.y; lse[4 * q + 2] = x.z; lse[4 * q + 3] = x.w;
        dl[4 * q] = y.x; dl[4 * q + 1] = y.y; dl[4 * q + 2] = y.z; dl[4 * q + 3] = y.w;
      }
      s8v pb[KQ][2], db[KQ][2];
#pragma unroll
      for (int u = 0; u < KQ; ++u) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[u][e] = exp2_(fmaf(s[u][e], sc, -lse[e]));
          dp[u][e] = s[u][e] * (dp[u][e] - dl[e]);
        }
        if (MASK && part) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int row = (e & 3) + 8 * (e >> 2);
            const uint32_t lo = __builtin_amdgcn_readlane(cur[n][u], row);
            const uint32_t hi = __builtin_amdgcn_readlane(cur[n][u], row + 4);
            const bool ok = __builtin_amdgcn_inverse_ballot_w64(((unsigned long long)hi << 32) | lo);
            s[u][e] = ok ? s[u][e] : 0.f;
            dp[u][e] = ok ? dp[u][e] : 0.f;
          }
        }
        if (edge) {
          const int from = rmin[u] - r0 - 4 * h;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const bool ok = (e & 3) + 8 * (e >> 2) >= from;
            s[u][e] = ok ? s[u][e] : 0.f;
            dp[u][e] = ok ? dp[u][e] : 0.f;
          }
        }
        pb[u][0] = pack_b<T>(s[u], 0);
        pb[u][1] = pack_b<T>(s[u], 1);
        db[u][0] = pack_b<T>(dp[u], 0);
        db[u][1] = pack_b<T>(dp[u], 1);
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const s8v a = frag_t<DP>(sg, 32 * n + 16 * ks, d, lane);
#pragma unroll
          for (int u = 0; u < KQ; ++u) dv[d][u] = T::mma(a, pb[u][ks], dv[d][u]);
        }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const s8v a = frag_t<DP>(sq, 32 * n + 16 * ks, d, lane);
#pragma unroll
          for (int u = 0; u < KQ; ++u) dk[d][u] = T::mma(a, db[u][ks], dk[d][u]);
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    buf ^= 1;
    t = tn;
  }
#pragma unroll
  for (int u = 0; u < KQ; ++u) {
    const int key = wkey0 + 32 * u + c;
    bf16_t* ko = reinterpret_cast<bf16_t*>(p.dk.p) + b * p.dk.sb + key * p.dk.ss + hk * p.dk.sh;
    bf16_t* vo = reinterpret_cast<bf16_t*>(p.dv.p) + b * p.dv.sb + key * p.dv.ss + hk * p.dv.sh;
    if (key >= len) {                                        // padding behind the image's keys
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[d][u][e] = dv[d][u][e] = 0.f;
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      if (p.dk.p) store_row<T>(ko, dk[d][u], p.scale, d, p.D, h, key < p.Sk);
      if (p.dv.p) store_row<T>(vo, dv[d][u], 1.f, d, p.D, h, key < p.Sk);
    }
  }
}

template <class T, int DP, bool MASK>
void bwd(const AttnParams& p, hipStream_t st) {
  const unsigned nq = (unsigned)((p.M + 127) / 128 * (int64_t)p.B * p.Hkv);
  attn_dq_kernel<T, DP, 1, MASK><<<nq, 256, 0, st>>>(p);
  if (p.dk.p == nullptr && p.dv.p == nullptr) return;
  const unsigned nk = (unsigned)((p.Sk + 127) / 128 * (int64_t)p.B * p.Hkv);
  if (nk) attn_dkv_kernel<T, DP, 1, MASK><<<nk, 256, 0, st>>>(p);
}

template <class T, bool MASK>
void bwd_d(const AttnParams& p, hipStream_t st) {
  if (p.D <= 32) bwd<T, 32, MASK>(p, st);
  else if (p.D <= 64) bwd<T, 64, MASK>(p, st);
  else if (p.D <= 96) bwd<T, 96, MASK>(p, st);
  else bwd<T, 128, MASK>(p, st);
}

}  // namespace

int attn_bwd(const AttnParams& p, hipStream_t st) {
  if (p.D < 8 || p.D > 128 || p.D % 8 || p.M < 1 || p.Sk < 0) return 1;
  if ((p.M + 127) / 128 * (int64_t)p.B * p.Hkv > 0x7fffffff || (p.Sk + 127) / 128 * (int64_t)p.B * p.Hkv > 0x7fffffff)
    return 2;
  if (p.mask.bits) {
    if (p.fp16) bwd_d<FP16, true>(p, st);
    else bwd_d<BF16, true>(p, st);
  } else {
    if (p.fp16) bwd_d<FP16, false>(p, st);
    else bwd_d<BF16, false>(p, st);
  }
  return hipGetLastError() == hipSuccess ? 0 : 3;
}
