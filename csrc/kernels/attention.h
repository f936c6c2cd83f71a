// Shared parts of the attention kernels (attention.hip: forward, attention_bwd.hip: backward).
//
// Rows. The queries of the G = Hq / Hkv heads that share a key head are packed into one row axis, row r = i * G + g
// (query i, head hkv * G + g), M = Sq * G rows per (image, key head). One block then reads a key head once for all of
// them, gradients of a shared head are plain sums over its rows, and a few queries still fill a tile.
//
// MFMA layouts (v_mfma_f32_32x32x16): lane l = (c = l % 32, h = l / 32).
//   A operand: row c, reduction slots 8h + j       B operand: column c, reduction slots 8h + j       (j = 0..7)
//   result:    column c, element e (0..15) is row rowof(e) = (e & 3) + 8 * (e >> 2) + 4 * h
// Both products of a pair are arranged so that the first one's result IS the second one's B operand: elements
// 8s .. 8s + 7 of a result are 16 of its 32 rows (16s + {0-3, 8-11} + 4h), so with the A operand's slots taken in the
// same order (two transposing LDS reads of 4 rows each) no lane exchanges anything between the products.
#pragma once
#include "common.h"
#include "launch.h"

#include <type_traits>

namespace attn {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));

struct BF16 {
  static constexpr bool NARROW = false;         // fp32's exponents: nothing that is finite leaves the range
  static constexpr float UP = 0.f, P_UP = 0.f, REST = 1.f;
  static constexpr short INF = 0x7f80, ONE = 0x3f80;
  static CFL_DEVICE f16v mma(const s8v& a, const s8v& b, const f16v& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8v, a), __builtin_bit_cast(bf8v, b), c, 0, 0,
                                                   0);
  }
  static CFL_DEVICE uint32_t pack2(float a, float b) { return pack2bf(a, b); }
  static CFL_DEVICE float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static CFL_DEVICE float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
};

struct FP16 {
  // Its numbers end at 65,504 and lose bits below 2^-14, so the softmax weights are held times a power of two, in the
  // exponent, where it costs nothing. Forward 2^UP: weights down to 2^-21 of the row's largest keep their bits, and
  // those that lag the maximum (attention.hip SLACK) reach 2^15. Backward, where they are normalised, 2^P_UP: down to
  // 2^-28, and the largest is 2^14. lse2 is kept less P_UP, so that exp2(s - lse2) is P times it. What the rounding of
  // the output took away, at most 2^-11 of it, is kept times REST.
  static constexpr bool NARROW = true;
  static constexpr float UP = 7.f, P_UP = ATTN_FP16_P_UP, REST = 2048.f;
  static constexpr short INF = 0x7c00, ONE = 0x3c00;
  static CFL_DEVICE f16v mma(const s8v& a, const s8v& b, const f16v& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
  }
  static CFL_DEVICE uint32_t pack2(float a, float b) {
    const f32x2_t v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2v));
  }
  static CFL_DEVICE float lo(uint32_t w) { return (float)__builtin_bit_cast(h2v, w)[0]; }
  static CFL_DEVICE float hi(uint32_t w) { return (float)__builtin_bit_cast(h2v, w)[1]; }
};

// what a call allows: every key up to the image's length; the causal ones of those; a boolean mask, causal or not
enum Kind { ATTN_PLAIN = 0, ATTN_CAUSAL = 1, ATTN_MASK = 2 };

CFL_DEVICE int rowof(int e, int h) { return (e & 3) + 8 * (e >> 2) + 4 * h; }

CFL_DEVICE float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// 2^-P_UP
template <class T>
CFL_DEVICE constexpr float p_undo() { return T::NARROW ? 1.f / (1 << (int)T::P_UP) : 1.f; }

// value of the lane 32 away
CFL_DEVICE float other_half(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (threadIdx.x & 32) ? (unsigned)r[0] : (unsigned)r[1]);
}

// LDS image of a tile of token rows, DP 16-bit values each: row-major without padding (an LDS-DMA load writes 16
// bytes a lane, lanes in order), the 16-byte chunks of a row permuted by its index. 64 banks of 4 bytes serve a 256-byte
// line per cycle, so that
//   - a fragment read (ds_read_b128, 16 lanes a cycle: rows that differ modulo 16, one chunk) needs 16 rows to hold a
//     chunk in the 16 places of a line,
//   - a transposing read (ds_read_b64_tr_b16, 32 lanes a cycle: rows 4a .. 4a + 3, one 64-byte quarter) needs four rows in
//     a row to hold a quarter in the four quarters of a line.
// Rows of 64 and 192 bytes alternate the quarters by themselves. (A permutation made for lines of 128 bytes left half of
// the LDS cycles to conflicts.)
template <int DP>
CFL_DEVICE int swz(int row) {
  if (DP == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
  if (DP == 64) return ((row & 2) << 1) | ((row >> 2) & 3);
  return (row >> 2) & 3;
}
template <int DP>
CFL_DEVICE int lds_at(int row, int chunk) { return row * DP + ((chunk ^ swz<DP>(row)) << 3); }

// A operand of a product that reduces over d: fragment kk of the token row whose chunk h is at element `at` of the tile
// (lds_at of row c; rows 32 apart are permuted alike)
template <int DP>
CFL_DEVICE s8v frag_x(const bf16_t* tile, int at, int kk) {
  if (DP % 64 == 0) return *reinterpret_cast<const s8v*>(tile + (at ^ (kk << 4)));
  return *reinterpret_cast<const s8v*>(tile + (at ^ ((kk & 1) << 4)) + ((kk >> 1) << 5));
}

CFL_DEVICE s4v tr4(const bf16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4v __attribute__((address_space(3)))*)(p));
}

// A operand of a product that reduces over token rows: operand row = channel 32 * dt + c, slots = token rows
// row0 + {0-3, 8-11} + 4h (row0 a multiple of 16). Rows 16 apart are permuted alike, so a lane's addresses are two per
// channel tile (TransAt), formed once, and offsets that the compiler puts into the instructions.
template <int DP>
struct TransAt {
  int at[DP / 32][2];
  CFL_DEVICE explicit TransAt(int lane) {
    const int p = lane & 15, row = ((lane >> 5) << 2) + (p >> 2);
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
      const int col = 32 * dt + (lane & 16) + ((p & 3) << 2);
      at[dt][0] = lds_at<DP>(row, col >> 3) + (col & 7);
      at[dt][1] = lds_at<DP>(row + 8, col >> 3) + (col & 7);
    }
  }
};
template <int DP>
CFL_DEVICE s8v frag_t(const bf16_t* rows, const TransAt<DP>& t, int dt) {
  const s4v a = tr4(rows + t.at[dt][0]), b = tr4(rows + t.at[dt][1]);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// the same from the first channel tile's addresses: two registers where the second walk has no more
template <int DP>
CFL_DEVICE s8v frag_t2(const bf16_t* rows, const TransAt<DP>& t, int dt) {
  int x = t.at[0][0], y = t.at[0][1];
  asm volatile("" : "+v"(x), "+v"(y));                     // not formed ahead of the loop, for all tiles at once
  const int d = 32 * dt;
  const s4v a = tr4(rows + (DP % 64 == 0 ? x ^ d : x + d)), b = tr4(rows + (DP % 64 == 0 ? y ^ d : y + d));
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Values that are not finite, where pairs are not allowed. A product over token rows gives such a pair the factor 0, but
// 0 * inf and 0 * NaN are NaN: what a key holds where no query may attend it would show in every row. So after its walk
// a block with any mask looks whether its sums are finite (they are, in all but broken calls) and if not walks again
// with the operand's values replaced by 0 (clean), and those of pairs with a probability put back: `poison` adds +inf /
// -inf to the sums whose pairs of p > 0 in fp32 (the bits of `weighed`) hold +inf or NaN / -inf or NaN (both: NaN).
template <class T>
CFL_DEVICE s8v clean(const s8v& a, s8v& pos, s8v& neg) {
  s8v r;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const short m = (short)(a[j] & 0x7fff);
    const bool fin = m < T::INF, nan = m > T::INF;
    r[j] = fin ? a[j] : (short)0;
    pos[j] = !fin && (nan || a[j] >= 0) ? T::ONE : (short)0;
    neg[j] = !fin && (nan || a[j] < 0) ? T::ONE : (short)0;
  }
  return r;
}
template <class T>
CFL_DEVICE void poison(f16v& acc, const s8v& pos, const s8v& neg, uint32_t some) {
  s8v one;
#pragma unroll
  for (int j = 0; j < 8; ++j) one[j] = some >> j & 1 ? T::ONE : (short)0;
  f16v z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = 0.f;
  const f16v a = T::mma(pos, one, z);
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] += a[e] > 0.f ? INFINITY : 0.f;
  const f16v b = T::mma(neg, one, z);
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] -= b[e] > 0.f ? INFINITY : 0.f;
}
CFL_DEVICE uint32_t weighed(const f16v& p) {
  uint32_t r = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) r |= p[e] != 0.f ? 1u << e : 0;
  return r;
}
// 0, or NaN if any element is not finite
CFL_DEVICE float finite_sum(const f16v& v) {
  float t = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) t = fmaf(v[e], 0.f, t);
  return t;
}

// eight elements 8s .. 8s + 7 of a result, rounded to 16 bits: the B operand of the second product; and (FINE) what
// that rounding took away, rounded itself: as a second operand it leaves the product with little more than the error
// of fp32, for twice the second products (attn_fine).
template <class T, bool FINE>
struct Packed {
  s8v hi, lo;
  CFL_DEVICE void set(const f16v& v, int s) {
    u4v w, x = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a = v[8 * s + 2 * j], b = v[8 * s + 2 * j + 1];
      if (FINE) asm("" : "+v"(a), "+v"(b));                // a product, if it is one, not fused into the difference:
                                                           // the same bits in both walks
      w[j] = T::pack2(a, b);
      if (FINE) x[j] = T::pack2(a - T::lo(w[j]), b - T::hi(w[j]));
    }
    hi = __builtin_bit_cast(s8v, w);
    if (FINE) lo = __builtin_bit_cast(s8v, x);
  }
  CFL_DEVICE f16v mma(const s8v& a, f16v c) const {
    c = T::mma(a, hi, c);
    return FINE ? T::mma(a, lo, c) : c;
  }
};

// 32 channels 32 * dt .. + 31 of one token row per lane pair (c, c + 32): four quads each, exchanged between the
// halves so that a lane stores 16 contiguous bytes (lane half h: channels 16s + 8h .. + 7). rest: if given, what the
// rounding took away, times REST, rounded itself. zero: zeros are stored, whatever v holds.
template <class T>
CFL_DEVICE void store_row(bf16_t* row, const f16v& v, float mul, int dt, int D, int h, bool ok,
                          bf16_t* rest = nullptr, bool zero = false) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    unsigned w[4], x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = zero ? 0.f : v[8 * s + 2 * j] * mul, b = zero ? 0.f : v[8 * s + 2 * j + 1] * mul;
      w[j] = T::pack2(a, b);
      x[j] = T::pack2((a - T::lo(w[j])) * T::REST, (b - T::hi(w[j])) * T::REST);
    }
    const int d = 32 * dt + 16 * s + 8 * h;
    const auto p = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    const auto q = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    if (ok && d < D) *reinterpret_cast<uint4*>(row + d) = make_uint4(p[0], q[0], p[1], q[1]);
    if (rest != nullptr) {
      const auto y = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false);
      const auto z = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
      if (ok && d < D) *reinterpret_cast<uint4*>(rest + d) = make_uint4(y[0], z[0], y[1], z[1]);
    }
  }
}

// the same channels of a part of a sum, fp32, rows of DP
template <int DP>
CFL_DEVICE void store_part(float* row, const f16v& v, float mul, int dt, int h, bool ok) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (ok)
      *reinterpret_cast<float4*>(row + 32 * dt + 8 * q + 4 * h) =
          make_float4(v[4 * q] * mul, v[4 * q + 1] * mul, v[4 * q + 2] * mul, v[4 * q + 3] * mul);
}

// 16 bytes of the buffer at byte offset `off` -> LDS at the wave-uniform `lds` + 16 * lane; an offset past the range
// writes zeros. Inline asm: with the builtin the compiler orders every later LDS read behind all loads in flight. The
// caller waits with wait_vm() before the barrier that publishes the tile.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
CFL_DEVICE void dma16(const u4v& rs, uint32_t off, const bf16_t* lds) {
  const uint32_t a =
      __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)lds);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(a), "v"(off), "s"(rs)
               : "memory", "m0");
}
CFL_DEVICE void dma4(const u4v& rs, uint32_t off, const float* lds) {      // the same, 4 bytes a lane
  const uint32_t a =
      __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)lds);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(a), "v"(off), "s"(rs)
               : "memory", "m0");
}
#pragma clang diagnostic pop
CFL_DEVICE void wait_vm() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

CFL_DEVICE u4v rsrc(const void* base) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  u4v r;
  r.x = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  r.y = __builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xffffu));
  r.z = CFL_OOB - 1;
  r.w = 0x00020000;
  return r;
}

CFL_DEVICE int fdiv(int x, const FastDiv& f) { return fdiv32(x, f); }

// max of a value and the one 32 lanes away
CFL_DEVICE float max_halves(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}

// dS as fp16 operands. ds = p (dp - delta) is about |do| sqrt(D) / Sk: below the normal range (2^-14) where the gradients,
// sums of many, are in it, or above 65,504 where they are not. A lane holds ds of one row (dq) or one key (dk), and its
// sums are that row's or key's: so they carry a power of two, f = 2^ef, as a softmax carries its maximum, and are divided
// by it when they are stored. f starts so high that any ds which counts (2^-59 and more) brings it down; from then on the
// largest ds so far is 2^-4 to 2, and what two parts cannot hold is below 2^-21 of it: 8 comparisons for 16 of them, and a
// branch that is seldom taken (16 images x 8 heads x 1,024 tokens of 64 channels: dq 82 -> 84 us, dk and dv 125 -> 136).
template <class T>
struct Fit {
  float f, ef;
  CFL_DEVICE void start() {
    f = T::NARROW ? 0x1p46f : 1.f;                         // P has P_UP = 14 more
    ef = T::NARROW ? 46.f : 0.f;
  }
  // x: 16 of the lane's ds times f -> ds; lower(g): called where f falls, to scale the lane's sums by g (1: not this
  // lane's). What a lane does goes by its own values alone.
  template <bool FINE, class F>
  CFL_DEVICE void pack(f16v& x, Packed<T, FINE>* ds, const F& lower) {
    if constexpr (T::NARROW) {
      float mx = fabsf(x[0]);                              // NaN is passed over; an infinity stays one and lowers nothing
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, fabsf(x[e]));
      if (__any(mx >= 2.f)) {
        mx = max_halves(mx);
        const int down = mx >= 2.f && mx < INFINITY ? -3 - __builtin_amdgcn_frexp_expf(mx) : 0;
        const float g = ldexpf(1.f, down);
        f *= g;
        ef += (float)down;
        lower(g);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] *= g;
      }
    }
    ds[0].set(x, 0);
    ds[1].set(x, 1);
  }
  CFL_DEVICE float undo(float mul) const { return T::NARROW ? mul / f * p_undo<T>() : mul; }
};

// Which of `n` blocks of an (image, key head), which of bhn of those and which of `splits` parts this workgroup is.
// Where all blocks have the same work, XCD by XCD: the blocks that read one head's tokens share an L2 (16 heads, 4,096
// tokens, 128 channels, weights in one part as below: 292 us forward against 302). Where they differ (causal: block 0 must be the longest; lengths;
// masks by image) that order gives some XCDs the long ones: then block by block over all heads, the longest first, the
// heads rotated so that no XCD keeps one (the same shape, causal: 157 us against 199).
CFL_DEVICE void locate(const AttnParams& p, int n, int bhn, int splits, int& blk, int& bh, int& sp) {
  const int heads = bhn * splits;
  int rest;
  if (p.uneven) {
    blk = (int)blockIdx.x / heads;
    rest = ((int)blockIdx.x - blk * heads + blk) % heads;
  } else {
    const int lin = xcd_swizzle(blockIdx.x, gridDim.x);
    rest = lin / n;
    blk = lin - rest * n;
  }
  sp = rest / bhn;
  bh = rest - sp * bhn;
}

// Which tiles of a block's walk hold any allowed pair, and which only allowed ones: a byte a tile in LDS, filled from the
// mask's classes at the start. Tiles past the table count as partly allowed.
constexpr int MASK_TILES = 2048;
struct TileMask {
  const uint8_t* tab;            // MASK_TILES + 64 bytes
  bool part;                     // the tile that next() returned holds pairs that are not allowed

  // f(t, i0, i1, w0, w1): queries i0 .. i1 and mask words w0 .. w1 of tile t
  template <class F>
  CFL_DEVICE void fill(const AttnParams& p, int b, int hk, uint8_t* t8, int tiles, const F& f) {
    tab = t8;
    const int nib = (p.mask.rows + 31) >> 5, heads = p.mask.sh ? p.G : 1;
    // sb / sh count mask rows, `rows` of them for each (image, head) entry
    const int64_t lead = (b * p.mask.sb + (int64_t)hk * p.G * p.mask.sh) / p.mask.rows;
    for (int t = threadIdx.x; t < MASK_TILES + 64; t += blockDim.x) {
      bool any = false, all = true;
      if (t < tiles && t < MASK_TILES) {
        int i0, i1, w0, w1;
        f(t, i0, i1, w0, w1);
        const int b0 = p.mask.rows > 1 ? i0 >> 5 : 0, b1 = p.mask.rows > 1 ? i1 >> 5 : 0;
        // at most 128 queries and 128 keys: five class rows of two words, all of their loads under way together
        for (int g = 0; g < heads; ++g) {
          const uint8_t* c = p.mask.cls + (lead + g) * nib * p.mask.words;
          int k[10];
#pragma unroll
          for (int j = 0; j < 10; ++j) k[j] = c[(int64_t)imin(b0 + (j >> 1), b1) * p.mask.words + (j & 1 ? w1 : w0)];
#pragma unroll
          for (int j = 0; j < 10; ++j) {
            any |= k[j] != 0;
            all &= k[j] == 2;
          }
        }
      }
      t8[t] = any ? (all ? 2 : 1) : 0;
    }
    __syncthreads();
  }
  // first tile at or after t with an allowed pair, t1 if there is none before it
  CFL_DEVICE int next(int t, int t1) {
    part = true;
    while (t < t1) {
      if (t >= MASK_TILES) return t;
      const int k = tab[t + (int)(threadIdx.x & 63)];
      const unsigned long long live = __ballot(k != 0), whole = __ballot(k == 2);
      if (live) {
        const int n = __builtin_ctzll(live);
        part = !((whole >> n) & 1);
        return imin(t + n, t1);
      }
      t = imin(t + 64, imax(t + 1, MASK_TILES));
    }
    return t1;
  }
};

}  // namespace attn
