// Attention over the 8-bit key/value cache: what its two kernels share
// (rnsmx_kv_rows.hip for few rows, rnsmx_kv_tiles.hip for prompts).
#pragma once

#include "rnsmx_kv.hpp"

namespace rnsmx {

// Two stored bytes (code + 128) as halves code / 512: a byte alone in a half's
// low bits is that many 2^-24, so one multiply by 2^15 and one subtraction of
// 128 / 512 give it, both exact.
template <int LO, int HI>
__device__ __forceinline__ h16x2 kv_halves(uint32_t lo, uint32_t hi) {
  constexpr uint32_t sel = LO | 0x0C00u | (static_cast<uint32_t>(4 + HI) << 16) | 0x0C000000u;
  const h16x2 u = __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(hi, lo, sel));
  const h16x2 up = {static_cast<_Float16>(32768.0f), static_cast<_Float16>(32768.0f)};
  const h16x2 off = {static_cast<_Float16>(-0.25f), static_cast<_Float16>(-0.25f)};
  return __builtin_elementwise_fma(u, up, off);
}
constexpr float kKvUnit = 512.0f;

__device__ __forceinline__ h16x8 kv_join(h16x2 a, h16x2 b, h16x2 c, h16x2 d) {
  return h16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Eight consecutive codes of a row.
__device__ __forceinline__ h16x8 kv_row8(uint32_t w0, uint32_t w1) {
  return kv_join(kv_halves<0, 1>(w0, w0), kv_halves<2, 3>(w0, w0), kv_halves<0, 1>(w1, w1), kv_halves<2, 3>(w1, w1));
}

constexpr float kKvLog2e = 1.44269504088896340736f;
// A row's reference is put 10 below its largest weight's exponent and follows
// when one passes 15.75: weights stay below 2^15.75 (float16 ends at 2^16), and
// those 2^-24 of the largest keep all their bits, as float16 does from 2^-14 on.
// What is far below the largest matters where that has small values: 4095 tokens
// 16 below one whose codes are zero come out within 1e-3 of themselves so, and
// with the largest at 2^4 (limit 2^12) within 8e-2.  The room above decides how
// often rows are rescaled: one prompt of 2048, 32 heads of 128, in short runs takes
// 67.8 us with 8 of it, 68.6 so, 71.2 with 4.
constexpr float kKvBelow = 10.0f, kKvAbove = 15.75f;

// 16-bit calls round their weights to float16's 11 bits, three more than bfloat16
// outputs keep and as many as float16's: against 64 bits their error is 1 % and 30 %
// above that of the output's rounding alone.  A second half would cost half the
// products again (decode 200 us to 214, one token of 131072 56.8 to 58.8, a prompt
// of 2048 71 to 92); float32 queries have it.
//
// A weight's exponent is fma(product, page's factor, page's part - reference): the
// product is not rounded, its row's largest was when it became the reference, and
// past 2^27 that half of a last place alone takes a weight past float16.  Rows whose
// reference has 2^20 (a last place of 2^-3) and more, and a wave's others with them,
// take the product as the reference had it, rounded, and the difference before the
// page's part.
constexpr float kKvFar = 1048576.0f;
__device__ __forceinline__ float kv_apart(float product, float factor, float reference) {
  float x = product * factor;
  asm("" : "+v"(x));  // kept from joining the subtraction
  return x - reference;
}

// Float32 calls have weights in two halves: h, and what is left of w times 2^11,
// as large as h was, against codes times 2^-11, which float16 holds exactly (code
// 2^-20).  22 bits down to 2^-24 of the largest, 11 down to 2^-35; at the same
// unit as h it would end where h does.
constexpr float kKvLow = 2048.0f;
__device__ __forceinline__ _Float16 kv_low(float w, _Float16 h) {
  return static_cast<_Float16>((w - static_cast<float>(h)) * kKvLow);
}
__device__ __forceinline__ h16x8 kv_low_codes(h16x8 v) { return v * static_cast<_Float16>(1.0f / kKvLow); }

struct F32x2 {
  float x, y;
};

// A row's queries as float32, S groups of 8 from column first(s) on, zeros past
// the head dimension.  Every load is issued before the first is waited for: no
// branch but on what is one for the call, columns past the end read the last.
template <int S, bool SPLIT, typename F>
__device__ __forceinline__ void kv_query(float (&x)[S][8], const KvAttnArgs &a, int64_t at, F &&first) {
  const int32_t dim = a.b.dim;
  if (a.vec) {
    kv_for<S>([&](auto G) {
      constexpr int g = G;
      const int32_t d = min(first(G), dim - 8);
      if constexpr (SPLIT) {
        const f32x4 *p = reinterpret_cast<const f32x4 *>(static_cast<const float *>(a.q) + at + d);
        const f32x4 lo = p[0], hi = p[1];
        kv_for<4>([&](auto J) {
          constexpr int j = J;
          x[g][j] = lo[j];
          x[g][j + 4] = hi[j];
        });
      } else {
        // two halves to a word until all are here
        const f32x4 w = *reinterpret_cast<const f32x4 *>(static_cast<const uint16_t *>(a.q) + at + d);
        kv_for<4>([&](auto J) {
          constexpr int j = J;
          x[g][j] = w[j];
        });
      }
    });
  } else {
    kv_for<S>([&](auto G) {
      constexpr int g = G;
      kv_for<8>([&](auto J) {
        constexpr int j = J;
        const int64_t i = at + min(first(G) + j, dim - 1);
        if constexpr (SPLIT) {
          x[g][j] = static_cast<const float *>(a.q)[i];
        } else {
          const uint32_t bits = static_cast<const uint16_t *>(a.q)[i];
          x[g][j / 2] = __uint_as_float(j % 2 ? __float_as_uint(x[g][j / 2]) | bits << 16 : bits);
        }
      });
    });
  }
  kv_for<S>([&](auto G) {
    constexpr int g = G;
    if constexpr (!SPLIT) {
      uint32_t w[4];
      kv_for<4>([&](auto J) { w[J] = __float_as_uint(x[g][J]); });
      if (a.dtype == RNSMX_FLOAT16) {
        kv_for<8>([&](auto J) {
          constexpr int j = J;
          x[g][j] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[j / 2] >> (16 * (j % 2)))));
        });
      } else {
        kv_for<8>([&](auto J) {
          constexpr int j = J;
          x[g][j] = __uint_as_float(j % 2 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
        });
      }
    }
    kv_for<8>([&](auto J) {
      constexpr int j = J;
      x[g][j] = first(G) + j < dim ? x[g][j] : 0.0f;
    });
  });
}

// The power of two that brings a row's largest query below 2^15 (as its
// exponent); a row of zeros or with an infinity stays as it is.
__device__ __forceinline__ int32_t kv_query_exponent(float top) {
  return max(top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 15 : 0, -120);
}

// Eight tokens of a mask's row from t on, as they are stored: loads that do not
// depend on each other or on what is seen.  Tokens in a row of a mask that covers
// the step up to `end` come in one load or two; else one by one, the last
// column's in the place of those past it (0 of a mask without columns).
__device__ __forceinline__ void kv_mask_load(uint32_t (&m)[8], const KvAttnArgs &a, int64_t row, int32_t q_head, int32_t t,
                                             int32_t end) {
  const int64_t at = row * a.mask_rs + static_cast<int64_t>(q_head) * a.mask_hs;
  const int32_t size = a.mask_dtype == RNSMX_INT8 ? 1 : a.mask_dtype == RNSMX_FLOAT32 ? 4 : 2;
  if (a.mask_ts == 1 && end <= a.mask_len) {
    const uint8_t *p = static_cast<const uint8_t *>(a.mask) + (at + t) * size;
    uint32_t w[8];
    if (size == 1) {
      __builtin_memcpy(w, p, 8);
      kv_for<8>([&](auto J) { m[J] = w[J / 4] >> (8 * (J % 4)) & 0xFFu; });
    } else if (size == 2) {
      __builtin_memcpy(w, p, 16);
      kv_for<8>([&](auto J) { m[J] = w[J / 2] >> (16 * (J % 2)) & 0xFFFFu; });
    } else {
      __builtin_memcpy(m, p, 32);
    }
    return;
  }
  auto load = [&](auto *p) {
    kv_for<8>([&](auto J) {
      constexpr int j = J;
      m[j] = p[at + static_cast<int64_t>(min(t + j, a.mask_len - 1)) * a.mask_ts];
    });
  };
  if (a.mask_len <= 0)
    kv_for<8>([&](auto J) { m[J] = 0; });
  else if (size == 1)
    load(static_cast<const uint8_t *>(a.mask));
  else if (size == 4)
    load(static_cast<const uint32_t *>(a.mask));
  else
    load(static_cast<const uint16_t *>(a.mask));
}
// Which of eight tokens from t on the mask shows (bit j: token t + j); an additive
// mask's values go onto the scores.  `end` as kv_mask_load had it.
__device__ __forceinline__ uint32_t kv_mask_shows(const KvAttnArgs &a, const uint32_t (&m)[8], int32_t t, int32_t end,
                                                  float (&x)[8]) {
  uint32_t shown = 0;
  if (a.mask_dtype == RNSMX_INT8) {
    kv_for<8>([&](auto J) { shown |= m[J] != 0 ? 1u << J : 0u; });
  } else {
    float v[8];
    if (a.mask_dtype == RNSMX_FLOAT32)
      kv_for<8>([&](auto J) { v[J] = __uint_as_float(m[J]); });
    else if (a.mask_dtype == RNSMX_FLOAT16)
      kv_for<8>([&](auto J) { v[J] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(m[J]))); });
    else
      kv_for<8>([&](auto J) { v[J] = kv_bf16(static_cast<uint16_t>(m[J])); });
    kv_for<8>([&](auto J) {
      x[J] += v[J];
      shown |= v[J] != -INFINITY ? 1u << J : 0u;
    });
  }
  if (end > a.mask_len) shown &= (1u << min(max(a.mask_len - t, 0), 8)) - 1u;
  return shown;
}

// The first token that a row at position p sees.  A row before its sequence's
// first token lies below zero, where p + 1 - window would pass 32 bits.
__device__ __forceinline__ int32_t kv_window_begin(const KvAttnArgs &a, int32_t p) {
  return a.window > 0 ? max(p + 1, a.window) - a.window : 0;
}

// Where a row at position p sees tokens of its sequence up to.
__device__ __forceinline__ int32_t kv_causal_end(const KvAttnArgs &a, const KvSeq &q, int32_t p) {
  return a.causal ? min(p + 1, q.len) : q.len;
}

// Zeros for a sequence's rows past max_rows.
__device__ __forceinline__ void kv_zero_rows(const KvAttnArgs &a, const KvSeq &q, int32_t head) {
  const int64_t wide = static_cast<int64_t>(a.by_group.d) * a.b.dim, count = (q.all - q.n) * wide;
  for (int64_t i = threadIdx.x; i < count; i += blockDim.x) {
    const int64_t r = i / wide;
    kv_store(a.out, (q.row + q.n + r) * a.q_heads * a.b.dim + head * wide + (i - r * wide), a.dtype, 0.0f);
  }
}

// Bits of those of eight tokens from t on that lie in [begin, end).
__device__ __forceinline__ uint32_t kv_between(int32_t t, int32_t begin, int32_t end) {
  const uint32_t below = (1u << min(max(end - t, 0), 8)) - 1u, before = (1u << min(max(begin - t, 0), 8)) - 1u;
  return below & ~before;
}

// One candidate (x, lv) for a row's reference against another, e and e2 being
// how far each lies above the present one: of those that pass kKvAbove the one
// with the larger sum, by the differences, as sums lose what is less than a last
// place of x; of equals the larger x, then the larger lv, so that lanes that exchange
// theirs take the same one.
template <bool MASK>
__device__ __forceinline__ void kv_higher(float &e, float &x, float &lv, float e2, float x2, float lv2) {
  constexpr float kNat = MASK ? kKvLog2e : 1.0f;
  const float more = (x2 - x) * kNat + (lv2 - lv);
  const bool take = !(e > kKvAbove) ? e2 > kKvAbove
                                    : (e2 > kKvAbove && (more > 0.0f || (more == 0.0f && (x2 > x || (x2 == x && lv2 > lv)))));
  e = take ? e2 : e;
  x = take ? x2 : x;
  lv = take ? lv2 : lv;
}

// Sums against different references: the higher of two, and what sums against
// one are multiplied by to be against another.  Not-a-numbers of a part without
// a reference go through the zero.
template <bool MASK>
__device__ __forceinline__ void kv_reference(float &mx, float &ml, float mx2, float ml2) {
  constexpr float kNat = MASK ? kKvLog2e : 1.0f;
  const float more = (mx2 - mx) * kNat + (ml2 - ml);
  const bool take =
      mx2 > -INFINITY && (!(mx > -INFINITY) || more > 0.0f || (more == 0.0f && (mx2 > mx || (mx2 == mx && ml2 > ml))));
  mx = take ? mx2 : mx;
  ml = take ? ml2 : ml;
}
template <bool MASK>
__device__ __forceinline__ float kv_factor(float mx, float ml, float to_mx, float to_ml) {
  constexpr float kNat = MASK ? kKvLog2e : 1.0f;
  return mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((mx - to_mx) * kNat + (ml - to_ml));
}

}  // namespace rnsmx
