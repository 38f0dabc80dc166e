// Attention of few query rows over the 8-bit key/value cache (built once per
// row size, RNSMX_KV_DIM).
#include "rnsmx_kv.hpp"

namespace rnsmx {

// v_mfma_f32_16x16x32_f16: lane l feeds row (l & 15) of A and column (l & 15)
// of B, both at k = 8 * (l >> 4) + 0..7, and gets rows 4 * (l >> 4) + 0..3 of
// column (l & 15).
__device__ __forceinline__ f32x4 kv_mfma(h16x8 a, h16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

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
// A row's reference is put 4 below its largest weight's exponent and follows
// when one passes 12: weights stay below 2^12 (float16 ends at 2^16), and those
// 2^-18 of the largest keep all their bits.
constexpr float kKvBelow = 4.0f, kKvAbove = 12.0f;

struct F32x2 {
  float x, y;
};

// A workgroup of four waves for 16 query rows (token-major over the heads of a
// group) of one sequence and key/value head, and one chunk of its tokens.  A
// wave takes 32 tokens a step:
//   S^T = K Q^T  two 16 x 16 tiles, the token of tile i, row r being 8 (r / 4) + 4 i + r % 4,
//                so that lane group g holds the products of tokens 8 g .. 8 g + 7
//   O^T += V^T P^T  P in the registers and order that S^T left it in
// Codes go into the products as they are (code / 512, exact in float16); a
// page's key scale multiplies its products, its value scale is an exponent
// added to them: with lv = log2(value scale),
//   w = 2^(x - mx + lv - ml),  O += w code,  l += w 2^(ml - lv) = 2^(x - mx)
// where x is the product in powers of two and (mx, ml) a row's reference.
template <int DT, bool SPLIT, bool MASK>
__global__ __launch_bounds__(256, 2) void kv_rows_kernel(const KvAttnArgs a) {
  constexpr int C64 = DT / 64, C32 = DT / 32 % 2;  // 64-value chunks of a row, and whether 32 are left
  constexpr int KS = DT / 32;                      // products' steps
  constexpr int VW = DT / 16;                      // bytes of a token that a lane takes: value tiles
  constexpr int QN = SPLIT ? 2 : 1;
  __shared__ float part_o[4][kKvRowTile][DT + 4];
  __shared__ float part_m[4][kKvRowTile], part_l[4][kKvRowTile], part_f[4][kKvRowTile], total[kKvRowTile];
  __shared__ int32_t last;

  const KvBatchArgs &b = a.b;
  int32_t id = blockIdx.x;
  const int32_t split = id % a.splits;
  const int32_t task = id / a.splits;
  id = task;
  const int32_t tile = id % a.row_tiles;
  id /= a.row_tiles;
  const int32_t head = id % b.heads, seq = id / b.heads;
  const KvSeq q = kv_seq(b, seq);
  const int32_t rows = q.n * a.group;
  if (tile * kKvRowTile >= rows) return;
  const int32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t col = lane & 15, g = lane >> 4;
  const int32_t row = min(tile * kKvRowTile + col, rows - 1);
  const int32_t t_row = row / a.group, q_head = head * a.group + (row - t_row * a.group);
  const int32_t base = q.len - q.n;  // position of the sequence's first row
  const int32_t end_row = a.causal ? base + t_row + 1 : q.len;
  const int32_t begin_row = a.window > 0 ? max(base + t_row + 1 - a.window, 0) : 0;
  const int32_t t_first = tile * kKvRowTile / a.group, t_last = min(tile * kKvRowTile + 15, rows - 1) / a.group;
  const int32_t hi = max(a.causal ? base + t_last + 1 : q.len, 0);
  const int32_t lo = a.window > 0 ? max(base + t_first + 1 - a.window, 0) & ~31 : 0;
  const int32_t full_hi = a.causal ? base + t_first + 1 : q.len;                       // seen by every row: below it
  const int32_t full_lo = a.window > 0 ? max(base + t_last + 1 - a.window, 0) : 0;     // and from it on
  const int32_t active = max((hi - lo + a.chunk - 1) / a.chunk, 1);
  if (split >= active) return;
  const int32_t c0 = lo + split * a.chunk, c1 = min(hi, c0 + a.chunk);

  // queries, scaled by a power of two each to lie below 2^15
  h16x8 qf[QN][KS];
  float q_scale;
  {
    float x[KS][8];
    const int64_t at = static_cast<int64_t>(q.row + t_row) * a.q_rs + static_cast<int64_t>(q_head) * a.q_hs;
    float top = 0.0f;
    kv_for<KS>([&](auto S_) { constexpr int S = decltype(S_)::value;
      // lane group g takes bytes 16 g .. of a 64-value chunk, the first eight in its first step
      const int32_t d = S < 2 * C64 ? 64 * (S / 2) + 16 * g + 8 * (S % 2) : 64 * C64 + 8 * g;
      if (a.vec && d < b.dim) {
        if (a.dtype == RNSMX_FLOAT32) {
          const f32x4 *p = reinterpret_cast<const f32x4 *>(static_cast<const float *>(a.q) + at + d);
          kv_for<4>([&](auto J_) { constexpr int J = decltype(J_)::value; x[S][J] = p[0][J], x[S][J + 4] = p[1][J]; });
        } else {
          const u32x4 w = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(a.q) + at + d);
          kv_for<8>([&](auto J_) { constexpr int J = decltype(J_)::value;
            const uint16_t bits = static_cast<uint16_t>(w[J / 2] >> (16 * (J % 2)));
            x[S][J] = a.dtype == RNSMX_FLOAT16 ? static_cast<float>(__builtin_bit_cast(_Float16, bits)) : kv_bf16(bits);
          });
        }
      } else {
        kv_for<8>([&](auto J_) { constexpr int J = decltype(J_)::value; x[S][J] = d + J < b.dim ? kv_load(a.q, at + d + J, a.dtype) : 0.0f; });
      }
      kv_for<8>([&](auto J_) { constexpr int J = decltype(J_)::value; top = fmaxf(top, fabsf(x[S][J])); });
    });
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    // top in [2^(e-1), 2^e); a row of zeros or with an infinity stays as it is
    int32_t e = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;
    e = max(e, -120);
    kv_for<KS>([&](auto S_) { constexpr int S = decltype(S_)::value;
      kv_for<8>([&](auto J_) { constexpr int J = decltype(J_)::value;
        const float v = ldexpf(x[S][J], -e);
        const _Float16 h = static_cast<_Float16>(v);
        qf[0][S][J] = h;
        if constexpr (SPLIT) qf[1][S][J] = static_cast<_Float16>(v - static_cast<float>(h));
      });
    });
    q_scale = ldexpf(a.scale * kKvUnit, e);
    if constexpr (!MASK) q_scale *= kKvLog2e;
  }

  f32x4 o[VW];
  kv_for<VW>([&](auto I_) { constexpr int I = decltype(I_)::value; o[I] = f32x4{0.0f, 0.0f, 0.0f, 0.0f}; });
  float mx = -INFINITY, ml = 0.0f, sum = 0.0f;

  struct Step {
    u32x4 k[2][C64 > 0 ? C64 : 1];
    u32x2 k8[2];
    uint32_t v[8][VW / 4 + 1];
    float ks, vs;
    bool there;
  };
  // page numbers of the lane's key row and of its eight tokens
  const int32_t key_token = 8 * (col >> 2) + (col & 3);  // of tile 0; tile 1: 4 tokens on
  auto pages_of = [&](int32_t t0, int32_t &pk, int32_t &pv) {
    const int32_t *row_table = b.table + seq * b.table_stride;
    pk = row_table[min((t0 + key_token) >> b.log_page, b.table_width - 1)];
    pv = row_table[min((t0 + 8 * g) >> b.log_page, b.table_width - 1)];
  };
  const int32_t in_page = (1 << b.log_page) - 1;
  auto load_step = [&](Step &s, int32_t t0, int32_t pk, int32_t pv) {
    s.there = static_cast<uint32_t>(pv) < static_cast<uint32_t>(b.blocks);
    const int64_t slot_k = static_cast<int64_t>(min(max(pk, 0), b.blocks - 1)) * b.heads + head;
    const int64_t slot_v = static_cast<int64_t>(s.there ? pv : 0) * b.heads + head;
    const uint8_t *kp = b.k + ((slot_k << b.log_page) + ((t0 + key_token) & in_page)) * DT;
    const uint8_t *vp = b.v + ((slot_v << b.log_page) + ((t0 + 8 * g) & in_page)) * DT;
    kv_for<2>([&](auto I_) { constexpr int I = decltype(I_)::value;
      kv_for<C64>([&](auto C_) { constexpr int C = decltype(C_)::value;
        s.k[I][C] = *reinterpret_cast<const u32x4 *>(kp + I * 4 * DT + C * 64 + 16 * g);
      });
      if constexpr (C32 != 0) s.k8[I] = *reinterpret_cast<const u32x2 *>(kp + I * 4 * DT + C64 * 64 + 8 * g);
    });
    kv_for<8>([&](auto J_) { constexpr int J = decltype(J_)::value;
      const uint8_t *p = vp + J * DT;
      // pieces of 16, 8, 4 and 2 bytes a lane, VW in all, each over 16 lanes
      constexpr int W16 = VW / 16, W8 = VW / 8 % 2, W4 = VW / 4 % 2, W2 = VW / 2 % 2;
      if constexpr (W16 != 0) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(p + 16 * col);
        kv_for<4>([&](auto W_) { constexpr int W = decltype(W_)::value; s.v[J][W] = w[W]; });
      }
      if constexpr (W8 != 0) {
        const u32x2 w = *reinterpret_cast<const u32x2 *>(p + 256 * W16 + 8 * col);
        kv_for<2>([&](auto W_) { constexpr int W = decltype(W_)::value; s.v[J][4 * W16 + W] = w[W]; });
      }
      if constexpr (W4 != 0)
        s.v[J][4 * W16 + 2 * W8] = *reinterpret_cast<const uint32_t *>(p + 256 * W16 + 128 * W8 + 4 * col);
      if constexpr (W2 != 0)
        s.v[J][4 * W16 + 2 * W8 + W4] =
            *reinterpret_cast<const uint16_t *>(p + 256 * W16 + 128 * W8 + 64 * W4 + 2 * col);
    });
    const F32x2 sc = *reinterpret_cast<const F32x2 *>(b.scales + slot_v * 2);
    s.ks = sc.x;
    s.vs = sc.y;
  };

  auto compute = [&](const Step &s, int32_t t0) {
    f32x4 acc[2];
    kv_for<2>([&](auto I_) { constexpr int I = decltype(I_)::value;
      acc[I] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      kv_for<KS>([&](auto S_) { constexpr int S = decltype(S_)::value;
        h16x8 k;
        if constexpr (S < 2 * C64)
          k = kv_row8(s.k[I][S / 2][2 * (S % 2)], s.k[I][S / 2][2 * (S % 2) + 1]);
        else
          k = kv_row8(s.k8[I][0], s.k8[I][1]);
        kv_for<QN>([&](auto N_) { constexpr int N = decltype(N_)::value; acc[I] = kv_mfma(k, qf[N][S], acc[I]); });
      });
    });
    const float c = q_scale * s.ks, lv = __builtin_amdgcn_logf(s.vs);
    const int32_t t8 = t0 + 8 * g;
    // what every row of the tile sees needs no look at single tokens
    const bool full = !MASK && t0 >= full_lo && t0 + 32 <= full_hi && __all(s.there);
    float w[8];
    uint32_t seen = 0xFFu;
    float xm;
    if (full) {
      kv_for<8>([&](auto J_) { constexpr int J = decltype(J_)::value; w[J] = acc[J / 4][J % 4]; });
      xm = w[0];
      kv_for<7>([&](auto J_) { constexpr int J = decltype(J_)::value; xm = fmaxf(xm, w[J + 1]); });
      xm *= c;
    } else {
      seen = 0;
      kv_for<8>([&](auto J_) { constexpr int J = decltype(J_)::value;
        if (s.there && t8 + J < end_row && t8 + J >= begin_row) seen |= 1u << J;
      });
      xm = -INFINITY;
      kv_for<8>([&](auto J_) { constexpr int J = decltype(J_)::value;
        float x = acc[J / 4][J % 4];
        if constexpr (MASK) {
          x *= c;
          const int32_t t = t8 + J;
          if (t >= a.mask_len) seen &= ~(1u << J);
          if (seen >> J & 1u) {
            const int64_t at = static_cast<int64_t>(q.row + t_row) * a.mask_rs + static_cast<int64_t>(q_head) * a.mask_hs +
                               static_cast<int64_t>(t) * a.mask_ts;
            if (a.mask_dtype == RNSMX_INT8) {
              if (static_cast<const uint8_t *>(a.mask)[at] == 0) seen &= ~(1u << J);
            } else {
              const float m = kv_load(a.mask, at, a.mask_dtype);
              if (m == -INFINITY) seen &= ~(1u << J);
              x += m;
            }
          }
        }
        w[J] = x;
        if (seen >> J & 1u) xm = fmaxf(xm, x);
      });
      if constexpr (!MASK) {
        // no token seen leaves minus infinity, whatever the scale
        xm = seen ? xm * c : -INFINITY;
      }
    }
    // exponents are (x - mx) + lv - ml, in powers of two; x of masked calls is natural
    constexpr float kNat = MASK ? kKvLog2e : 1.0f;
    const float em = (xm - mx) * kNat + (lv - ml);
    if (__any(em > kKvAbove)) {
      float best = em, bx = xm, bl = lv;
      kv_for<2>([&](auto I_) { constexpr int I = decltype(I_)::value;
        const float e2 = __shfl_xor(best, 16 << I), x2 = __shfl_xor(bx, 16 << I), l2 = __shfl_xor(bl, 16 << I);
        // the pair with the larger sum, of equals the larger x, then the larger lv: all four lane groups take the same one
        const float s1 = bx * kNat + bl, s2 = x2 * kNat + l2;
        const bool take = !(best > kKvAbove) ? e2 > kKvAbove : (e2 > kKvAbove && (s2 > s1 || (s2 == s1 && (x2 > bx || (x2 == bx && l2 > bl)))));
        best = take ? e2 : best;
        bx = take ? x2 : bx;
        bl = take ? l2 : bl;
      });
      if (best > kKvAbove) {
        const float nl = bl - kKvBelow;
        const float fx = __builtin_amdgcn_exp2f((mx - bx) * kNat);
        const float fo = __builtin_amdgcn_exp2f((mx - bx) * kNat + (ml - nl));
        sum *= fx;
        kv_for<VW>([&](auto I_) { constexpr int I = decltype(I_)::value; kv_for<4>([&](auto T_) { constexpr int T = decltype(T_)::value; o[I][T] *= fo; }); });
        mx = bx;
        ml = nl;
      }
    }
    float part = 0.0f;
    if (full) {
      const float off = lv - ml - mx;
      kv_for<8>([&](auto J_) { constexpr int J = decltype(J_)::value;
        w[J] = __builtin_amdgcn_exp2f(fmaf(w[J], c, off));
        part += w[J];
      });
    } else {
      kv_for<8>([&](auto J_) { constexpr int J = decltype(J_)::value;
        const float x = MASK ? w[J] : w[J] * c;
        const float e = (x - mx) * kNat + (lv - ml);
        w[J] = seen >> J & 1u ? __builtin_amdgcn_exp2f(e) : 0.0f;
        part += w[J];
      });
    }
    // a group of tokens that none is seen of may lie in a page that holds anything
    sum = seen ? fmaf(part, __builtin_amdgcn_exp2f(ml - lv), sum) : sum;
    h16x8 p[QN];
    kv_for<8>([&](auto J_) { constexpr int J = decltype(J_)::value;
      const _Float16 h = static_cast<_Float16>(w[J]);
      p[0][J] = h;
      if constexpr (SPLIT) p[1][J] = static_cast<_Float16>(w[J] - static_cast<float>(h));
    });
    kv_for<VW>([&](auto I_) { constexpr int I = decltype(I_)::value;
      constexpr int word = I / 4, byte = I % 4;
      const h16x8 v = kv_join(kv_halves<byte, byte>(s.v[0][word], s.v[1][word]), kv_halves<byte, byte>(s.v[2][word], s.v[3][word]),
                              kv_halves<byte, byte>(s.v[4][word], s.v[5][word]), kv_halves<byte, byte>(s.v[6][word], s.v[7][word]));
      kv_for<QN>([&](auto N_) { constexpr int N = decltype(N_)::value; o[I] = kv_mfma(v, p[N], o[I]); });
    });
  };

  // two steps of loads in flight, page numbers a step further ahead
  {
    Step s0, s1;
    int32_t pk, pv;
    int32_t t0 = c0 + 32 * wave;
    if (t0 < c1) {
      pages_of(t0, pk, pv);
      load_step(s0, t0, pk, pv);
      pages_of(t0 + kKvChunkUnit, pk, pv);
      while (true) {
        if (t0 + kKvChunkUnit < c1) load_step(s1, t0 + kKvChunkUnit, pk, pv);
        pages_of(t0 + 2 * kKvChunkUnit, pk, pv);
        compute(s0, t0);
        t0 += kKvChunkUnit;
        if (t0 >= c1) break;
        if (t0 + kKvChunkUnit < c1) load_step(s0, t0 + kKvChunkUnit, pk, pv);
        pages_of(t0 + 2 * kKvChunkUnit, pk, pv);
        compute(s1, t0);
        t0 += kKvChunkUnit;
        if (t0 >= c1) break;
      }
    }
  }

  // the four waves' parts: natural units of the codes from here on
  constexpr float kNat = MASK ? kKvLog2e : 1.0f;
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  const float unit = __builtin_amdgcn_exp2f(ml) * kKvUnit;
  kv_for<VW>([&](auto I_) { constexpr int I = decltype(I_)::value;
    // value tile I of a piece of W bytes a lane holds its columns W r + I
    constexpr int W16 = VW / 16, W8 = VW / 8 % 2, W4 = VW / 4 % 2;
    constexpr int P16 = 16 * W16, P8 = P16 + 8 * W8, P4 = P8 + 4 * W4;
    constexpr int width = I < P16 ? 16 : I < P8 ? 8 : I < P4 ? 4 : 2;
    constexpr int first = I < P16 ? 0 : I < P8 ? P16 : I < P4 ? P8 : P4;
    kv_for<4>([&](auto T_) { constexpr int T = decltype(T_)::value;
      part_o[wave][col][16 * first + width * (4 * g + T) + (I - first)] = o[I][T] * unit;
    });
  });
  if (g == 0) {
    part_m[wave][col] = mx;
    part_l[wave][col] = sum;
  }
  __syncthreads();
  // rows' reference and sum over the waves
  if (tid < kKvRowTile) {
    float m = part_m[0][tid];
    kv_for<3>([&](auto W_) { constexpr int W = decltype(W_)::value; m = fmaxf(m, part_m[W + 1][tid]); });
    float l = 0.0f;
    kv_for<4>([&](auto W_) { constexpr int W = decltype(W_)::value;
      const float mw = part_m[W][tid];
      const float f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((mw - m) * kNat);
      part_f[W][tid] = f;
      l += part_l[W][tid] * f;
    });
    part_m[0][tid] = m;
    total[tid] = l;
  }
  __syncthreads();
  const int32_t live = min(rows - tile * kKvRowTile, kKvRowTile);
  auto row_out = [&](int32_t r) {
    const int32_t i = tile * kKvRowTile + r, t = i / a.group;
    return (static_cast<int64_t>(q.row + t) * a.q_heads + head * a.group + (i - t * a.group)) * b.dim;
  };
  auto joined = [&](int32_t r, int32_t d) {
    float v = 0.0f;
    kv_for<4>([&](auto W_) { constexpr int W = decltype(W_)::value; v += part_o[W][r][d] * part_f[W][r]; });
    return v;
  };
  if (active == 1) {
    for (int32_t i = tid; i < live * DT; i += 256) {
      const int32_t r = i / DT, d = i - r * DT;
      const float l = total[r];
      if (d < b.dim) kv_store(a.out, row_out(r) + d, a.dtype, l == 0.0f ? 0.0f : joined(r, d) / l);
    }
    return;
  }

  // A split's part goes to its place in the workspace; the workgroup that
  // draws a task's last ticket joins them.  Written and read with agent-scope
  // accesses, which go past the XCDs' own caches, the stores complete before
  // the ticket is drawn; no workgroup waits for another.
  constexpr int64_t kPart = static_cast<int64_t>(kKvRowTile) * (DT + 2);
  float *to = a.partial + (static_cast<int64_t>(task) * a.splits + split) * kPart;
  for (int32_t i = tid; i < live * DT; i += 256) {
    const int32_t r = i / DT, d = i - r * DT;
    __hip_atomic_store(to + i, joined(r, d), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (tid < kKvRowTile) {
    __hip_atomic_store(to + kKvRowTile * DT + tid, part_m[0][tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(to + kKvRowTile * DT + 16 + tid, total[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const uint32_t old = __hip_atomic_fetch_add(a.tickets + task, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = old == static_cast<uint32_t>(active - 1);
    if (last) __hip_atomic_store(a.tickets + task, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  asm volatile("" ::: "memory");
  const float *from = a.partial + static_cast<int64_t>(task) * a.splits * kPart;
  auto get = [&](int64_t i) {
    return __hip_atomic_load(const_cast<float *>(from) + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  if (tid < kKvRowTile) {
    float m = -INFINITY;
    for (int32_t s = 0; s < active; ++s) m = fmaxf(m, get(s * kPart + kKvRowTile * DT + tid));
    float l = 0.0f;
    for (int32_t s = 0; s < active; ++s) {
      const float ms = get(s * kPart + kKvRowTile * DT + tid);
      l += get(s * kPart + kKvRowTile * DT + 16 + tid) * (ms == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((ms - m) * kNat));
    }
    part_m[0][tid] = m;
    total[tid] = l;
  }
  __syncthreads();
  for (int32_t i = tid; i < live * DT; i += 256) {
    const int32_t r = i / DT, d = i - r * DT;
    const float m = part_m[0][r], l = total[r];
    float v = 0.0f;
    for (int32_t s = 0; s < active; ++s) {
      const float ms = get(s * kPart + kKvRowTile * DT + r);
      v += get(s * kPart + i) * (ms == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((ms - m) * kNat));
    }
    if (d < b.dim) kv_store(a.out, row_out(r) + d, a.dtype, l == 0.0f ? 0.0f : v / l);
  }
}

template <int DT>
void launch_kv_rows(const KvAttnArgs &a, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.b.seqs) * a.b.heads * a.row_tiles * a.splits)), block(256);
  const bool split = a.dtype == RNSMX_FLOAT32;
  if (a.mask) {
    if (split)
      hipLaunchKernelGGL((kv_rows_kernel<DT, true, true>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((kv_rows_kernel<DT, false, true>), grid, block, 0, st, a);
  } else if (split) {
    hipLaunchKernelGGL((kv_rows_kernel<DT, true, false>), grid, block, 0, st, a);
  } else {
    hipLaunchKernelGGL((kv_rows_kernel<DT, false, false>), grid, block, 0, st, a);
  }
}

template void launch_kv_rows<RNSMX_KV_DIM>(const KvAttnArgs &a, hipStream_t st);

}  // namespace rnsmx
