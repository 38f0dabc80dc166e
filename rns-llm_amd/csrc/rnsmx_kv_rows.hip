// Attention of few query rows over the 8-bit key/value cache (built once per
// row size, RNSMX_KV_DIM).
#include "rnsmx_kv_attn.hpp"

namespace rnsmx {

// v_mfma_f32_16x16x32_f16: lane l feeds row (l & 15) of A and column (l & 15)
// of B, both at k = 8 * (l >> 4) + 0..7, and gets rows 4 * (l >> 4) + 0..3 of
// column (l & 15).
__device__ __forceinline__ f32x4 kv_mfma(h16x8 a, h16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// A workgroup of NW waves for 16 query rows (token-major over the heads of a
// group) of one sequence and key/value head, and one chunk of its tokens.  A
// wave takes 32 tokens a step:
//   S^T = K Q^T  two 16 x 16 tiles, the token of tile i, row r being 8 (r / 4) + 4 i + r % 4,
//                so that lane group g holds the products of tokens 8 g .. 8 g + 7
//   O^T += V^T P^T  P in the registers and order that S^T left it in
// Codes go into the products as they are (code / 512, exact in float16); a
// page's key scale multiplies its products, its value scale is an exponent
// added to them: with lv = log2(value scale),
//   w = 2^(x - mx + lv - ml),  O += w code,  l += w / value scale = 2^(x - mx - ml)
// where x is the product in powers of two and (mx, ml) a row's reference.
// Bound by memory where codes are many: 62 sequences of up to 4096 tokens, 32 heads of
// 128 (1181 MB) in 189 to 202 us, 5.8 to 6.2 TB/s, one row of 8 heads over 131071 tokens (268
// MB) in 50 to 57, its waves waiting 46 to 48 % of their time.  The 16 rows cost what
// one does, as a product of 16 x 16 has no smaller form, so grouped heads and drafted
// tokens come for nothing.  Codes are loaded from memory into the operands' places,
// without a pass through shared memory: no wave reads what another does.  Small calls
// are chains: 129 tokens, 12 heads 5.2 us, 16 sequences of 777 with 5 masked rows 10.4,
// about 2000 cycles for each 256 tokens of eight waves, most of them waits.
// STREAM: the values' codes are read past the caches; the keys' are not, as a load
// takes half a line of 128, which has to stay for the other half (62 sequences of
// up to 4096 tokens, 32 heads: 212 us through the caches, 200 so, 219 with the keys).
template <int DT, int NW, bool SPLIT, bool MASK, bool STREAM>
__global__ __launch_bounds__(64 * NW, NW == 8 || DT <= 160 ? 2 : 1) void kv_rows_kernel(const KvAttnArgs a) {
  constexpr int C64 = DT / 64, C32 = DT / 32 % 2;  // 64-value chunks of a row, and whether 32 are left
  constexpr int KS = DT / 32;                      // products' steps
  constexpr int VW = DT / 16;                      // bytes of a token that a lane takes: value tiles
  // pieces of 16, 8, 4 and 2 bytes a lane, VW in all, each over 16 lanes
  constexpr int W16 = VW / 16, W8 = VW / 8 % 2, W4 = VW / 4 % 2, W2 = VW / 2 % 2;
  constexpr int QN = SPLIT ? 2 : 1, ROWS = kKvRows, THREADS = 64 * NW;
  constexpr int kUnit = 32 * NW;  // tokens of a step of all waves
  __shared__ float part_o[NW][ROWS][DT + 4];
  __shared__ float part_m[NW][ROWS], part_l[NW][ROWS], part_f[NW][ROWS], total[ROWS];
  __shared__ int32_t last;

  const KvBatchArgs &b = a.b;
  const KvPlace place = kv_place(a, false);
  const int32_t split = place.split, task = place.task, tile = place.tile, head = place.head, seq = place.seq;
  const int32_t group = a.by_group.d;
  const KvSeq q = kv_seq(b, seq);
  auto token_of = [&](int32_t r) { return static_cast<int32_t>(kv_quot(a.by_group, r)); };  // of a row
  if (q.all > q.n && tile == 0 && split == 0) kv_zero_rows(a, q, head);
  const int32_t rows = q.n * group, row0 = tile * ROWS;
  if (row0 >= rows) return;
  const int32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t col = lane & 15, g = lane >> 4;
  const int32_t base = q.base;
  const int32_t t_first = token_of(row0), t_last = token_of(min(row0 + ROWS, rows) - 1);
  const int32_t hi = max(kv_causal_end(a, q, base + t_last), 0);
  const int32_t lo = min(kv_window_begin(a, base + t_first), q.len) & ~31;
  const int32_t full_hi = kv_causal_end(a, q, base + t_first);  // seen by every row: below it
  const int32_t full_lo = kv_window_begin(a, base + t_last);    // and from it on
  const int32_t c0 = lo + split * a.chunk;
  if (split > 0 && c0 >= hi) return;
  const int32_t c1 = min(hi, c0 + a.chunk);

  // this lane's row: its place and what it sees
  const int32_t row = min(row0 + col, rows - 1), t_row = token_of(row), q_head = head * group + (row - t_row * group);
  const int32_t end_row = kv_causal_end(a, q, base + t_row);
  const int32_t begin_row = kv_window_begin(a, base + t_row);

  struct Step {
    u32x4 k[2][C64];
    u32x2 k8[2];
    uint32_t v[8][VW / 4 + 1];
    uint32_t m[8];
    float ks, vs;
    bool there;
  };
  // page numbers of the lane's key row and of its eight tokens
  const int32_t key_token = 8 * (col >> 2) + (col & 3);  // of tile 0; tile 1: 4 tokens on
  const int32_t *pages = b.table + seq * b.table_stride;
  auto pages_of = [&](int32_t t0, int32_t &pk, int32_t &pv) {
    pk = pages[min((t0 + key_token) >> b.log_page, b.table_width - 1)];
    pv = pages[min((t0 + 8 * g) >> b.log_page, b.table_width - 1)];
  };
  const int32_t in_page = (1 << b.log_page) - 1;
  auto load_step = [&](Step &s, int32_t t0, int32_t pk, int32_t pv) {
    s.there = static_cast<uint32_t>(pv) < static_cast<uint32_t>(b.blocks);
    const int64_t slot_k = static_cast<int64_t>(min(max(pk, 0), b.blocks - 1)) * b.heads + head;
    const int64_t slot_v = static_cast<int64_t>(s.there ? pv : 0) * b.heads + head;
    const uint8_t *kp = b.k + ((slot_k << b.log_page) + ((t0 + key_token) & in_page)) * DT;
    const uint8_t *vp = b.v + ((slot_v << b.log_page) + ((t0 + 8 * g) & in_page)) * DT;
    kv_for<2>([&](auto I) {
      constexpr int i = I;
      kv_for<C64>([&](auto C) {
        constexpr int c = C;
        s.k[i][c] = *reinterpret_cast<const u32x4 *>(kp + i * 4 * DT + c * 64 + 16 * g);
      });
      if constexpr (C32 != 0) s.k8[i] = *reinterpret_cast<const u32x2 *>(kp + i * 4 * DT + C64 * 64 + 8 * g);
    });
    kv_for<8>([&](auto J) {
      constexpr int j = J;
      const uint8_t *p = vp + j * DT;
      if constexpr (W16 != 0) {
        const u32x4 w = kv_fetch<STREAM>(reinterpret_cast<const u32x4 *>(p + 16 * col));
        kv_for<4>([&](auto W) { s.v[j][W] = w[static_cast<int>(W)]; });
      }
      if constexpr (W8 != 0) {
        const u32x2 w = kv_fetch<STREAM>(reinterpret_cast<const u32x2 *>(p + 256 * W16 + 8 * col));
        s.v[j][4 * W16] = w[0];
        s.v[j][4 * W16 + 1] = w[1];
      }
      if constexpr (W4 != 0)
        s.v[j][4 * W16 + 2 * W8] = kv_fetch<STREAM>(reinterpret_cast<const uint32_t *>(p + 256 * W16 + 128 * W8 + 4 * col));
      if constexpr (W2 != 0)
        s.v[j][4 * W16 + 2 * W8 + W4] =
            *reinterpret_cast<const uint16_t *>(p + 256 * W16 + 128 * W8 + 64 * W4 + 2 * col);
    });
    const F32x2 sc = *reinterpret_cast<const F32x2 *>(b.scales + slot_v * 2);
    s.ks = sc.x;
    s.vs = sc.y;
    if constexpr (MASK) kv_mask_load(s.m, a, q.row + t_row, q_head, t0 + 8 * g, t0 + 32);
  };

  // The first step's loads go out before the queries', one wait for both, where
  // the registers hold the two.
  constexpr bool kEarly = DT <= 160;
  Step s0, s1;
  int32_t pk, pv, pk2 = 0, pv2 = 0;
  int32_t t0 = c0 + 32 * wave;
  if (t0 < c1) {
    pages_of(t0, pk, pv);
    pages_of(t0 + kUnit, pk2, pv2);
    if constexpr (kEarly) load_step(s0, t0, pk, pv);
  }

  // the row's queries, scaled by a power of two to lie below 2^15
  h16x8 qf[QN][KS];
  float q_scale;
  {
    float x[KS][8];
    const int64_t at = static_cast<int64_t>(q.row + t_row) * a.q_rs + static_cast<int64_t>(q_head) * a.q_hs;
    float top = 0.0f;
    // lane group g takes bytes 16 g .. of a 64-value chunk, the first eight in its first step
    kv_query<KS, SPLIT>(x, a, at, [&](auto S) {
      constexpr int s = S;
      return s < 2 * C64 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 64 * C64 + 8 * g;
    });
    kv_for<KS>([&](auto S) { kv_for<8>([&](auto J) { top = fmaxf(top, fabsf(x[S][J])); }); });
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const int32_t e = kv_query_exponent(top);
    kv_for<KS>([&](auto S) {
      constexpr int s = S;
      kv_for<8>([&](auto J) {
        constexpr int j = J;
        const float v = ldexpf(x[s][j], -e);
        const _Float16 h = static_cast<_Float16>(v);
        qf[0][s][j] = h;
        if constexpr (SPLIT) qf[1][s][j] = static_cast<_Float16>(v - static_cast<float>(h));
      });
    });
    q_scale = ldexpf(a.scale * kKvUnit, e);
    if constexpr (!MASK) q_scale *= kKvLog2e;
  }
  if constexpr (!kEarly)
    if (t0 < c1) load_step(s0, t0, pk, pv);

  // exponents are (x - mx) kNat + lv - ml in powers of two: x of masked calls is natural
  constexpr float kNat = MASK ? kKvLog2e : 1.0f;
  f32x4 o[VW];
  kv_for<VW>([&](auto I) { o[I] = f32x4{0.0f, 0.0f, 0.0f, 0.0f}; });
  // the row's reference, and its weights over the value scales, in units of 2^-ml
  float mx = -INFINITY, ml = 0.0f, sum = 0.0f;
  // what its products are less: mx; 0 of a row without a reference, which has nothing
  // but minus infinities (and not-a-numbers) so far, and of a wave that has far ones.
  // Kept from step to step, but in masked calls, which lack the register.
  float held = 0.0f;
  uint64_t far = 0;

  auto compute = [&](const Step &s, int32_t t0) {
    f32x4 acc[2];
    kv_for<2>([&](auto I) {
      constexpr int i = I;
      acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      kv_for<KS>([&](auto S) {
        constexpr int st = S;
        h16x8 k;
        if constexpr (st < 2 * C64)
          k = kv_row8(s.k[i][st / 2][2 * (st % 2)], s.k[i][st / 2][2 * (st % 2) + 1]);
        else
          k = kv_row8(s.k8[i][0], s.k8[i][1]);
        kv_for<QN>([&](auto P) { acc[i] = kv_mfma(k, qf[P][st], acc[i]); });
      });
    });
    float c = q_scale * s.ks, lv = __builtin_amdgcn_logf(s.vs), rv = __builtin_amdgcn_rcpf(s.vs);
    float w[8];
    kv_for<8>([&](auto J) {
      constexpr int j = J;
      w[j] = MASK ? acc[j / 4][j % 4] * c : acc[j / 4][j % 4];
    });
    // what every row of the tile sees needs no look at single tokens
    if (MASK || t0 < full_lo || t0 + 32 > full_hi || !__all(s.there)) {
      // scores of what is not seen are minus infinity; a lane that sees none of
      // its eight tokens does without their page's scales, which may be anything
      const int32_t t8 = t0 + 8 * g;
      uint32_t seen = s.there ? kv_between(t8, begin_row, end_row) : 0u;
      if constexpr (MASK) seen &= kv_mask_shows(a, s.m, t8, t0 + 32, w);
      kv_for<8>([&](auto J) { w[J] = seen >> J & 1u ? w[J] : -INFINITY; });
      const bool any = seen != 0;
      c = any ? c : 1.0f;
      lv = any ? lv : 0.0f;
      rv = any ? rv : 0.0f;
    }
    float xm = w[0];
    kv_for<7>([&](auto J) { xm = fmaxf(xm, w[J + 1]); });
    if constexpr (!MASK) xm *= c;
    const float em = (xm - mx) * kNat + (lv - ml);
    if ((__ballot(em > kKvAbove) | far) != 0) {
      float best = em, bx = xm, bl = lv;
      kv_for<2>([&](auto I) {
        constexpr int step = 16 << I;
        kv_higher<MASK>(best, bx, bl, __shfl_xor(best, step), __shfl_xor(bx, step), __shfl_xor(bl, step));
      });
      if (best > kKvAbove) {
        const float nl = bl - kKvBelow;
        const float fo = __builtin_amdgcn_exp2f((mx - bx) * kNat + (ml - nl));
        sum *= fo;
        kv_for<VW>([&](auto I) { o[I] *= fo; });
        mx = bx;
        ml = nl;
      }
      if constexpr (!MASK) {
        held = mx == -INFINITY ? 0.0f : mx;
        far |= __ballot(fabsf(held) >= kKvFar);
        if (far != 0) {
          kv_for<8>([&](auto J) { w[J] = kv_apart(w[J], c, held); });
          c = 1.0f;
          held = 0.0f;
        }
      }
    }
    const float ref = !MASK ? held : mx == -INFINITY ? 0.0f : mx, off = MASK ? lv - ml : lv - ml - ref;
    float part = 0.0f;
    kv_for<8>([&](auto J) {
      constexpr int j = J;
      w[j] = __builtin_amdgcn_exp2f(MASK ? fmaf(w[j] - ref, kNat, off) : fmaf(w[j], c, off));
      part += w[j];
    });
    sum = fmaf(part, rv, sum);
    h16x8 p[QN];
    kv_for<8>([&](auto J) {
      constexpr int j = J;
      const _Float16 h = static_cast<_Float16>(w[j]);
      p[0][j] = h;
      if constexpr (SPLIT) p[1][j] = kv_low(w[j], h);
    });
    kv_for<VW>([&](auto I) {
      constexpr int i = I, word = i / 4, byte = i % 4;
      const h16x8 v = kv_join(kv_halves<byte, byte>(s.v[0][word], s.v[1][word]), kv_halves<byte, byte>(s.v[2][word], s.v[3][word]),
                              kv_halves<byte, byte>(s.v[4][word], s.v[5][word]), kv_halves<byte, byte>(s.v[6][word], s.v[7][word]));
      o[i] = kv_mfma(v, p[0], o[i]);
      if constexpr (SPLIT) o[i] = kv_mfma(kv_low_codes(v), p[1], o[i]);
    });
  };

  // Two steps of loads in flight.  Page numbers are loaded two steps ahead and
  // before that step's codes: loads return in order, so waiting for them leaves
  // the codes in flight.
  if (t0 < c1)
    while (true) {
      pages_of(t0 + 2 * kUnit, pk, pv);
      if (t0 + kUnit < c1) load_step(s1, t0 + kUnit, pk2, pv2);
      compute(s0, t0);
      t0 += kUnit;
      if (t0 >= c1) break;
      pages_of(t0 + 2 * kUnit, pk2, pv2);
      if (t0 + kUnit < c1) load_step(s0, t0 + kUnit, pk, pv);
      compute(s1, t0);
      t0 += kUnit;
      if (t0 >= c1) break;
    }

  // The waves' parts: their reference mx and sums in natural units.
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  const float unit = __builtin_amdgcn_exp2f(ml);
  if (g == 0) {
    part_m[wave][col] = mx;
    part_l[wave][col] = sum * unit;
  }
  kv_for<VW>([&](auto I) {
    // value tile i of a piece of W bytes a lane holds its columns W r + i
    constexpr int i = I, P16 = 16 * W16, P8 = P16 + 8 * W8, P4 = P8 + 4 * W4;
    constexpr int width = i < P16 ? 16 : i < P8 ? 8 : i < P4 ? 4 : 2;
    constexpr int first = i < P16 ? 0 : i < P8 ? P16 : i < P4 ? P8 : P4;
    kv_for<4>([&](auto T) {
      constexpr int t = T;
      part_o[wave][col][16 * first + width * (4 * g + t) + (i - first)] = o[i][t] * (unit * kKvUnit);
    });
  });
  const int32_t live = min(rows - row0, ROWS);
  const int32_t active = a.splits == 1 ? 1 : max((hi - lo + a.chunk - 1) / a.chunk, 1);
  constexpr int64_t kPart = static_cast<int64_t>(ROWS) * (DT + 2);
  float *to = a.partial + (static_cast<int64_t>(task) * a.splits + split) * kPart;
  __syncthreads();
  // rows' reference and sum over the waves
  if (tid < ROWS) {
    float m = part_m[0][tid];
    kv_for<NW - 1>([&](auto W) { m = fmaxf(m, part_m[W + 1][tid]); });
    float l = 0.0f;
    kv_for<NW>([&](auto W) {
      const float mw = part_m[W][tid];
      const float f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((mw - m) * kNat);
      part_f[W][tid] = f;
      l += part_l[W][tid] * f;
    });
    total[tid] = l;
    if (active > 1) {
      __hip_atomic_store(to + ROWS * DT + tid, m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(to + ROWS * DT + ROWS + tid, l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();
  auto row_out = [&](int32_t r) {
    const int32_t i = row0 + r, t = token_of(i);
    return (static_cast<int64_t>(q.row + t) * a.q_heads + head * group + (i - t * group)) * b.dim;
  };
  for (int32_t i = tid; i < live * DT; i += THREADS) {
    const int32_t r = i / DT, d = i - r * DT;
    float v = 0.0f;
    kv_for<NW>([&](auto W) { v += part_o[W][r][d] * part_f[W][r]; });
    if (active > 1) {
      __hip_atomic_store(to + i, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else if (d < b.dim) {
      const float l = total[r];
      kv_store(a.out, row_out(r) + d, a.dtype, l == 0.0f ? 0.0f : v / l);
    }
  }
  if (active == 1) return;

  // A split's part lies in its place in the workspace; the workgroup that
  // draws a task's last ticket joins them.  The parts are written with
  // agent-scope accesses, which go past the XCDs' own caches, and are complete
  // before the ticket is drawn; the reader drops what its caches hold of older
  // ones first.  No workgroup waits for another.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const uint32_t old = __hip_atomic_fetch_add(a.tickets + task, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = old == static_cast<uint32_t>(active - 1);
    if (last) __hip_atomic_store(a.tickets + task, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  const float *from = a.partial + static_cast<int64_t>(task) * a.splits * kPart;
  // four values a thread, eight splits' loads at a time, one wait for all of
  // what they need: references, sums and values
  for (int32_t i = tid * 4; i < live * DT; i += THREADS * 4) {
    const int32_t r = i / DT, d = i - r * DT;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    for (int32_t s0 = 0; s0 < active; s0 += 8) {
      f32x4 vs[8];
      float ms[8], ls[8], top = m;
      kv_for<8>([&](auto S) {
        const float *p = from + min(s0 + S, active - 1) * kPart;
        vs[S] = *reinterpret_cast<const f32x4 *>(p + i);
        ms[S] = p[ROWS * DT + r];
        ls[S] = p[ROWS * DT + ROWS + r];
      });
      kv_for<8>([&](auto S) { top = fmaxf(top, ms[S]); });
      const float old = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - top) * kNat);
      v *= old;
      l *= old;
      kv_for<8>([&](auto S) {
        const float f = s0 + S >= active || ms[S] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((ms[S] - top) * kNat);
        if (s0 + S < active) {
          v += vs[S] * f;
          l += ls[S] * f;
        }
      });
      m = top;
    }
    kv_for<4>([&](auto J) {
      constexpr int j = J;
      if (d + j < b.dim) kv_store(a.out, row_out(r) + d + j, a.dtype, l == 0.0f ? 0.0f : v[j] / l);
    });
  }
}

template <int DT, int NW>
static void launch_waves(const KvAttnArgs &a, uint32_t groups, hipStream_t st) {
  const dim3 grid(groups), block(64 * NW);
  auto launch = [&](auto split) {
    constexpr bool S = decltype(split)::value;
    if (a.mask)
      hipLaunchKernelGGL((kv_rows_kernel<DT, NW, S, true, false>), grid, block, 0, st, a);
    else if (a.stream)
      hipLaunchKernelGGL((kv_rows_kernel<DT, NW, S, false, kv_whole(DT)>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((kv_rows_kernel<DT, NW, S, false, false>), grid, block, 0, st, a);
  };
  if (a.dtype == RNSMX_FLOAT32)
    launch(std::true_type{});
  else
    launch(std::false_type{});
}

template <int DT>
void launch_kv_rows(const KvAttnArgs &a, uint32_t groups, hipStream_t st) {
  if (a.waves == 8 && kv_wide(DT))
    launch_waves<DT, kv_wide(DT) ? 8 : 4>(a, groups, st);
  else
    launch_waves<DT, 4>(a, groups, st);
}

template void launch_kv_rows<RNSMX_KV_DIM>(const KvAttnArgs &a, uint32_t groups, hipStream_t st);

}  // namespace rnsmx
