// Attention of many query rows (prompts) over the 8-bit key/value cache (built
// once per row size, RNSMX_KV_DIM).
#include "rnsmx_kv_attn.hpp"

namespace rnsmx {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// v_mfma_f32_32x32x16_f16: lane l feeds row (l & 31) of A and column (l & 31)
// of B, both at k = 8 * (l >> 5) + 0..7, and gets rows 8 (i / 4) + 4 (l >> 5) +
// i % 4, i = 0..15, of column (l & 31).
__device__ __forceinline__ f32x16 kv_mfma32(h16x8 a, h16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

constexpr int kStep = 64;  // tokens of a step

// The token of A's row r that leaves lane half h tokens 8 h .. 8 h + 7 and 16 +
// 8 h .. of 32 in its 16 results, in order: what P^T's operand wants.
__device__ __forceinline__ int32_t tile_token(int32_t r) {
  const int32_t i = 4 * (r >> 3) + (r & 3);
  return 16 * (i >> 3) + 8 * ((r >> 2) & 1) + (i & 7);
}
// 16-byte columns of the staged tiles are exchanged by these, so that the eight
// lanes that the shared memory serves at a time meet eight of its columns: keys
// are read by tile_token's rows and written along a row, values read down eight
// rows and written four rows apart.
__device__ __forceinline__ int32_t key_swap(int32_t t) { return (t & 3) | ((t >> 3 & 1) << 2); }
__device__ __forceinline__ int32_t value_swap(int32_t d) { return (d & 7) ^ (d >> 2 & 7); }

// A workgroup of four waves for 128 query rows (32 a wave, token-major over the
// heads of a group) of one sequence and key/value head.  Steps of 64 tokens are
// staged for all four as halves, keys by token and values by column, each code
// converted once; wave w loads and converts tokens 16 w .. 16 w + 15, which lie
// in one page.  The products and the weights are as kv_rows_kernel's, with
// 32 x 32 products: a row is one lane pair's.
//
// Bound by what surrounds the products (weights, conversions, waits) more than by
// them: at 8192 tokens, 32 heads of 128 (550 GFLOP) 630 to 700 us, 0.79 to 0.87 PFLOP/s of the 1.23
// that a large library product reaches here, vector units busy half of the time, matrix
// units and shared memory a third each.  2048 tokens, 32 heads (34 GFLOP) take 62 to 70
// us: 512 tiles go in one round, so the longest chain decides, 32 steps of some 4200
// cycles; waves wait 30 % of their time and are issue-blocked 25 %.
//
// HALVES 2: eight waves, the second four with the same rows and every other
// step, staged apart; they join in the shared memory at the end.  A step's chain
// (load, products, weights, products, conversions: some 4000 cycles, twice that
// of its longest part) is then run through half as often by the longest tiles,
// which a call of few workgroups waits for.
template <int DT, int HALVES, bool SPLIT, bool MASK>
__global__ __launch_bounds__(256 * HALVES, (DT <= 128 ? 2 : 1)) void kv_tiles_kernel(const KvAttnArgs a) {
  constexpr int KS = DT / 16, DB = DT / 32, QN = SPLIT ? 2 : 1;
  constexpr int KROW = (DT + 63) / 64 * 64;  // halves of a staged key
  constexpr int KR = DT / 32;                // loads of 8 codes a lane and step, keys
  constexpr int VD = DT == 64 ? 2 : DT == 256 ? 8 : 4;  // columns of 8 tokens that a lane converts
  constexpr int VG = DT / VD, VR = (2 * VG + 63) / 64;  // of a token group, and rounds
  // each half's two buffers of keys and of values
  constexpr int kKeys = kStep * KROW, kValues = DT * kStep;
  __shared__ __attribute__((aligned(128))) _Float16 staged[HALVES][2 * kKeys + 2 * kValues];
  // key scale, log2 and reciprocal of the value scale, whether it is there
  __shared__ __attribute__((aligned(16))) float page_scales[HALVES][2][4][4];
  __shared__ int32_t last;

  const KvBatchArgs &b = a.b;
  const KvPlace place = kv_place(a, HALVES == 1);
  const int32_t split = place.split, task = place.task, tile = place.tile, head = place.head, seq = place.seq;
  const int32_t group = a.by_group.d;
  const KvSeq q = kv_seq(b, seq);
  if (q.all > q.n && tile == 0 && split == 0) kv_zero_rows(a, q, head);
  const int32_t rows = q.n * group, row0 = tile * kKvTileRows;
  if (row0 >= rows) return;
  const int32_t tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t half = HALVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  _Float16 *const keys = staged[half], *const values = keys + 2 * kKeys;
  float (*const pages_of_step)[4][4] = page_scales[half];
  const int32_t col = lane & 31, h = lane >> 5;
  const int32_t base = q.base;
  auto kv_of = [&](int32_t r) { return static_cast<int32_t>(kv_quot(a.by_group, r)); };  // the token of a row
  // what the workgroup's rows see, and this wave's
  const int32_t last_row = min(row0 + kKvTileRows, rows) - 1;
  const int32_t hi = max(kv_causal_end(a, q, base + kv_of(last_row)), 0);
  const int32_t lo = min(kv_window_begin(a, base + kv_of(row0)), q.len) & ~(kStep - 1);
  const int32_t c0 = lo + split * a.chunk;
  if (split > 0 && c0 >= hi) return;
  const int32_t c1 = min(hi, c0 + a.chunk);
  const int32_t w_first = row0 + 32 * wave, w_last = min(w_first + 31, rows - 1);
  const bool w_any = w_first < rows;
  const int32_t t_first = kv_of(w_first), t_last = kv_of(w_last);
  const int32_t full_hi = min(kv_causal_end(a, q, base + t_first), c1);
  const int32_t full_lo = kv_window_begin(a, base + t_last);

  const int32_t row = min(w_first + col, rows - 1);
  const int32_t t_row = kv_of(row), q_head = head * group + (row - t_row * group);
  const int32_t end_row = min(kv_causal_end(a, q, base + t_row), c1);
  const int32_t begin_row = kv_window_begin(a, base + t_row);

  // loads of a step: this wave's 16 tokens
  u32x2 kr[KR];
  uint32_t vr[VR][8][VD / 4 + 1];
  F32x2 sr;
  bool there = false;
  // read through the scalar cache: one number a wave, whose wait leaves the
  // codes' loads in flight
  const kv_const_i32 *table = (const kv_const_i32 *)(b.table + seq * b.table_stride);
  const int32_t in_page = (1 << b.log_page) - 1;
  auto page_of = [&](int32_t t0) {
    return table[min((t0 + 16 * wave) >> b.log_page, b.table_width - 1)];
  };
  auto load_step = [&](int32_t t0, int32_t page) {
    there = static_cast<uint32_t>(page) < static_cast<uint32_t>(b.blocks);
    const int64_t slot = static_cast<int64_t>(there ? page : 0) * b.heads + head;
    const int64_t at = ((slot << b.log_page) + ((t0 + 16 * wave) & in_page)) * DT;
    kv_for<KR>([&](auto R) {
      constexpr int r = R;
      kr[r] = *reinterpret_cast<const u32x2 *>(b.k + at + lane * 8 + r * 512);
    });
    kv_for<VR>([&](auto R) {
      constexpr int r = R;
      const int32_t item = lane + 64 * r;
      if (2 * VG % 64 == 0 || item < 2 * VG) {
        const uint8_t *p = b.v + at + (item / VG) * 8 * DT + (item % VG) * VD;
        kv_for<8>([&](auto J) {
          constexpr int j = J;
          if constexpr (VD == 8) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(p + j * DT);
            vr[r][j][0] = w[0];
            vr[r][j][1] = w[1];
          } else if constexpr (VD == 4) {
            vr[r][j][0] = *reinterpret_cast<const uint32_t *>(p + j * DT);
          } else {
            vr[r][j][0] = *reinterpret_cast<const uint16_t *>(p + j * DT);
          }
        });
      }
    });
    sr = *reinterpret_cast<const F32x2 *>(b.scales + slot * 2);
  };
  auto stage = [&](int32_t buf) {
    kv_for<KR>([&](auto R) {
      constexpr int r = R;
      const int32_t item = lane + 64 * r, t = 16 * wave + item / (DT / 8), c = item % (DT / 8);
      *reinterpret_cast<h16x8 *>(&keys[buf * kKeys + t * KROW + (c ^ key_swap(t)) * 8]) = kv_row8(kr[r][0], kr[r][1]);
    });
    kv_for<VR>([&](auto R) {
      constexpr int r = R;
      const int32_t item = lane + 64 * r;
      if (2 * VG % 64 == 0 || item < 2 * VG) {
        const int32_t group = 2 * wave + item / VG, d0 = (item % VG) * VD;
        kv_for<VD>([&](auto I) {
          constexpr int i = I, w = i / 4, byte = i % 4;
          const auto &v = vr[r];
          const h16x8 x = kv_join(kv_halves<byte, byte>(v[0][w], v[1][w]), kv_halves<byte, byte>(v[2][w], v[3][w]),
                                  kv_halves<byte, byte>(v[4][w], v[5][w]), kv_halves<byte, byte>(v[6][w], v[7][w]));
          *reinterpret_cast<h16x8 *>(&values[buf * kValues + (d0 + i) * kStep + (group ^ value_swap(d0 + i)) * 8]) = x;
        });
      }
    });
    if (lane == 0) {
      pages_of_step[buf][wave][0] = sr.x;
      pages_of_step[buf][wave][1] = __builtin_amdgcn_logf(sr.y);
      pages_of_step[buf][wave][2] = __builtin_amdgcn_rcpf(sr.y);
      pages_of_step[buf][wave][3] = there ? 1.0f : 0.0f;
    }
  };

  // a half's steps; past the chunk's end it goes on with the last one, all hidden
  constexpr int32_t kStride = HALVES * kStep;
  auto step_at = [&](int32_t t0) { return min(t0, c1 - 1) & ~(kStep - 1); };
  const int32_t first = c0 + kStep * half;
  int32_t page = 0;
  if (c0 < c1) {
    load_step(step_at(first), page_of(step_at(first)));
    page = page_of(step_at(first + kStride));
  }

  h16x8 qf[QN][KS];
  float q_scale;
  {
    float x[KS][8];
    const int64_t at = static_cast<int64_t>(q.row + t_row) * a.q_rs + static_cast<int64_t>(q_head) * a.q_hs;
    float top = 0.0f;
    kv_query<KS, SPLIT>(x, a, at, [&](auto S) { return 16 * S + 8 * h; });
    kv_for<KS>([&](auto S) { kv_for<8>([&](auto J) { top = fmaxf(top, fabsf(x[S][J])); }); });
    top = fmaxf(top, __shfl_xor(top, 32));
    const int32_t e = kv_query_exponent(top);
    kv_for<KS>([&](auto S) {
      constexpr int s = S;
      kv_for<8>([&](auto J) {
        constexpr int j = J;
        const float v = ldexpf(x[s][j], -e);
        const _Float16 half = static_cast<_Float16>(v);
        qf[0][s][j] = half;
        if constexpr (SPLIT) qf[1][s][j] = static_cast<_Float16>(v - static_cast<float>(half));
      });
    });
    q_scale = ldexpf(a.scale * kKvUnit, e);
    if constexpr (!MASK) q_scale *= kKvLog2e;
  }

  f32x16 o[DB];
  kv_for<DB>([&](auto I) { kv_for<16>([&](auto J) { o[I][static_cast<int>(J)] = 0.0f; }); });
  // the row's reference and its weights' sum over the value scale, in units of 2^ml
  float mx = -INFINITY, ml = 0.0f, sum = 0.0f;
  // what its products are less (kv_rows_kernel has which)
  float held = 0.0f;
  uint64_t far = 0;
  constexpr float kNat = MASK ? kKvLog2e : 1.0f;

  auto compute = [&](int32_t buf, int32_t t0) {
    f32x16 acc[2];
    kv_for<2>([&](auto B) { kv_for<16>([&](auto J) { acc[B][static_cast<int>(J)] = 0.0f; }); });
    const int32_t kt = tile_token(col), swap = key_swap(kt);
    kv_for<KS>([&](auto S) {
      constexpr int s = S;
      kv_for<2>([&](auto B) {
        constexpr int sub = B;
        const h16x8 k = *reinterpret_cast<const h16x8 *>(&keys[buf * kKeys + (32 * sub + kt) * KROW + (((2 * s + h)) ^ swap) * 8]);
        kv_for<QN>([&](auto P) { acc[sub] = kv_mfma32(k, qf[P][s], acc[sub]); });
      });
    });
    float c[4], lv[4], rv[4], w[4][8], xm[4];
    bool there[4], all_there = true;
    kv_for<4>([&](auto G) {
      constexpr int g = G;
      const f32x4 sc = *reinterpret_cast<const f32x4 *>(pages_of_step[buf][g]);
      c[g] = q_scale * sc[0];
      lv[g] = sc[1];
      rv[g] = sc[2];
      there[g] = sc[3] != 0.0f;
      all_there = all_there && there[g];
      // results i of a product are tokens 16 (i / 8) + 8 h + i % 8: four groups of eight
      kv_for<8>([&](auto J) {
        constexpr int j = J;
        const float x = acc[g / 2][8 * (g % 2) + j];
        w[g][j] = MASK ? x * c[g] : x;
      });
    });
    // what every row of the wave sees needs no look at single tokens
    if (MASK || t0 < full_lo || t0 + kStep > full_hi || !__all(all_there))
      // scores of what is not seen are minus infinity; a lane that sees none of
      // a group does without its page's scales, which may be anything
      kv_for<4>([&](auto G) {
        constexpr int g = G;
        const int32_t t8 = t0 + 16 * g + 8 * h;
        uint32_t m[8];
        if constexpr (MASK) kv_mask_load(m, a, q.row + t_row, q_head, t8, t0 + kStep);
        uint32_t seen = there[g] ? kv_between(t8, begin_row, end_row) : 0u;
        if constexpr (MASK) seen &= kv_mask_shows(a, m, t8, t0 + kStep, w[g]);
        kv_for<8>([&](auto J) { w[g][J] = seen >> J & 1u ? w[g][J] : -INFINITY; });
        const bool any = seen != 0;
        c[g] = any ? c[g] : 1.0f;
        lv[g] = any ? lv[g] : 0.0f;
        rv[g] = any ? rv[g] : 0.0f;
      });
    kv_for<4>([&](auto G) {
      constexpr int g = G;
      xm[g] = w[g][0];
      kv_for<7>([&](auto J) { xm[g] = fmaxf(xm[g], w[g][J + 1]); });
      if constexpr (!MASK) xm[g] *= c[g];
    });
    float em[4];
    bool above = false;
    kv_for<4>([&](auto G) {
      constexpr int g = G;
      em[g] = (xm[g] - mx) * kNat + (lv[g] - ml);
      above |= em[g] > kKvAbove;
    });
    if ((__ballot(above) | far) != 0) {
      float best = em[0], bx = xm[0], bl = lv[0];
      kv_for<3>([&](auto G) { kv_higher<MASK>(best, bx, bl, em[G + 1], xm[G + 1], lv[G + 1]); });
      kv_higher<MASK>(best, bx, bl, __shfl_xor(best, 32), __shfl_xor(bx, 32), __shfl_xor(bl, 32));
      if (best > kKvAbove) {
        const float nl = bl - kKvBelow;
        const float fo = __builtin_amdgcn_exp2f((mx - bx) * kNat + (ml - nl));
        sum *= fo;
        kv_for<DB>([&](auto I) { o[I] *= fo; });
        mx = bx;
        ml = nl;
      }
      if constexpr (!MASK) {
        held = mx == -INFINITY ? 0.0f : mx;
        far |= __ballot(fabsf(held) >= kKvFar);
        if (far != 0) {
          kv_for<4>([&](auto G) {
            constexpr int g = G;
            kv_for<8>([&](auto J) { w[g][J] = kv_apart(w[g][J], c[g], held); });
            c[g] = 1.0f;
          });
          held = 0.0f;
        }
      }
    }
    // A group's weights, then its products, whose time on the matrix cores the
    // next group's weights fill (and the next step's codes after the last).
    const float ref = !MASK ? held : mx == -INFINITY ? 0.0f : mx;
    kv_for<4>([&](auto G) {
      constexpr int g = G;
      const float off = MASK ? lv[g] - ml : lv[g] - ml - ref;
      float part = 0.0f;
      kv_for<8>([&](auto J) {
        constexpr int j = J;
        w[g][j] = __builtin_amdgcn_exp2f(MASK ? fmaf(w[g][j] - ref, kNat, off) : fmaf(w[g][j], c[g], off));
        part += w[g][j];
      });
      sum = fmaf(part, rv[g], sum);
      h16x8 p[QN];
      kv_for<8>([&](auto J) {
        constexpr int j = J;
        const _Float16 half = static_cast<_Float16>(w[g][j]);
        p[0][j] = half;
        if constexpr (SPLIT) p[1][j] = kv_low(w[g][j], half);
      });
      kv_for<DB>([&](auto I) {
        constexpr int i = I;
        const int32_t d = 32 * i + col;
        const h16x8 v = *reinterpret_cast<const h16x8 *>(&values[buf * kValues + d * kStep + ((2 * g + h) ^ value_swap(d)) * 8]);
        o[i] = kv_mfma32(v, p[0], o[i]);
        if constexpr (SPLIT) o[i] = kv_mfma32(kv_low_codes(v), p[1], o[i]);
      });
    });
  };

  if (c0 < c1) {
    stage(0);
    int32_t buf = 0;
    for (int32_t at = c0; at < c1; at += kStride, buf ^= 1) {
      __syncthreads();  // this step is staged, and the other buffer's readers are done
      // The next step's codes (the last step's again after it: no branch parts
      // the products from the conversions).  A wave whose rows see nothing of a
      // step goes through it all the same, beside those that do.
      const int32_t t0 = at + kStep * half;
      load_step(step_at(t0 + kStride), page);
      page = page_of(step_at(t0 + 2 * kStride));
      compute(buf, t0);
      stage(buf ^ 1);
    }
  }
  sum += __shfl_xor(sum, 32);

  if constexpr (HALVES == 2) {
    // the second half's sums as its lanes hold them, into the buffers of both
    float *const sums = reinterpret_cast<float *>(staged[1]) + tid * 4;
    float *const refs = reinterpret_cast<float *>(staged[0]) + tid;
    static_assert(sizeof(staged[0]) >= 256 * 4 * 4 * DB * sizeof(float), "a half's sums");
    __syncthreads();
    if (half == 1) {
      kv_for<4 * DB>([&](auto K) {
        constexpr int k = K, i = k / 4, r = 4 * (k % 4);
        *reinterpret_cast<f32x4 *>(sums + k * 1024) = f32x4{o[i][r], o[i][r + 1], o[i][r + 2], o[i][r + 3]};
      });
      refs[0] = mx;
      refs[256] = ml;
      refs[512] = sum;
    }
    __syncthreads();
    if (half == 0) {
      const float mx2 = refs[0], ml2 = refs[256], mx1 = mx, ml1 = ml;
      kv_reference<MASK>(mx, ml, mx2, ml2);
      const float f1 = kv_factor<MASK>(mx1, ml1, mx, ml), f2 = kv_factor<MASK>(mx2, ml2, mx, ml);
      sum = sum * f1 + refs[512] * f2;
      kv_for<4 * DB>([&](auto K) {
        constexpr int k = K, i = k / 4, r = 4 * (k % 4);
        const f32x4 v = *reinterpret_cast<const f32x4 *>(sums + k * 1024);
        kv_for<4>([&](auto J) {
          constexpr int j = J;
          o[i][r + j] = o[i][r + j] * f1 + v[j] * f2;
        });
      });
    }
  }
  const bool mine = w_any && half == 0;  // the waves that go on with the rows

  // Split over its tokens, a workgroup leaves its sums in the workspace as the
  // lanes hold them, two at a time; the one that draws the task's last ticket
  // joins them, in the order of the splits (kv_rows_kernel has the protocol).
  const int32_t active = a.splits == 1 ? 1 : max((hi - lo + a.chunk - 1) / a.chunk, 1);
  if (active > 1) {
    constexpr int64_t kPart = kv_tile_floats(DT);
    float *at = a.partial + static_cast<int64_t>(task) * a.splits * kPart + tid * 2;
    auto put = [&](int64_t i, float x, float y) {
      __hip_atomic_store(reinterpret_cast<uint64_t *>(at + split * kPart + i),
                         static_cast<uint64_t>(__float_as_uint(y)) << 32 | __float_as_uint(x), __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    };
    if (mine) {
      kv_for<DB>([&](auto I) {
        kv_for<8>([&](auto J) {
          constexpr int i = I, j = J;
          put((8 * i + j) * 512, o[i][2 * j], o[i][2 * j + 1]);
        });
      });
      put(8 * DB * 512, mx, ml);
      put((8 * DB + 1) * 512, sum, 0.0f);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
      const uint32_t old = __hip_atomic_fetch_add(a.tickets + task, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = old == static_cast<uint32_t>(active - 1);
      if (last) __hip_atomic_store(a.tickets + task, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last || !mine) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    auto get = [&](int32_t s, int64_t i) { return *reinterpret_cast<const F32x2 *>(at + s * kPart + i); };
    // the highest reference of all, the references of four parts at a time; then
    // the parts in their order, this workgroup's own as it still holds it
    f32x16 own[DB];
    kv_for<DB>([&](auto I) {
      own[I] = o[I];
      kv_for<16>([&](auto J) { o[I][static_cast<int>(J)] = 0.0f; });
    });
    const float own_sum = sum;
    mx = -INFINITY;
    ml = sum = 0.0f;
    for (int32_t s0 = 0; s0 < active; s0 += 4) {
      F32x2 r[4];
      kv_for<4>([&](auto S) { r[S] = get(min(s0 + S, active - 1), 8 * DB * 512); });
      kv_for<4>([&](auto S) { kv_reference<MASK>(mx, ml, r[S].x, r[S].y); });
    }
    for (int32_t s = 0; s < active; ++s) {
      const F32x2 r = get(s, 8 * DB * 512);
      if (s == split) {
        const float f = kv_factor<MASK>(r.x, r.y, mx, ml);
        sum = fmaf(own_sum, f, sum);
        kv_for<DB>([&](auto I) {
          kv_for<16>([&](auto J) {
            constexpr int i = I, j = J;
            o[i][j] = fmaf(own[i][j], f, o[i][j]);
          });
        });
      } else {
        const F32x2 t = get(s, (8 * DB + 1) * 512);
        F32x2 v[8 * DB];
        kv_for<8 * DB>([&](auto K) { v[K] = get(s, K * 512); });
        const float f = kv_factor<MASK>(r.x, r.y, mx, ml);
        sum = fmaf(t.x, f, sum);
        kv_for<8 * DB>([&](auto K) {
          constexpr int k = K, i = k / 8, j = 2 * (k % 8);
          o[i][j] = fmaf(v[k].x, f, o[i][j]);
          o[i][j + 1] = fmaf(v[k].y, f, o[i][j + 1]);
        });
      }
    }
  }

  if (!mine || w_first + col >= rows) return;
  // l = sum 2^ml, and the codes' unit
  const float f = sum == 0.0f ? 0.0f : kKvUnit / sum;
  const int64_t out = (static_cast<int64_t>(q.row + t_row) * a.q_heads + q_head) * b.dim;
  kv_for<DB>([&](auto I) {
    kv_for<4>([&](auto R) {
      constexpr int i = I, r = R;
      const int32_t d = 32 * i + 8 * r + 4 * h;
      float y[4];
      kv_for<4>([&](auto J) {
        constexpr int j = J;
        y[j] = sum == 0.0f ? 0.0f : o[i][4 * r + j] * f;
      });
      if (a.out_vec && b.dim % 4 == 0) {
        if (d >= b.dim) return;
        if (a.dtype == RNSMX_FLOAT32) {
          *reinterpret_cast<f32x4 *>(static_cast<float *>(a.out) + out + d) = f32x4{y[0], y[1], y[2], y[3]};
        } else {
          uint16_t bits[4];
          kv_for<4>([&](auto J) {
            constexpr int j = J;
            bits[j] = a.dtype == RNSMX_FLOAT16 ? __builtin_bit_cast(uint16_t, static_cast<_Float16>(y[j])) : kv_to_bf16(y[j]);
          });
          *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.out) + out + d) =
              u32x2{bits[0] | static_cast<uint32_t>(bits[1]) << 16, bits[2] | static_cast<uint32_t>(bits[3]) << 16};
        }
      } else {
        kv_for<4>([&](auto J) {
          constexpr int j = J;
          if (d + j < b.dim) kv_store(a.out, out + d + j, a.dtype, y[j]);
        });
      }
    });
  });
}

template <int DT, int HALVES>
static void launch_halves(const KvAttnArgs &a, uint32_t groups, hipStream_t st) {
  const dim3 grid(groups), block(256 * HALVES);
  const bool split = a.dtype == RNSMX_FLOAT32;
  if (a.mask) {
    if (split)
      hipLaunchKernelGGL((kv_tiles_kernel<DT, HALVES, true, true>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((kv_tiles_kernel<DT, HALVES, false, true>), grid, block, 0, st, a);
  } else if (split) {
    hipLaunchKernelGGL((kv_tiles_kernel<DT, HALVES, true, false>), grid, block, 0, st, a);
  } else {
    hipLaunchKernelGGL((kv_tiles_kernel<DT, HALVES, false, false>), grid, block, 0, st, a);
  }
}

template <int DT>
void launch_kv_tiles(const KvAttnArgs &a, uint32_t groups, hipStream_t st) {
  if (a.waves == 8)
    launch_halves<DT, kv_tile_halves(DT)>(a, groups, st);
  else
    launch_halves<DT, 1>(a, groups, st);
}

template void launch_kv_tiles<RNSMX_KV_DIM>(const KvAttnArgs &a, uint32_t groups, hipStream_t st);

}  // namespace rnsmx
