// The 8-bit key/value cache: what its kernels share (rnsmx_kv_cache.hip writes
// and reads pages, rnsmx_kv_rows.hip attends with few rows).
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <utility>

#include "rnsmx_common.hpp"

namespace rnsmx {

typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(4))) int32_t kv_const_i32;

template <typename F, int... I>
__device__ __forceinline__ void kv_for_impl(F &&f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void kv_for(F &&f) {
  kv_for_impl(f, std::make_integer_sequence<int, N>{});
}

// Quotients by a divisor known on the host, for n below 2^31: with s = ceil(log2
// d) and mul = floor(2^32 (2^s - d) / d) + 1 (Granlund and Montgomery's method),
// n / d = (mulhi(mul, n) + n) >> s.  A division in scalar code takes some 250
// cycles, and a workgroup finds its place with half a dozen.
struct KvDiv {
  uint32_t mul, shift, d;
};
inline KvDiv kv_div(uint32_t d) {
  KvDiv r{0, 0, d};
  while ((1ull << r.shift) < d) ++r.shift;
  r.mul = static_cast<uint32_t>((((1ull << r.shift) - d) << 32) / d + 1);
  return r;
}
__device__ __forceinline__ uint32_t kv_quot(const KvDiv &v, uint32_t n) { return (__umulhi(v.mul, n) + n) >> v.shift; }
// n becomes the quotient; the remainder
__device__ __forceinline__ uint32_t kv_rem(const KvDiv &v, uint32_t &n) {
  const uint32_t q = kv_quot(v, n), r = n - q * v.d;
  n = q;
  return r;
}

// A launch has fewer than 2^32 threads, which a prompt beside many sequences passes
// (128 of them, 32 heads, 131072 tokens in pages of 16): f(first workgroup, how many)
// for each launch of a call's, all but the last a multiple of 512, so that kv_place's
// order goes on from one to the next.
template <typename F>
inline void kv_launches(uint32_t groups, uint32_t threads, F &&f) {
  const uint32_t most = (0xFFFFFFFFu / threads) & ~511u;
  for (uint32_t first = 0; first < groups; first += std::min(most, groups - first)) f(first, std::min(most, groups - first));
}

// Row sizes the attention kernels are built for; a head dimension takes the
// next one (codes of zero past it).
constexpr int kKvDims[] = {64, 96, 128, 160, 192, 256};

// Cache and sequences as the kernels read them.
struct KvBatchArgs {
  uint8_t *k, *v;
  float *scales;
  const int32_t *table, *lengths, *starts;
  int64_t table_stride;
  int32_t blocks, log_page, heads, dim, row_bytes;
  int32_t seqs, table_width, rows, max_rows, max_length;
};

// One sequence: its tokens and rows as far as the host was told of them.  `base`,
// the position of its first row, is that of what the device holds, so that a cut
// drops tokens or rows and moves none.
struct KvSeq {
  int32_t len, row, n, base;
  int32_t all;  // its rows, those past max_rows too
};
__device__ __forceinline__ KvSeq kv_seq(const KvBatchArgs &a, int32_t s) {
  KvSeq r;
  // through the scalar cache: s is one for the workgroup
  const kv_const_i32 *lengths = (const kv_const_i32 *)a.lengths, *starts = (const kv_const_i32 *)a.starts;
  const int32_t length = max(lengths[s], 0);
  r.len = min(length, a.max_length);
  if (a.starts) {
    r.row = min(max(starts[s], 0), a.rows);
    r.all = min(max(starts[s + 1], r.row), a.rows) - r.row;
  } else {
    r.row = s;
    r.all = 1;
  }
  r.n = min(r.all, a.max_rows);
  r.base = length - r.all;
  return r;
}

// STREAM: past the caches, for what one call reads or writes once and is too much
// for them.
template <bool STREAM, typename V>
__device__ __forceinline__ V kv_fetch(const V *p) {
  if constexpr (STREAM)
    return __builtin_nontemporal_load(p);
  else
    return *p;
}

// Element access for float32 / float16 / bfloat16 rows (dtype: rnsmx_dtype).
__device__ __forceinline__ float kv_bf16(uint16_t b) { return __uint_as_float(static_cast<uint32_t>(b) << 16); }
__device__ __forceinline__ float kv_load(const void *p, int64_t i, int32_t dtype) {
  if (dtype == RNSMX_FLOAT32) return static_cast<const float *>(p)[i];
  if (dtype == RNSMX_FLOAT16) return static_cast<float>(static_cast<const _Float16 *>(p)[i]);
  return kv_bf16(static_cast<const uint16_t *>(p)[i]);
}
// Rounded to nearest even; a NaN stays one.
__device__ __forceinline__ uint16_t kv_to_bf16(float v) {
  const uint32_t u = __float_as_uint(v);
  return static_cast<uint16_t>(v != v ? 0x7FC0u : (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ void kv_store(void *p, int64_t i, int32_t dtype, float v) {
  if (dtype == RNSMX_FLOAT32)
    static_cast<float *>(p)[i] = v;
  else if (dtype == RNSMX_FLOAT16)
    static_cast<_Float16 *>(p)[i] = static_cast<_Float16>(v);
  else
    static_cast<uint16_t *>(p)[i] = kv_to_bf16(v);
}

// Arguments of the attention kernels.
struct KvAttnArgs {
  KvBatchArgs b;
  const void *q;
  void *out;
  const void *mask;
  float *partial;     // [tasks][splits] partial results, tasks = seqs * heads * row tiles
  uint32_t *tickets;  // one arrival counter per task
  int64_t q_rs, q_hs, mask_rs, mask_hs, mask_ts;
  int32_t q_heads, dtype, mask_dtype, mask_len;
  int32_t stream;  // values' codes are read past the caches
  int32_t causal, window, vec, out_vec;  // vec: q rows are read 16 bytes at a time; out_vec: out starts on 16 bytes
  int32_t chunk, splits, waves;  // waves of a workgroup, 4 or 8
  int32_t tile_rows, row_tiles;  // rows of a workgroup (which says the kernel), workgroups over a sequence's rows
  // group: query heads of a key/value head; units: a pair's workgroups; pairs: those that run side by side
  KvDiv by_group, by_splits, by_units, by_heads, by_pairs;
  uint32_t first, groups;  // a launch's first workgroup, and those of all the call's launches
  float scale;
};

constexpr int kKvRows = 16;          // query rows of a workgroup of kv_rows_kernel
// Whether it is built with eight waves: row sizes whose waves are two to a SIMD.
constexpr bool kv_wide(int row_bytes) { return row_bytes <= 160; }

// Whether its values' codes are loaded in pieces of 64 bytes and more.
constexpr bool kv_whole(int row_bytes) { return row_bytes % 64 == 0; }

// Floats of one split's partial result.  Of kv_rows_kernel: rows of row_bytes
// values, then each row's reference and sum; of kv_tiles_kernel: what the 256
// lanes hold, row_bytes / 2 values, a reference of two and a sum each.
constexpr int64_t kv_row_floats(int row_bytes) { return kKvRows * (static_cast<int64_t>(row_bytes) + 2); }
constexpr int64_t kv_tile_floats(int row_bytes) { return 256 * (static_cast<int64_t>(row_bytes) / 2 + 4); }

// A workgroup's part of the work: sequence and head (a pair), tile of rows,
// split of the tokens; task numbers pairs' tiles.  Neighbours are different
// pairs, so that each of the 8 XCDs, which workgroups go to in turn, gets as many
// long and short parts as the others (72 pairs of sequences of 400 to 2500
// tokens: 78 us with the pairs one after the other in eighths, 44 so; a prompt of
// 2048, 32 heads: 84, 69), and where the pairs divide by 8 each is one XCD's, whose
// L2 its tiles share.  Tiles run from the longest down; with two workgroups to a CU
// (turn) every other 32 (an XCD's CUs) are reversed, so that a long one shares its
// CU with a short one (two prompts of 1024, 32 heads on 8: 39.7 us without, 38.0
// with).
struct KvPlace {
  int32_t seq, head, tile, split, task;
};
__device__ __forceinline__ KvPlace kv_place(const KvAttnArgs &a, bool turn) {
  const uint32_t count = a.groups;
  uint32_t id = a.first + blockIdx.x;
  if (turn) {
    const uint32_t xcd = id & 7, size = (count >> 3) + (xcd < (count & 7) ? 1 : 0);
    uint32_t n = id >> 3;
    if ((n & 32) && (n | 31) < size) id = (n ^ 31) << 3 | xcd;
  }
  uint32_t rest = id;
  const uint32_t in_group = kv_rem(a.by_pairs, rest);
  uint32_t unit = kv_rem(a.by_units, rest);
  uint32_t pair = rest * a.by_pairs.d + in_group;
  KvPlace p;
  p.split = kv_rem(a.by_splits, unit);
  p.tile = a.row_tiles - 1 - static_cast<int32_t>(unit);
  p.task = pair * a.row_tiles + p.tile;
  p.head = kv_rem(a.by_heads, pair);
  p.seq = pair;
  return p;
}

// rnsmx_kv_rows.hip, one object per row size
template <int DT>
void launch_kv_rows(const KvAttnArgs &a, uint32_t groups, hipStream_t st);

// rnsmx_kv_tiles.hip, one object per row size
constexpr int kKvTileRows = 128;  // query rows of a workgroup of kv_tiles_kernel
// Row sizes whose staged steps fit the shared memory twice run on eight waves too.
constexpr int kv_tile_halves(int row_bytes) { return row_bytes <= 128 ? 2 : 1; }
template <int DT>
void launch_kv_tiles(const KvAttnArgs &a, uint32_t groups, hipStream_t st);

}  // namespace rnsmx
