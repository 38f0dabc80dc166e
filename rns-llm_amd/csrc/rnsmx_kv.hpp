// The 8-bit key/value cache: what its kernels share (rnsmx_kv_cache.hip writes
// and reads pages, rnsmx_kv_rows.hip attends with few rows).
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <utility>

#include "rnsmx_common.hpp"

namespace rnsmx {

typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename F, int... I>
__device__ __forceinline__ void kv_for_impl(F &&f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void kv_for(F &&f) {
  kv_for_impl(f, std::make_integer_sequence<int, N>{});
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

// One sequence's length and rows, cut to what the host was told.
struct KvSeq {
  int32_t len, row, n;
};
__device__ __forceinline__ KvSeq kv_seq(const KvBatchArgs &a, int32_t s) {
  KvSeq r;
  r.len = min(max(a.lengths[s], 0), a.max_length);
  if (a.starts) {
    r.row = min(max(a.starts[s], 0), a.rows);
    r.n = min(max(a.starts[s + 1] - r.row, 0), min(a.max_rows, a.rows - r.row));
  } else {
    r.row = s;
    r.n = 1;
  }
  return r;
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
  int32_t q_heads, group, dtype, mask_dtype, mask_len;
  int32_t causal, window, vec;  // vec: q rows are read 16 bytes at a time
  int32_t chunk, splits, row_tiles;
  float scale;
};

constexpr int kKvRowTile = 16;   // query rows of a workgroup of kv_rows_kernel
constexpr int kKvChunkUnit = 128;  // tokens four waves take per step

// Floats of one split's partial result: 16 rows of row_bytes values, then each
// row's reference and sum.
inline int64_t kv_partial_floats(int32_t row_bytes) { return kKvRowTile * (static_cast<int64_t>(row_bytes) + 2); }

// rnsmx_kv_rows.hip, one object per row size
template <int DT>
void launch_kv_rows(const KvAttnArgs &a, hipStream_t st);

}  // namespace rnsmx
