// The 8-bit key/value cache: quantising tokens into pages, reading them back,
// and the host side of its C ABI.
#include <algorithm>
#include <cmath>

#include "rnsmx_kv.hpp"

namespace rnsmx {

struct KvAppendArgs {
  KvBatchArgs b;
  const void *src[2];
  int64_t row_stride[2], head_stride[2];
  int32_t vec;              // rows are read 16 bytes at a time
  KvDiv by_heads, by_pages;  // pages: most of one sequence that the rows touch
  uint32_t first;            // a launch's first workgroup
};

struct KvReadArgs {
  KvBatchArgs b;
  void *dst[2];
  int32_t vec;
  KvDiv by_heads, by_pages;
  uint32_t first;
};

constexpr float kKvMax = 127.0f;
constexpr int kKvHeld = 4;  // groups of 8 values a thread of kv_append_kernel holds

template <bool STREAM, typename T>
__device__ __forceinline__ void kv_load8(float (&x)[8], const T *p, int32_t left, bool vec) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const f32x4 a = reinterpret_cast<const f32x4 *>(p)[0], b = reinterpret_cast<const f32x4 *>(p)[1];
      kv_for<4>([&](auto I) {
        constexpr int i = I;
        x[i] = a[i];
        x[i + 4] = b[i];
      });
    } else {
      const u32x4 a = kv_fetch<STREAM>(reinterpret_cast<const u32x4 *>(p));
      kv_for<8>([&](auto I) {
        constexpr int i = I;
        const uint16_t bits = static_cast<uint16_t>(a[i / 2] >> (16 * (i % 2)));
        if constexpr (std::is_same<T, _Float16>::value)
          x[i] = static_cast<float>(__builtin_bit_cast(_Float16, bits));
        else
          x[i] = kv_bf16(bits);
      });
    }
    return;
  }
  kv_for<8>([&](auto I) {
    constexpr int i = I;
    float v = 0.0f;
    if (i < left) {
      if constexpr (std::is_same<T, uint16_t>::value)
        v = kv_bf16(p[i]);
      else
        v = static_cast<float>(p[i]);
    }
    x[i] = v;
  });
}

// Codes plus 128 of eight values at the scale s, each rint of the correctly
// rounded quotient x / s.  With r the correctly rounded 1 / s, q = x r is within
// an ulp of it and q + (x - q s) r, both products fused, is it (Markstein's
// theorem); where the remainder underflows x / s is far below a half.  Adding 1.5
// 2^23 leaves the integer in the low byte, rounded to even.  |x| <= 127.01 s, as s
// comes from the largest: no code needs a clamp.  A quarter of what divisions and
// conversions cost, which bounded prompts (10454 tokens, 32 heads of 128: 87 us with
// them, 66 so).
// At a scale that is not finite every code is zero.
__device__ __forceinline__ u32x2 kv_codes(const float (&x)[8], float s) {
  if (!(s < INFINITY)) return u32x2{0x80808080u, 0x80808080u};
  const float r = 1.0f / s;
  uint32_t n[8];
  kv_for<8>([&](auto I) {
    constexpr int i = I;
    const float q = x[i] * r;
    n[i] = __float_as_uint(fmaf(fmaf(-q, s, x[i]), r, q) + 12582912.0f);
  });
  u32x2 c;
  kv_for<2>([&](auto I) {
    constexpr int i = I;
    const uint32_t lo = __builtin_amdgcn_perm(n[4 * i + 1], n[4 * i], 0x0C0C0400u);
    const uint32_t hi = __builtin_amdgcn_perm(n[4 * i + 3], n[4 * i + 2], 0x04000C0Cu);
    c[i] = (lo | hi) ^ 0x80808080u;
  });
  return c;
}

// code * scale in float32.  The product is kept apart from a conversion to
// float16 after it: the compiler would join them into one operation, which
// rounds once, where the definition has float32 values.
__device__ __forceinline__ float kv_value(uint32_t c, int i, float s) {
  float v = static_cast<float>(static_cast<int32_t>((c >> (8 * i)) & 0xFFu) - 128) * s;
  asm("" : "+v"(v));
  return v;
}

// The end of those of a sequence's tokens that its rows are, up to max_rows of them.
__device__ __forceinline__ int32_t kv_rows_end(const KvSeq &q) { return min(q.base + q.n, q.len); }

// The tokens of one page that a sequence's rows are: `old` to end - 1, from row
// `row` on; nothing where the page is past their end.
struct KvSpan {
  int32_t page, old, end, row;
};
__device__ __forceinline__ KvSpan kv_span(const KvBatchArgs &b, const KvSeq &q, int32_t seq, int32_t index) {
  const int32_t from = max(q.base, 0), to = kv_rows_end(q), pg = (from >> b.log_page) + index;
  KvSpan r{-1, 0, 0, 0};
  if (to <= from || pg > (to - 1) >> b.log_page) return r;
  const int32_t start = pg << b.log_page;
  r.old = max(from - start, 0);
  r.end = min(to - start, 1 << b.log_page);
  r.row = q.row + (start + r.old) - q.base;
  r.page = ((const kv_const_i32 *)b.table)[seq * b.table_stride + pg];
  return r;
}

// One workgroup for the new tokens of one page and head, keys or values: a page's
// scale is one maximum over them, so they are read once and wait for it in registers,
// up to four groups of eight a thread (two: 1 % slower), and only a page that held
// tokens before and whose scale grows is read and written again.  Bound by memory:
// two or four bytes read and one written a value, 10454 tokens, 32 heads of 128 in
// bfloat16 (257 MB) in 49 us, 5.2 TB/s, waves waiting for loads 69 % of their time; a
// single token of 12 heads takes 3.2 us, which is the launch and three loads in turn
// (length, page, values).
template <int DT, typename T, bool STREAM>
__global__ __launch_bounds__(1024) void kv_append_kernel(const KvAppendArgs a) {
  constexpr int CPT = DT / 8;
  __shared__ uint32_t tops[16];
  const KvBatchArgs &b = a.b;
  uint32_t id = a.first + blockIdx.x;
  const int32_t part = id & 1;
  id >>= 1;
  const int32_t head = kv_rem(a.by_heads, id), index = kv_rem(a.by_pages, id), seq = id;
  const KvSeq q = kv_seq(b, seq);
  const KvSpan p = kv_span(b, q, seq, index);
  if (p.end == 0 || static_cast<uint32_t>(p.page) >= static_cast<uint32_t>(b.blocks)) return;
  const int64_t slot = static_cast<int64_t>(p.page) * b.heads + head;
  uint8_t *page = (part ? b.v : b.k) + (slot << b.log_page) * DT;
  const int64_t rs = part ? a.row_stride[1] : a.row_stride[0], hs = part ? a.head_stride[1] : a.head_stride[0];
  const T *src = static_cast<const T *>(part ? a.src[1] : a.src[0]) + p.row * rs + head * hs;
  const int32_t groups = (p.end - p.old) * CPT;

  float x[kKvHeld][8];
  uint32_t top = 0;  // of |x| as bits: ordered as the values are, a NaN above all
  kv_for<kKvHeld>([&](auto J) {
    constexpr int j = J;
    const int32_t c = threadIdx.x + j * blockDim.x;
    const int32_t t = c / CPT, d = (c - t * CPT) * 8;
    if (c < groups && d < b.dim) {
      kv_load8<STREAM>(x[j], src + t * rs + d, b.dim - d, a.vec);
    } else {
      kv_for<8>([&](auto I) { x[j][I] = 0.0f; });
    }
  });
  float *scale = b.scales + slot * 2 + part;
  const float held = p.old > 0 ? *scale : 0.0f;
  kv_for<kKvHeld>([&](auto J) { kv_for<8>([&](auto I) { top = max(top, __float_as_uint(x[J][I]) & 0x7FFFFFFFu); }); });
  kv_for<6>([&](auto I) { top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1 << I))); });
  if (blockDim.x > 64) {
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    for (uint32_t w = 0; w < blockDim.x / 64; ++w) top = max(top, tops[w]);
  }
  const float amax = __uint_as_float(top);
  float s = amax != amax ? amax : fmaxf(amax * (1.0f / kKvMax), 1.1920928955078125e-07f);
  if (p.old > 0) s = (s != s || held != held) ? __builtin_nanf("") : fmaxf(s, held);
  if (threadIdx.x == 0) *scale = s;
  kv_for<kKvHeld>([&](auto J) {
    const int32_t c = threadIdx.x + J * blockDim.x;
    if (c < groups) *reinterpret_cast<u32x2 *>(page + p.old * DT + c * 8) = kv_codes(x[J], s);
  });
  if (p.old > 0 && s != held)  // the older tokens' codes, to the larger scale
    for (int32_t c = threadIdx.x; c < p.old * CPT; c += blockDim.x) {
      u32x2 *at = reinterpret_cast<u32x2 *>(page + c * 8);
      const u32x2 code = *at;
      float v[8];
      kv_for<8>([&](auto I) {
        constexpr int i = I;
        v[i] = kv_value(code[i / 4], i % 4, held);
      });
      *at = kv_codes(v, s);
    }
}

// One workgroup for the rows of one page and head, keys and values: two groups of
// eight of each in flight a thread, as a page of 64 tokens of 128 values gives 256
// threads four.  Bound by memory: 16 sequences of up to 4095 tokens, 32 heads of 128 to
// bfloat16 (979 MB) in 190 us, 5.2 TB/s, a copy's rate; 257 tokens of 12 heads 3.1 us.
template <int DT, typename T, bool STREAM>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvReadArgs a) {
  constexpr int CPT = DT / 8;
  const KvBatchArgs &b = a.b;
  uint32_t id = a.first + blockIdx.x;
  const int32_t head = kv_rem(a.by_heads, id), index = kv_rem(a.by_pages, id), seq = id;
  const KvSeq q = kv_seq(b, seq);
  const int64_t rs = static_cast<int64_t>(b.heads) * b.dim;
  T *dst[2] = {static_cast<T *>(a.dst[0]) + head * b.dim, static_cast<T *>(a.dst[1]) + head * b.dim};
  if (index == 0) {  // rows that have no token: `none` before the first, and those after the last
    const int32_t none = min(max(-q.base, 0), q.all), last = max(kv_rows_end(q) - q.base, none);
    const int32_t empty = none + q.all - last;
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(empty) * b.dim; i += 256) {
      const int64_t e = i / b.dim, r = e < none ? e : last + (e - none);
      kv_for<2>([&](auto P) { dst[P][(q.row + r) * rs + (i - e * b.dim)] = static_cast<T>(0); });
    }
  }
  const KvSpan p = kv_span(b, q, seq, index);
  if (p.end == 0) return;
  const bool there = static_cast<uint32_t>(p.page) < static_cast<uint32_t>(b.blocks);
  const int64_t slot = static_cast<int64_t>(there ? p.page : 0) * b.heads + head;
  const int64_t at = ((slot << b.log_page) + p.old) * DT;
  const float scale[2] = {b.scales[slot * 2], b.scales[slot * 2 + 1]};
  kv_for<2>([&](auto P) { dst[P] += p.row * rs; });
  const int32_t groups = (p.end - p.old) * CPT;
  for (int32_t c0 = threadIdx.x; c0 < groups; c0 += 512) {
    u32x2 code[2][2];
    kv_for<2>([&](auto U) {
      const int32_t c = min(c0 + 256 * U, groups - 1);
      code[0][U] = *reinterpret_cast<const u32x2 *>(b.k + at + c * 8);
      code[1][U] = *reinterpret_cast<const u32x2 *>(b.v + at + c * 8);
    });
    kv_for<2>([&](auto U) {
      const int32_t c = c0 + 256 * U, t = c / CPT, d = (c - t * CPT) * 8;
      if (c < groups && d < b.dim)
        kv_for<2>([&](auto P) {
          T y[8];
          kv_for<8>([&](auto I) {
            constexpr int i = I;
            const float v = there ? kv_value(code[P][U][i / 4], i % 4, scale[P]) : 0.0f;
            if constexpr (std::is_same<T, uint16_t>::value)
              y[i] = kv_to_bf16(v);
            else
              y[i] = static_cast<T>(v);
          });
          T *to = dst[P] + t * rs + d;
          if (a.vec) {
            kv_for<sizeof(T) / 2>([&](auto I) {
              if constexpr (STREAM)
                __builtin_nontemporal_store(reinterpret_cast<u32x4 *>(y)[I], reinterpret_cast<u32x4 *>(to) + I);
              else
                reinterpret_cast<u32x4 *>(to)[I] = reinterpret_cast<u32x4 *>(y)[I];
            });
          } else {
            kv_for<8>([&](auto I) {
              if (d + I < b.dim) to[I] = y[I];
            });
          }
        });
    });
  }
}

static int32_t kv_row_bytes(int32_t dim) {
  for (int d : kKvDims)
    if (dim >= 1 && dim <= d) return d;
  return -1;
}

static int32_t kv_check(const char *what) {
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return RNSMX_OK;
  set_error("%s: %s", what, hipGetErrorString(err));
  return RNSMX_ELAUNCH;
}

static bool aligned(const void *p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

static int64_t dtype_bytes(int32_t dtype) { return dtype == RNSMX_FLOAT32 ? 4 : dtype == RNSMX_INT8 ? 1 : 2; }
static bool is_float(int32_t dtype) {
  return dtype == RNSMX_FLOAT32 || dtype == RNSMX_FLOAT16 || dtype == RNSMX_BFLOAT16;
}

static int32_t kv_batch_args(const rnsmx_kv_cache_t *cache, const rnsmx_kv_batch_t *batch, KvBatchArgs &a) {
  if (!cache || !batch) return fail(RNSMX_EINVAL, "null cache or batch");
  if (cache->page != 16 && cache->page != 32 && cache->page != 64 && cache->page != 128)
    return fail(RNSMX_EINVAL, "a page holds 16, 32, 64 or 128 tokens");
  if (cache->blocks < 1 || cache->heads < 1) return fail(RNSMX_EINVAL, "a cache has at least one page and one head");
  if (kv_row_bytes(cache->head_dim) < 0) return fail(RNSMX_EINVAL, "head dimensions are 1 to 256");
  if (cache->row_bytes != kv_row_bytes(cache->head_dim)) return fail(RNSMX_EINVAL, "row_bytes is not the head dimension's");
  if (!cache->k_dev || !cache->v_dev || !cache->scales_dev) return fail(RNSMX_EINVAL, "null cache pointer");
  if (!aligned(cache->k_dev, 16) || !aligned(cache->v_dev, 16) || !aligned(cache->scales_dev, 8))
    return fail(RNSMX_EINVAL, "codes start on 16-byte boundaries, scales on 8-byte ones");
  if (batch->seqs < 0 || batch->rows < 0 || batch->max_rows < 0 || batch->max_length < 0 || batch->table_width < 1 ||
      batch->table_stride < 0)
    return fail(RNSMX_EINVAL, "bad batch sizes");
  if (batch->max_length > 1 << 30) return fail(RNSMX_EINVAL, "sequences hold at most 2^30 tokens");
  if (batch->max_length > static_cast<int64_t>(batch->table_width) * cache->page)
    return fail(RNSMX_EINVAL, "max_length is past the block table");
  if (static_cast<int64_t>(batch->seqs) * cache->heads > 0x7FFFFFFFLL) return fail(RNSMX_EINVAL, "too many sequences and heads");
  if (batch->seqs > 0 && (!batch->table_dev || !batch->lengths_dev)) return fail(RNSMX_EINVAL, "null batch pointer");
  if (!aligned(batch->table_dev, 4) || !aligned(batch->lengths_dev, 4) || !aligned(batch->starts_dev, 4))
    return fail(RNSMX_EINVAL, "batch pointers are not on 4-byte boundaries");
  if (!batch->starts_dev && batch->rows != batch->seqs) return fail(RNSMX_EINVAL, "one row a sequence without row starts");
  a.k = cache->k_dev;
  a.v = cache->v_dev;
  a.scales = cache->scales_dev;
  a.table = batch->table_dev;
  a.lengths = batch->lengths_dev;
  a.starts = batch->starts_dev;
  a.table_stride = batch->table_stride;
  a.blocks = cache->blocks;
  a.log_page = cache->page == 16 ? 4 : cache->page == 32 ? 5 : cache->page == 64 ? 6 : 7;
  a.heads = cache->heads;
  a.dim = cache->head_dim;
  a.row_bytes = cache->row_bytes;
  a.seqs = batch->seqs;
  a.table_width = batch->table_width;
  a.rows = batch->rows;
  a.max_rows = batch->starts_dev ? std::min(batch->max_rows, batch->rows) : 1;
  a.max_length = batch->max_length;
  return RNSMX_OK;
}

// Most pages that max_rows tokens in a row can lie in.
static int64_t pages_touched(const KvBatchArgs &a) {
  const int64_t page = 1 << a.log_page, n = std::min(a.max_rows, a.max_length);
  return n < 1 ? 1 : (n + page - 2) / page + 1;
}

// Whether a call's bytes go past the caches: where the 256 MB behind the L2s would
// not keep them for the next reader, and a load or store takes its lines whole.  Keys
// and values of 20736 tokens, 32 heads of 128 (340 MB) in bfloat16: appended 95 us so,
// 105 through the caches, read 81 and 105; of 10368 tokens (170 MB) appended and read
// after each other 92 and 101, of 7296 tokens (120 MB) 73 both.  Float32 goes through
// them (a load takes half of its lines: 14592 tokens, 8 heads of 128, appended 36, 27
// through them, read 59, 29), and so do rows of other sizes (46848 tokens, 8 heads of
// 80: 53, 50 and 64, 35; rows of 192 bytes appended 114, 109, but read 81, 134).
// Attention (codes of 134 MB, 16 sequences of 4096 tokens, 8 heads of 128): 36 so, 40
// through the caches; rows of 64: 27, 30; of 160: 117, 107 (48 sequences).
constexpr int64_t kStreamBytes = 128ll << 20;
static bool streams(double bytes, bool whole) { return whole && bytes >= kStreamBytes; }
// Values of a call's rows, keys or values: past 64 bits for sizes that the checks take.
static double kv_values(const KvBatchArgs &b) { return static_cast<double>(b.rows) * b.heads * b.dim; }

// f(a value of the type, whether past the caches as a constant)
template <typename F>
static void kv_of_type(int32_t dtype, bool stream, F &&f) {
  auto with = [&](auto t) {
    if (stream)
      f(t, std::true_type{});
    else
      f(t, std::false_type{});
  };
  if (dtype == RNSMX_FLOAT32)
    f(float{}, std::false_type{});
  else if (dtype == RNSMX_FLOAT16)
    with(_Float16{});
  else
    with(uint16_t{});
}

static int32_t grid_of(int64_t groups, unsigned &grid) {
  if (groups > 0x7FFFFFFFLL) return fail(RNSMX_EINVAL, "too many sequences, pages and heads for one call");
  grid = static_cast<unsigned>(groups);
  return RNSMX_OK;
}

#define RNSMX_KV_DIM_CASE(D, ...) \
  case D: {                       \
    constexpr int DT = D;         \
    __VA_ARGS__;                  \
    break;                        \
  }
// the statement with DT the row size
#define RNSMX_KV_DIMS(dim, ...)          \
  switch (dim) {                         \
    RNSMX_KV_DIM_CASE(64, __VA_ARGS__)   \
    RNSMX_KV_DIM_CASE(96, __VA_ARGS__)   \
    RNSMX_KV_DIM_CASE(128, __VA_ARGS__)  \
    RNSMX_KV_DIM_CASE(160, __VA_ARGS__)  \
    RNSMX_KV_DIM_CASE(192, __VA_ARGS__)  \
    RNSMX_KV_DIM_CASE(256, __VA_ARGS__)  \
  }

// How a call's tokens are split over waves and workgroups (device time, 32-wide
// pages and up).  Eight waves take a step of 256 tokens where the workgroups
// leave room for them on the chip (24 x 8 heads of 80, window 1023: 13.5 us, 15.3
// with four) or sequences are long (62 x 32 heads of 128, up to 4096 tokens: 200,
// 204); many short ones take four (256 x 12 heads of 64, 512 tokens: 29.3, 39.7
// with eight).  Splitting costs the parts' way through memory and the ticket's,
// some 5 us: not past a workgroup a CU (one token against 131071, 8 heads: 58 us,
// 65 with twice as many), and not below 1024 tokens each (32 heads, 1024 tokens:
// 11.0 whole, 14.2 in two).
constexpr int64_t kSplitGroups = 256, kSplitTokens = 1024, kWideTasks = 512, kWideTokens = 4096;
// Prompts: eight waves where the tiles leave room for them (72 pairs of parts of
// prompts, 288 tiles: 44 us, 56 with four) or are few and long (8192 tokens, 8
// heads, 512 tiles: 195, 212), four where two workgroups to a CU hide each other's
// waits (8192 tokens, 32 heads: 654, 726 with eight; 2048 tokens, 32 heads: 69,
// 75).  Tokens are split only up to a workgroup a CU: a part is 64 KB at 128
// values a head (16 heads of 256, 1024 tokens, 128 tiles: 57 us in two, 72 whole;
// 2048 tokens, 32 heads, 512 tiles: 72 in two, 69 whole).
constexpr int64_t kTileGroups = 256, kTileTokens = 512, kHalvesTasks = 384;
// Most tokens between a workgroup's first and its last: a window's, the rows of one
// sequence that it may have, and what its first step starts before them.
static int64_t kv_tokens(const KvAttnArgs &a) {
  return a.window > 0 ? std::min<int64_t>(a.b.max_length, static_cast<int64_t>(a.window) + a.b.max_rows + 64) : a.b.max_length;
}
static void kv_split(KvAttnArgs &a) {
  const int64_t span = kv_tokens(a);
  const int64_t tasks = static_cast<int64_t>(a.b.seqs) * a.b.heads * a.row_tiles;
  const bool few = a.tile_rows == kKvRows;
  if (few)
    a.waves = kv_wide(a.b.row_bytes) && span > 128 && (tasks < kWideTasks || span >= kWideTokens) ? 8 : 4;
  else
    a.waves = kv_tile_halves(a.b.row_bytes) == 2 &&
                      (tasks <= kHalvesTasks || (tasks <= 512 && span >= kWideTokens))
                  ? 8
                  : 4;
  const int64_t unit = few ? 32 * a.waves : 64;
  const int64_t steps = std::max<int64_t>(1, (span + unit - 1) / unit);
  int64_t splits = 1;
  if (tasks > 0 && tasks <= RNSMX_KV_TICKETS)
    splits = few ? std::min(span / kSplitTokens, kSplitGroups / tasks) : std::min(span / kTileTokens, kTileGroups / tasks);
  splits = std::max<int64_t>(splits, 1);
  const int64_t each = (steps + splits - 1) / splits;
  a.chunk = static_cast<int32_t>(std::min<int64_t>(each * unit, 1 << 30));
  a.splits = static_cast<int32_t>((steps + each - 1) / each);
}

// Whether a call runs 16 rows to a workgroup: up to kFewRows rows of a sequence and
// key/value head, and past them while the work is too little to fill the chip with
// tiles of 128: kFewGroups workgroups of 16 rows, each seeing so many tokens that
// together they see kFewTokens.  One sequence of 8000 tokens, 8 heads, 128 rows: 27
// us so, 53 in tiles, 512 rows: 58 and 54; 32 sequences of 2000, 8 heads, 48 rows: 39
// and 54, 96 rows: 65 and 55; 4 of 500, 12 heads of 64, 400 rows: 11 and 17; prompts
// of 1024 in float32, 32 heads: 58 and 44.  Half as many groups of heads wider than
// 160, whose waves are one to a SIMD (1024 tokens, 16 heads of 256: 70 and 60).
constexpr int64_t kFewRows = 32, kFewGroups = 1280, kFewTokens = 1750000;
static bool few_rows(const KvBatchArgs &b, int64_t rows, int64_t span) {
  if (rows <= kFewRows) return true;
  const int64_t groups = static_cast<int64_t>(b.seqs) * b.heads * ((rows + kKvRows - 1) / kKvRows);
  return groups <= (kv_wide(b.row_bytes) ? kFewGroups : kFewGroups / 2) && groups * std::max<int64_t>(span - b.max_rows / 2, 1) <= kFewTokens;
}

// Pairs of sequences and heads whose workgroups run side by side: all, or where
// there are many a divisor of their number, so that an XCD's part of them stays
// in its L2 from one tile of rows to the next.
static int64_t pairs_at_once(int64_t pairs) {
  if (pairs <= 256) return std::max<int64_t>(pairs, 1);
  for (int64_t n = 256; n >= 64; n -= 8)
    if (pairs % n == 0) return n;
  return pairs;
}

static int32_t kv_attn_args(const rnsmx_kv_cache_t *cache, const rnsmx_kv_batch_t *batch, const rnsmx_kv_query_t *query,
                            KvAttnArgs &a) {
  if (int32_t rc = kv_batch_args(cache, batch, a.b)) return rc;
  if (!query) return fail(RNSMX_EINVAL, "null query");
  if (!is_float(query->dtype)) return fail(RNSMX_EINVAL, "queries are float32, float16 or bfloat16");
  if (query->q_heads < 1 || query->q_heads % cache->heads != 0)
    return fail(RNSMX_EINVAL, "query heads are a multiple of the cache's heads");
  if (!(query->scale > 0.0f) || !std::isfinite(query->scale)) return fail(RNSMX_EINVAL, "the scale is positive and finite");
  if (query->window < 0 || (query->window > 0 && !query->causal)) return fail(RNSMX_EINVAL, "a window needs causal rows");
  a.q_rs = query->row_stride;
  a.q_hs = query->head_stride;
  a.mask_rs = query->mask_row_stride;
  a.mask_hs = query->mask_head_stride;
  a.mask_ts = query->mask_token_stride;
  a.mask_dtype = query->mask_dtype;
  a.mask_len = query->mask_len;
  a.q_heads = query->q_heads;
  a.dtype = query->dtype;
  a.causal = query->causal != 0;
  a.window = query->window;
  a.scale = query->scale;
  const int64_t rows = static_cast<int64_t>(a.b.max_rows) * (query->q_heads / cache->heads);
  if (rows > 0x7FFFFFFF - kKvTileRows) return fail(RNSMX_EINVAL, "too many rows");  // of 32 bits in the kernels
  a.tile_rows = few_rows(a.b, rows, kv_tokens(a)) ? kKvRows : kKvTileRows;
  a.row_tiles = static_cast<int32_t>((rows + a.tile_rows - 1) / a.tile_rows);
  kv_split(a);
  a.row_tiles = std::max(a.row_tiles, 1);  // what zeroes a sequence's rows past max_rows 0
  a.by_group = kv_div(query->q_heads / cache->heads);
  a.by_splits = kv_div(a.splits);
  a.by_units = kv_div(a.row_tiles * a.splits);
  a.by_pairs = kv_div(static_cast<uint32_t>(pairs_at_once(static_cast<int64_t>(a.b.seqs) * cache->heads)));
  a.by_heads = kv_div(cache->heads);
  return RNSMX_OK;
}

// Each code is read by one workgroup alone, and they are many.
static bool kv_past_caches(const KvAttnArgs &a, bool masked) {
  return !masked && a.tile_rows == kKvRows && a.row_tiles == 1 &&
         streams(2.0 * a.b.row_bytes * a.b.heads * a.b.seqs * kv_tokens(a), kv_whole(a.b.row_bytes));
}

static int64_t kv_tasks(const KvAttnArgs &a) { return static_cast<int64_t>(a.b.seqs) * a.b.heads * a.row_tiles; }

static int64_t kv_workspace(const KvAttnArgs &a) {
  if (a.splits < 2) return 0;
  return RNSMX_KV_TICKETS * 4 +
         kv_tasks(a) * a.splits * (a.tile_rows == kKvRows ? kv_row_floats(a.b.row_bytes) : kv_tile_floats(a.b.row_bytes)) * 4;
}

}  // namespace rnsmx

using namespace rnsmx;

extern "C" {

int32_t rnsmx_kv_row_bytes(int32_t head_dim) { return kv_row_bytes(head_dim); }

int32_t rnsmx_kv_append(const rnsmx_kv_cache_t *cache, const rnsmx_kv_batch_t *batch, const void *k_dev,
                        const void *v_dev, int32_t dtype, int64_t k_row_stride, int64_t k_head_stride,
                        int64_t v_row_stride, int64_t v_head_stride, void *stream) {
  clear_error();
  KvAppendArgs a{};
  if (int32_t rc = kv_batch_args(cache, batch, a.b)) return rc;
  if (!is_float(dtype)) return fail(RNSMX_EINVAL, "keys and values are float32, float16 or bfloat16");
  if (a.b.rows == 0 || a.b.seqs == 0) return RNSMX_OK;
  const int64_t size = dtype_bytes(dtype);
  if (!k_dev || !v_dev || !aligned(k_dev, size) || !aligned(v_dev, size))
    return fail(RNSMX_EINVAL, "keys or values null or not aligned to their type");
  a.src[0] = k_dev;
  a.src[1] = v_dev;
  a.row_stride[0] = k_row_stride;
  a.row_stride[1] = v_row_stride;
  a.head_stride[0] = k_head_stride;
  a.head_stride[1] = v_head_stride;
  a.vec = a.b.dim % 8 == 0 && aligned(k_dev, 16) && aligned(v_dev, 16) && k_row_stride * size % 16 == 0 &&
          v_row_stride * size % 16 == 0 && k_head_stride * size % 16 == 0 && v_head_stride * size % 16 == 0;
  const int64_t pages = pages_touched(a.b);
  a.by_heads = kv_div(a.b.heads);
  a.by_pages = kv_div(static_cast<uint32_t>(pages));
  unsigned grid;
  if (int32_t rc = grid_of(a.b.seqs * pages * a.b.heads * 2, grid)) return rc;
  // every thread holds kKvHeld groups of 8 values of the tokens that a page can get
  const int64_t tokens = std::min<int64_t>(cache->page, a.b.max_rows);
  const int64_t groups = (tokens * (a.b.row_bytes / 8) + kKvHeld - 1) / kKvHeld;
  const unsigned threads = static_cast<unsigned>(std::max<int64_t>(64, (groups + 63) / 64 * 64));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool whole = size == 2 && a.vec && a.b.dim % 64 == 0 && aligned(k_dev, 128) && aligned(v_dev, 128) &&
                     k_row_stride % 64 == 0 && v_row_stride % 64 == 0 && k_head_stride % 64 == 0 && v_head_stride % 64 == 0;
  kv_of_type(dtype, streams(2.0 * size * kv_values(a.b), whole), [&](auto t, auto stream) {
    using T = decltype(t);
    kv_launches(grid, threads, [&](uint32_t first, uint32_t groups) {
      a.first = first;
      RNSMX_KV_DIMS(a.b.row_bytes, hipLaunchKernelGGL((kv_append_kernel<DT, T, decltype(stream)::value>), dim3(groups), dim3(threads), 0, st, a))
    });
  });
  return kv_check("kv_append");
}

int32_t rnsmx_kv_read(const rnsmx_kv_cache_t *cache, const rnsmx_kv_batch_t *batch, void *k_dev, void *v_dev,
                      int32_t dtype, void *stream) {
  clear_error();
  KvReadArgs a{};
  if (int32_t rc = kv_batch_args(cache, batch, a.b)) return rc;
  if (!is_float(dtype)) return fail(RNSMX_EINVAL, "values are read as float32, float16 or bfloat16");
  if (a.b.rows == 0 || a.b.seqs == 0) return RNSMX_OK;
  const int64_t size = dtype_bytes(dtype);
  if (!k_dev || !v_dev || !aligned(k_dev, size) || !aligned(v_dev, size))
    return fail(RNSMX_EINVAL, "keys or values null or not aligned to their type");
  a.dst[0] = k_dev;
  a.dst[1] = v_dev;
  a.vec = a.b.dim % 8 == 0 && aligned(k_dev, 16) && aligned(v_dev, 16);
  const int64_t pages = pages_touched(a.b);
  a.by_heads = kv_div(a.b.heads);
  a.by_pages = kv_div(static_cast<uint32_t>(pages));
  unsigned grid;
  if (int32_t rc = grid_of(a.b.seqs * pages * a.b.heads, grid)) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool whole = size == 2 && a.vec && a.b.dim % 32 == 0 && aligned(k_dev, 64) && aligned(v_dev, 64);
  kv_of_type(dtype, streams(2.0 * size * kv_values(a.b), whole), [&](auto t, auto stream) {
    using T = decltype(t);
    kv_launches(grid, 256, [&](uint32_t first, uint32_t groups) {
      a.first = first;
      RNSMX_KV_DIMS(a.b.row_bytes, hipLaunchKernelGGL((kv_read_kernel<DT, T, decltype(stream)::value>), dim3(groups), dim3(256), 0, st, a))
    });
  });
  return kv_check("kv_read");
}

int64_t rnsmx_kv_attention_workspace_bytes(const rnsmx_kv_cache_t *cache, const rnsmx_kv_batch_t *batch,
                                           const rnsmx_kv_query_t *query) {
  clear_error();
  KvAttnArgs a{};
  if (kv_attn_args(cache, batch, query, a)) return -1;
  return kv_workspace(a);
}

int32_t rnsmx_kv_attention_plan(const rnsmx_kv_cache_t *cache, const rnsmx_kv_batch_t *batch,
                                const rnsmx_kv_query_t *query, int32_t masked, rnsmx_kv_plan_t *out) {
  clear_error();
  if (!out) return fail(RNSMX_EINVAL, "null plan");
  KvAttnArgs a{};
  if (int32_t rc = kv_attn_args(cache, batch, query, a)) return rc;
  *out = rnsmx_kv_plan_t{a.tile_rows, a.row_tiles, a.waves, a.splits, a.chunk, kv_past_caches(a, masked != 0)};
  return RNSMX_OK;
}

int32_t rnsmx_kv_attention(const rnsmx_kv_cache_t *cache, const rnsmx_kv_batch_t *batch, const rnsmx_kv_query_t *query,
                           const void *q_dev, const void *mask_dev, void *workspace_dev, int64_t workspace_bytes,
                           void *out_dev, void *stream) {
  clear_error();
  KvAttnArgs a{};
  if (int32_t rc = kv_attn_args(cache, batch, query, a)) return rc;
  if (a.b.rows == 0 || a.b.seqs == 0) return RNSMX_OK;
  const int64_t size = dtype_bytes(a.dtype);
  if (!q_dev || !aligned(q_dev, size)) return fail(RNSMX_EINVAL, "queries null or not aligned to their type");
  if (mask_dev) {
    if (query->mask_dtype != RNSMX_INT8 && !is_float(query->mask_dtype))
      return fail(RNSMX_EINVAL, "masks are bytes, float32, float16 or bfloat16");
    if (query->mask_len < 0) return fail(RNSMX_EINVAL, "bad mask length");
    if (!aligned(mask_dev, dtype_bytes(query->mask_dtype))) return fail(RNSMX_EINVAL, "the mask is not aligned to its type");
  }
  a.q = q_dev;
  a.mask = mask_dev;
  a.vec = cache->head_dim % 8 == 0 && aligned(q_dev, 16) && query->row_stride * size % 16 == 0 &&
          query->head_stride * size % 16 == 0;
  if (!out_dev || !aligned(out_dev, size)) return fail(RNSMX_EINVAL, "output null or not aligned to its type");
  const int64_t need = kv_workspace(a);
  if (need > 0) {
    if (!workspace_dev || !aligned(workspace_dev, 16)) return fail(RNSMX_EINVAL, "workspace null or not on a 16-byte boundary");
    if (workspace_bytes < need) return fail(RNSMX_ESPACE, "workspace too small");
    a.tickets = static_cast<uint32_t *>(workspace_dev);
    a.partial = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace_dev) + RNSMX_KV_TICKETS * 4);
  }
  a.out = out_dev;
  a.stream = kv_past_caches(a, a.mask != nullptr);
  unsigned grid;
  if (int32_t rc = grid_of(kv_tasks(a) * a.splits, grid)) return rc;
  if (grid == 0) return RNSMX_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  a.out_vec = aligned(out_dev, 16);
  a.groups = grid;
  kv_launches(grid, 64 * a.waves, [&](uint32_t first, uint32_t groups) {
    a.first = first;
    if (a.tile_rows == kKvTileRows) {
      RNSMX_KV_DIMS(a.b.row_bytes, launch_kv_tiles<DT>(a, groups, st))
    } else {
      RNSMX_KV_DIMS(a.b.row_bytes, launch_kv_rows<DT>(a, groups, st))
    }
  });
  return kv_check("kv_attention");
}

}  // extern "C"
