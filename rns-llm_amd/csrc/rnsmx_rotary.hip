// Rotary positions: queries and keys turned by their positions' angles.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <type_traits>

#include "rnsmx_kv_attn.hpp"

namespace rnsmx {

// One of the two tensors of a call: heads of `dim` values at its strides.
struct RotaryPart {
  const void *src;
  void *dst;
  int64_t src_rs, src_hs, dst_rs, dst_hs;
};

struct RotaryArgs {
  RotaryPart part[2];
  const uint64_t *steps;
  const void *positions;
  int64_t rows, first;  // a launch's first row
  int32_t wide;  // positions of 64 bits
  int32_t q_heads, heads, pairs, dim;
  int32_t pieces;     // of a head: its pairs, then what is copied
  int32_t turning;    // of them those of pairs
  int32_t per_row;    // pieces of a row
  int32_t row_tile;   // rows of a workgroup
  int32_t head_tile;  // heads of a workgroup
  KvDiv by_pieces, by_row, by_pairs;
  float magnitude, sign;
};

constexpr int kRotaryTable = 1024;  // angles of a workgroup

// Cosine and sine of a position's angle.  position * step mod 2^64 is the fraction
// of a turn, exact but for the step's own last place (2^-65 turns a position, below the
// 2^-32 that is kept up to position 2^32).  Its upper half is cut into quarters, so that what
// is converted to float32 is below an eighth of a turn and keeps its bits.
__device__ __forceinline__ F32x2 rotary_angle(int64_t position, uint64_t step) {
  const uint32_t turn = static_cast<uint32_t>((static_cast<uint64_t>(position) * step) >> 32);
  const uint32_t quarter = (turn + 0x20000000u) >> 30;
  const float x = static_cast<float>(static_cast<int32_t>(turn - (quarter << 30))) * 4.656612873077393e-10f;  // 2^-31
  float s, c;
  sincospif(x, &s, &c);
  const float co = quarter & 1 ? s : c, si = quarter & 1 ? c : s;
  return F32x2{(quarter == 1 || quarter == 2) ? -co : co, quarter >= 2 ? -si : si};
}

template <typename T>
__device__ __forceinline__ float rotary_load(T v) {
  if constexpr (std::is_same<T, uint16_t>::value)
    return kv_bf16(v);
  else
    return static_cast<float>(v);
}
template <typename T>
__device__ __forceinline__ T rotary_round(float v) {
  if constexpr (std::is_same<T, uint16_t>::value)
    return kv_to_bf16(v);
  else
    return static_cast<T>(v);
}

// f(where, how many) for the first `left` of N values: all of them, or fours, a two and a one.
template <int N, typename F>
__device__ __forceinline__ void rotary_parts(int32_t left, F &&f) {
  using std::integral_constant;
  if (left >= N) return f(integral_constant<int, 0>{}, integral_constant<int, N>{});
  kv_for<N / 4>([&](auto Q) {
    constexpr int q = 4 * Q;
    if (left >= q + 4) {
      f(integral_constant<int, q>{}, integral_constant<int, 4>{});
    } else if (left >= q + 2) {
      f(integral_constant<int, q>{}, integral_constant<int, 2>{});
      if (left == q + 3) f(integral_constant<int, q + 2>{}, integral_constant<int, 1>{});
    } else if (left == q + 1) {
      f(integral_constant<int, q>{}, integral_constant<int, 1>{});
    }
  });
}
// 16 bytes at p, of whose values those from `left` on are not there.  Whole ones are one load or
// store from wherever they begin (6909 rows of 64 heads of 65 in 16 bits: 36 us, 69 by values).
template <bool VEC, bool STREAM, typename T, int N>
__device__ __forceinline__ void rotary_get(T (&x)[N], const T *p, int32_t left) {
  if constexpr (VEC) {
    *reinterpret_cast<u32x4 *>(x) = kv_fetch<STREAM>(reinterpret_cast<const u32x4 *>(p));
  } else {
    rotary_parts<N>(left, [&](auto at, auto n) { __builtin_memcpy(x + at, p + at, n * sizeof(T)); });
  }
}
template <bool VEC, bool STREAM, typename T, int N>
__device__ __forceinline__ void rotary_put(T *p, const T (&x)[N], int32_t left) {
  if constexpr (VEC && STREAM) {
    __builtin_nontemporal_store(*reinterpret_cast<const u32x4 *>(x), reinterpret_cast<u32x4 *>(p));
  } else if constexpr (VEC) {
    *reinterpret_cast<u32x4 *>(p) = *reinterpret_cast<const u32x4 *>(x);
  } else {
    rotary_parts<N>(left, [&](auto at, auto n) { __builtin_memcpy(p + at, x + at, n * sizeof(T)); });
  }
}

// A workgroup takes some rows and heads: the rows' angles once into shared memory,
// then a piece a thread and step: the pairs of two loads of 16 bytes.  A thread reads what it writes before it writes
// it, so a call may be in place.
template <typename T, bool VEC, bool NEIGHBOURS, bool STREAM>
__global__ __launch_bounds__(256) void rotate_kernel(const RotaryArgs a) {
  constexpr int N = 16 / sizeof(T);  // values of a load, pairs of a piece
  __shared__ __attribute__((aligned(16))) F32x2 angles[kRotaryTable];
  const int64_t row0 = a.first + static_cast<int64_t>(blockIdx.x) * a.row_tile;
  const int32_t rows = static_cast<int32_t>(min(static_cast<int64_t>(a.row_tile), a.rows - row0));
  const int32_t head0 = blockIdx.y * a.head_tile;
  const int32_t count = rows * a.per_row;
  const int32_t half = a.pairs;

  struct Piece {
    alignas(16) T x[2][N] = {};
    const T *from;
    T *to;
    int32_t at[2], left[2], row;  // columns and how many of them are there
    bool there, turned;
  };
  auto load = [&](Piece &p, int32_t i) {
    p.there = i < count;
    uint32_t n = static_cast<uint32_t>(min(i, count - 1));
    const int32_t in_row = kv_rem(a.by_row, n);
    p.row = n;
    n = in_row;
    const int32_t piece = kv_rem(a.by_pieces, n), head = head0 + n;
    const bool second = head >= a.q_heads;
    p.there = p.there && head < a.q_heads + a.heads;
    const int32_t h = p.there ? head - (second ? a.q_heads : 0) : 0;
    const int64_t row = row0 + p.row;
    const RotaryPart &u = a.part[0], &v = a.part[1];
    p.from = static_cast<const T *>(second ? v.src : u.src) + (row * (second ? v.src_rs : u.src_rs) + h * (second ? v.src_hs : u.src_hs));
    p.to = static_cast<T *>(second ? v.dst : u.dst) + (row * (second ? v.dst_rs : u.dst_rs) + h * (second ? v.dst_hs : u.dst_hs));
    p.turned = piece < a.turning;
    // A load of neighbours or of what is copied lies beside that of the next thread, and a
    // piece's second as far behind it as there are pieces (side by side they take their lines by
    // halves: 12000 rows of 64 heads of 128 neighbours in 16 bits 168 us, 66 so).
    if (p.turned && !NEIGHBOURS) {
      p.at[0] = N * piece;
      p.at[1] = half + N * piece;
      p.left[0] = p.left[1] = half - N * piece;
    } else {
      p.at[0] = p.turned ? N * piece : 2 * half + N * (piece - a.turning);
      p.at[1] = p.at[0] + N * (p.turned ? a.turning : a.pieces - a.turning);
      const int32_t end = p.turned ? 2 * half : a.dim;
      p.left[0] = end - p.at[0];
      p.left[1] = end - p.at[1];
    }
    kv_for<2>([&](auto K) {
      // whole or not at all where loads are
      if (p.there && p.left[K] > 0) rotary_get<VEC, STREAM>(p.x[K], p.from + p.at[K], p.left[K]);
    });
  };
  auto store = [&](Piece &p) {
    if (!p.there) return;
    if (p.turned) {
      const F32x2 *const t = angles + p.row * half;
      kv_for<N>([&](auto I) {
        constexpr int i = I;
        // neighbours: pair i lies in values 2 i, 2 i + 1 of the two loads
        constexpr int ka = NEIGHBOURS ? (2 * i) / N : 0, ia = NEIGHBOURS ? (2 * i) % N : i;
        constexpr int kb = NEIGHBOURS ? (2 * i + 1) / N : 1, ib = NEIGHBOURS ? (2 * i + 1) % N : i;
        const int32_t pair = NEIGHBOURS ? p.at[ka] / 2 + ia / 2 : p.at[0] + i;
        const F32x2 cs = VEC || pair < half ? t[pair] : F32x2{1.0f, 0.0f};
        const float u = rotary_load(p.x[ka][ia]), v = rotary_load(p.x[kb][ib]);
        p.x[ka][ia] = rotary_round<T>(fmaf(u, cs.x, -(v * cs.y)));
        p.x[kb][ib] = rotary_round<T>(fmaf(v, cs.x, u * cs.y));
      });
    }
    kv_for<2>([&](auto K) {
      if (p.left[K] > 0) rotary_put<VEC, STREAM>(p.to + p.at[K], p.x[K], p.left[K]);
    });
  };

  Piece first;
  load(first, threadIdx.x);
  for (int32_t i = threadIdx.x; i < rows * half; i += 256) {
    uint32_t r = i;
    const int32_t pair = kv_rem(a.by_pairs, r);
    const int64_t row = row0 + r;
    const int64_t position = a.wide ? static_cast<const int64_t *>(a.positions)[row] : static_cast<const int32_t *>(a.positions)[row];
    const F32x2 t = rotary_angle(position, a.steps[pair]);
    angles[i] = F32x2{t.x * a.magnitude, t.y * (a.magnitude * a.sign)};
  }
  __syncthreads();
  store(first);
  for (int32_t i = threadIdx.x + 256; i < count; i += 512) {
    Piece p, q;
    load(p, i);
    load(q, i + 256);
    store(p);
    store(q);
  }
}

// Whether every row and head begins at a multiple of `bytes`.
static bool rotary_on(int64_t bytes, int64_t size, const void *p, int64_t rs, int64_t hs) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && rs % bytes * size % bytes == 0 && hs % bytes * size % bytes == 0;
}

// Bytes from the first to past the last of a tensor's rows.
static int64_t rotary_extent(int64_t rows, int64_t heads, int64_t dim, int64_t rs, int64_t hs, int64_t size) {
  return ((rows - 1) * rs + (heads - 1) * hs + dim) * size;
}

// No address space has 2^57 bytes, and below that no extent wraps.
static bool rotary_addressed(int64_t rows, int64_t heads, int64_t dim, int64_t rs, int64_t hs, int64_t size) {
  return (static_cast<double>(rows - 1) * rs + static_cast<double>(heads - 1) * hs + dim) * size < 0x1p57;
}

// Whether `a` and `b`, rows and heads of `dim` values each at its strides and as many rows, share no
// value: apart as a whole, blocks side by side in steps of one stride (columns of one product, whose
// rows or, transposed, heads are that far apart), or, rows being one stride apart, no two heads
// the same.  Rows at other strides that lie among each other are taken to share.
struct RotaryGrid {
  const void *p;
  int64_t rs, hs, rows, heads;
};
static bool rotary_apart(const RotaryGrid &a, const RotaryGrid &b, int64_t dim, int64_t size) {
  if (!ranges_meet(a.p, rotary_extent(a.rows, a.heads, dim, a.rs, a.hs, size), b.p, rotary_extent(b.rows, b.heads, dim, b.rs, b.hs, size)))
    return true;
  const int64_t bytes = static_cast<const char *>(b.p) - static_cast<const char *>(a.p);
  if (bytes % size != 0) return false;
  // what lies within one step of the stride, from a's start on, around its end
  auto fit = [&](int64_t stride, int64_t span_a, int64_t span_b) {
    if (stride <= 0) return false;
    const int64_t at = ((bytes / size) % stride + stride) % stride;
    return at >= span_a && at + span_b <= stride;
  };
  const int64_t rs = a.rows == 1 ? 0 : a.rs;
  if (a.hs == b.hs && fit(a.hs, (a.rows - 1) * a.rs + dim, (b.rows - 1) * b.rs + dim)) return true;
  if ((a.rows > 1 && a.rs != b.rs) || (a.rows > 1 && rs < dim)) return false;
  if (fit(rs, (a.heads - 1) * a.hs + dim, (b.heads - 1) * b.hs + dim)) return true;
  // a head of b begins `at` past one of a, and `rows` strides more in other rows
  auto meet = [&](int64_t at) {
    if (rs == 0) return std::abs(at) < dim;
    const int64_t over = (at % rs + rs) % rs, down = (at - over) / rs;  // at - down * rs = over, the row before: over - rs
    return (over < dim && std::abs(down) < a.rows) || (rs - over < dim && std::abs(down + 1) < a.rows);
  };
  for (int64_t h = 0; h < b.heads; ++h) {
    if (meet(bytes / size + h * b.hs)) return false;
    // at one stride of heads only how far they are apart counts
    for (int64_t g = 1; g < (a.hs == b.hs && h > 0 ? 0 : a.heads); ++g)
      if (meet(bytes / size + h * b.hs - g * a.hs)) return false;
  }
  return true;
}

}  // namespace rnsmx

using namespace rnsmx;

extern "C" {

int32_t rnsmx_rotate(const rnsmx_rotary_t *rotary, const rnsmx_rotary_rows_t *rows, const void *positions_dev, const void *q_dev,
                     const void *k_dev, void *q_out_dev, void *k_out_dev, void *stream) {
  clear_error();
  if (!rotary || !rows) return fail(RNSMX_EINVAL, "null rotary or rows");
  if (rows->dtype != RNSMX_FLOAT32 && rows->dtype != RNSMX_FLOAT16 && rows->dtype != RNSMX_BFLOAT16)
    return fail(RNSMX_EINVAL, "queries and keys are float32, float16 or bfloat16");
  if (rows->positions_dtype != RNSMX_INT32 && rows->positions_dtype != RNSMX_INT64)
    return fail(RNSMX_EINVAL, "positions are int32 or int64");
  if (rows->rows < 0 || rows->q_heads < 0 || rows->k_heads < 0 || rows->head_dim < 1 || rows->head_dim > RNSMX_ROTARY_MAX_DIM ||
      static_cast<int64_t>(rows->q_heads) + rows->k_heads > RNSMX_ROTARY_MAX_HEADS)
    return fail(RNSMX_EINVAL, "bad row sizes");
  if (rotary->pairs < 1 || 2 * static_cast<int64_t>(rotary->pairs) > rows->head_dim)
    return fail(RNSMX_EINVAL, "the pairs are more than a head has");
  if (!std::isfinite(rotary->magnitude)) return fail(RNSMX_EINVAL, "the magnitude is not finite");
  for (const int64_t s : {rows->q_row_stride, rows->q_head_stride, rows->k_row_stride, rows->k_head_stride, rows->q_out_row_stride,
                          rows->q_out_head_stride, rows->k_out_row_stride, rows->k_out_head_stride})
    if (s < 0) return fail(RNSMX_EINVAL, "negative strides");
  const int32_t heads = rows->q_heads + rows->k_heads;
  if (rows->rows == 0 || heads == 0) return RNSMX_OK;
  if (rows->rows > 0x7FFFFFFFLL) return fail(RNSMX_EINVAL, "too many rows");
  const int64_t size = rows->dtype == RNSMX_FLOAT32 ? 4 : 2;
  if (!rotary->steps_dev || reinterpret_cast<uintptr_t>(rotary->steps_dev) % 8 != 0 || !positions_dev ||
      reinterpret_cast<uintptr_t>(positions_dev) % (rows->positions_dtype == RNSMX_INT64 ? 8 : 4) != 0)
    return fail(RNSMX_EINVAL, "steps or positions null or not aligned to their type");

  RotaryArgs a{};
  a.part[0] = {q_dev, q_out_dev, rows->q_row_stride, rows->q_head_stride, rows->q_out_row_stride, rows->q_out_head_stride};
  a.part[1] = {k_dev, k_out_dev, rows->k_row_stride, rows->k_head_stride, rows->k_out_row_stride, rows->k_out_head_stride};
  const int32_t part_heads[2] = {rows->q_heads, rows->k_heads};
  const int32_t step = static_cast<int32_t>(16 / size);  // values of a load
  for (int i = 0; i < 2; ++i)
    if (part_heads[i] > 0 && !(rotary_addressed(rows->rows, part_heads[i], rows->head_dim, a.part[i].src_rs, a.part[i].src_hs, size) &&
                               rotary_addressed(rows->rows, part_heads[i], rows->head_dim, a.part[i].dst_rs, a.part[i].dst_hs, size)))
      return fail(RNSMX_EINVAL, "strides past the address space");
  bool vec = rotary->pairs % step == 0 && rows->head_dim % step == 0, copied = false, lines = true;
  if (part_heads[0] > 0 && part_heads[1] > 0 && q_out_dev && k_out_dev &&
      !rotary_apart({q_out_dev, rows->q_out_row_stride, rows->q_out_head_stride, rows->rows, rows->q_heads},
                    {k_out_dev, rows->k_out_row_stride, rows->k_out_head_stride, rows->rows, rows->k_heads}, rows->head_dim, size))
    return fail(RNSMX_EINVAL, "the outputs of queries and keys share values, or lie among each other's rows at another row stride");
  for (int i = 0; i < 2; ++i) {
    if (part_heads[i] == 0) continue;
    const RotaryPart &p = a.part[i];
    if (!p.src || !p.dst || reinterpret_cast<uintptr_t>(p.src) % size != 0 || reinterpret_cast<uintptr_t>(p.dst) % size != 0)
      return fail(RNSMX_EINVAL, "queries, keys or outputs null or not aligned to their type");
    const bool in_place = p.src == p.dst && p.src_rs == p.dst_rs && p.src_hs == p.dst_hs;
    copied = copied || !in_place;
    vec = vec && rotary_on(16, size, p.src, p.src_rs, p.src_hs) && rotary_on(16, size, p.dst, p.dst_rs, p.dst_hs);
    lines = lines && rotary_on(128, size, p.src, p.src_rs, p.src_hs) && rotary_on(128, size, p.dst, p.dst_rs, p.dst_hs);
    // Outputs meet an input's memory only where they are it; columns of one
    // product interleave without sharing a value, which ranges cannot tell.
    for (int j = 0; j < 2; ++j) {
      if (part_heads[j] == 0 || (in_place && j == i)) continue;
      const RotaryPart &other = a.part[j];
      if (in_place ? !rotary_apart({p.dst, p.dst_rs, p.dst_hs, rows->rows, part_heads[i]},
                                   {other.src, other.src_rs, other.src_hs, rows->rows, part_heads[j]}, rows->head_dim, size)
                   : ranges_meet(p.dst, rotary_extent(rows->rows, part_heads[i], rows->head_dim, p.dst_rs, p.dst_hs, size), other.src,
                                 rotary_extent(rows->rows, part_heads[j], rows->head_dim, other.src_rs, other.src_hs, size)))
        return fail(RNSMX_EINVAL, "outputs lie over queries or keys without being them");
    }
  }
  a.steps = rotary->steps_dev;
  a.positions = positions_dev;
  a.rows = rows->rows;
  a.wide = rows->positions_dtype == RNSMX_INT64;
  a.q_heads = rows->q_heads;
  a.heads = rows->k_heads;
  a.pairs = rotary->pairs;
  a.dim = rows->head_dim;
  a.magnitude = rotary->magnitude;
  a.sign = rows->back ? -1.0f : 1.0f;
  a.turning = (a.pairs + step - 1) / step;
  a.pieces = a.turning + (copied ? (a.dim - 2 * a.pairs + 2 * step - 1) / (2 * step) : 0);

  // Inputs and outputs that the 256 MB behind the L2s would not hold go past the caches: 16384 rows
  // of 40 heads of 128 in 16 bits (336 MB) 60 us so, 65 through them, 12288 (252 MB) 46 and 43.
  // The same in float32: 6909 rows of 64 heads of 128 (453 MB) 80 us so, 87 through them.
  // But only where neighbouring threads' loads, a head's pairs or half of what is copied, take whole
  // lines of 128 bytes, or few in parts: a line taken by halves travels twice.  340 MB of 40 heads, us so
  // and through the caches: heads of 64 in 16 bits (64 bytes) 82 and 71, 64 of 128 turned 82 and 69, heads
  // of 80 and 96 130 and 72, 160 (160 bytes) 89 and 70, 192 68 and 68 (900 MB: 175 and 166), 320 (320 bytes) 68
  // and 70; in float32 heads of 64 (128 bytes) 60 and 66, 80 90 and 67, 160 65 and 68, 32 of 128 69 and
  // 67.  Heads of 128 in 16 bits that begin 16 bytes off a line 67 and 65, in float32 61 and 64.
  constexpr int64_t kRotaryStream = 256ll << 20;
  auto whole = [&](int64_t bytes) { return bytes >= 256 || (bytes % 128 == 0 && lines); };
  const bool past = rows->rows * static_cast<double>(heads) * a.dim * size * 2 >= kRotaryStream && whole(a.pairs * size) &&
                    (a.pieces == a.turning || whole(16 * (a.pieces - a.turning)));

  // A workgroup takes rows of some kRotaryPieces pieces, which share the angles' cost (16383 rows
  // of 40 heads of 128, 320 pieces each, through the caches: 66.7 us with 2 rows, 66.9 with 4, 69.2
  // with 8, 80 with 16), but no more than leave the chip kRotaryGroups workgroups; where rows are fewer than
  // that their heads are split.
  constexpr int64_t kRotaryGroups = 1024, kRotaryPieces = 640;
  const int64_t most_rows = std::min<int64_t>(kRotaryTable / a.pairs, std::max<int64_t>(1, kRotaryPieces / (static_cast<int64_t>(heads) * a.pieces)));
  a.row_tile = static_cast<int32_t>(std::max<int64_t>(1, std::min(most_rows, a.rows / kRotaryGroups)));
  const int64_t row_tiles = (a.rows + a.row_tile - 1) / a.row_tile;
  a.head_tile = heads;
  if (row_tiles < 256) {
    // down to 128 pieces
    const int64_t least = std::max<int64_t>(1, 128 / a.pieces), parts = std::max<int64_t>(1, std::min<int64_t>(512 / row_tiles, heads / least));
    a.head_tile = static_cast<int32_t>((heads + parts - 1) / parts);
  }
  a.per_row = a.head_tile * a.pieces;
  a.by_pieces = kv_div(a.pieces);
  a.by_row = kv_div(a.per_row);
  a.by_pairs = kv_div(a.pairs);
  const unsigned head_tiles = (heads + a.head_tile - 1) / a.head_tile;
  hipStream_t st = static_cast<hipStream_t>(stream);
  // a launch has fewer than 2^32 threads
  const int64_t most = (1 << 23) / head_tiles;
  auto run = [&](auto kernel) {
    for (int64_t tile = 0; tile < row_tiles; tile += most) {
      a.first = tile * a.row_tile;
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(std::min(most, row_tiles - tile)), head_tiles), dim3(256), 0, st, a);
    }
  };
  auto with = [&](auto t, auto vector, auto streams) {
    using T = decltype(t);
    constexpr bool V = decltype(vector)::value, S = decltype(streams)::value;
    if (rotary->interleaved)
      run(rotate_kernel<T, V, true, S>);
    else
      run(rotate_kernel<T, V, false, S>);
  };
  auto launch = [&](auto t) {
    if (!vec) return with(t, std::false_type{}, std::false_type{});
    if (past) return with(t, std::true_type{}, std::true_type{});
    with(t, std::true_type{}, std::false_type{});
  };
  if (rows->dtype == RNSMX_FLOAT32)
    launch(float{});
  else if (rows->dtype == RNSMX_FLOAT16)
    launch(_Float16{});
  else
    launch(uint16_t{});
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return RNSMX_OK;
  set_error("rotate: %s", hipGetErrorString(err));
  return RNSMX_ELAUNCH;
}

}  // extern "C"
