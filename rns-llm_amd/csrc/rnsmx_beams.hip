// Beam search's selection: the best continuations of each request's beams.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "rnsmx_kv_attn.hpp"

namespace rnsmx {

struct BeamArgs {
  const void *logits;
  const float *scores;
  const uint8_t *finished;
  int64_t request_stride, beam_stride;
  uint64_t *partial;   // [requests * beams][splits][k + 2]: the chunk's best, then its reference and sum
  uint32_t *tickets;   // an arrival counter a request of the launch, `apart` words from the next
  float *out_scores;
  int32_t *out_tokens, *out_parents;
  int32_t first, apart;  // first: a launch's first request
  int32_t beams, vocabulary, k, end_token;
  int32_t chunk, splits;  // values of a workgroup, and workgroups of a beam
  KvDiv by_splits, by_beams;
};

constexpr int kBeamMost = 256 * 64;  // values of a workgroup at most
constexpr int kBeamList = 512;    // of a workgroup's or request's values those that reach its bound
// Continuations up to which the maxima of 64 lanes give a chunk's bound: some 44 of its values reach
// it with 32, but 270 with 64, past which those of 256 threads do, 74 with 64 (12 x 16 beams of 128257
// in float32, k 64: 338 us with lanes, 37 with threads; k 32: 30.3 and 31.2).
constexpr int kBeamLanes = 32;
// Of a request's offers as many are put in order as they are, which takes the square of their
// number, and more get a higher bound first, 1 us (56 x 16 beams of 8328, k 16, 256 offers: 31.4 us
// without it, 17.3 with it; 14 of these requests, of whose offers few reach the first bound: 11.7 and 12.9).
constexpr int kBeamFew = 96;
constexpr int kBeamChunks = 1024; // of a request at most
constexpr int kBeamHeld = 1024;   // results of a request that shared memory holds all

// Numbers whose order as unsigned ones is that of the values; zeros are one.
__device__ __forceinline__ uint32_t beam_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float beam_logit(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
constexpr uint32_t kBeamNone = 0x007FFFFFu;  // of minus infinity, which is no candidate
__device__ __forceinline__ uint64_t beam_score_key(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);
  return u ^ (static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double beam_score(uint64_t key) {
  return __builtin_bit_cast(double, key >> 63 ? key ^ 0x8000000000000000ull : ~key);
}

// The largest of a wave's numbers, in every lane: rows of 16, then across them.
__device__ __forceinline__ uint32_t beam_wave_max(uint32_t v) {
  auto step = [&](auto ctrl, auto rows) {
    constexpr int c = ctrl, r = rows;
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), c, r, 0xF, false)));
  };
  using std::integral_constant;
  step(integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});  // row_shr:1
  step(integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
  step(integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
  step(integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
  step(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});  // row_bcast:15
  step(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});  // row_bcast:31
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}

// A number that at least k lanes' reach (0 if fewer have any), no higher than the
// k-th largest: its bits from the highest down until just k are left.
__device__ __forceinline__ uint32_t beam_bound(uint32_t v, int32_t k) {
  uint32_t bound = 0;
  for (uint32_t bit = 0x80000000u; bit != 0; bit >>= 1) {
    const int32_t n = __popcll(__ballot(v >= (bound | bit)));
    if (n >= k) bound |= bit;
    if (n == k) break;
  }
  return bound;
}

// The same of four numbers a lane.
__device__ __forceinline__ uint32_t beam_bound(const uint32_t (&v)[4], int32_t k) {
  uint32_t bound = 0;
  for (uint32_t bit = 0x80000000u; bit != 0; bit >>= 1) {
    int32_t n = 0;
    kv_for<4>([&](auto W) { n += __popcll(__ballot(v[W] >= (bound | bit))); });
    if (n >= k) bound |= bit;
    if (n == k) break;
  }
  return bound;
}

// A continuation that a request's beams offer.  key: of its score, 0: none.  tie: what
// goes first of equal ones, the beam from below, the logit's key, the token from below.
struct __attribute__((aligned(16))) BeamOffer {
  uint64_t key, tie;
};
__device__ __forceinline__ bool beam_better(const BeamOffer &p, const BeamOffer &q) {
  return p.key > q.key || (p.key == q.key && p.tie > q.tie);
}

// How many of n numbers in shared memory are larger than one, each of four neighbouring
// lanes asking a quarter of them.
__device__ __forceinline__ int32_t beam_larger(const uint64_t *of, int32_t n, uint64_t one) {
  int32_t larger = 0;
  for (int32_t j0 = threadIdx.x & 3; j0 < n; j0 += 16) {
    uint64_t v[4];
    kv_for<4>([&](auto U) { v[U] = of[min(j0 + 4 * U, n - 1)]; });
    kv_for<4>([&](auto U) { larger += j0 + 4 * U < n && v[U] > one ? 1 : 0; });
  }
  kv_for<2>([&](auto I) { larger += __shfl_xor(larger, 1 << I); });
  return larger;
}

template <typename T>
__device__ __forceinline__ float beam_float(T v) {
  if constexpr (std::is_same<T, uint16_t>::value)
    return kv_bf16(v);
  else
    return static_cast<float>(v);
}
// A value of a load's raw words.
template <typename T>
__device__ __forceinline__ float beam_value(const u32x4 &raw, int i) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(raw[i]);
  const uint32_t w = raw[i / 2];
  if constexpr (std::is_same<T, uint16_t>::value) return __uint_as_float(i % 2 ? w & 0xFFFF0000u : w << 16);
  return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(i % 2 ? w >> 16 : w)));
}

// One workgroup for a chunk of one beam's logits, which are read once, all loads in
// flight, and stay in registers as they are stored.  They give the largest, the sum of
// exponentials against it and the chunk's k best.  Exponentials are float32, up to 33 of which are
// added in float32: scores have no more bits when they come out, and what it leaves open is the
// order of different beams' continuations nearer than some 1e-5.  A bound that at least k of them
// reach: the k-th largest of 64 maxima, one for each lane over the four waves, or of the
// threads' 256; of what lies below it nothing more is asked, eight values at a time.  The few that reach it are put
// in order by counting.  Where they are many (logits that are equal, or in an order that puts
// the largest side by side) the k-th largest itself is found digit by digit, from the logits
// read again.  The workgroup that comes last of a request's joins the chunks, in the same manner.
// 4 beams of 50272 in float16: 9.6 us, a chain of loads, bound, list and ticket (6) and the
// join (4).  256 rows of 50272 in bfloat16 (26 MB): 15.1, to 10 of it without joins, some ten
// instructions a value and an exponential that takes four's time.  192 rows of 128257 in float32
// (98 MB, a fifth of them finished) with k 32: 27, memory to 19 and the last joins, 8 each of
// which 2 are trips to memory, after it.
template <typename T, int N>
__global__ __launch_bounds__(256, 4) void beam_kernel(const BeamArgs a) {
  constexpr int G = 16 / sizeof(T);  // values of a load, of which a thread has N
  extern __shared__ __attribute__((aligned(16))) uint64_t shared[];
  uint64_t *const list = shared;
  u32x4 *const load_of = reinterpret_cast<u32x4 *>(list + kBeamList);
  int32_t *const load_at = reinterpret_cast<int32_t *>(load_of + kBeamList);
  __shared__ uint32_t column[4][64];
  __shared__ double wave_sum[4], total[64], score[64];
  __shared__ bool over[64];
  __shared__ uint32_t shared_bound;
  __shared__ uint64_t result[RNSMX_BEAMS_MAX + 2];
  __shared__ int32_t count, loads, digit[4], last;
  const int32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint32_t id = blockIdx.x;
  const int32_t split = kv_rem(a.by_splits, id), beam = kv_rem(a.by_beams, id), place = id, request = a.first + place;
  const int32_t k = a.k, lists = a.beams * a.splits;
  const int64_t row = static_cast<int64_t>(request) * a.beams + beam, row0 = static_cast<int64_t>(request) * a.beams;
  uint64_t *to = a.partial + (row * a.splits + split) * (k + 2);
  if (tid == 0) count = loads = 0;

  if (!(a.finished && a.finished[row])) {
    const T *p = static_cast<const T *>(a.logits) + request * a.request_stride + beam * a.beam_stride;
    // Loads of 16 bytes from wherever the row begins: which value is whose does not depend on
    // its address, so that beams of the same logits have the same sums.
    const int64_t first = static_cast<int64_t>(split) * a.chunk;
    const int64_t end = min(first + a.chunk, static_cast<int64_t>(a.vocabulary));
    // what is past the row's end is as little a candidate as minus infinity
    constexpr uint32_t none = sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, uint16_t>::value ? 0xFF80FF80u : 0xFC00FC00u;
    u32x4 raw[N];
    const T *const base = p + first;
    const int32_t size = static_cast<int32_t>(end - first);
    kv_for<N>([&](auto J) {
      const int32_t e = (J * 256 + tid) * G;
      raw[J] = u32x4{none, none, none, none};
      if (e + G <= size) __builtin_memcpy(&raw[J], base + e, 16);
    });
    // the values after the last whole load, one a lane
    const int32_t edge_place = size / G * G + lane;
    float edge = -INFINITY;
    if (wave == 0 && edge_place < size) edge = beam_float(base[edge_place]);
    auto place_of = [&](int j, int i) { return (j * 256 + tid) * G + i; };  // in the chunk
    // f(value, place in the chunk)
    auto each = [&](auto &&f) {
      kv_for<N>([&](auto J) { kv_for<G>([&](auto I) { f(beam_value<T>(raw[J], I), place_of(J, I)); }); });
      f(edge, edge_place);
    };
    float top[N], most = -INFINITY;
    kv_for<N>([&](auto J) {
      top[J] = beam_value<T>(raw[J], 0);
      kv_for<G - 1>([&](auto I) { top[J] = fmaxf(top[J], beam_value<T>(raw[J], I + 1)); });
      most = fmaxf(most, top[J]);
    });
    most = fmaxf(most, edge);
    column[wave][lane] = beam_key(most);
    // The values stay as they are stored, and what is asked of them is asked anew each time:
    // 64 values or answers more would halve the waves that the registers hold.
    auto keep_raw = [&]() {
      kv_for<N>([&](auto J) {
        u32x4 &words = raw[J];
        asm volatile("" : "+v"(words));
      });
    };
    keep_raw();
    __syncthreads();
    const uint32_t four[4] = {column[0][lane], column[1][lane], column[2][lane], column[3][lane]};
    const uint32_t mine = max(max(four[0], four[1]), max(four[2], four[3]));
    const float largest = beam_logit(beam_wave_max(mine)), reference = largest == -INFINITY ? 0.0f : largest;
    if (wave == 0) {
      const uint32_t bound = k > kBeamLanes ? beam_bound(four, k) : beam_bound(mine, k);
      if (lane == 0) shared_bound = bound;
    }
    float part[2] = {0.0f, 0.0f};
    each([&](float x, int32_t at) { part[at & 1] += __builtin_amdgcn_exp2f((x - reference) * kKvLog2e); });
    double sum = static_cast<double>(part[0]) + part[1];
    kv_for<6>([&](auto I) { sum += __shfl_xor(sum, 1 << I); });
    if (lane == 0) wave_sum[wave] = sum;
    keep_raw();
    __syncthreads();
    auto enter = [&](float x, int32_t place) {
      const int32_t at = atomicAdd(&count, 1);
      if (at < kBeamList) list[at] = static_cast<uint64_t>(beam_key(x)) << 32 | ~static_cast<uint32_t>(first + place);
    };
    // whole loads with one that reaches the bound, then their values, one a thread
    const float least = shared_bound > kBeamNone ? beam_logit(shared_bound) : -INFINITY;
    kv_for<N>([&](auto J) {
      if (top[J] >= least && top[J] > -INFINITY) {
        const int32_t at = atomicAdd(&loads, 1);
        if (at < kBeamList) {
          load_of[at] = raw[J];
          load_at[at] = J * 256 + tid;
        }
      }
    });
    if (edge >= least && edge > -INFINITY) enter(edge, edge_place);
    __syncthreads();
    const int32_t held = loads;
    for (int32_t i = tid; i < min(held, kBeamList) * G; i += 256) {
      const float x = beam_float(reinterpret_cast<const T *>(load_of)[i]);
      if (x >= least && x > -INFINITY) enter(x, load_at[i / G] * G + i % G);
    }
    __syncthreads();
    int32_t n = count;
    if (held > kBeamList || n > kBeamList) {
      // Digit by digit the key of the k-th largest, and how many that are it belong to the k.
      auto key_at = [&](int32_t i) { return i < size ? beam_key(beam_float(base[i])) : 0u; };
      int32_t *const bins = reinterpret_cast<int32_t *>(column);
      uint32_t kth = 0;
      int32_t wanted = k;
      for (int32_t shift = 24; shift >= 0; shift -= 8) {
        bins[tid] = 0;
        __syncthreads();
        for (int32_t i = tid; i < size; i += 256) {
          const uint32_t key = key_at(i);
          if (key > kBeamNone && (shift == 24 || key >> (shift + 8) == kth >> (shift + 8))) atomicAdd(&bins[key >> shift & 255], 1);
        }
        __syncthreads();
        int32_t larger = 0;
        for (int32_t j = tid + 1; j < 256; ++j) larger += bins[j];
        if (larger < wanted && wanted <= larger + bins[tid]) {
          digit[0] = tid;
          digit[1] = wanted - larger;
        }
        __syncthreads();
        kth |= static_cast<uint32_t>(digit[0]) << shift;
        wanted = digit[1];
      }
      if (tid == 0) count = 0;
      __syncthreads();
      // the larger ones, and in the order of the tokens as many equal ones as are wanted
      int32_t before_these = 0;
      for (int32_t i0 = 0; i0 < size; i0 += 256) {
        const uint32_t key = key_at(i0 + tid);
        if (key > kth) enter(beam_logit(key), i0 + tid);
        if (before_these >= wanted) continue;
        const uint64_t equal = __ballot(key == kth);
        __syncthreads();
        if (lane == 0) digit[wave] = __popcll(equal);
        __syncthreads();
        int32_t rank = before_these + __popcll(equal & ((1ull << lane) - 1));
        for (int32_t w = 0; w < 4; ++w) {
          rank += w < wave ? digit[w] : 0;
          before_these += digit[w];
        }
        if (key == kth && rank < wanted) enter(beam_logit(key), i0 + tid);
      }
      __syncthreads();
      n = count;
    }
    for (int32_t i = tid >> 2; i < n; i += 64) {  // four lanes an item
      const uint64_t item = list[i];
      const int32_t rank = beam_larger(list, n, item);
      if (rank < k && (tid & 3) == 0) result[rank] = item;
    }
    if (tid >= n && tid < k) result[tid] = 0;
    if (tid == 0) {
      result[k] = __float_as_uint(largest);
      result[k + 1] = __builtin_bit_cast(uint64_t, wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3]);
    }
    __syncthreads();
    if (tid < k + 2) __hip_atomic_store(to + tid, result[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }

  // The last workgroup of a request (kv_rows_kernel has the protocol).
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const uint32_t old = __hip_atomic_fetch_add(a.tickets + place * a.apart, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = old == static_cast<uint32_t>(lists - 1);
    if (last) __hip_atomic_store(a.tickets + place * a.apart, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    count = 0;
  }
  __syncthreads();
  if (!last) return;
  // The chunks' results are read past this XCD's caches, each once: a fence that drops what
  // the caches hold would cost some 20 us with 64 requests joining at once.
  const uint64_t *from = a.partial + row0 * a.splits * (k + 2);
  auto get = [&](int32_t i, int32_t n) {
    return __hip_atomic_load(from + static_cast<int64_t>(i) * (k + 2) + n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  const int64_t out = static_cast<int64_t>(request) * k;
  // few results are all held in shared memory, of many each chunk's best
  const bool whole = lists * (k + 2) <= kBeamHeld;
  const int32_t each_held = whole ? k + 2 : 1;
  BeamOffer *const offers = reinterpret_cast<BeamOffer *>(shared);
  uint64_t *const held = reinterpret_cast<uint64_t *>(offers + kBeamList);
  double *const sums = reinterpret_cast<double *>(held + lists * each_held);
  float *const tops = reinterpret_cast<float *>(sums + lists);
  int32_t *const chosen = reinterpret_cast<int32_t *>(tops + lists);
  if (whole) {
    for (int32_t i = tid; i < lists * (k + 2); i += 256)
      held[i] = __hip_atomic_load(from + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
  }
  auto item_at = [&](int32_t i, int32_t n) { return whole ? held[i * (k + 2) + n] : n == 0 ? held[i] : get(i, n); };
  for (int32_t i = tid; i < lists; i += 256) {
    uint32_t b = i;
    const int32_t s = kv_rem(a.by_splits, b);
    if (a.finished && a.finished[row0 + b]) {  // one candidate, the beam itself
      held[i * each_held] = s == 0 ? ~static_cast<uint32_t>(a.end_token) : 0;
    } else {
      const uint64_t m = whole ? held[i * (k + 2) + k] : get(i, k), v = whole ? held[i * (k + 2) + k + 1] : get(i, k + 1);
      if (!whole) held[i] = get(i, 0);
      tops[i] = __uint_as_float(static_cast<uint32_t>(m));
      sums[i] = __builtin_bit_cast(double, v);
    }
  }
  __syncthreads();

  // each beam's logarithm of its exponentials' sum, by sixteen lanes
  for (int32_t b0 = 0; b0 < a.beams; b0 += 16) {
    const int32_t b = b0 + (tid >> 4), in_group = tid & 15;
    const bool ended = b < a.beams && a.finished && a.finished[row0 + b];
    const int32_t first = b * a.splits, chunks = b < a.beams && !ended ? a.splits : 0;
    float largest = -INFINITY;
    for (int32_t s = in_group; s < chunks; s += 16) largest = fmaxf(largest, tops[first + s]);
    kv_for<4>([&](auto I) { largest = fmaxf(largest, __shfl_xor(largest, 1 << I)); });
    double sum = 0.0;
    for (int32_t s = in_group; s < chunks; s += 16) {
      const float m = tops[first + s];
      // a chunk without anything above minus infinity has a sum of 0, or not-a-numbers
      sum += m == -INFINITY ? sums[first + s] : sums[first + s] * exp(static_cast<double>(m) - static_cast<double>(largest));
    }
    kv_for<4>([&](auto I) { sum += __shfl_xor(sum, 1 << I); });
    if (in_group == 0 && b < a.beams) {
      total[b] = static_cast<double>(largest) + log(sum);
      score[b] = a.scores[row0 + b];
      over[b] = ended;
    }
  }
  __syncthreads();

  auto offer = [&](int32_t i, uint64_t item) {  // an item of chunk i
    const int32_t b = static_cast<int32_t>(kv_quot(a.by_splits, i));
    if (item == 0) return BeamOffer{0, 0};
    const double v = over[b] ? score[b] : score[b] + (static_cast<double>(beam_logit(static_cast<uint32_t>(item >> 32))) - total[b]);
    // a token has 24 bits (kBeamChunks of kBeamMost)
    return BeamOffer{fabs(v) < INFINITY ? beam_score_key(v) : 0,
                     static_cast<uint64_t>(RNSMX_BEAMS_MAX - 1 - b) << 56 | item >> 32 << 24 | (item & 0xFFFFFFu)};
  };
  auto write = [&](int32_t j, const BeamOffer &o) {
    a.out_scores[out + j] = static_cast<float>(beam_score(o.key));
    a.out_tokens[out + j] = static_cast<int32_t>(~o.tie & 0xFFFFFFu);
    a.out_parents[out + j] = static_cast<int32_t>(row0) + RNSMX_BEAMS_MAX - 1 - static_cast<int32_t>(o.tie >> 56);
  };

  // A bound from the largest that each thread has, or each lane over the four waves, which
  // is lower but found sooner.
  auto settle = [&](uint32_t most, auto lanes) {
    __syncthreads();
    column[wave][lane] = most;
    __syncthreads();
    const uint32_t all[4] = {column[0][lane], column[1][lane], column[2][lane], column[3][lane]};
    if constexpr (decltype(lanes)::value) return max(beam_bound(max(max(all[0], all[1]), max(all[2], all[3])), k), 1u);
    return max(beam_bound(all, k), 1u);
  };
  auto best_of = [&](int32_t i) { return static_cast<uint32_t>(offer(i, held[i * each_held]).key >> 32); };
  uint32_t most_here = 0;
  for (int32_t i = tid; i < lists; i += 256) most_here = max(most_here, best_of(i));
  if (tid == 0) loads = 0;
  uint32_t least = settle(most_here, std::true_type{});
  for (int32_t i = tid; i < lists; i += 256)
    if (best_of(i) >= least) chosen[atomicAdd(&loads, 1)] = i;
  __syncthreads();
  // Only chunks whose best reaches the bound are looked at further, by eight lanes each and
  // eight results at a time: they are in order, so the rest of a chunk whose eighth does not
  // reach it need not be read.  Where there are many, the first that are read
  // give a higher bound (33 to 54 chunks with k 32: 32 to 41 results left of 46 to 1027, 27.2 us;
  // 30.2 with all of the chunks' results read and put in order).
  const int32_t chunks = loads, in_eight = tid & 7;
  bool measure = false, again = false;
  for (;;) {
    for (int32_t c0 = 0; c0 < chunks; c0 += 128) {
      bool more[4] = {true, true, true, true};
      for (int32_t n0 = 0; n0 < k; n0 += 8) {
        const int32_t n = n0 + in_eight;
        uint64_t item[4];
        int32_t chunk[4];
        kv_for<4>([&](auto U) {
          item[U] = chunk[U] = 0;
          if (c0 + 32 * U < chunks) {
            chunk[U] = chosen[min(c0 + 32 * U + (tid >> 3), chunks - 1)];
            item[U] = item_at(chunk[U], min(n, k - 1));
          }
        });
        BeamOffer o[4];
        kv_for<4>([&](auto U) {
          o[U] = BeamOffer{0, 0};
          if (c0 + 32 * U < chunks) {
            const bool there = more[U] && c0 + 32 * U + (tid >> 3) < chunks && n < k &&
                               (n == 0 || !over[kv_quot(a.by_splits, chunk[U])]);
            o[U] = offer(chunk[U], there ? item[U] : 0);
          }
        });
        if (c0 + n0 == 0 || measure) {
          uint32_t most = 0;
          kv_for<4>([&](auto U) { most = max(most, static_cast<uint32_t>(o[U].key >> 32)); });
          most_here = c0 + n0 == 0 ? most : max(most_here, most);
        }
        if (!measure) {
          if (c0 + n0 == 0 && chunks * min(k, 8) > kBeamFew) least = max(least, settle(most_here, std::false_type{}));
          kv_for<4>([&](auto U) {
            if (static_cast<uint32_t>(o[U].key >> 32) >= least) {
              const int32_t at = atomicAdd(&count, 1);
              if (at < kBeamList) offers[at] = o[U];
            }
          });
        }
        bool any = false;
        kv_for<4>([&](auto U) {
          more[U] = __shfl(static_cast<int>(static_cast<uint32_t>(o[U].key >> 32) >= least), lane | 7) != 0;
          any = any || more[U];
        });
        if (!__any(any)) break;
      }
    }
    if (measure) {
      measure = false;
      least = max(least, settle(most_here, std::false_type{}));
      if (tid == 0) count = 0;
      __syncthreads();
      continue;
    }
    __syncthreads();
    const int32_t n = count;
    if (n > kBeamList && !again) {  // all that reach it give a higher one
      measure = again = true;
      continue;
    }
    if (n > kBeamFew && n <= kBeamList) {  // so do those in the list
      BeamOffer o[2];
      kv_for<2>([&](auto U) { o[U] = tid + 256 * U < n ? offers[tid + 256 * U] : BeamOffer{0, 0}; });
      least = max(least, settle(static_cast<uint32_t>(max(o[0].key, o[1].key) >> 32), std::false_type{}));
      if (tid == 0) count = 0;
      __syncthreads();
      kv_for<2>([&](auto U) {
        if (static_cast<uint32_t>(o[U].key >> 32) >= least) offers[atomicAdd(&count, 1)] = o[U];
      });
      __syncthreads();
    }
    break;
  }
  const int32_t n = count;
  if (n <= kBeamList) {
    for (int32_t i = tid >> 2; i < n; i += 64) {  // four lanes an offer
      const BeamOffer o = offers[i];
      int32_t rank = 0;
      for (int32_t j0 = tid & 3; j0 < n; j0 += 16) {
        BeamOffer other[4];
        kv_for<4>([&](auto U) { other[U] = offers[min(j0 + 4 * U, n - 1)]; });
        kv_for<4>([&](auto U) { rank += j0 + 4 * U < n && beam_better(other[U], o) ? 1 : 0; });
      }
      kv_for<2>([&](auto I) { rank += __shfl_xor(rank, 1 << I); });
      if (rank < k && (tid & 3) == 0) write(rank, o);
    }
    for (int32_t j = n + tid; j < k; j += 256) {
      a.out_scores[out + j] = -INFINITY;
      a.out_tokens[out + j] = max(a.end_token, 0);
      a.out_parents[out + j] = static_cast<int32_t>(row0) + j % a.beams;
    }
    return;
  }
  // Too many that are equal, and more than are wanted: k rounds, in which each thread
  // offers the best of its chunks' next ones.
  int32_t *const taken = chosen;
  __syncthreads();
  for (int32_t i = tid; i < lists; i += 256) taken[i] = 0;
  __syncthreads();
  auto next = [&](int32_t &from_chunk) {
    BeamOffer most{0, 0};
    for (int32_t i = tid; i < lists; i += 256)
      if (taken[i] < (over[kv_quot(a.by_splits, i)] ? 1 : k)) {
        const BeamOffer o = offer(i, item_at(i, taken[i]));
        if (o.key != 0 && beam_better(o, most)) {
          most = o;
          from_chunk = i;
        }
      }
    return most;
  };
  int32_t from_chunk = 0;
  BeamOffer mine = next(from_chunk);
  __shared__ BeamOffer wave_best[4];
  for (int32_t j = 0; j < k; ++j) {
    BeamOffer most = mine;
    kv_for<6>([&](auto I) {
      auto other = [&](uint64_t v) { return static_cast<uint64_t>(__shfl_xor(static_cast<long long>(v), 1 << I)); };
      const BeamOffer o{other(most.key), other(most.tie)};
      if (beam_better(o, most)) most = o;
    });
    if (lane == 0) wave_best[wave] = most;
    __syncthreads();
    kv_for<4>([&](auto W) {
      if (beam_better(wave_best[W], most)) most = wave_best[W];
    });
    if (tid == 0) write(j, most);
    if (mine.key != 0 && most.key == mine.key && most.tie == mine.tie) {
      ++taken[from_chunk];
      mine = next(from_chunk);
    }
    __syncthreads();
  }
}

// Bytes of a workgroup's shared memory: what its own values need, or the join of `lists` chunks.
static size_t beam_shared(int64_t lists, int32_t k) {
  const int64_t held = lists * (k + 2) <= kBeamHeld ? lists * (k + 2) : lists;
  return std::max<size_t>(kBeamList * (8 + 16 + 4), kBeamList * 16 + held * 8 + lists * (8 + 4 + 4));
}

// Chunks of a beam: as many as give the chip kBeamGroups workgroups, but no smaller than
// kBeamLeast values and no larger than the registers hold.
constexpr int64_t kBeamGroups = 1024, kBeamLeast = 4096;
static void beam_chunks(const rnsmx_beams_t &b, int32_t &chunk, int32_t &splits) {
  const int64_t per = b.dtype == RNSMX_FLOAT32 ? 4 : 8, values = b.vocabulary;
  const int64_t rows = std::max<int64_t>(static_cast<int64_t>(b.requests) * b.beams, 1);
  const int64_t least = (values + kBeamMost - 1) / kBeamMost, most = (values + kBeamLeast - 1) / kBeamLeast;
  const int64_t n = std::max(least, std::min({most, kBeamGroups / rows, kBeamChunks / static_cast<int64_t>(b.beams)}));
  chunk = static_cast<int32_t>(round_up((values + n - 1) / n, per));
  splits = static_cast<int32_t>((values + chunk - 1) / chunk);
}

// The kernel of the fewest loads a thread that take a chunk, by eighths of the most.
template <typename T, int N = kBeamMost / 256 * static_cast<int>(sizeof(T)) / 16>
static void launch_beams(const BeamArgs &a, dim3 grid, size_t shared, hipStream_t st) {
  constexpr int step = sizeof(T) == 4 ? 2 : 1, values = 256 * 16 / static_cast<int>(sizeof(T));
  if constexpr (N > step) {
    if (a.chunk <= (N - step) * values) return launch_beams<T, N - step>(a, grid, shared, st);
  }
  hipLaunchKernelGGL((beam_kernel<T, N>), grid, dim3(256), shared, st, a);
}

static int32_t beam_check(const rnsmx_beams_t *b) {
  if (!b) return fail(RNSMX_EINVAL, "null beams");
  if (b->dtype != RNSMX_FLOAT32 && b->dtype != RNSMX_FLOAT16 && b->dtype != RNSMX_BFLOAT16)
    return fail(RNSMX_EINVAL, "logits are float32, float16 or bfloat16");
  if (b->requests < 0 || b->beams < 1 || b->beams > RNSMX_BEAMS_MAX || b->vocabulary < 1 || b->k < 1 || b->k > RNSMX_BEAMS_MAX)
    return fail(RNSMX_EINVAL, "1 to 64 beams, 1 to 64 continuations, at least one token");
  if (b->request_stride < 0 || b->beam_stride < 0) return fail(RNSMX_EINVAL, "negative strides");
  int32_t chunk, splits;
  beam_chunks(*b, chunk, splits);
  if (static_cast<int64_t>(b->beams) * splits > kBeamChunks) return fail(RNSMX_EINVAL, "too many tokens and beams");
  if (static_cast<int64_t>(b->requests) * b->beams > 0x7FFFFFFFLL) return fail(RNSMX_EINVAL, "too many requests and beams");
  return RNSMX_OK;
}

}  // namespace rnsmx

using namespace rnsmx;

extern "C" {

int64_t rnsmx_beam_workspace_bytes(const rnsmx_beams_t *beams) {
  clear_error();
  if (beam_check(beams)) return -1;
  int32_t chunk, splits;
  beam_chunks(*beams, chunk, splits);
  return RNSMX_KV_TICKETS * 4 + static_cast<int64_t>(beams->requests) * beams->beams * splits * (beams->k + 2) * 8;
}

int32_t rnsmx_beam_select(const rnsmx_beams_t *beams, const void *logits_dev, const float *scores_dev, const uint8_t *finished_dev,
                          void *workspace_dev, int64_t workspace_bytes, float *out_scores_dev, int32_t *out_tokens_dev,
                          int32_t *out_parents_dev, void *stream) {
  clear_error();
  if (int32_t rc = beam_check(beams)) return rc;
  if (beams->requests == 0) return RNSMX_OK;
  const int64_t size = beams->dtype == RNSMX_FLOAT32 ? 4 : 2;
  auto on = [](const void *p, int64_t n) { return p && reinterpret_cast<uintptr_t>(p) % n == 0; };
  if (!on(logits_dev, size) || !on(scores_dev, 4)) return fail(RNSMX_EINVAL, "logits or scores null or not aligned to their type");
  if (finished_dev && (beams->end_token < 0 || beams->end_token >= beams->vocabulary))
    return fail(RNSMX_EINVAL, "finished beams need an end token of the vocabulary");
  if (!on(out_scores_dev, 4) || !on(out_tokens_dev, 4) || !on(out_parents_dev, 4))
    return fail(RNSMX_EINVAL, "an output is null or not on a 4-byte boundary");
  if (!on(workspace_dev, 16)) return fail(RNSMX_EINVAL, "workspace null or not on a 16-byte boundary");
  if (workspace_bytes < rnsmx_beam_workspace_bytes(beams)) return fail(RNSMX_ESPACE, "workspace too small");
  BeamArgs a{};
  a.logits = logits_dev;
  a.scores = scores_dev;
  a.finished = finished_dev;
  a.request_stride = beams->request_stride;
  a.beam_stride = beams->beam_stride;
  a.tickets = static_cast<uint32_t *>(workspace_dev);
  a.partial = reinterpret_cast<uint64_t *>(static_cast<uint8_t *>(workspace_dev) + RNSMX_KV_TICKETS * 4);
  a.out_scores = out_scores_dev;
  a.out_tokens = out_tokens_dev;
  a.out_parents = out_parents_dev;
  a.beams = beams->beams;
  a.vocabulary = beams->vocabulary;
  a.k = beams->k;
  beam_chunks(*beams, a.chunk, a.splits);
  a.end_token = beams->end_token;
  a.by_splits = kv_div(a.splits);
  a.by_beams = kv_div(a.beams);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t lists = static_cast<int64_t>(a.beams) * a.splits;
  // a ticket a request, and fewer than 2^32 threads
  const int64_t most = std::min<int64_t>(RNSMX_KV_TICKETS, std::max<int64_t>(1, (1 << 23) / lists));
  // Counters a line of 128 bytes apart, as far as there are so many: on one line they wait for each
  // other (1024 workgroups of 64 requests 2.8 us, 1536 of 12 some 6).
  a.apart = 32;
  while (a.apart > 1 && std::min<int64_t>(most, beams->requests) * a.apart > RNSMX_KV_TICKETS) a.apart /= 2;
  for (int64_t first = 0; first < beams->requests; first += most) {
    a.first = static_cast<int32_t>(first);
    const dim3 grid(static_cast<unsigned>(std::min(most, beams->requests - first) * lists));
    const size_t shared = beam_shared(lists, a.k);
    if (beams->dtype == RNSMX_FLOAT32)
      launch_beams<float>(a, grid, shared, st);
    else if (beams->dtype == RNSMX_FLOAT16)
      launch_beams<_Float16>(a, grid, shared, st);
    else
      launch_beams<uint16_t>(a, grid, shared, st);
  }
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return RNSMX_OK;
  set_error("beam_select: %s", hipGetErrorString(err));
  return RNSMX_ELAUNCH;
}

}  // extern "C"
