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
  uint64_t *partial;   // [requests * beams][splits][k + 2]
  uint32_t *tickets;   // an arrival counter a request of the launch
  float *out_scores;
  int32_t *out_tokens, *out_parents;
  int32_t first;       // a launch's first request
  int32_t beams, vocabulary, k, splits, end_token;
  KvDiv by_splits, by_beams;
};

constexpr int kBeamValues = 16;                    // of a thread
constexpr int kBeamChunk = 256 * kBeamValues;      // of a workgroup
constexpr int kBeamLists = 16384;                  // chunks of a request
// Entries of a workgroup's list: no more than kBeamValues of each of k lanes of its four
// waves lie above their common bound, and k at it.
constexpr int beam_list(int k) { return (4 * kBeamValues + 1) * k; }

// Numbers whose order as unsigned ones is that of the values; zeros are one.
__device__ __forceinline__ uint32_t beam_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float beam_logit(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ uint64_t beam_score_key(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);
  return u ^ (static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | 0x8000000000000000ull);
}

__device__ __forceinline__ uint64_t beam_shuffle(uint64_t v, int lanes) {
  return static_cast<uint64_t>(__shfl_xor(static_cast<long long>(v), lanes));
}

// One workgroup for a chunk of one beam's logits: read once into registers, they give
// the largest, the sum of exponentials against it and the chunk's k best.  A bound that
// at least k of them reach is the k-th largest of a wave's 64 lane maxima, the highest of
// the four waves'; the few that reach it are put in order by counting.  The workgroup that
// comes last of a request's joins the chunks.
template <typename T>
__global__ __launch_bounds__(256) void beam_kernel(const BeamArgs a) {
  constexpr int G = 16 / sizeof(T), N = kBeamValues / G;  // values of a load, loads of a thread
  extern __shared__ uint64_t list[];  // and, once it is written out, how many of each chunk's are taken
  uint8_t *const taken = reinterpret_cast<uint8_t *>(list);
  __shared__ uint32_t wave_key[4], wave_bound[4];
  __shared__ double wave_sum[4], total[64];
  __shared__ int32_t count, last;
  const int32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint32_t id = blockIdx.x;
  const int32_t split = kv_rem(a.by_splits, id), beam = kv_rem(a.by_beams, id), place = id, request = a.first + place;
  const int32_t k = a.k, lists = a.beams * a.splits;
  const int64_t row = static_cast<int64_t>(request) * a.beams + beam;
  uint64_t *to = a.partial + (row * a.splits + split) * (k + 2);
  auto put = [&](int32_t i, uint64_t v) { __hip_atomic_store(to + i, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };

  if (!(a.finished && a.finished[row])) {
    const T *p = static_cast<const T *>(a.logits) + request * a.request_stride + beam * a.beam_stride;
    const int32_t before = static_cast<int32_t>(reinterpret_cast<uintptr_t>(p) / sizeof(T) % G);  // to the load's boundary
    const int64_t first = static_cast<int64_t>(split) * kBeamChunk - before;
    float x[kBeamValues];
    uint32_t there = 0;  // a bit a value
    kv_for<N>([&](auto J) {
      constexpr int j = J;
      const int64_t e = first + (j * 256 + tid) * G;
      T v[G];
      if (e >= 0 && e + G <= a.vocabulary) {
        *reinterpret_cast<u32x4 *>(v) = *reinterpret_cast<const u32x4 *>(p + e);
        there |= ((1u << G) - 1u) << (j * G);
      } else {
        kv_for<G>([&](auto I) {
          const bool in = e + I >= 0 && e + I < a.vocabulary;
          v[I] = in ? p[e + I] : T(0);
          there |= in ? 1u << (j * G + I) : 0u;
        });
      }
      kv_for<G>([&](auto I) {
        if constexpr (std::is_same<T, uint16_t>::value)
          x[j * G + I] = kv_bf16(v[I]);
        else
          x[j * G + I] = static_cast<float>(v[I]);
      });
    });
    uint32_t top = 0;
    kv_for<kBeamValues>([&](auto I) { top = max(top, there >> I & 1u ? beam_key(x[I]) : 0u); });
    uint32_t most = top;
    kv_for<6>([&](auto I) { most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 1 << I))); });
    // the k-th largest lane maximum, from its highest bit down
    uint32_t bound = 0;
    for (uint32_t bit = 0x80000000u; bit != 0; bit >>= 1) {
      const int32_t n = __popcll(__ballot(top >= (bound | bit)));
      if (n >= k) bound |= bit;
      if (n == k) break;
    }
    if (lane == 0) {
      wave_key[wave] = most;
      wave_bound[wave] = bound;
    }
    if (tid == 0) count = 0;
    __syncthreads();
    most = max(max(wave_key[0], wave_key[1]), max(wave_key[2], wave_key[3]));
    bound = max(max(wave_bound[0], wave_bound[1]), max(wave_bound[2], wave_bound[3]));
    const float largest = most == 0 ? -INFINITY : beam_logit(most), reference = largest == -INFINITY ? 0.0f : largest;
    float part = 0.0f;
    kv_for<kBeamValues>([&](auto I) {
      part += there >> I & 1u ? __builtin_amdgcn_exp2f((x[I] - reference) * kKvLog2e) : 0.0f;
    });
    double sum = part;
    kv_for<6>([&](auto I) { sum += __shfl_xor(sum, 1 << I); });
    if (lane == 0) wave_sum[wave] = sum;
    // those above the bound, and, where they are few, those at it
    uint32_t above = 0, equal = 0;
    kv_for<kBeamValues>([&](auto I) {
      const uint32_t key = beam_key(x[I]);
      above |= (there >> I & 1u) && key > bound ? 1u << I : 0u;
      equal |= (there >> I & 1u) && key == bound ? 1u << I : 0u;
    });
    auto token = [&](int32_t i) { return static_cast<uint32_t>(first + ((i / G) * 256 + tid) * G + i % G); };
    auto enter = [&](uint32_t which) {
      if (which != 0) {
        int32_t at = atomicAdd(&count, __popc(which));
        kv_for<kBeamValues>([&](auto I) {
          if (which >> I & 1u) list[at++] = static_cast<uint64_t>(beam_key(x[I])) << 32 | ~token(I);
        });
      }
    };
    enter(above);
    __syncthreads();
    const int32_t larger = count;
    const double chunk_sum = wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3];
    __syncthreads();
    // equal ones: as many as there are, counted together with the larger
    if (larger < k) {
      if (equal != 0) atomicAdd(&count, __popc(equal));
      __syncthreads();
      const int32_t all = count;
      __syncthreads();
      if (tid == 0) count = larger;
      __syncthreads();
      if (all > beam_list(k)) {
        // too many: the k lowest tokens of them, by halving
        int32_t low = -1, high = kBeamChunk - 1;  // in the chunk; k of them lie up to `high`
        while (high - low > 1) {
          const int32_t mid = (low + high) >> 1;
          int32_t n = 0;
          kv_for<kBeamValues>([&](auto I) {
            constexpr int i = I;
            n += (equal >> i & 1u) && ((i / G) * 256 + tid) * G + i % G <= mid ? 1 : 0;
          });
          if (tid == 0) last = 0;
          __syncthreads();
          if (n != 0) atomicAdd(&last, n);
          __syncthreads();
          if (last >= k)
            high = mid;
          else
            low = mid;
          __syncthreads();
        }
        kv_for<kBeamValues>([&](auto I) {
          constexpr int i = I;
          if (((i / G) * 256 + tid) * G + i % G > high) equal &= ~(1u << i);
        });
      }
      enter(equal);
      __syncthreads();
    }
    const int32_t n = count;
    for (int32_t i = tid; i < n; i += 256) {
      const uint64_t mine = list[i];
      int32_t rank = 0;
      for (int32_t j = 0; j < n; ++j) rank += list[j] > mine ? 1 : 0;
      if (rank < k) put(rank, mine);
    }
    for (int32_t i = n + tid; i < k; i += 256) put(i, 0);
    if (tid == 0) {
      put(k, __float_as_uint(largest));
      put(k + 1, __builtin_bit_cast(uint64_t, chunk_sum));
    }
  }

  // The last workgroup of a request (kv_rows_kernel has the protocol).
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const uint32_t old = __hip_atomic_fetch_add(a.tickets + place, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = old == static_cast<uint32_t>(lists - 1);
    if (last) __hip_atomic_store(a.tickets + place, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  const int64_t row0 = static_cast<int64_t>(request) * a.beams;
  const uint64_t *from = a.partial + row0 * a.splits * (k + 2);

  // each beam's logarithm of its exponentials' sum; not a number: no candidates
  for (int32_t b = wave; b < a.beams; b += 4) {
    if (a.finished && a.finished[row0 + b]) continue;
    float largest = -INFINITY;
    bool bad = false;
    for (int32_t s = lane; s < a.splits; s += 64) {
      const float m = __uint_as_float(static_cast<uint32_t>(from[(b * a.splits + s) * static_cast<int64_t>(k + 2) + k]));
      bad = bad || m != m;
      largest = fmaxf(largest, m);
    }
    kv_for<6>([&](auto I) { largest = fmaxf(largest, __shfl_xor(largest, 1 << I)); });
    double sum = 0.0;
    for (int32_t s = lane; s < a.splits; s += 64) {
      const uint64_t *e = from + (b * a.splits + s) * static_cast<int64_t>(k + 2) + k;
      const float m = __uint_as_float(static_cast<uint32_t>(e[0]));
      const double v = __builtin_bit_cast(double, e[1]);
      sum += m == -INFINITY ? v : v * exp(static_cast<double>(m) - static_cast<double>(largest));
    }
    kv_for<6>([&](auto I) { sum += __shfl_xor(sum, 1 << I); });
    const bool dead = __any(bad) || !(fabsf(largest) < INFINITY);
    if (lane == 0) total[b] = dead ? __builtin_nan("") : static_cast<double>(largest) + log(sum);
  }
  for (int32_t i = tid; i < lists; i += 256) taken[i] = 0;
  __syncthreads();

  // k rounds: each thread offers the best of its chunks' next ones
  struct Offer {
    uint64_t key;   // of the score, 0: none
    uint64_t item;  // key of the logit and the token, as the lists have them
    int32_t beam, list;
  };
  auto better = [](const Offer &p, const Offer &q) {
    if (p.key != q.key) return p.key > q.key;
    if (p.beam != q.beam) return p.beam < q.beam;
    return p.item > q.item;
  };
  auto offer = [&]() {
    Offer best{0, 0, INT_MAX, 0};
    for (int32_t i = tid; i < lists; i += 256) {
      const int32_t b = i / a.splits, s = i - b * a.splits, n = taken[i];
      const double score = a.scores[row0 + b];
      Offer o{0, 0, b, i};
      if (a.finished && a.finished[row0 + b]) {
        if (s != 0 || n != 0) continue;
        o.item = ~static_cast<uint32_t>(a.end_token);
        o.key = fabs(score) < INFINITY ? beam_score_key(score) : 0;
      } else {
        if (n >= k) continue;
        o.item = from[i * static_cast<int64_t>(k + 2) + n];
        const double v = score + (static_cast<double>(beam_logit(static_cast<uint32_t>(o.item >> 32))) - total[b]);
        o.key = o.item != 0 && fabs(v) < INFINITY ? beam_score_key(v) : 0;
      }
      if (o.key != 0 && better(o, best)) best = o;
    }
    return best;
  };
  Offer mine = offer();
  __shared__ Offer wave_best[4];
  for (int32_t j = 0; j < k; ++j) {
    Offer best = mine;
    kv_for<6>([&](auto I) {
      Offer o{beam_shuffle(best.key, 1 << I), beam_shuffle(best.item, 1 << I), __shfl_xor(best.beam, 1 << I), __shfl_xor(best.list, 1 << I)};
      if (better(o, best)) best = o;
    });
    if (lane == 0) wave_best[wave] = best;
    __syncthreads();
    kv_for<4>([&](auto W) {
      if (better(wave_best[W], best)) best = wave_best[W];
    });
    const int64_t at = static_cast<int64_t>(request) * k + j;
    if (best.key == 0) {  // nothing left: this place and those after it have none
      if (tid < k - j) {
        a.out_scores[at + tid] = -INFINITY;
        a.out_tokens[at + tid] = max(a.end_token, 0);
        a.out_parents[at + tid] = static_cast<int32_t>(row0) + (j + tid) % a.beams;
      }
      break;
    }
    if (tid == 0) {
      const uint64_t u = best.key;
      a.out_scores[at] = static_cast<float>(__builtin_bit_cast(double, u >> 63 ? u ^ 0x8000000000000000ull : ~u));
      a.out_tokens[at] = static_cast<int32_t>(~static_cast<uint32_t>(best.item));
      a.out_parents[at] = static_cast<int32_t>(row0) + best.beam;
    }
    if (best.list == mine.list && mine.key != 0) {
      ++taken[mine.list];
      mine = offer();
    }
    __syncthreads();
  }
}

static int32_t beam_splits(int32_t vocabulary) {
  // a row starts up to seven values into its first load
  return static_cast<int32_t>((static_cast<int64_t>(vocabulary) + 7 + kBeamChunk - 1) / kBeamChunk);
}

static int32_t beam_check(const rnsmx_beams_t *b) {
  if (!b) return fail(RNSMX_EINVAL, "null beams");
  if (b->dtype != RNSMX_FLOAT32 && b->dtype != RNSMX_FLOAT16 && b->dtype != RNSMX_BFLOAT16)
    return fail(RNSMX_EINVAL, "logits are float32, float16 or bfloat16");
  if (b->requests < 0 || b->beams < 1 || b->beams > RNSMX_BEAMS_MAX || b->vocabulary < 1 || b->k < 1 || b->k > RNSMX_BEAMS_MAX)
    return fail(RNSMX_EINVAL, "1 to 64 beams, 1 to 64 continuations, at least one token");
  if (b->request_stride < 0 || b->beam_stride < 0) return fail(RNSMX_EINVAL, "negative strides");
  if (static_cast<int64_t>(b->beams) * beam_splits(b->vocabulary) > kBeamLists) return fail(RNSMX_EINVAL, "too many tokens and beams");
  if (static_cast<int64_t>(b->requests) * b->beams > 0x7FFFFFFFLL) return fail(RNSMX_EINVAL, "too many requests and beams");
  return RNSMX_OK;
}

}  // namespace rnsmx

using namespace rnsmx;

extern "C" {

int64_t rnsmx_beam_workspace_bytes(const rnsmx_beams_t *beams) {
  clear_error();
  if (beam_check(beams)) return -1;
  return RNSMX_KV_TICKETS * 4 +
         static_cast<int64_t>(beams->requests) * beams->beams * beam_splits(beams->vocabulary) * (beams->k + 2) * 8;
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
  a.splits = beam_splits(beams->vocabulary);
  a.end_token = beams->end_token;
  a.by_splits = kv_div(a.splits);
  a.by_beams = kv_div(a.beams);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t lists = static_cast<int64_t>(a.beams) * a.splits;
  // a ticket a request, and fewer than 2^32 threads
  const int64_t most = std::min<int64_t>(RNSMX_KV_TICKETS, std::max<int64_t>(1, (1 << 23) / lists));
  for (int64_t first = 0; first < beams->requests; first += most) {
    a.first = static_cast<int32_t>(first);
    const dim3 grid(static_cast<unsigned>(std::min(most, beams->requests - first) * lists));
    const size_t shared = std::max<size_t>(static_cast<size_t>(beam_list(a.k)) * 8, lists);
    if (beams->dtype == RNSMX_FLOAT32)
      hipLaunchKernelGGL(beam_kernel<float>, grid, dim3(256), shared, st, a);
    else if (beams->dtype == RNSMX_FLOAT16)
      hipLaunchKernelGGL(beam_kernel<_Float16>, grid, dim3(256), shared, st, a);
    else
      hipLaunchKernelGGL(beam_kernel<uint16_t>, grid, dim3(256), shared, st, a);
  }
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return RNSMX_OK;
  set_error("beam_select: %s", hipGetErrorString(err));
  return RNSMX_ELAUNCH;
}

}  // extern "C"
