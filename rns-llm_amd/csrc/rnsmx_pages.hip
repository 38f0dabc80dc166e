// Pages handed out on the device: block tables, reference counts and slot maps
// of sequences that grow, shrink and share, and copies of shared pages.
#include <algorithm>
#include <climits>

#include "rnsmx_kv.hpp"

namespace rnsmx {

struct PoolArgs {
  int32_t *table, *lengths, *refs;
  uint8_t *free;                   // 1 where nobody holds a page, by sixteens (0 past the last)
  int32_t *going, *first;          // scratch, [blocks] each: zeros and INT32_MAX between calls
  int32_t *before;                 // scratch, [blocks]: free pages before each word of them
  int32_t *spare, *spare_lengths;  // scratch of kv_reorder: a table and lengths
  int32_t blocks, words, log_page, seqs, width;  // words: sixteens of pages
};

struct AssignArgs {
  PoolArgs p;
  const int32_t *asked;  // new tokens of each sequence; null: one each
  int32_t *seen, *starts, *copies, *missing;
  int32_t rows, max_rows, max_length;
};

__device__ __forceinline__ int32_t pool_pages(const PoolArgs &p, int32_t n) {  // that n tokens lie in
  return static_cast<int32_t>((static_cast<uint32_t>(n) + (1u << p.log_page) - 1u) >> p.log_page);
}
__device__ __forceinline__ bool pool_has(const PoolArgs &p, int32_t page) {
  return static_cast<uint32_t>(page) < static_cast<uint32_t>(p.blocks);
}
// A holder less; a page without one is free.  A byte a page: bits would be set by
// atomics, some 30 to a word where pages lie side by side, as those of prompts do (515
// sequences with 18800 pages cut to nothing: 11.8 us).
__device__ __forceinline__ void pool_drop(const PoolArgs &p, int32_t page) {
  if (!pool_has(p, page)) return;
  if (__hip_atomic_fetch_add(p.refs + page, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 1)
    p.free[page] = 1;
}

// The sum of a value over the lanes up to each: within rows of 16, then across them.
__device__ __forceinline__ int64_t pool_lanes(int64_t v) {
  auto step = [&](auto ctrl, auto rows) {
    constexpr int c = ctrl, r = rows;
    const uint32_t low = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), c, r, 0xF, false);
    const uint32_t high = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), c, r, 0xF, false);
    v += static_cast<int64_t>(static_cast<uint64_t>(high) << 32 | low);
  };
  using std::integral_constant;
  step(integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});  // row_shr:1
  step(integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
  step(integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
  step(integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
  step(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});  // row_bcast:15
  step(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});  // row_bcast:31
  return v;
}
__device__ __forceinline__ int64_t pool_lane(int64_t v, int32_t lane) {
  const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(v), lane);
  const uint32_t high = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
  return static_cast<int64_t>(static_cast<uint64_t>(high) << 32 | low);
}

// Sums of N values a thread over the threads before it, and over all.  The waves' sums are summed by
// a wave's lanes (every thread reading them one after the other took 1.3 us of 16 waves' call).
template <int N>
__device__ __forceinline__ void pool_scan(int64_t (&before)[N], int64_t (&all)[N], int64_t (*wave)[N]) {
  const int32_t lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  int64_t sum[N];
  kv_for<N>([&](auto K) { sum[K] = pool_lanes(before[K]); });
  __syncthreads();
  if (lane == 63) kv_for<N>([&](auto K) { wave[w][K] = sum[K]; });
  __syncthreads();
  kv_for<N>([&](auto K) {
    const int64_t past = pool_lanes(lane < waves ? wave[lane][K] : 0);
    before[K] = sum[K] - before[K] + (w > 0 ? pool_lane(past, max(w - 1, 0)) : 0);
    all[K] = pool_lane(past, waves - 1);
  });
}

// The last sequence that starts at a number or before it, from `low` on, which does, and before
// `high`: of a wave's one number, by 64 steps at a time, and of a number a lane.
__device__ __forceinline__ int32_t find_wave(const int32_t *starts, int32_t low, int32_t high, int64_t number) {
  const int32_t lane = threadIdx.x & 63;
  while (high - low > 1) {
    // up to 2^31 + 62
    const uint32_t step = ((high - low - 1) >> 6) + 1, end = high, at = low + step * (lane + 1);
    const uint32_t n = __popcll(__ballot(at < end && starts[min(at, end)] <= number));
    high = static_cast<int32_t>(min(end, low + step * (n + 1)));
    low += static_cast<int32_t>(step * n);
  }
  return __builtin_amdgcn_readfirstlane(low);
}
__device__ __forceinline__ int32_t find_lane(const int32_t *starts, int32_t low, int32_t high, int64_t number) {
  while (high - low > 1) {
    const int32_t mid = (low + high) >> 1;
    if (starts[mid] <= number)
      low = mid;
    else
      high = mid;
  }
  return low;
}

constexpr int32_t kPoolPicked = 4096;  // page numbers in shared memory
constexpr int32_t kPoolOwn = 2;        // pages of a sequence that its thread enters, a wave together the others
constexpr int32_t kPoolMost = INT_MAX;

// The free ones of sixteen pages, a bit each; what lies past the last page is none.
__device__ __forceinline__ uint32_t pool_free(const PoolArgs &p, int32_t w, const u32x4 &words) {
  uint32_t bits = 0;
  kv_for<4>([&](auto I) {  // four bytes' lowest bits side by side
    constexpr int i = I;
    const uint32_t v = words[i] & 0x01010101u;
    bits |= ((v | v >> 7 | v >> 14 | v >> 21) & 15u) << (4 * i);
  });
  const int32_t left = p.blocks - 16 * w;
  return left < 16 ? bits & ((1u << left) - 1u) : bits;
}
__device__ __forceinline__ uint32_t pool_free(const PoolArgs &p, int32_t w) {
  return pool_free(p, w, reinterpret_cast<const u32x4 *>(p.free)[w]);
}

struct PoolInfo {
  int32_t seq, old, n, inside;  // tokens held, new, and of the held ones those on the last page
  int32_t source;               // the page copied, -1: none
  int32_t begin, need;          // pages wanted from column `begin` on
  int32_t rank;                 // the first of them among all
};
__device__ __forceinline__ int32_t pool_room(const AssignArgs &a) { return min(a.p.width << a.p.log_page, a.max_length); }
__device__ __forceinline__ PoolInfo pool_held(const AssignArgs &a, int32_t s) {
  PoolInfo i{s, 0, 0, 0, -1, 0, 0, 0};
  if (s < a.p.seqs) {
    i.old = min(max(a.p.lengths[s], 0), a.p.width << a.p.log_page);
    i.n = min(a.asked ? max(a.asked[s], 0) : 1, a.max_rows);
    i.inside = i.old & ((1 << a.p.log_page) - 1);
  }
  return i;
}
// Its last page where it goes on in it and others hold it too.
__device__ __forceinline__ int32_t pool_tail(const PoolArgs &p, const PoolInfo &i) {
  if (i.n == 0 || i.inside == 0) return -1;
  const int32_t t = p.table[static_cast<int64_t>(i.seq) * p.width + (i.old >> p.log_page)];
  return pool_has(p, t) && p.refs[t] > 1 ? t : -1;
}
__device__ __forceinline__ void pool_want(const AssignArgs &a, PoolInfo &i) {
  i.begin = pool_pages(a.p, i.old) - (i.source >= 0 ? 1 : 0);
  i.need = i.n > 0 && i.n <= pool_room(a) - i.old ? pool_pages(a.p, i.old + i.n) - i.begin : 0;
}

// One workgroup for a call, as the pages of every sequence depend on those of all
// before it.  What a call needs is counted before anything is changed, so one that
// the pool has no room for changes nothing.  LOCAL: the page numbers go through shared
// memory into the tables; else, where they may be more than it holds, through memory, and
// kv_enter_kernel enters them.
// Bound by its chain: lengths, tails' entries and counts, a sum over the workgroup,
// page numbers into the tables.  One token each of 67 sequences 4.8 us, of 256 beams that all
// copy a page 5.9, 18800 pages of 515 sequences 7.0 and kv_enter_kernel's 4.3.
template <bool LOCAL>
__global__ __launch_bounds__(1024) void kv_assign_kernel(const AssignArgs a) {
  __shared__ int32_t held[LOCAL ? kPoolPicked : 1];
  __shared__ int64_t sums[16][3];
  __shared__ int32_t any, past;
  const PoolArgs &p = a.p;
  const int32_t threads = blockDim.x, tid = threadIdx.x, lane = tid & 63;
  const int32_t room = pool_room(a);
  const bool once = p.seqs <= threads;  // a sequence a thread, kept in registers

  // this thread's words of the free pages
  const int32_t each = (p.words + threads - 1) / threads;
  const int32_t word0 = min(tid * each, p.words), word1 = min(word0 + each, p.words);
  // the first two, mostly all, are kept
  u32x4 raw[2] = {};
  kv_for<2>([&](auto J) {
    if (word0 + J < word1) raw[J] = reinterpret_cast<const u32x4 *>(p.free)[word0 + J];
  });
  if (tid == 0) any = past = 0;
  __syncthreads();
  PoolInfo mine{};
  int32_t tail = -1;
  for (int32_t s0 = 0; s0 < p.seqs; s0 += threads) {
    mine = pool_held(a, s0 + tid);
    mine.source = tail = pool_tail(p, mine);
    if (mine.n > 0 && mine.n > room - mine.old) past = 1;
    if (mine.source >= 0) {
      any = 1;
      __hip_atomic_fetch_add(p.going + mine.source, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_fetch_min(p.first + mine.source, mine.seq, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  int64_t wanted = 0, rows = 0, free_before = 0, free_all = 0;
  uint32_t own[2];
  kv_for<2>([&](auto J) { own[J] = word0 + J < word1 ? pool_free(p, word0 + J, raw[J]) : 0; });
  auto free_of = [&](int32_t w) { return w == word0 ? own[0] : w == word0 + 1 ? own[1] : pool_free(p, w); };
  for (int32_t w = word0; w < word1; ++w) free_before += __popc(free_of(w));
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  const bool shared = any != 0;
  for (int32_t s0 = 0; s0 < p.seqs; s0 += threads) {
    if (!once) {
      mine = pool_held(a, s0 + tid);
      mine.source = pool_tail(p, mine);
    }
    if (shared && mine.source >= 0) {
      // the first of a page's holders keeps it if all of them go on
      const int32_t going = __hip_atomic_load(p.going + mine.source, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const int32_t first = __hip_atomic_load(p.first + mine.source, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (going == p.refs[mine.source] && first == mine.seq) mine.source = -1;
    }
    pool_want(a, mine);
    int64_t before[3] = {mine.need, mine.n, s0 == 0 ? free_before : 0}, total[3];
    pool_scan(before, total, sums);
    if (s0 == 0) {
      free_before = before[2];
      free_all = total[2];
    }
    mine.rank = static_cast<int32_t>(min(wanted + before[0], static_cast<int64_t>(kPoolMost)));
    if (mine.seq < p.seqs) {
      if (a.starts) a.starts[mine.seq] = static_cast<int32_t>(min(rows + before[1], static_cast<int64_t>(kPoolMost)));
      if (!once) {  // what was settled waits in the outputs
        int32_t *c = a.copies + 3 * static_cast<int64_t>(mine.seq);
        c[0] = mine.source;
        c[1] = mine.rank;
      }
    }
    wanted += total[0];
    rows += total[1];
  }
  const int32_t missing = rows > a.rows ? -2
                          : past != 0   ? -1
                                        : static_cast<int32_t>(min(max(wanted - free_all, static_cast<int64_t>(0)), static_cast<int64_t>(kPoolMost)));
  if (tid == 0) {
    if (a.starts) a.starts[p.seqs] = static_cast<int32_t>(min(rows, static_cast<int64_t>(kPoolMost)));
    *a.missing = missing;
  }
  const bool ok = missing == 0;
  const int32_t count = ok ? static_cast<int32_t>(wanted) : 0;
  __syncthreads();  // marks and counts are read by all before they change
  if (shared)
    for (int32_t s0 = 0; s0 < p.seqs; s0 += threads) {
      const int32_t t = once ? tail : pool_tail(p, pool_held(a, s0 + tid));
      if (t >= 0) {
        p.going[t] = 0;
        p.first[t] = INT_MAX;
      }
    }
  __syncthreads();

  // the lowest free pages, in their order
  if constexpr (LOCAL) {
    int64_t rank = free_before;
    for (int32_t w = word0; w < word1 && rank < count; ++w)
      for (uint32_t bits = free_of(w); bits != 0 && rank < count; bits &= bits - 1) {
        const int32_t number = 16 * w + __ffs(bits) - 1;
        held[rank++] = number;
        p.refs[number] = 1;
        p.free[number] = 0;
      }
    __syncthreads();
  } else {
    int64_t rank = free_before;
    for (int32_t w = word0; w < word1; ++w) {
      p.before[w] = static_cast<int32_t>(rank);
      rank += __popc(free_of(w));
    }
    if (tid == 0) p.spare[p.seqs] = count;
  }
  for (int32_t s0 = 0; s0 < p.seqs; s0 += threads) {
    if (!once) {
      mine = pool_held(a, s0 + tid);
      if (mine.seq < p.seqs) {
        mine.source = a.copies[3 * static_cast<int64_t>(mine.seq)];
        mine.rank = a.copies[3 * static_cast<int64_t>(mine.seq) + 1];
      }
      pool_want(a, mine);
    }
    if (count == 0) mine.need = 0;
    if constexpr (LOCAL) {
      kv_for<kPoolOwn>([&](auto J) {
        if (J < mine.need) p.table[static_cast<int64_t>(mine.seq) * p.width + mine.begin + J] = held[mine.rank + J];
      });
      uint64_t many = __ballot(mine.need > kPoolOwn);
      while (many != 0) {
        const int32_t l = __ffsll(static_cast<unsigned long long>(many)) - 1;
        many &= many - 1;
        const int32_t need = __shfl(mine.need, l), first = __shfl(mine.rank, l);
        int32_t *to = p.table + static_cast<int64_t>(__shfl(mine.seq, l)) * p.width + __shfl(mine.begin, l);
        for (int32_t j = kPoolOwn + lane; j < need; j += 64) to[j] = held[first + j];
      }
    }
    const int32_t s = mine.seq;
    if (s >= p.seqs) continue;
    const bool copied = ok && mine.source >= 0;
    int32_t *c = a.copies + 3 * static_cast<int64_t>(s);
    c[0] = copied ? mine.source : -1;
    c[1] = -1;
    if constexpr (LOCAL)
      if (copied) c[1] = held[mine.rank];
    c[2] = copied ? mine.inside : 0;
    if (copied) __hip_atomic_fetch_add(p.refs + mine.source, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    a.seen[s] = ok && mine.n > 0 ? mine.old + mine.n : 0;
    if (ok && mine.n > 0) p.lengths[s] = mine.old + mine.n;
    if constexpr (!LOCAL) p.spare[s] = mine.rank;
  }
}

// A thread a page: the free ones of the lowest ranks are taken, each by the sequence in whose
// part of the ranks it lies (searched for a wave's first and last page first: no faster).
__global__ __launch_bounds__(256) void kv_enter_kernel(const AssignArgs a) {
  const PoolArgs &p = a.p;
  const int64_t b = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int32_t w = static_cast<int32_t>(b >> 4), count = p.spare[p.seqs];
  if (w >= p.words || count == 0) return;
  const uint32_t bits = pool_free(p, w);
  const int32_t bit = static_cast<int32_t>(b & 15), rank = p.before[w] + __popc(bits & ((1u << bit) - 1u));
  if (!(bits >> bit & 1u) || rank >= count) return;
  const int32_t page = static_cast<int32_t>(b), low = find_lane(p.spare, 0, p.seqs, rank);
  const int32_t first = p.spare[low], need = p.spare[low + 1] - first;
  p.refs[page] = 1;
  p.free[page] = 0;
  p.table[static_cast<int64_t>(low) * p.width + (pool_pages(p, p.lengths[low]) - need) + (rank - first)] = page;
  int32_t *c = a.copies + 3 * static_cast<int64_t>(low);
  if (rank == first && c[0] >= 0) c[1] = page;
}

// A workgroup for a sequence: the pages past `to` tokens are let go.
__global__ __launch_bounds__(256) void kv_trim_kernel(const PoolArgs p, const int32_t *to, uint32_t first) {
  const int32_t s = first + blockIdx.x;
  const int32_t old = min(max(p.lengths[s], 0), p.width << p.log_page), n = min(old, max(to[s], 0));
  if (n == old) return;
  int32_t *row = p.table + static_cast<int64_t>(s) * p.width;
  for (int32_t w = pool_pages(p, n) + threadIdx.x; w < pool_pages(p, old); w += blockDim.x) {
    const int32_t page = row[w];
    row[w] = -1;
    pool_drop(p, page);
  }
  __syncthreads();  // every thread has read the length
  if (threadIdx.x == 0) p.lengths[s] = n;
}

// A sequence that goes on from itself is left alone, and a page that stays where it
// was is neither counted up nor down.
__device__ __forceinline__ int32_t pool_parent(const PoolArgs &p, const int32_t *parents, int32_t s) {
  const int32_t from = parents[s];
  return static_cast<uint32_t>(from) < static_cast<uint32_t>(p.seqs) ? from : -1;
}
// Two launches, a workgroup for a sequence each: what every sequence becomes is laid
// aside and held once more; then it takes its place and what was there is let go, after all
// that stays is held.  256 sequences of 512 pages 3.4 and 2.8 us, two launches' own time.
__global__ __launch_bounds__(256) void kv_gather_kernel(const PoolArgs p, const int32_t *parents, uint32_t first) {
  const int32_t s = first + blockIdx.x, from = pool_parent(p, parents, s);
  if (from == s) return;
  const int32_t *row = p.table + static_cast<int64_t>(s) * p.width, *source = p.table + static_cast<int64_t>(max(from, 0)) * p.width;
  int32_t *to = p.spare + static_cast<int64_t>(s) * p.width;
  for (int32_t w = threadIdx.x; w < p.width; w += blockDim.x) {
    const int32_t page = from < 0 ? -1 : source[w];
    to[w] = page;
    if (page != row[w] && pool_has(p, page)) __hip_atomic_fetch_add(p.refs + page, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (threadIdx.x == 0) p.spare_lengths[s] = from < 0 ? 0 : p.lengths[from];
}
__global__ __launch_bounds__(256) void kv_settle_kernel(const PoolArgs p, const int32_t *parents, uint32_t first) {
  const int32_t s = first + blockIdx.x, from = pool_parent(p, parents, s);
  if (from == s) return;
  int32_t *row = p.table + static_cast<int64_t>(s) * p.width;
  const int32_t *source = p.spare + static_cast<int64_t>(s) * p.width;
  for (int32_t w = threadIdx.x; w < p.width; w += blockDim.x) {
    const int32_t page = source[w], old = row[w];
    if (page == old) continue;
    row[w] = page;
    pool_drop(p, old);
  }
  if (threadIdx.x == 0) p.lengths[s] = p.spare_lengths[s];
}

// Small tables in one launch of one workgroup, which holds what every sequence becomes in
// registers until all that stays is held.
constexpr int kReorderEach = 8;
__global__ __launch_bounds__(1024) void kv_reorder_kernel(const PoolArgs p, const int32_t *parents, const KvDiv by_width) {
  const int32_t threads = blockDim.x, count = p.seqs * p.width;
  // loads that wait for each other do so once for all of a thread's entries
  int32_t from[kReorderEach], page[kReorderEach], old[kReorderEach], whose[kReorderEach], length[kReorderEach];
  kv_for<kReorderEach>([&](auto J) {
    const int32_t e = min(static_cast<int32_t>(threadIdx.x) + J * threads, count - 1);
    uint32_t s = e;
    kv_rem(by_width, s);
    from[J] = pool_parent(p, parents, s);
    old[J] = p.table[e];
    whose[J] = pool_parent(p, parents, min(e, p.seqs - 1));
  });
  kv_for<kReorderEach>([&](auto J) {
    const int32_t e = min(static_cast<int32_t>(threadIdx.x) + J * threads, count - 1);
    uint32_t s = e;
    const int32_t w = kv_rem(by_width, s);
    page[J] = p.table[static_cast<int64_t>(max(from[J], 0)) * p.width + w];
    if (from[J] < 0) page[J] = -1;
    length[J] = p.lengths[max(whose[J], 0)];
    if (whose[J] < 0) length[J] = 0;
  });
  kv_for<kReorderEach>([&](auto J) {
    if (static_cast<int32_t>(threadIdx.x) + J * threads < count && page[J] != old[J] && pool_has(p, page[J]))
      __hip_atomic_fetch_add(p.refs + page[J], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  });
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  kv_for<kReorderEach>([&](auto J) {
    const int32_t e = threadIdx.x + J * threads;
    if (e < count && page[J] != old[J]) {
      p.table[e] = page[J];
      pool_drop(p, old[J]);
    }
    if (e < p.seqs) p.lengths[e] = length[J];
  });
}

constexpr int32_t kSlotStarts = 4096;  // row starts held in shared memory

// A wave for GROUPS groups of 64 rows.  The sequences of a group's first and last row are found
// by 64 steps at a time among the row starts, which a workgroup reads once where they fit; a
// group of one sequence, which those of prompts mostly are, asks no more, else each row
// finds its own by halving between the two.  1.2 million rows of 515 sequences 9.2 us (without the stores
// 6.5, without the table's entries 8.6, without the searches 8.1), 64 rows of 67 2.7; every first row by
// halving among all 10.0 and 2.8, the next 64 row starts asked one after the other, in registers, 9.0 and 7.1.
template <int GROUPS>
__global__ __launch_bounds__(256) void kv_slots_kernel(const KvBatchArgs b, int32_t *positions, int64_t *slots) {
  __shared__ int32_t held[kSlotStarts];
  const bool few = b.starts && b.seqs < kSlotStarts;
  if (few) {
    for (int32_t i0 = threadIdx.x; i0 <= b.seqs; i0 += 1024) {  // four loads at a time
      int32_t v[4];
      kv_for<4>([&](auto U) { v[U] = b.starts[min(i0 + 256 * U, b.seqs)]; });
      kv_for<4>([&](auto U) {
        if (i0 + 256 * U <= b.seqs) held[i0 + 256 * U] = v[U];
      });
    }
    __syncthreads();
  }
  const int32_t *const starts = few ? held : b.starts;
  const int32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t wave_row = (static_cast<int64_t>(blockIdx.x) * 4 + wave) * (64 * GROUPS);
  if (wave_row >= b.rows) return;
  // sequences of all groups first, then their lengths, then their pages: loads that wait for
  // each other do so once
  int32_t seq[GROUPS], length[GROUPS], page[GROUPS], place[GROUPS], position[GROUPS];
  int32_t known = b.starts ? find_wave(starts, -1, b.seqs, wave_row) : 0;
  kv_for<GROUPS>([&](auto I) {
    const int64_t row0 = wave_row + 64 * I, row = row0 + lane;
    seq[I] = b.starts ? known : static_cast<int32_t>(min(row, static_cast<int64_t>(b.seqs)));
    if (b.starts && !(known >= 0 && known + 1 < b.seqs && starts[known + 1] > row0 + 63)) {
      const int32_t last = find_wave(starts, known, b.seqs, row0 + 63);
      seq[I] = find_lane(starts, known, last + 1, row);
      known = last;
    }
    const bool any = seq[I] >= 0 && seq[I] < b.seqs && row < b.rows;
    if (!any) seq[I] = -1;
    length[I] = any ? max(b.lengths[seq[I]], 0) : 0;
  });
  kv_for<GROUPS>([&](auto I) {
    const int64_t row = wave_row + 64 * I + lane;
    position[I] = 0;
    place[I] = 0;
    page[I] = -1;
    if (seq[I] >= 0) {
      int32_t first = static_cast<int32_t>(row), all = 1;
      if (b.starts) {
        first = min(max(starts[seq[I]], 0), b.rows);
        all = min(max(starts[seq[I] + 1], first), b.rows) - first;
      }
      const int32_t n = static_cast<int32_t>(row) - first, at = length[I] - all + n;
      if (n < all) {
        position[I] = max(at, 0);
        if (at >= 0 && n < b.max_rows && at < b.max_length) {
          page[I] = b.table[seq[I] * b.table_stride + (at >> b.log_page)];
          place[I] = at & ((1 << b.log_page) - 1);
        }
      }
    }
  });
  kv_for<GROUPS>([&](auto I) {
    const int64_t row = wave_row + 64 * I + lane;
    if (row < b.rows) {
      positions[row] = position[I];
      slots[row] = static_cast<uint32_t>(page[I]) < static_cast<uint32_t>(b.blocks)
                       ? (static_cast<int64_t>(page[I]) << b.log_page) + place[I]
                       : -1;
    }
  });
}

struct CopyArgs {
  uint8_t *k, *v;
  float *scales;
  const int32_t *copies;
  int32_t blocks, log_page, heads, row_bytes;
  KvDiv by_heads;
  uint32_t first;
};

// A workgroup for a sequence's copy of one head: the page's first tokens, keys and
// values, and its scales.  Bound by memory; most workgroups of a step find nothing to copy.
__global__ __launch_bounds__(256) void kv_copy_kernel(const CopyArgs a) {
  uint32_t id = a.first + blockIdx.x;
  const int32_t head = kv_rem(a.by_heads, id);
  const kv_const_i32 *c = (const kv_const_i32 *)a.copies + 3 * static_cast<int64_t>(id);
  const int32_t source = c[0], target = c[1], tokens = min(c[2], 1 << a.log_page);
  if (static_cast<uint32_t>(source) >= static_cast<uint32_t>(a.blocks) || static_cast<uint32_t>(target) >= static_cast<uint32_t>(a.blocks) ||
      source == target)
    return;
  const int64_t from = static_cast<int64_t>(source) * a.heads + head, to = static_cast<int64_t>(target) * a.heads + head;
  const int64_t size = static_cast<int64_t>(a.row_bytes) << a.log_page;
  const u32x4 *ks = reinterpret_cast<const u32x4 *>(a.k + from * size), *vs = reinterpret_cast<const u32x4 *>(a.v + from * size);
  u32x4 *kt = reinterpret_cast<u32x4 *>(a.k + to * size), *vt = reinterpret_cast<u32x4 *>(a.v + to * size);
  const int32_t count = tokens * a.row_bytes / 16;
  if (threadIdx.x < 2) a.scales[2 * to + threadIdx.x] = a.scales[2 * from + threadIdx.x];
  for (int32_t i = threadIdx.x; i < count; i += 512) {
    const int32_t j = i + 256;
    const u32x4 k0 = ks[i], v0 = vs[i];
    if (j < count) {
      const u32x4 k1 = ks[j], v1 = vs[j];
      kt[j] = k1;
      vt[j] = v1;
    }
    kt[i] = k0;
    vt[i] = v0;
  }
}

static int32_t pages_check(const char *what) {
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return RNSMX_OK;
  set_error("%s: %s", what, hipGetErrorString(err));
  return RNSMX_ELAUNCH;
}
static bool on(const void *p, int64_t n) { return p && reinterpret_cast<uintptr_t>(p) % n == 0; }
static int32_t log_of(int32_t page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1; }

static int64_t scratch_words(int32_t blocks, int32_t seqs, int32_t width) {
  return 3 * static_cast<int64_t>(blocks) + static_cast<int64_t>(seqs) * width + static_cast<int64_t>(seqs);
}

static int32_t pool_args(const rnsmx_kv_pool_t *pool, PoolArgs &a) {
  if (!pool) return fail(RNSMX_EINVAL, "null pool");
  a.log_page = log_of(pool->page);
  if (a.log_page < 0) return fail(RNSMX_EINVAL, "a page holds 16, 32, 64 or 128 tokens");
  if (pool->blocks < 1 || pool->seqs < 1 || pool->width < 1) return fail(RNSMX_EINVAL, "a pool has pages, sequences and a table");
  if ((static_cast<int64_t>(pool->width) << a.log_page) > 1 << 30) return fail(RNSMX_EINVAL, "sequences hold at most 2^30 tokens");
  if (!on(pool->table_dev, 4) || !on(pool->lengths_dev, 4) || !on(pool->refs_dev, 4) || !on(pool->free_dev, 16) || !on(pool->scratch_dev, 4))
    return fail(RNSMX_EINVAL, "a pool's pointer is null or not on a 4-byte (free_dev 16-byte) boundary");
  a.table = pool->table_dev;
  a.lengths = pool->lengths_dev;
  a.refs = pool->refs_dev;
  a.free = pool->free_dev;
  a.going = pool->scratch_dev;
  a.first = a.going + pool->blocks;
  a.before = a.first + pool->blocks;
  a.spare = a.before + pool->blocks;
  a.spare_lengths = a.spare + static_cast<int64_t>(pool->seqs) * pool->width;
  a.blocks = pool->blocks;
  a.words = static_cast<int32_t>((static_cast<int64_t>(pool->blocks) + 15) / 16);
  a.seqs = pool->seqs;
  a.width = pool->width;
  return RNSMX_OK;
}

// A workgroup for each sequence's row of the table, of the threads that it needs; several launches
// from 2^26 (rows past 64 pages: 2^24) sequences on.
template <typename K>
static void launch_rows(K kernel, const PoolArgs &a, const int32_t *numbers, void *stream) {
  const unsigned threads = a.width <= 64 ? 64 : 256;
  kv_launches(a.seqs, threads, [&](uint32_t first, uint32_t groups) {
    hipLaunchKernelGGL(kernel, dim3(groups), dim3(threads), 0, static_cast<hipStream_t>(stream), a, numbers, first);
  });
}

}  // namespace rnsmx

using namespace rnsmx;

extern "C" {

int64_t rnsmx_kv_pool_scratch_words(int32_t blocks, int32_t seqs, int32_t width) {
  return blocks < 1 || seqs < 1 || width < 1 ? -1 : scratch_words(blocks, seqs, width);
}

int32_t rnsmx_kv_assign(const rnsmx_kv_pool_t *pool, const rnsmx_kv_step_t *step, const int32_t *new_dev, void *stream) {
  clear_error();
  AssignArgs a{};
  if (int32_t rc = pool_args(pool, a.p)) return rc;
  if (!step) return fail(RNSMX_EINVAL, "null step");
  if (step->rows < 0 || step->max_rows < 0 || step->max_length < 0) return fail(RNSMX_EINVAL, "bad step sizes");
  if (!on(step->lengths_dev, 4) || !on(step->copies_dev, 4) || !on(step->missing_dev, 4) ||
      (step->starts_dev && !on(step->starts_dev, 4)) || (new_dev && !on(new_dev, 4)))
    return fail(RNSMX_EINVAL, "a step's pointer is null or not on a 4-byte boundary");
  a.asked = new_dev;
  a.seen = step->lengths_dev;
  a.starts = step->starts_dev;
  a.copies = step->copies_dev;
  a.missing = step->missing_dev;
  a.rows = step->rows;
  a.max_rows = step->max_rows;
  a.max_length = step->max_length;
  // a sequence and two words of free pages a thread
  const int64_t work = std::max<int64_t>(a.p.seqs, a.p.words / 2);
  const unsigned threads = static_cast<unsigned>(std::min<int64_t>(1024, (work + 63) / 64 * 64));
  // Most pages that a call can hand out: those of whole pages of rows, and for each sequence a
  // copy and a page that its rows begin or end.
  const int64_t most = std::min<int64_t>(a.p.blocks, (a.rows >> a.p.log_page) + 2 * std::min<int64_t>(a.p.seqs, a.rows));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (most <= kPoolPicked) {
    hipLaunchKernelGGL(kv_assign_kernel<true>, dim3(1), dim3(threads), 0, st, a);
  } else {
    hipLaunchKernelGGL(kv_assign_kernel<false>, dim3(1), dim3(1024), 0, st, a);
    hipLaunchKernelGGL(kv_enter_kernel, dim3((a.p.words + 15) / 16), dim3(256), 0, st, a);
  }
  return pages_check("kv_assign");
}

int32_t rnsmx_kv_trim(const rnsmx_kv_pool_t *pool, const int32_t *lengths_dev, void *stream) {
  clear_error();
  PoolArgs a{};
  if (int32_t rc = pool_args(pool, a)) return rc;
  if (!on(lengths_dev, 4)) return fail(RNSMX_EINVAL, "lengths null or not on a 4-byte boundary");
  launch_rows(kv_trim_kernel, a, lengths_dev, stream);
  return pages_check("kv_trim");
}

int32_t rnsmx_kv_reorder(const rnsmx_kv_pool_t *pool, const int32_t *parents_dev, void *stream) {
  clear_error();
  PoolArgs a{};
  if (int32_t rc = pool_args(pool, a)) return rc;
  if (!on(parents_dev, 4)) return fail(RNSMX_EINVAL, "parents null or not on a 4-byte boundary");
  const int64_t entries = static_cast<int64_t>(a.seqs) * a.width;
  if (entries <= kReorderEach * 1024) {
    const unsigned threads = static_cast<unsigned>(std::min<int64_t>(1024, (entries + 63) / 64 * 64));
    hipLaunchKernelGGL(kv_reorder_kernel, dim3(1), dim3(threads), 0, static_cast<hipStream_t>(stream), a, parents_dev, kv_div(a.width));
    return pages_check("kv_reorder");
  }
  launch_rows(kv_gather_kernel, a, parents_dev, stream);
  launch_rows(kv_settle_kernel, a, parents_dev, stream);
  return pages_check("kv_reorder");
}

int32_t rnsmx_kv_slots(const rnsmx_kv_batch_t *batch, int32_t blocks, int32_t page, int32_t *positions_dev, int64_t *slots_dev,
                       void *stream) {
  clear_error();
  if (!batch) return fail(RNSMX_EINVAL, "null batch");
  KvBatchArgs b{};
  b.log_page = log_of(page);
  if (b.log_page < 0) return fail(RNSMX_EINVAL, "a page holds 16, 32, 64 or 128 tokens");
  if (blocks < 1 || batch->seqs < 0 || batch->seqs == 0x7FFFFFFF || batch->rows < 0 || batch->max_rows < 0 || batch->max_length < 0 || batch->table_width < 1 ||
      batch->table_stride < 0)
    return fail(RNSMX_EINVAL, "bad batch sizes");
  if (batch->max_length > 1 << 30 || batch->max_length > static_cast<int64_t>(batch->table_width) << b.log_page)
    return fail(RNSMX_EINVAL, "max_length is past the block table");
  if (!batch->starts_dev && batch->rows != batch->seqs) return fail(RNSMX_EINVAL, "one row a sequence without row starts");
  if (batch->rows == 0) return RNSMX_OK;
  if (batch->seqs > 0 && (!on(batch->table_dev, 4) || !on(batch->lengths_dev, 4)))
    return fail(RNSMX_EINVAL, "a batch's pointer is null or not on a 4-byte boundary");
  if ((batch->starts_dev && !on(batch->starts_dev, 4)) || !on(positions_dev, 4) || !on(slots_dev, 8))
    return fail(RNSMX_EINVAL, "starts, positions or slots null or not aligned to their type");
  b.table = batch->table_dev;
  b.lengths = batch->lengths_dev;
  b.starts = batch->starts_dev;
  b.table_stride = batch->table_stride;
  b.blocks = blocks;
  b.seqs = batch->seqs;
  b.rows = batch->rows;
  b.max_rows = batch->starts_dev ? batch->max_rows : 1;
  b.max_length = batch->max_length;
  // a group a wave where that leaves some of the chip's waves free
  const int64_t each = 256 * (b.rows >= 1 << 18 ? 4 : 1);
  const dim3 grid(static_cast<unsigned>((b.rows + each - 1) / each));
  if (each > 256)
    hipLaunchKernelGGL(kv_slots_kernel<4>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), b, positions_dev, slots_dev);
  else
    hipLaunchKernelGGL(kv_slots_kernel<1>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), b, positions_dev, slots_dev);
  return pages_check("kv_slots");
}

int32_t rnsmx_kv_copy(const rnsmx_kv_cache_t *cache, const int32_t *copies_dev, int32_t count, void *stream) {
  clear_error();
  if (!cache) return fail(RNSMX_EINVAL, "null cache");
  CopyArgs a{};
  a.log_page = log_of(cache->page);
  if (a.log_page < 0 || cache->blocks < 1 || cache->heads < 1 || cache->row_bytes != rnsmx_kv_row_bytes(cache->head_dim) ||
      cache->row_bytes < 1)
    return fail(RNSMX_EINVAL, "bad cache sizes");
  if (!on(cache->k_dev, 16) || !on(cache->v_dev, 16) || !on(cache->scales_dev, 8))
    return fail(RNSMX_EINVAL, "codes start on 16-byte boundaries, scales on 8-byte ones");
  if (count < 0 || static_cast<int64_t>(count) * cache->heads > 0x7FFFFFFFLL) return fail(RNSMX_EINVAL, "too many copies and heads for one call");
  if (count == 0) return RNSMX_OK;
  if (!on(copies_dev, 4)) return fail(RNSMX_EINVAL, "copies null or not on a 4-byte boundary");
  a.k = cache->k_dev;
  a.v = cache->v_dev;
  a.scales = cache->scales_dev;
  a.copies = copies_dev;
  a.blocks = cache->blocks;
  a.heads = cache->heads;
  a.row_bytes = cache->row_bytes;
  a.by_heads = kv_div(cache->heads);
  kv_launches(static_cast<uint32_t>(count) * cache->heads, 256, [&](uint32_t first, uint32_t groups) {
    a.first = first;
    hipLaunchKernelGGL(kv_copy_kernel, dim3(groups), dim3(256), 0, static_cast<hipStream_t>(stream), a);
  });
  return pages_check("kv_copy");
}

}  // extern "C"
