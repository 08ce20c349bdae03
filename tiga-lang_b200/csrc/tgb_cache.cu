// The paged cache of keys and values: new tokens' rows into their pages, and
// eviction down to a budget by accumulated attention weight.
//
// Append: a copy.  One token per sequence (a decoding step): one block per
// sequence copies its rows and then moves that sequence's length on, so a step is
// one launch.  Runs of tokens (prompts): warps over all tokens read the old
// lengths, and a second kernel moves them on (8 prompts, 153 MB moved: 31 us, as a
// plain copy of as many bytes).
//
// Eviction: one block (or a cluster of them) per (sequence, head) finds the
// budget-th largest weight by a radix selection over the weights' order-preserving
// bit patterns (11 bits a pass, ranks and histogram in shared memory), then walks the
// places once in order, writing which place each kept row goes to; a second kernel
// moves the rows.  In place only as many rows move as places below the budget were
// freed: attention does not depend on the order of places, so a kept place below the
// budget stays where it is and no row is both read and written.  8 prompts of up to
// 16384 places and 8 heads of 128 to 2048: 18 us for the selection and 24 us for 134 MB
// of rows (a plain copy: 28 us).  The selection waits for its loads (5.3 clocks an
// instruction) more than at its barriers (2.1), with 1.6 % of the memory's rate: the
// cluster's size follows the capacity, so the longest sequence has 2 blocks of 1024
// threads left for itself when those of the short ones have ended.
#include <cooperative_groups.h>

#include <initializer_list>

#include "tgb_cache.cuh"

namespace tgb {
namespace {

__device__ __forceinline__ uint4 load16(const void *p) { return __ldcs(static_cast<const uint4 *>(p)); }

// ---- append -----------------------------------------------------------------
struct AppendArgs {
  tgb_paged_cache cache;
  const unsigned char *key, *value;
  int64_t key_token_stride, key_head_stride, value_token_stride, value_head_stride;   // bytes
  int64_t tokens;
  const int32_t *bounds, *start;
};

// where sequence b's run begins; faults are clamped
__device__ __forceinline__ int append_start(const AppendArgs &a, int b, int length) {
  if (!a.start) return length;
  const int start = a.start[b];
  if (start < 0 || start > length) {
    cache_fault(a.cache, TGB_CACHE_BAD_START);
    return start < 0 ? 0 : length;
  }
  return start;
}

// where a new token goes: row -1 where it goes nowhere; a tracking cache's state is set on the way
__device__ __forceinline__ int64_t append_row(const AppendArgs &a, int b, int64_t place) {
  const tgb_paged_cache &c = a.cache;
  if (place >= cache_capacity(c)) {
    cache_fault(c, TGB_CACHE_FULL);
    return -1;
  }
  return cache_row(c, b, (int)place);
}
__device__ __forceinline__ void append_state(const AppendArgs &a, int b, int place, int number, int thread, int threads) {
  const tgb_paged_cache &c = a.cache;
  for (int h = thread; h < c.heads; h += threads) {
    const int64_t at = ((int64_t)b * c.heads + h) * cache_capacity(c) + place;
    c.weight[at] = 0.f, c.position[at] = number;
  }
}

// a token's key and value, `thread` of `threads` 16-byte pieces at a time; PACKED: the heads of a row follow each
// other on both sides
template <bool PACKED>
__device__ __forceinline__ void append_copy(const AppendArgs &a, int64_t token, int64_t row, int thread, int threads) {
  const tgb_paged_cache &c = a.cache;
  const int pieces = c.dim / 8, all = c.heads * pieces;
  const unsigned char *key = a.key + token * a.key_token_stride, *value = a.value + token * a.value_token_stride;
  unsigned char *to_key = static_cast<unsigned char *>(c.key) + row * c.key_slot_stride * 2;
  unsigned char *to_value = static_cast<unsigned char *>(c.value) + row * c.value_slot_stride * 2;
  constexpr int kUnroll = 4;
  for (int first = thread; first < all; first += kUnroll * threads) {
    uint4 k[kUnroll], v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = first + u * threads, h = PACKED ? 0 : i / pieces, p = i - h * pieces;
      if (i < all) k[u] = load16(key + h * a.key_head_stride + p * 16), v[u] = load16(value + h * a.value_head_stride + p * 16);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = first + u * threads, h = PACKED ? 0 : i / pieces, p = i - h * pieces;
      if (i >= all) break;
      *reinterpret_cast<uint4 *>(to_key + h * c.key_head_stride * 2 + p * 16) = k[u];
      *reinterpret_cast<uint4 *>(to_value + h * c.value_head_stride * 2 + p * 16) = v[u];
    }
  }
}

__device__ __forceinline__ void append_lengths(const AppendArgs &a, int b, int length, int start, int64_t run) {
  const tgb_paged_cache &c = a.cache;
  const int64_t room = cache_capacity(c) - start, taken = run < room ? run : room;
  if (c.seen) c.seen[b] += start + (int)taken - length;
  c.lengths[b] = start + (int)taken;
}

template <bool PACKED> __global__ void __launch_bounds__(256) k_append_step(const __grid_constant__ AppendArgs a) {
  const int b = blockIdx.x;
  wait_for_previous();
  const int length = cache_length(a.cache, b), start = append_start(a, b, length);
  const int number = a.cache.seen ? a.cache.seen[b] + start - length : 0;
  __syncthreads();                           // everyone has the old length before it changes
  const int64_t row = append_row(a, b, start);
  if (a.cache.weight && start < cache_capacity(a.cache)) append_state(a, b, start, number, threadIdx.x, blockDim.x);
  if (row >= 0) append_copy<PACKED>(a, b, row, threadIdx.x, blockDim.x);
  if (threadIdx.x == 0) append_lengths(a, b, length, start, 1);
}

// where the run of sequence b begins, or the last one ends, inside [0, tokens]
__device__ __forceinline__ int64_t append_bound(const AppendArgs &a, int b) {
  const int64_t v = a.bounds[b];
  return v < 0 ? 0 : v > a.tokens ? a.tokens : v;
}

constexpr int kAppendWarps = 8;

// A warp takes `each` tokens in a row: its lanes find out at once where they go, then all of them copy one token
// after the other.
template <bool PACKED>
__global__ void __launch_bounds__(kAppendWarps * 32, PACKED ? 4 : 1) k_append_runs(const __grid_constant__ AppendArgs a, int each) {
  const int lane = threadIdx.x % 32;
  wait_for_previous();
  const int64_t first_token = ((int64_t)blockIdx.x * kAppendWarps + threadIdx.x / 32) * each;
  if (first_token >= a.tokens) return;
  const int count = (int)(a.tokens - first_token < each ? a.tokens - first_token : each);
  int64_t row = -1;
  int sequence = 0, place = -1, number = 0;  // place >= 0: a place of the sequence
  if (lane < count) {
    const int64_t token = first_token + lane;
    int low = 0, high = a.cache.sequences;   // the last sequence whose run begins at or before the token
    while (low < high) {
      const int middle = (low + high + 1) / 2;
      if (middle < a.cache.sequences && append_bound(a, middle) <= token) low = middle;
      else high = middle - 1;
    }
    const int64_t first = append_bound(a, low), last = append_bound(a, low + 1);
    if (token >= first && token < last) {
      const int length = cache_length(a.cache, low), start = append_start(a, low, length);
      const int64_t at = start + (token - first);
      sequence = low;
      row = append_row(a, low, at);
      place = at < cache_capacity(a.cache) ? (int)at : -1;
      number = a.cache.seen ? (int)(a.cache.seen[low] + (at - length)) : 0;
    }
  }
  for (int i = 0; i < count; ++i) {
    const int64_t to = __shfl_sync(0xffffffffu, row, i);
    if (to >= 0) append_copy<PACKED>(a, first_token + i, to, lane, 32);
  }
  if (!a.cache.weight) return;
  for (int i = 0; i < count; ++i) {
    const int b = __shfl_sync(0xffffffffu, sequence, i), at = __shfl_sync(0xffffffffu, place, i);
    const int n = __shfl_sync(0xffffffffu, number, i);
    if (at >= 0) append_state(a, b, at, n, lane, 32);
  }
}

__global__ void __launch_bounds__(256) k_append_lengths(const __grid_constant__ AppendArgs a) {
  wait_for_previous();
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= a.cache.sequences) return;
  const int length = cache_length(a.cache, b), start = append_start(a, b, length);
  // runs that overlap or leave the tokens: some of their places were not written
  if (a.bounds[b] < 0 || a.bounds[b] > a.bounds[b + 1] || a.bounds[b + 1] > a.tokens) cache_fault(a.cache, TGB_CACHE_BAD_BOUNDS);
  const int64_t run = append_bound(a, b + 1) - append_bound(a, b);
  append_lengths(a, b, length, start, run > 0 ? run : 0);
}

// ---- eviction -----------------------------------------------------------------
struct EvictArgs {
  tgb_paged_cache cache, into;
  int32_t in_place, budget, recent;
  int32_t list;                              // entries of a list of one (sequence, head)
  int32_t *from;                             // [sequences * heads][list] places of rows that move
  int32_t *to;                               // in place: [sequences * heads][list] freed places
  int32_t *moves;                            // [sequences * heads] rows that move
};

constexpr int kItems = 4;                    // places a thread takes of one stretch
constexpr int kDigits = 3;                   // of a rank: 11, 11 and 10 bits from the top
constexpr int kBins = 2048;

// order of a place: larger is kept first
__device__ __forceinline__ uint32_t evict_rank(float weight, int position, int newest) {
  if (position >= newest) return 0xffffffffu;
  if (weight != weight) return 0;
  const uint32_t bits = __float_as_uint(weight + 0.f);        // -0 counts as 0
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// exclusive prefix sums of two counts over the block's threads, packed in 32 + 32 bits; total in `all`
template <int THREADS>
__device__ __forceinline__ unsigned long long block_before(unsigned long long v, unsigned long long *warps,
                                                           unsigned long long &all) {
  constexpr int kWarps = THREADS / 32;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  unsigned long long sum = v;
#pragma unroll
  for (int step = 1; step < 32; step <<= 1) {
    const unsigned long long other = __shfl_up_sync(0xffffffffu, sum, step);
    if (lane >= step) sum += other;
  }
  if (lane == 31) warps[warp] = sum;
  __syncthreads();
  unsigned long long through = lane < kWarps ? warps[lane] : 0;      // every warp scans the warps' sums for itself
#pragma unroll
  for (int step = 1; step < kWarps; step <<= 1) {
    const unsigned long long other = __shfl_up_sync(0xffffffffu, through, step);
    if (lane >= step) through += other;
  }
  all = __shfl_sync(0xffffffffu, through, kWarps - 1);
  const unsigned long long before = __shfl_sync(0xffffffffu, through, warp ? warp - 1 : 0);
  __syncthreads();
  return (warp ? before : 0) + sum - v;
}

constexpr int kFew = 8;

// Where at most kFew places go, as in every step of a cache held at its budget, they are found one after the other:
// the smallest (rank, -place) above the last one. One block does it. (64 sequences and 8 heads of 2049 places: append and
// eviction 12.8 us, 23.3 with the selection by digits.)
template <int THREADS>
__device__ void evict_few(const EvictArgs &a, int id, int length, const uint32_t *ranks, int32_t *from, int32_t *to) {
  __shared__ unsigned long long least[THREADS / 32];
  __shared__ int gone[kFew];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, few = length - a.budget;
  unsigned long long last = 0;               // smallest key that may go; a key is never 0: no place is 2^32 - 1
  for (int i = 0; i < few; ++i) {
    unsigned long long best = ~0ull;
    for (int t = threadIdx.x; t < length; t += THREADS) {
      const unsigned long long key = (unsigned long long)ranks[t] << 32 | (0xffffffffu - (uint32_t)t);
      if (key >= last && key < best) best = key;
    }
    const uint32_t rank = __reduce_min_sync(0xffffffffu, (uint32_t)(best >> 32));
    const uint32_t place = __reduce_min_sync(0xffffffffu, (uint32_t)(best >> 32) == rank ? (uint32_t)best : 0xffffffffu);
    if (lane == 0) least[warp] = (unsigned long long)rank << 32 | place;
    __syncthreads();
    best = least[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) best = least[w] < best ? least[w] : best;
    last = best + 1;
    if (threadIdx.x == 0) gone[i] = (int)(0xffffffffu - (uint32_t)best);
    __syncthreads();
  }
  auto goes = [&](int t) {
    bool found = false;
    for (int i = 0; i < few; ++i) found = found || gone[i] == t;
    return found;
  };
  if (!a.in_place) {
    for (int t = threadIdx.x; t < length; t += THREADS) {
      int before = 0;
      for (int i = 0; i < few; ++i) before += gone[i] < t;
      if (!goes(t)) from[t - before] = t;
    }
    if (threadIdx.x == 0) a.moves[id] = a.budget;
  } else if (threadIdx.x == 0) {
    int moves = 0, free = 0;
    for (int t = length - 1; t >= a.budget; --t)             // listed from the last kept place
      if (!goes(t)) from[moves++] = t;
    for (int least_free = -1; free < moves; ++free) {
      int next = length;
      for (int i = 0; i < few; ++i)
        if (gone[i] > least_free && gone[i] < next) next = gone[i];
      to[free] = least_free = next;
    }
    a.moves[id] = moves;
  }
}

// One cluster of blocks per (sequence, head), each block with an equal run of the places.  The ranks of the
// first `cached` places are kept in shared memory, so that weights and positions are read once; a longer
// sequence computes the others again for every digit.
template <int THREADS>
__global__ void __launch_bounds__(THREADS) k_evict_select(const __grid_constant__ EvictArgs a, int cached) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint32_t ranks[];
  __shared__ uint32_t histograms[2][kBins];
  __shared__ uint32_t chosen[4];
  __shared__ unsigned long long warps[THREADS / 32];
  const cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), block = cluster.block_rank();
  const tgb_paged_cache &c = a.cache;
  const int id = blockIdx.x / blocks, b = id / c.heads;
  wait_for_previous();
  const int length = cache_length(c, b);
  const int64_t base = (int64_t)id * cache_capacity(c);
  int32_t *from = a.from + (int64_t)id * a.list, *to = a.to + (int64_t)id * a.list;
  if (length <= a.budget) {                  // everything stays
    if (!a.in_place)
      for (int t = block * THREADS + threadIdx.x; t < length; t += blocks * THREADS) from[t] = t;
    if (block == 0 && threadIdx.x == 0) a.moves[id] = a.in_place ? 0 : length;
    return;
  }
  const float *weight = c.weight + base;
  const int32_t *position = c.position + base;
  const long long first_new = (long long)c.seen[b] - a.recent;
  const int newest = (int)(first_new < -2147483647ll ? -2147483647ll : first_new);
  if (length - a.budget <= kFew && length <= cached) {
    if (block) return;
#pragma unroll 4
    for (int t = threadIdx.x; t < length; t += THREADS) ranks[t] = evict_rank(weight[t], position[t], newest);
    __syncthreads();
    evict_few<THREADS>(a, id, length, ranks, from, to);
    return;
  }
  // this block's places, a multiple of kItems each; rank of one of them
  const int share = ((length + blocks - 1) / blocks + kItems - 1) / kItems * kItems;
  const int begin = min(block * share, length), end = min(begin + share, length);
  auto rank_of = [&](int t) {
    return t - begin < cached ? ranks[t - begin] : evict_rank(weight[t], position[t], newest);
  };

  // the budget-th largest rank, digit by digit from the top
  uint32_t prefix = 0, wanted = a.budget;    // how many of the places whose upper digits are `prefix` stay
  unsigned long long done = 0;               // places above the rank, places equal to it (32 + 32 bits), in the blocks before
  for (int digit = 0; digit < kDigits; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bits = digit == 2 ? 10 : 11;
    uint32_t *histogram = histograms[digit & 1];              // the other one may still be read by the cluster
    for (int i = threadIdx.x; i < kBins; i += THREADS) histogram[i] = 0;
    __syncthreads();
    if (digit == 0) {
#pragma unroll 4
      for (int t = begin + threadIdx.x; t < end; t += THREADS) {
        const uint32_t rank = evict_rank(weight[t], position[t], newest);
        if (t - begin < cached) ranks[t - begin] = rank;
        atomicAdd(&histogram[rank >> 21], 1u);
      }
    } else {
#pragma unroll 4
      for (int t = begin + threadIdx.x; t < end; t += THREADS) {
        const uint32_t rank = rank_of(t);
        if (rank >> (shift + bits) == prefix) atomicAdd(&histogram[rank >> shift & ((1u << bits) - 1)], 1u);
      }
    }
    cluster.sync();
    constexpr int kEach = kBins / THREADS;   // bins of a thread, the largest digits first
    uint32_t counts[kEach] = {}, lower[kEach] = {}, sum = 0, lower_sum = 0;      // of all blocks, of the blocks before
    for (int r = 0; r < blocks; ++r) {
      const uint32_t *other = cluster.map_shared_rank(histogram, r);
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const uint32_t n = other[kBins - 1 - kEach * threadIdx.x - i];
        counts[i] += n, lower[i] += r < block ? n : 0;
      }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += counts[i], lower_sum += lower[i];
    unsigned long long all;
    const unsigned long long both = block_before<THREADS>((unsigned long long)lower_sum << 32 | sum, warps, all);
    uint32_t before = (uint32_t)both, lower_before = (uint32_t)(both >> 32);
    if (before < wanted && wanted <= before + sum) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (before < wanted && wanted <= before + counts[i]) {
          chosen[0] = prefix << bits | (kBins - 1 - kEach * threadIdx.x - i), chosen[1] = wanted - before;
          chosen[2] = lower_before, chosen[3] = lower[i];
        }
        before += counts[i], lower_before += lower[i];
      }
    }
    __syncthreads();
    prefix = chosen[0], wanted = chosen[1];
    done += (unsigned long long)chosen[2] << 32;
    if (digit + 1 == kDigits) done += chosen[3];
  }
  // nobody leaves while its shared memory is read; all reading is done
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");

  // ranks above `prefix` stay, and the first `wanted` places of rank `prefix`
  auto count_of = [&](uint32_t rank) { return rank > prefix ? 1ull << 32 : rank == prefix ? 1ull : 0ull; };
  for (int stretch = begin; stretch < end; stretch += THREADS * kItems) {
    const int t0 = stretch + threadIdx.x * kItems;
    uint32_t rank[kItems];
    unsigned long long counts = 0;
    if (t0 - begin + kItems <= cached && t0 + kItems <= end) {
      const uint4 four = *reinterpret_cast<const uint4 *>(ranks + t0 - begin);
      rank[0] = four.x, rank[1] = four.y, rank[2] = four.z, rank[3] = four.w;
    } else {
#pragma unroll
      for (int i = 0; i < kItems; ++i) rank[i] = t0 + i < end ? rank_of(t0 + i) : 0;
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (t0 + i < end) counts += count_of(rank[i]);
    unsigned long long all;
    unsigned long long before = done + block_before<THREADS>(counts, warps, all);
    done += all;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int t = t0 + i;
      if (t >= end) break;
      const uint32_t above = (uint32_t)(before >> 32), equal = (uint32_t)before;
      const bool keep = rank[i] > prefix || (rank[i] == prefix && equal < wanted);
      const int kept = (int)(above + min(equal, wanted));       // kept places before this one
      if (a.in_place && t == a.budget) a.moves[id] = a.budget - kept;      // as many as are kept from here on
      if (keep) {
        if (!a.in_place) from[kept] = t;
        else if (t >= a.budget) from[a.budget - 1 - kept] = t;  // counted from the last kept place
      } else if (a.in_place && t < a.budget) {
        to[t - kept] = t;
      }
      before += count_of(rank[i]);
    }
  }
  if (!a.in_place && block == 0 && threadIdx.x == 0) a.moves[id] = a.budget;
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

constexpr int kMoveWarps = 8;

constexpr int kMoveRows = 32;                // of a warp

// A warp looks up its rows' moves at once, a lane each, and carries their weights and positions over; then its
// lanes copy the rows' 16-byte pieces, four loads in flight each.
__global__ void __launch_bounds__(kMoveWarps * 32) k_evict_move(const __grid_constant__ EvictArgs a) {
  const tgb_paged_cache &c = a.cache, &g = a.into;
  const int id = blockIdx.x, b = id / c.heads, h = id % c.heads;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  wait_for_previous();
  const int moves = a.moves[id], capacity = cache_capacity(c), target_capacity = cache_capacity(g);
  const int32_t *from = a.from + (int64_t)id * a.list, *to = a.to + (int64_t)id * a.list;
  // a row's key pieces, then its value pieces; short rows several at a time
  const int pieces = c.dim / 8, both = 2 * pieces, rows_at_once = both < 32 ? 32 / both : 1;
  const int my_row = both < 32 ? lane / both : 0;
  const uint64_t key_stride = c.key_slot_stride * 2, value_stride = c.value_slot_stride * 2;
  const uint64_t to_key_stride = g.key_slot_stride * 2, to_value_stride = g.value_slot_stride * 2;
  for (int first = (blockIdx.y * kMoveWarps + warp) * kMoveRows; first < moves; first += gridDim.y * kMoveWarps * kMoveRows) {
    const int n = min(kMoveRows, moves - first);
    int row = -1, target = -1;
    if (lane < n) {
      const int i = first + lane;
      const int source = from[a.in_place ? moves - 1 - i : i], place = a.in_place ? to[i] : i;
      row = (int)cache_row(c, b, source), target = (int)cache_row(g, b, place);
      if (g.weight) {
        const int64_t s = (int64_t)id * capacity + source, t = (int64_t)id * target_capacity + place;
        g.weight[t] = c.weight[s], g.position[t] = c.position[s];
      }
      if (row < 0 || target < 0) row = target = -1;
    }
    for (int q = 0; q < both; q += 32) {     // every lane takes every round: rows are handed out by shuffle
      const int p = both < 32 ? lane % both : q + lane;
      const bool works = p < both && my_row < rows_at_once, is_key = p < pieces;
      const unsigned char *in = is_key ? static_cast<unsigned char *>(c.key) + (h * c.key_head_stride + p * 8) * 2
                                       : static_cast<unsigned char *>(c.value) + (h * c.value_head_stride + (p - pieces) * 8) * 2;
      unsigned char *out = is_key ? static_cast<unsigned char *>(g.key) + (h * g.key_head_stride + p * 8) * 2
                                  : static_cast<unsigned char *>(g.value) + (h * g.value_head_stride + (p - pieces) * 8) * 2;
      const uint64_t stride = is_key ? key_stride : value_stride, to_stride = is_key ? to_key_stride : to_value_stride;
      constexpr int kUnroll = 4;
      for (int r0 = 0; r0 < n; r0 += rows_at_once * kUnroll) {
        uint4 v[kUnroll];
        int put[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int r = r0 + u * rows_at_once + my_row;
          const int s = __shfl_sync(0xffffffffu, row, r & 31);
          put[u] = __shfl_sync(0xffffffffu, target, r & 31);
          if (r >= n || !works) put[u] = -1;
          if (put[u] >= 0) v[u] = *reinterpret_cast<const uint4 *>(in + s * stride);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (put[u] >= 0) *reinterpret_cast<uint4 *>(out + put[u] * to_stride) = v[u];
      }
    }
  }
  if (h == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
    // the select kernel is done with lengths; other blocks of this one read none
    const int length = cache_length(c, b);
    g.lengths[b] = length < a.budget ? length : a.budget;
    if (!a.in_place && g.seen) g.seen[b] = c.seen[b];
  }
}

template <int THREADS>
int32_t launch_select(const EvictArgs &a, int64_t rows, int64_t capacity, int cluster, cudaStream_t stream) {
  constexpr int kMost = 48 * 1024 - 2048;    // ranks that fit into shared memory next to the histograms
  const int cached = (int)(capacity < kMost ? capacity : kMost);
  const size_t bytes = align_up(4 * (uint64_t)cached, 16);
  static std::atomic<uint64_t> asked{0};
  TGB_CUDA(allow_shared(k_evict_select<THREADS>, 4 * kMost, asked));
  TGB_CUDA(launch_clusters(k_evict_select<THREADS>, cluster, dim3((unsigned)(rows * cluster)), dim3(THREADS), bytes, stream,
                           a, cached));
  return TGB_STATUS_OK;
}

int32_t evict_list(const tgb_paged_cache &c, int32_t budget) {
  const int64_t capacity = (int64_t)c.pages_per_sequence * c.page_size;
  return (int32_t)(budget < capacity ? budget : capacity);
}

}  // namespace

int32_t check_cache(const tgb_paged_cache *c) {
  if (!c) TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "null cache");
  if (c->dtype != TGB_DTYPE_BF16 && c->dtype != TGB_DTYPE_F16) TGB_FAIL(TGB_STATUS_UNSUPPORTED, "a paged cache holds bfloat16 or float16");
  if (c->dim < 8 || c->dim > 256 || c->dim % 8) TGB_FAIL(TGB_STATUS_UNSUPPORTED, "head size must be a multiple of 8 up to 256, got %d", c->dim);
  if (c->sequences < 0 || c->heads < 1 || c->heads > (1 << 16) || c->page_size < 1 || c->pages_per_sequence < 0 || c->num_pages < 1)
    TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "sequences >= 0, heads in [1, 65536], page_size >= 1, pages_per_sequence >= 0 and num_pages >= 1 expected");
  if ((int64_t)c->pages_per_sequence * c->page_size > (1 << 30)) TGB_FAIL(TGB_STATUS_UNSUPPORTED, "a sequence has at most 2^30 places");
  if (c->page_size > (1 << 30) || c->num_pages > ((1ll << 31) - 1) / c->page_size)
    TGB_FAIL(TGB_STATUS_UNSUPPORTED, "a cache has fewer than 2^31 slots");
  for (const int64_t stride : {c->key_slot_stride, c->value_slot_stride})
    if (stride < 0 || stride > (1 << 30)) TGB_FAIL(TGB_STATUS_UNSUPPORTED, "slot strides are non-negative and at most 2^30 values");
  if ((int64_t)c->sequences * c->heads > (1 << 30)) TGB_FAIL(TGB_STATUS_UNSUPPORTED, "at most 2^30 pairs of sequence and head");
  if (!c->key || !c->value || !c->fault || (c->sequences && (!c->lengths || (c->pages_per_sequence && !c->page_table))))
    TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "null cache pointer");
  // memory of no places may have no address
  const bool places = c->sequences && c->pages_per_sequence;
  if (places ? !c->weight != !c->seen || !c->position != !c->seen : (c->weight || c->position) && !c->seen)
    TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "weight, position and seen come together");
  if (reinterpret_cast<uintptr_t>(c->key) % 16 || reinterpret_cast<uintptr_t>(c->value) % 16 || c->key_slot_stride % 8 ||
      c->key_head_stride % 8 || c->value_slot_stride % 8 || c->value_head_stride % 8)
    TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "cache rows must be 16-byte aligned");
  return TGB_STATUS_OK;
}

}  // namespace tgb

extern "C" {

int32_t tgb_cache_append(const tgb_paged_cache *cache, const void *key, const void *value, int64_t key_token_stride,
                         int64_t key_head_stride, int64_t value_token_stride, int64_t value_head_stride, int64_t tokens,
                         const void *bounds, const void *start, uint64_t stream_handle) {
  const int32_t status = tgb::check_cache(cache);
  if (status) return status;
  if (tokens < 0 || (!bounds && tokens != cache->sequences))
    TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "without bounds there is one token per sequence");
  if (!cache->sequences) return TGB_STATUS_OK;
  if (tokens && (!key || !value)) TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "null key or value");
  if (reinterpret_cast<uintptr_t>(key) % 16 || reinterpret_cast<uintptr_t>(value) % 16 || key_token_stride % 8 ||
      key_head_stride % 8 || value_token_stride % 8 || value_head_stride % 8)
    TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "new rows must be 16-byte aligned");
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
  const tgb::AppendArgs a{*cache, static_cast<const unsigned char *>(key), static_cast<const unsigned char *>(value),
                          2 * key_token_stride, 2 * key_head_stride, 2 * value_token_stride, 2 * value_head_stride, tokens,
                          static_cast<const int32_t *>(bounds), static_cast<const int32_t *>(start)};
  const bool packed = key_head_stride == cache->dim && value_head_stride == cache->dim &&
                      cache->key_head_stride == cache->dim && cache->value_head_stride == cache->dim;
  if (!bounds) {
    const int pieces = cache->heads * (cache->dim / 8);
    const int threads = pieces >= 256 ? 256 : pieces >= 128 ? 128 : 64;
    TGB_CUDA(tgb::launch_dependent(packed ? tgb::k_append_step<true> : tgb::k_append_step<false>, dim3(cache->sequences),
                                   dim3(threads), 0, stream, a));
    return TGB_STATUS_OK;
  }
  if (tokens) {
    // one round of resident warps where that leaves each of them at most 8 tokens
    const int64_t share = tgb::ceil_div(tokens, 148 * 32);
    const int each = (int)(share < 8 ? share : 8);
    const int64_t blocks = tgb::ceil_div(tokens, (int64_t)each * tgb::kAppendWarps);
    if (blocks > 0x7fffffff) TGB_FAIL(TGB_STATUS_UNSUPPORTED, "too many tokens");
    TGB_CUDA(tgb::launch_dependent(packed ? tgb::k_append_runs<true> : tgb::k_append_runs<false>, dim3((unsigned)blocks),
                                   dim3(tgb::kAppendWarps * 32), 0, stream, a, each));
  }
  TGB_CUDA(tgb::launch_dependent(tgb::k_append_lengths, dim3((unsigned)tgb::ceil_div(cache->sequences, 256)), dim3(256), 0,
                                 stream, a));
  return TGB_STATUS_OK;
}

int32_t tgb_cache_evict_scratch_bytes(const tgb_paged_cache *cache, int32_t budget, uint64_t *bytes) {
  const int32_t status = tgb::check_cache(cache);
  if (status) return status;
  if (!bytes || budget < 0) TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "null bytes or negative budget");
  const uint64_t rows = (uint64_t)cache->sequences * cache->heads;
  *bytes = 4 * rows + 8 * rows * tgb::evict_list(*cache, budget);
  return TGB_STATUS_OK;
}

int32_t tgb_cache_evict(const tgb_paged_cache *cache, const tgb_paged_cache *into, int32_t budget, int32_t recent,
                        void *scratch, uint64_t scratch_bytes, uint64_t stream_handle) {
  uint64_t need = 0;
  int32_t status = tgb_cache_evict_scratch_bytes(cache, budget, &need);
  if (status) return status;
  const bool in_place = !into || into == cache;
  if (cache->sequences && !cache->seen) TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "the cache does not track attention weights");
  if (budget < 1 || recent < 0 || recent > budget)
    TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "budget must be positive and recent in [0, budget]");
  const int32_t list = tgb::evict_list(*cache, budget);
  if (!in_place) {
    status = tgb::check_cache(into);
    if (status) return status;
    if (into->sequences != cache->sequences || into->heads != cache->heads || into->dim != cache->dim || into->dtype != cache->dtype)
      TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "both caches need the same sequences, heads, head size and dtype");
    if ((int64_t)into->pages_per_sequence * into->page_size < list)
      TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "the cache evicted into has fewer places than the budget");
  }
  if (!cache->sequences) return TGB_STATUS_OK;
  if (!scratch || scratch_bytes < need || reinterpret_cast<uintptr_t>(scratch) % 8)
    TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "eviction needs %llu bytes of scratch", (unsigned long long)need);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
  const int64_t rows = (int64_t)cache->sequences * cache->heads;
  tgb::EvictArgs a;
  a.cache = *cache, a.into = in_place ? *cache : *into;
  a.in_place = in_place, a.budget = budget, a.recent = recent, a.list = list;
  a.moves = static_cast<int32_t *>(scratch);
  a.from = a.moves + rows;
  a.to = a.from + rows * list;
  const int64_t capacity = (int64_t)cache->pages_per_sequence * cache->page_size;
  // More sequences and heads than SMs, of few places each: small blocks, several to an SM, whose barriers cost less (a
  // decoding step of 64 sequences and 8 heads of 2049 places: 12.8 us against 24.9; 2000 places down to 500: 60.6
  // against 64.8). Otherwise large ones (8 sequences and 8 heads of 4000 places: 29 us against 38), and a cluster of them
  // per head where SMs are left over and places many (16384 places: 18.5 us against 25.7 for the selection).
  int cluster = 1;
  while (cluster < 8 && rows * cluster * 2 <= 148 && capacity / (cluster * 2) >= 4096) cluster *= 2;
  status = rows > 148 && capacity <= 4096 ? tgb::launch_select<256>(a, rows, capacity, 1, stream)
                                          : tgb::launch_select<1024>(a, rows, capacity, cluster, stream);
  if (status) return status;
  // rows that can move at most, dealt to enough blocks to fill the machine
  const int64_t most = in_place ? (list < capacity - list ? list : capacity - list) : list;
  int64_t parts = tgb::ceil_div(148 * 8, rows);
  const int64_t enough = tgb::ceil_div(most > 0 ? most : 1, tgb::kMoveWarps * tgb::kMoveRows);
  parts = parts < enough ? parts : enough;
  TGB_CUDA(tgb::launch_dependent(tgb::k_evict_move, dim3((unsigned)rows, (unsigned)parts), dim3(tgb::kMoveWarps * 32), 0,
                                 stream, a));
  return TGB_STATUS_OK;
}

}  // extern "C"
