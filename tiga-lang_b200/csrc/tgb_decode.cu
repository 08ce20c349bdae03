// Attention of one query token per sequence over a paged cache of keys and
// values: out[b, h] = sum_t p[t] value[t], p = softmax_t(scale * q . key[t]).
//
// Bandwidth bound: every key and value row is read once, 4 * group flops per
// 2-byte value (16 sequences of 65536 places, 8 heads of 128: 590 us, 7.3 TB/s; 64
// ragged ones up to 8192: 121 us, 6.5 TB/s).  Keys stand on the 16-row side of mma.m16n8k16 and the queries
// that share them on the 8-column side (S^T = K Q^T, O^T = V^T P^T), so up to 8
// query heads cost one pass of the matrix pipe without padding; tensor memory and
// tcgen05 would pad the queries to 64 rows or more and buy nothing, the pipe is
// idle most of the time here.
//
// The places of all sequences form one list of units of 64 places, cut into equal
// runs; a run is taken by as many blocks as there are heads, next to each other, so
// that the heads of a row are read at about the same time (a head's part of a row is
// 128 to 512 bytes, and memory is fetched by more than that). A ragged batch is as
// balanced as an even one and a single long sequence fills the machine. A block that
// does not hold the whole of a sequence writes its maximum, denominator and
// numerator; a second kernel joins them in the order of the runs. The cut is
// computed on the device from `lengths`, which the host need not know.  Caches so
// small that launches are what they cost take a cluster of blocks per (sequence,
// head) instead, and one launch.
//
// Each warp streams its own 16 places of a unit through a ring of cp.async
// stages, with no block-wide barrier until its run leaves a sequence;
// the ring reads on into the next one. Softmax state is float32. A softmax
// weight enters the second product as the sum of two 16-bit values (its upper part
// and what that left), because rounding it once costs as much as the output's own
// rounding does; the extra product is free next to the loads. The sum has 15 bits
// of a bf16 cache's weight and 21 of an fp16 cache's, where float32 has 24: a bf16 output
// of a plain float32 evaluation may round the other way now and then.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tgb_cache.cuh"

namespace tgb {
namespace {

constexpr int kTile = 16;                   // places a warp takes at a time
constexpr int kQueries = 8;                 // columns of one matrix product
constexpr float kLog2e = 1.4426950408889634f;

struct DecodeArgs {
  tgb_paged_cache cache;
  const void *query;
  int64_t query_token_stride, query_head_stride;
  void *out;
  int32_t q_heads, group, head_tiles;       // queries per key head, and tiles of NT * 8 of them
  int32_t accumulate;
  float scale;                              // times log2(e)
  uint32_t page_factor, page_shift;         // t / page_size = t * page_factor >> page_shift for t < 2^30
  // scratch
  int64_t *first_unit;                      // accumulate: [sequences + 1]
  int4 *cuts;                               // [blocks]: the sequence that a block's run begins inside of (-1: none),
                                            // and its first and last run
  float2 *part_state;                       // [2 * blocks][NT * 8] (maximum, denominator)
  float *part_sum;                          // [2 * blocks][NT * 8][dim]
  float2 *state;                            // accumulate: [sequences, q_heads] of pieces that were whole
  float *scores;                            // accumulate: [sequences, q_heads, capacity], log2 domain
  int32_t blocks, runs;                     // runs of the unit list, and their blocks: one per head tile
};

__device__ __forceinline__ uint32_t shared_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void copy16(uint32_t to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy16_or_zeros(uint32_t to, const void *from, bool valid) {
  const int bytes = valid ? 16 : 0;         // 0: nothing is read, the 16 bytes are filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ uint32_t transpose_matrix(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <typename T> struct Matrix;
template <> struct Matrix<__nv_bfloat16> {
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  // (a, b) cut down to 16 bits, and in a, b what that left. Both parts of a weight are positive wherever the weight is, so
  // that an infinite value keeps its sign in both products and meets a 0 in neither; a weight of 0 (a score of -inf, or one
  // further below the maximum than float32 reaches) is 0 in both
  static __device__ __forceinline__ uint32_t split(float &a, float &b) {
    constexpr float kTiny = 1.1754944e-38f;
    const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
    a = a == 0.f ? 0.f : fmaxf(a - __uint_as_float(x & 0xffff0000u), kTiny);
    b = b == 0.f ? 0.f : fmaxf(b - __uint_as_float(y & 0xffff0000u), kTiny);
    return __byte_perm(x, y, 0x7632);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  // softmax weights are held times 2^-24 (denominator and numerator alike): the numerator of as many places of the largest
  // bf16 value is still finite, and a weight down to 2^-102 of the largest one still a normal number
  static constexpr float kLift = -24.f;
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Matrix<__half> {
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t split(float &a, float &b) {
    // 2^-24, the smallest fp16, next to weights of up to 2^15: a weight below 2^-39 of the largest is held as 2^-38 of it,
    // and what is left of any other as 2^-39 at least. n places are off by n * 2^-38 of the largest value at most
    constexpr float kTiny = 5.9604645e-8f;
    uint32_t bits;
    asm("cvt.rz.f16x2.f32 %0, %2, %1;" : "=r"(bits) : "f"(a), "f"(b));
    bits = __vmaxu2(bits, (a > 0.f ? 1u : 0u) | (b > 0.f ? 0x10000u : 0u));
    const __half2 v = *reinterpret_cast<const __half2 *>(&bits);
    a = a == 0.f ? 0.f : fmaxf(a - __low2float(v), kTiny);
    b = b == 0.f ? 0.f : fmaxf(b - __high2float(v), kTiny);
    return bits;
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  // softmax weights are held times 2^15 (denominator and numerator alike): the largest is then 2^15 and
  // one 2^-29 times smaller still a normal number
  static constexpr float kLift = 15.f;
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// the maximum to subtract: a row whose scores are all -inf keeps weights of 0
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// a sequence without places, or with scores of -inf alone, has a denominator of 0 and a result of 0
__device__ __forceinline__ float over(float sum, float denominator) { return denominator == 0.f ? 0.f : sum / denominator; }

// How the kernel for heads of up to D values is laid out on an SM. A warp's time per tile is a chain of some 370
// dependent instructions, so what counts is warps per SM: two stages of many warps beat three of few (a ragged batch
// of 64 sequences, 8 heads of 128: 132 us at 8 warps, 127 at 12; 16 queries on heads of 256: 338 at 4, 213 at 6).
template <int D, int NT> struct Layout {
  static constexpr int kWarps = D <= 192 ? 4 : 3;
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr int kBlocks = D <= 96 ? (NT == 1 ? 4 : 3) : D == 128 ? (NT == 1 ? 3 : 2) : 2;    // resident on an SM
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kUnit = kWarps * kTile;                  // places of a unit of work
  static constexpr int kRing = kWarps * kStages * kTile * D * 2 * 2;
  static constexpr int kHalf = D / 2;                           // columns that are joined at a time
  static constexpr int kShared = kRing + kWarps * kQueries * (kHalf + 2) * 4;
  static_assert(kBlocks * (kShared + 256 + 24 * kQueries * NT + 1024) <= 228 * 1024, "the blocks of a round are resident together");
  // 16-byte pieces of a row are permuted so that the same piece of 8 rows in a row lies in 8 different bank groups: by
  // the row's low bits where a row is a multiple of 128 bytes, by higher ones where rows shift each other
  static constexpr int kMask = D * 2 % 128 == 0 ? 7 : D * 2 % 64 == 0 ? 3 : 1;
  static constexpr int kShift = kMask == 7 ? 0 : kMask == 3 ? 1 : 2;
  static __host__ __device__ constexpr int permute(int row) { return row >> kShift & kMask; }
};

__host__ __device__ __forceinline__ int units_of(int length, int unit) { return (length + unit - 1) / unit; }

// runs of the unit list: block c of n takes [start(c), start(c + 1))
__device__ __forceinline__ int64_t run_start(int64_t units, int64_t c, int64_t n) { return units * c / n; }
__device__ __forceinline__ int64_t run_of(int64_t units, int64_t u, int64_t n) {
  const int64_t top = (u + 1) * n - 1;
  return ((uint64_t)(top | units) >> 32) == 0 ? (int64_t)((uint32_t)top / (uint32_t)units) : top / units;
}

// where in the list a warp stands
template <int UNIT> struct Cursor {
  int b, unit, units, length;               // sequence, unit of it, its units, its places
  __device__ __forceinline__ void next(const tgb_paged_cache &cache) {
    if (++unit < units) return;
    unit = 0;
    do {                                    // sequences without places have no units
      if (++b >= cache.sequences) {
        length = 0;
        return;
      }
      length = cache_length(cache, b);
      units = units_of(length, UNIT);
    } while (!units);
  }
};

// CLUSTER: a cluster of blocks has one (sequence, head tile), an equal run of units each, and joins its pieces through
// distributed shared memory: one launch and no scratch, for caches so small that launches are what they cost.
template <typename T, int D, int NT, bool CLUSTER>
__global__ void __launch_bounds__(Layout<D, NT>::kThreads, Layout<D, NT>::kBlocks)
k_decode(const __grid_constant__ DecodeArgs a) {
  using L = Layout<D, NT>;
  constexpr int kWarps = L::kWarps, kThreads = L::kThreads, kUnit = L::kUnit, STAGES = L::kStages;
  constexpr int kRowBytes = D * 2;
  constexpr int kTileBytes = kTile * kRowBytes;
  constexpr int kChunks = D / 8;            // 16-byte pieces of a row
  extern __shared__ __align__(128) unsigned char shared[];
  __shared__ int64_t scan[kWarps];
  __shared__ int64_t place_in_list[2];
  __shared__ float2 warp_state[kWarps][NT * kQueries];
  __shared__ float2 block_state[CLUSTER ? NT * kQueries : 1];
  float *block_sum = reinterpret_cast<float *>(shared);      // CLUSTER: over the ring, once it is empty
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const tgb_paged_cache &cache = a.cache;
  const int heads = cache.heads * a.head_tiles;
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  int64_t total_units = 0;
  // every run of the unit list is taken by `heads` blocks that follow each other, one per head tile
  const int hg = (CLUSTER ? blockIdx.x / cluster.num_blocks() : blockIdx.x) % heads, run = blockIdx.x / heads;
  const int hk = a.head_tiles == 1 ? hg : hg / a.head_tiles;
  const int first_query = (hg - hk * a.head_tiles) * NT * kQueries;            // of the key head's group
  wait_for_previous();
  int64_t begin, end;                       // this block's run (CLUSTER: of its sequence's units)
  if constexpr (CLUSTER) {
    const int b = blockIdx.x / cluster.num_blocks() / heads;
    const int units = units_of(cache_length(cache, b), kUnit);
    begin = run_start(units, cluster.block_rank(), cluster.num_blocks());
    end = run_start(units, cluster.block_rank() + 1, cluster.num_blocks());
    if (threadIdx.x == 0) place_in_list[0] = b, place_in_list[1] = begin;
  } else {
    // ---- the unit list: prefix sums over the sequences, and this block's run
    const int per = (cache.sequences + kThreads - 1) / kThreads;
    const int mine = min(threadIdx.x * per, cache.sequences), mine_end = min(mine + per, cache.sequences);
    int64_t sum = 0;
    for (int b = mine; b < mine_end; ++b) sum += units_of(cache_length(cache, b), kUnit);
    int64_t before = sum;
#pragma unroll
    for (int step = 1; step < 32; step <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, before, step);
      if (lane >= step) before += v;
    }
    if (lane == 31) scan[warp] = before;
    __syncthreads();
    int64_t total = 0;
    before -= sum;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    total_units = total;
    if (a.accumulate && blockIdx.x == 0) {
      int64_t at = before;
      for (int b = mine; b < mine_end; ++b) {
        a.first_unit[b] = at;
        at += units_of(cache_length(cache, b), kUnit);
      }
      if (threadIdx.x == 0) a.first_unit[cache.sequences] = total;
    }
    // sequences without places have no units: their rows are zeros
    for (int b = blockIdx.x; b < cache.sequences; b += gridDim.x)
      if (cache_length(cache, b) == 0)
        for (int i = threadIdx.x; i < a.q_heads * cache.dim; i += kThreads)
          static_cast<T *>(a.out)[(int64_t)b * a.q_heads * cache.dim + i] = Matrix<T>::from(0.f);
    const int64_t runs = min((int64_t)a.runs, total);
    if (threadIdx.x == 0) a.cuts[blockIdx.x].x = -1;
    if (run >= runs) return;
    begin = run_start(total, run, runs), end = run_start(total, run + 1, runs);
    if (begin >= before && begin < before + sum) {
      int64_t at = before;
      for (int b = mine; b < mine_end; ++b) {
        const int64_t n = units_of(cache_length(cache, b), kUnit);
        if (begin < at + n) {
          place_in_list[0] = b, place_in_list[1] = begin - at;
          break;
        }
        at += n;
      }
    }
  }
  const uint32_t ring = shared_address(shared) + warp * STAGES * 2 * kTileBytes;
  const int row_chunks = cache.dim / 8;
  if (row_chunks < kChunks)                 // columns that no copy fills
    for (int i = lane; i < STAGES * 2 * kTileBytes / 16; i += 32)
      *reinterpret_cast<uint4 *>(shared + warp * STAGES * 2 * kTileBytes + i * 16) = make_uint4(0, 0, 0, 0);
  __syncthreads();

  Cursor<kUnit> ahead;
  ahead.b = (int)place_in_list[0];
  ahead.length = cache_length(cache, ahead.b);
  ahead.units = units_of(ahead.length, kUnit);
  ahead.unit = (int)place_in_list[1];
  Cursor<kUnit> now = ahead;
  int64_t left_ahead = end - begin;
  if constexpr (!CLUSTER) {
    if (threadIdx.x == 0 && now.unit > 0) {
      const int64_t runs = min((int64_t)a.runs, total_units);
      a.cuts[blockIdx.x] = make_int4(now.b, (int)run_of(total_units, begin - now.unit, runs),
                                     (int)run_of(total_units, begin - now.unit + now.units - 1, runs), 0);
    }
  }

  // ---- the producer. A lane copies 16-byte piece lane % kChunks of rows lane / kChunks, + kRowsAtOnce, ...; kRowsAtOnce
  // is a power of two, so that the permutation of row i * kRowsAtOnce + lane / kChunks is an exclusive or of both parts'
  constexpr int kRowsAtOnce = kChunks <= 8 ? 4 : kChunks <= 16 ? 2 : 1;
  constexpr int kCopies = kTile / kRowsAtOnce;
  static_assert(kRowsAtOnce * kChunks <= 32, "a warp copies whole rows");
  const int my_row = lane / kChunks, my_chunk = lane % kChunks;
  const uint32_t my_slot = my_row * kRowBytes + ((my_chunk ^ L::permute(my_row)) * 16);
  const bool copies = my_chunk < row_chunks && my_row < kRowsAtOnce;
  const uint32_t key_stride = (uint32_t)cache.key_slot_stride * 2, value_stride = (uint32_t)cache.value_slot_stride * 2;
  const unsigned char *key = static_cast<const unsigned char *>(cache.key) + 2 * (hk * cache.key_head_stride + my_chunk * 8);
  const unsigned char *value = static_cast<const unsigned char *>(cache.value) + 2 * (hk * cache.value_head_stride + my_chunk * 8);
  int row_ahead = -1;                       // of this lane's place (lane % 16) of the unit to be fetched next
  auto look_up = [&]() {
    const int place = ahead.unit * kUnit + warp * kTile + lane % kTile;
    row_ahead = -1;
    if (place < ahead.length && left_ahead > 0) {
      const uint32_t page_at = (uint32_t)(((uint64_t)(uint32_t)place * a.page_factor) >> a.page_shift);
      const int page = cache.page_table[(int64_t)ahead.b * cache.pages_per_sequence + page_at];
      if ((uint32_t)page < (uint32_t)cache.num_pages)
        row_ahead = page * cache.page_size + (place - (int)page_at * cache.page_size);
      else
        cache_fault(cache, TGB_CACHE_BAD_PAGE);
    }
  };
  look_up();

  // issues the copies of the unit `ahead` into a stage and steps on
  auto fetch = [&](int stage) {
    if (left_ahead > 0) {
      const uint32_t to = ring + stage * 2 * kTileBytes + my_slot;
      if (__all_sync(0xffffffffu, row_ahead >= 0)) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const uint32_t row = __shfl_sync(0xffffffffu, row_ahead, i * kRowsAtOnce + my_row & 15);
          const uint32_t at = (to ^ (L::permute(i * kRowsAtOnce) * 16)) + i * kRowsAtOnce * kRowBytes;
          if (copies) {
            copy16(at, key + (uint64_t)row * key_stride);
            copy16(at + kTileBytes, value + (uint64_t)row * value_stride);
          }
        }
      } else {                              // the last unit of a sequence (or a page that does not exist)
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int row = __shfl_sync(0xffffffffu, row_ahead, i * kRowsAtOnce + my_row & 15);
          const uint32_t at = (to ^ (L::permute(i * kRowsAtOnce) * 16)) + i * kRowsAtOnce * kRowBytes;
          const uint64_t from = row < 0 ? 0 : row;
          if (copies) {
            copy16_or_zeros(at, key + from * key_stride, row >= 0);
            copy16_or_zeros(at + kTileBytes, value + from * value_stride, row >= 0);
          }
        }
      }
      ahead.next(cache);
      --left_ahead;
      look_up();
    }
    commit_copies();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch(s);

  // where a lane's ldmatrix rows begin: 16 keys by 8 values, and 8 places by 8 values of both halves
  const uint32_t key_lane = (lane % 16) * kRowBytes + ((lane / 16 ^ L::permute(lane % 16)) * 16);
  const int value_row = (lane / 16) * 8 + lane % 8;
  const uint32_t value_lane = value_row * kRowBytes + (((lane / 8 & 1) ^ L::permute(value_row)) * 16);
  uint32_t query[NT][D / 16][2];
  float *scores[NT];                        // accumulate: of the first of the lane's two queries at place lane / 4
  float m[NT][2], l[NT][2], o[NT][D / 16][4];
  int piece = now.unit;                     // first unit of the running piece
  bool fresh = true;
  int stage = 0;
  for (int64_t u = begin; u < end; ++u) {
    if (fresh) {
      fresh = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int g = first_query + t * kQueries + lane / 4;
        const T *q = static_cast<const T *>(a.query) + now.b * a.query_token_stride +
                     (int64_t)(hk * a.group + g) * a.query_head_stride;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int d = k * 16 + j * 8 + (lane % 4) * 2;
            query[t][k][j] = g < a.group && d < cache.dim ? *reinterpret_cast<const uint32_t *>(q + d) : 0u;
          }
        if (a.accumulate)
          scores[t] = a.scores + ((int64_t)now.b * a.q_heads + hk * a.group + first_query + t * kQueries + (lane % 4) * 2) *
                                     cache_capacity(cache) + lane / 4;
        m[t][0] = m[t][1] = -INFINITY;
        l[t][0] = l[t][1] = 0.f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[t][k][j] = 0.f;
      }
    }
    wait_copies<STAGES - 2>();
    __syncwarp();                           // everyone's copies have landed, and everyone is done with the oldest stage
    fetch(stage == 0 ? STAGES - 1 : stage - 1);
    const int place = now.unit * kUnit + warp * kTile;
    if (place < now.length) {
      const uint32_t keys = ring + stage * 2 * kTileBytes, values = keys + kTileBytes;
      float s[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
      {
        const uint32_t mine = keys + key_lane;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          uint32_t f[4];
          load_matrices(f, (mine ^ ((2 * k & L::kMask) * 16)) + (2 * k & ~L::kMask) * 16);
#pragma unroll
          for (int t = 0; t < NT; ++t) Matrix<T>::mma(s[t], f, query[t][k][0], query[t][k][1]);
        }
      }
      const bool whole_tile = place + kTile <= now.length;
      uint32_t high[NT][2], low[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = s[t][j] * a.scale;
        if (!whole_tile) {
          if (place + lane / 4 >= now.length) p[0] = p[1] = -INFINITY;
          if (place + 8 + lane / 4 >= now.length) p[2] = p[3] = -INFINITY;
        }
        if (a.accumulate) {
          const int g = first_query + t * kQueries + (lane % 4) * 2;
          float *to = scores[t] + place;
          if (g < a.group) {
            if (place + lane / 4 < now.length) to[0] = p[0];
            if (place + 8 + lane / 4 < now.length) to[8] = p[2];
          }
          if (g + 1 < a.group) {
            to += cache_capacity(cache);
            if (place + lane / 4 < now.length) to[0] = p[1];
            if (place + 8 + lane / 4 < now.length) to[8] = p[3];
          }
        }
        float shrink[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = fmaxf(p[j], p[j + 2]);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          top = fmaxf(top, m[t][j]);
          shrink[j] = exp2_of(m[t][j] - base_of(top));
          m[t][j] = top;
          const float lifted = base_of(top) - Matrix<T>::kLift;
          p[j] = exp2_of(p[j] - lifted);
          p[j + 2] = exp2_of(p[j + 2] - lifted);
          l[t][j] = l[t][j] * shrink[j] + (p[j] + p[j + 2]);
        }
        if (__any_sync(0xffffffffu, shrink[0] != 1.f || shrink[1] != 1.f)) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[t][k][j] *= shrink[j & 1];
        }
        high[t][0] = transpose_matrix(Matrix<T>::split(p[0], p[1]));
        high[t][1] = transpose_matrix(Matrix<T>::split(p[2], p[3]));
        low[t][0] = transpose_matrix(Matrix<T>::pack(p[0], p[1]));
        low[t][1] = transpose_matrix(Matrix<T>::pack(p[2], p[3]));
      }
      {
        const uint32_t mine = values + value_lane;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          uint32_t f[4];
          load_matrices_transposed(f, (mine ^ ((2 * k & L::kMask) * 16)) + (2 * k & ~L::kMask) * 16);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            Matrix<T>::mma(o[t][k], f, high[t][0], high[t][1]);
            Matrix<T>::mma(o[t][k], f, low[t][0], low[t][1]);
          }
        }
      }
    }
    stage = stage == STAGES - 1 ? 0 : stage + 1;

    if (now.unit + 1 == now.units || u + 1 == end) {
      // ---- the piece ends: join the four warps, then write the result or a partial one
      const bool whole = piece == 0 && now.unit + 1 == now.units;
      const int64_t slot = 2 * (int64_t)blockIdx.x + (piece == 0 ? 1 : 0);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float v = l[t][j];
          v += __shfl_xor_sync(0xffffffffu, v, 4);
          v += __shfl_xor_sync(0xffffffffu, v, 8);
          v += __shfl_xor_sync(0xffffffffu, v, 16);
          if (lane < 4) warp_state[warp][t * kQueries + lane * 2 + j] = make_float2(m[t][j], v);
        }
      __syncthreads();
      float *sums = reinterpret_cast<float *>(shared + L::kRing);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float factor[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int g = t * kQueries + (lane % 4) * 2 + j;
          float top = warp_state[0][g].x;
#pragma unroll
          for (int w = 1; w < kWarps; ++w) top = fmaxf(top, warp_state[w][g].x);
          factor[j] = exp2_of(m[t][j] - base_of(top));
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (t || half) __syncthreads();
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int column = k * 16 + (j < 2 ? 0 : 8);      // of lanes 0 to 3
              if (column / L::kHalf == half)
                sums[(warp * kQueries + (lane % 4) * 2 + (j & 1)) * (L::kHalf + 2) + column - half * L::kHalf + lane / 4] =
                    o[t][k][j] * factor[j & 1];
            }
          __syncthreads();
          for (int i = threadIdx.x; i < kQueries * (L::kHalf / 2); i += kThreads) {
            const int g = i / (L::kHalf / 2), column = i % (L::kHalf / 2) * 2, d = half * L::kHalf + column, gt = t * kQueries + g;
            if (first_query + gt >= a.group || d >= cache.dim) continue;
            float top = warp_state[0][gt].x, total_l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
            for (int w = 1; w < kWarps; ++w) top = fmaxf(top, warp_state[w][gt].x);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
              total_l += warp_state[w][gt].y * exp2_of(warp_state[w][gt].x - base_of(top));
              const float2 v = *reinterpret_cast<const float2 *>(&sums[(w * kQueries + g) * (L::kHalf + 2) + column]);
              x += v.x, y += v.y;
            }
            if constexpr (CLUSTER) {
              *reinterpret_cast<float2 *>(block_sum + gt * D + d) = make_float2(x, y);
              if (d == 0) block_state[gt] = make_float2(top, total_l);
            } else if (whole) {
              const int64_t head = (int64_t)now.b * a.q_heads + hk * a.group + first_query + gt;
              T *out = static_cast<T *>(a.out) + head * cache.dim + d;
              out[0] = Matrix<T>::from(over(x, total_l)), out[1] = Matrix<T>::from(over(y, total_l));
              if (a.accumulate && d == 0) a.state[head] = make_float2(top, total_l);
            } else {
              const int64_t at = slot * NT * kQueries + gt;
              *reinterpret_cast<float2 *>(a.part_sum + at * cache.dim + d) = make_float2(x, y);
              if (d == 0) a.part_state[at] = make_float2(top, total_l);
            }
          }
        }
      }
      __syncthreads();                      // warp_state and sums are free again
      fresh = true;
      piece = now.unit + 1 == now.units ? 0 : now.unit + 1;
    }
    now.next(cache);
  }
  wait_copies<0>();
  if constexpr (CLUSTER) {
    if (begin == end) {                     // no units: nothing to add
      for (int i = threadIdx.x; i < NT * kQueries * D; i += kThreads) block_sum[i] = 0.f;
      if (threadIdx.x < NT * kQueries) block_state[threadIdx.x] = make_float2(-INFINITY, 0.f);
    }
    cluster.sync();
    const int blocks = cluster.num_blocks(), b = blockIdx.x / blocks / heads;
    for (int i = cluster.block_rank() * kThreads + threadIdx.x; i < NT * kQueries * (D / 2); i += blocks * kThreads) {
      const int g = i / (D / 2), d = i % (D / 2) * 2;
      if (first_query + g >= a.group || d >= cache.dim) continue;
      float top = -INFINITY, sum = 0.f, x = 0.f, y = 0.f;
      for (int r = 0; r < blocks; ++r) top = fmaxf(top, cluster.map_shared_rank(block_state, r)[g].x);
      for (int r = 0; r < blocks; ++r) {
        const float2 state = cluster.map_shared_rank(block_state, r)[g];
        const float2 v = *reinterpret_cast<const float2 *>(cluster.map_shared_rank(block_sum, r) + g * D + d);
        const float f = exp2_of(state.x - base_of(top));
        sum = fmaf(f, state.y, sum), x = fmaf(f, v.x, x), y = fmaf(f, v.y, y);
      }
      T *out = static_cast<T *>(a.out) + ((int64_t)b * a.q_heads + hk * a.group + first_query + g) * cache.dim + d;
      out[0] = Matrix<T>::from(over(x, sum)), out[1] = Matrix<T>::from(over(y, sum));
    }
    cluster.sync();                         // nobody leaves while its shared memory is read
  }
}

// The pieces of a head tile `hg` and a sequence that runs first .. last left: a piece begins with its run, except
// the first one, which begins with the sequence.
struct Pieces {
  int heads, hg, first, last;
  template <int ALL> __device__ __forceinline__ int64_t at(int c) const {
    return (2 * ((int64_t)c * heads + hg) + (c == first)) * ALL;
  }
};

// The maximum and denominator of `n` queries: a warp each, a lane per piece.
template <int ALL, int THREADS>
__device__ __forceinline__ void join_states(const DecodeArgs &a, const Pieces &p, int n, float2 *joined) {
  const int lane = threadIdx.x % 32;
  for (int g = threadIdx.x / 32; g < n; g += THREADS / 32) {
    float top = -INFINITY, sum = 0.f;
    for (int c = p.first + lane; c <= p.last; c += 32) top = fmaxf(top, a.part_state[p.at<ALL>(c) + g].x);
#pragma unroll
    for (int step = 16; step; step >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, step));
    for (int c = p.first + lane; c <= p.last; c += 32) {
      const float2 s = a.part_state[p.at<ALL>(c) + g];
      sum += s.y * exp2_of(s.x - base_of(top));
    }
#pragma unroll
    for (int step = 16; step; step >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, step);
    if (lane == 0) joined[g] = make_float2(top, sum);
  }
  __syncthreads();
}

struct Joined {                             // two values of a query, with their maximum and denominator
  float top, sum, x, y;
  __device__ __forceinline__ void add(float2 state, float2 v) {
    const float larger = fmaxf(top, state.x), keep = exp2_of(top - base_of(larger)), f = exp2_of(state.x - base_of(larger));
    sum = fmaf(sum, keep, f * state.y), x = fmaf(x, keep, f * v.x), y = fmaf(y, keep, f * v.y);
    top = larger;
  }
};

// Share `part` of `parts` of the pairs of values of a tile's `n` queries. Where a share has fewer pairs than the block
// has threads, the pieces of a pair are dealt to several threads: a single sequence is cut into as many
// pieces as there are runs.
template <typename T, int ALL, int THREADS>
__device__ __forceinline__ void join_values(const DecodeArgs &a, const Pieces &p, int n, int part, int parts, T *out) {
  __shared__ Joined shares[THREADS];
  const int dim = a.cache.dim, all = n * (dim / 2), pieces = p.last - p.first + 1;
  const int begin = (int)((int64_t)all * part / parts), pairs = (int)((int64_t)all * (part + 1) / parts) - begin;
  if (!pairs) return;
  int splits = THREADS / pairs;
  splits = splits < 1 ? 1 : splits > pieces ? pieces : splits;
  const int split = splits > 1 ? threadIdx.x / pairs : 0;
  for (int i = splits > 1 ? threadIdx.x % pairs : threadIdx.x; i < pairs; i += splits > 1 ? pairs : THREADS) {
    const int g = (begin + i) / (dim / 2), d = (begin + i) % (dim / 2) * 2;
    Joined j = {-INFINITY, 0.f, 0.f, 0.f};
    if (split < splits) {
#pragma unroll 4
      for (int c = p.first + split; c <= p.last; c += splits) {
        const int64_t at = p.at<ALL>(c) + g;
        j.add(a.part_state[at], *reinterpret_cast<const float2 *>(a.part_sum + at * dim + d));
      }
    }
    if (splits > 1) {
      shares[threadIdx.x] = j;
      __syncthreads();
      if (split) break;
      for (int s = 1; s < splits; ++s) {
        const Joined &o = shares[s * pairs + i];
        j.add(make_float2(o.top, o.sum), make_float2(o.x, o.y));
      }
    }
    T *to = out + (int64_t)g * dim + d;
    to[0] = Matrix<T>::from(over(j.x, j.sum)), to[1] = Matrix<T>::from(over(j.y, j.sum));
  }
}

constexpr int kJoinThreads = 256, kWeightThreads = 128;

// The blocks whose runs begin inside of a sequence share the joining of its pieces.
template <typename T, int NT>
__global__ void __launch_bounds__(kJoinThreads) k_decode_join(const __grid_constant__ DecodeArgs a) {
  constexpr int kAll = NT * kQueries;
  const int heads = a.cache.heads * a.head_tiles, run = blockIdx.x / heads, hg = blockIdx.x - run * heads;
  const int hk = hg / a.head_tiles, first_query = (hg - hk * a.head_tiles) * kAll;
  const int queries = min(kAll, a.group - first_query);
  wait_for_previous();
  const int4 cut = a.cuts[blockIdx.x];
  if (cut.x < 0) return;
  const int64_t head = (int64_t)cut.x * a.q_heads + hk * a.group + first_query;
  join_values<T, kAll, kJoinThreads>(a, Pieces{heads, hg, cut.y, cut.z}, queries, run - cut.y - 1, cut.z - cut.y,
                                     static_cast<T *>(a.out) + head * a.cache.dim);
}

// The same for every (sequence, head tile) of a tracking call, and the softmax weights: block (x, y) adds those of
// places [y, y + 1) * span. The first tile of a key head adds the weights of all its queries, tile after tile: the same
// thread has a place each time, so the sum's order is fixed.
template <typename T, int NT>
__global__ void __launch_bounds__(kWeightThreads) k_decode_weights(const __grid_constant__ DecodeArgs a, int span) {
  constexpr int kAll = NT * kQueries;
  __shared__ float2 joined[kAll];
  const tgb_paged_cache &cache = a.cache;
  const int heads = cache.heads * a.head_tiles;
  const int b = blockIdx.x / heads, hg = blockIdx.x % heads;
  const int hk = hg / a.head_tiles, first_query = (hg - hk * a.head_tiles) * kAll;
  const int queries = min(kAll, a.group - first_query);
  const int64_t head0 = (int64_t)b * a.q_heads + hk * a.group + first_query;
  wait_for_previous();
  const int64_t total = a.first_unit[cache.sequences];
  const int64_t begin = a.first_unit[b], units = a.first_unit[b + 1] - begin;
  if (!units) return;
  const int64_t runs = min((int64_t)a.runs, total);
  const int c0 = (int)run_of(total, begin, runs), c1 = (int)run_of(total, begin + units - 1, runs);
  if (c0 != c1)
    join_values<T, kAll, kWeightThreads>(a, Pieces{heads, hg, c0, c1}, queries, blockIdx.y, gridDim.y,
                                         static_cast<T *>(a.out) + head0 * cache.dim);
  if (first_query) return;
  const int capacity = cache_capacity(cache), from = blockIdx.y * span + threadIdx.x;
  const int stop = min(cache_length(cache, b), (int)min((int64_t)(blockIdx.y + 1) * span, (int64_t)capacity));
  float *weight = cache.weight + ((int64_t)b * cache.heads + hk) * capacity;
  for (int tile = 0; tile < a.head_tiles; ++tile) {
    const int64_t head = head0 + tile * kAll;
    const int n = min(kAll, a.group - tile * kAll);
    if (c0 != c1) {
      join_states<kAll, kWeightThreads>(a, Pieces{heads, hg + tile, c0, c1}, n, joined);
    } else {
      if (threadIdx.x < n) joined[threadIdx.x] = a.state[head + threadIdx.x];
      __syncthreads();
    }
    constexpr int kUnroll = 4;
    for (int t = from; t < stop; t += kUnroll * kWeightThreads) {
      float sum[kUnroll] = {}, old[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) old[i] = t + i * kWeightThreads < stop ? weight[t + i * kWeightThreads] : 0.f;
      for (int g = 0; g < n; ++g) {
        const float top = base_of(joined[g].x) - Matrix<T>::kLift, share = over(1.f, joined[g].y);
        const float *score = a.scores + (head + g) * capacity + t;
        float s[kUnroll];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) s[i] = t + i * kWeightThreads < stop ? score[i * kWeightThreads] : 0.f;
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) sum[i] = fmaf(exp2_of(s[i] - top), share, sum[i]);
      }
#pragma unroll
      for (int i = 0; i < kUnroll; ++i)
        if (t + i * kWeightThreads < stop) weight[t + i * kWeightThreads] = old[i] + sum[i];
    }
    __syncthreads();
  }
}

struct Shape {
  int width;        // columns the kernel is built for
  int tiles;        // of 8 queries in one pass
  int head_tiles;   // passes over a key head
  int runs, blocks; // of the unit list: a round of resident blocks where the heads allow it
  int cluster;      // blocks of a cluster per head tile; 0: the unit list
};

template <typename F> void with_layout(int width, int tiles, F f) {
  auto with = [&](auto one, auto two) { tiles == 1 ? f(one) : f(two); };
  if (width == 64) with(Layout<64, 1>{}, Layout<64, 2>{});
  else if (width == 80) with(Layout<80, 1>{}, Layout<80, 2>{});
  else if (width == 96) with(Layout<96, 1>{}, Layout<96, 2>{});
  else if (width == 128) with(Layout<128, 1>{}, Layout<128, 2>{});
  else if (width == 192) with(Layout<192, 1>{}, Layout<192, 2>{});
  else with(Layout<256, 1>{}, Layout<256, 2>{});
}

void shape_of(const tgb_paged_cache &c, int q_heads, bool accumulate, Shape &s) {
  const int group = q_heads / c.heads;
  s.width = c.dim <= 64 ? 64 : c.dim <= 80 ? 80 : c.dim <= 96 ? 96 : c.dim <= 128 ? 128 : c.dim <= 192 ? 192 : 256;
  s.tiles = group <= kQueries ? 1 : 2;
  s.head_tiles = (int)ceil_div(group, s.tiles * kQueries);
  constexpr int sms = 148;                  // of the only device this is built for; a block needs no other to run
  int resident = 0;
  with_layout(s.width, s.tiles, [&](auto layout) { resident = sms * decltype(layout)::kBlocks; });
  const int heads = c.heads * s.head_tiles;
  s.runs = resident / heads > 1 ? resident / heads : 1;
  s.blocks = s.runs * heads;
  // A cluster per head tile where all its blocks are resident at once and one of them reads at most 220 KB more than a
  // block of the unit list would: it ends before the list's second launch does (8 heads of 128, us with a cluster and
  // with the list: 1 sequence of 1000 places 6.2 and 8.0, of 2048 8.3 and 8.9, of 4096 12.3 and 11.3, of 8192 21.7 and
  // 13.6; 4 of 4096 17.1 and 19.0; 16 of 500 10.0 and 13.5, of 2000 27.0 and 29.0). Never more than 512 KB: lengths are
  // not known here, and the longest sequence alone decides when its cluster ends.
  s.cluster = 0;
  const int64_t tiles = (int64_t)c.sequences * heads;
  int64_t cluster = 8;
  while (cluster > 1 && tiles * cluster > resident) cluster /= 2;
  const int64_t bytes = (int64_t)c.pages_per_sequence * c.page_size * c.dim * 4;          // of a tile's keys and values
  if (!accumulate && tiles * cluster <= resident && bytes / cluster <= (512 << 10) &&
      bytes / cluster <= (220 << 10) + bytes * tiles / resident)
    s.cluster = (int)cluster;
}

struct Scratch {
  uint64_t first_unit, cuts, part_state, part_sum, state, scores, bytes;
};
Scratch scratch_of(const tgb_paged_cache &c, int q_heads, const Shape &s, bool accumulate) {
  Scratch r = {};
  if (s.cluster) return r;
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at = align_up(at + bytes, 256);
    return here;
  };
  const uint64_t pieces = 2ull * s.blocks * s.tiles * kQueries;
  r.first_unit = take(accumulate ? 8ull * (c.sequences + 1) : 0);
  r.cuts = take(16ull * s.blocks);
  r.part_state = take(8 * pieces);
  r.part_sum = take(4 * pieces * c.dim);
  r.state = take(accumulate ? 8ull * c.sequences * q_heads : 0);
  r.scores = take(accumulate ? 4ull * c.sequences * q_heads * c.pages_per_sequence * c.page_size : 0);
  r.bytes = at;
  return r;
}

template <typename T, int D, int NT>
int32_t launch_cluster(const DecodeArgs &a, int cluster, cudaStream_t stream) {
  using L = Layout<D, NT>;
  auto kernel = k_decode<T, D, NT, true>;
  static std::atomic<uint64_t> asked{0};
  TGB_CUDA(allow_shared(kernel, L::kShared, asked));
  TGB_CUDA(launch_clusters(kernel, cluster, dim3((unsigned)(a.cache.sequences * a.cache.heads * a.head_tiles * cluster)),
                           dim3(L::kThreads), L::kShared, stream, a));
  return TGB_STATUS_OK;
}

template <typename T, int D, int NT>
int32_t launch(const DecodeArgs &a, int cluster, cudaStream_t stream) {
  using L = Layout<D, NT>;
  if (cluster) return launch_cluster<T, D, NT>(a, cluster, stream);
  auto kernel = k_decode<T, D, NT, false>;
  static std::atomic<uint64_t> asked{0};
  TGB_CUDA(allow_shared(kernel, L::kShared, asked));
  TGB_CUDA(launch_dependent(kernel, dim3(a.blocks), dim3(L::kThreads), L::kShared, stream, a));
  if (!a.accumulate) {
    TGB_CUDA(launch_dependent(k_decode_join<T, NT>, dim3(a.blocks), dim3(kJoinThreads), 0, stream, a));
    return TGB_STATUS_OK;
  }
  // one round of resident blocks, at least 512 places each
  const tgb_paged_cache &c = a.cache;
  const int capacity = c.pages_per_sequence * c.page_size > 0 ? c.pages_per_sequence * c.page_size : 1;
  const int64_t tiles = (int64_t)c.sequences * c.heads * a.head_tiles, parts = 148 * 8 / tiles;
  int span = (int)ceil_div(capacity, parts > 0 ? parts : 1);
  span = span < 512 ? 512 : span;
  TGB_CUDA(launch_dependent(k_decode_weights<T, NT>, dim3((unsigned)tiles, (unsigned)ceil_div(capacity, span)),
                            dim3(kWeightThreads), 0, stream, a, span));
  return TGB_STATUS_OK;
}

template <typename T, int D> int32_t launch_tiles(const DecodeArgs &a, const Shape &s, cudaStream_t stream) {
  return s.tiles == 1 ? launch<T, D, 1>(a, s.cluster, stream) : launch<T, D, 2>(a, s.cluster, stream);
}

template <typename T> int32_t dispatch(const DecodeArgs &a, const Shape &s, cudaStream_t stream) {
  switch (s.width) {
    case 64: return launch_tiles<T, 64>(a, s, stream);
    case 80: return launch_tiles<T, 80>(a, s, stream);
    case 96: return launch_tiles<T, 96>(a, s, stream);
    case 128: return launch_tiles<T, 128>(a, s, stream);
    case 192: return launch_tiles<T, 192>(a, s, stream);
    default: return launch_tiles<T, 256>(a, s, stream);
  }
}

int32_t check_heads(const tgb_paged_cache *cache, int32_t q_heads, int32_t accumulate) {
  const int32_t status = check_cache(cache);
  if (status) return status;
  if (q_heads < 1 || q_heads % cache->heads)
    TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "%d query heads are no multiple of %d key heads", q_heads, cache->heads);
  if (q_heads > (1 << 16)) TGB_FAIL(TGB_STATUS_UNSUPPORTED, "at most 65536 query heads");
  if (accumulate && cache->sequences && !cache->seen) TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "the cache does not track attention weights");
  return TGB_STATUS_OK;
}

}  // namespace
}  // namespace tgb

extern "C" {

int32_t tgb_cache_attend_scratch_bytes(const tgb_paged_cache *cache, int32_t q_heads, int32_t accumulate, uint64_t *bytes) {
  if (!bytes) TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "null bytes");
  const int32_t status = tgb::check_heads(cache, q_heads, accumulate);
  if (status) return status;
  tgb::Shape shape;
  tgb::shape_of(*cache, q_heads, accumulate, shape);
  *bytes = tgb::scratch_of(*cache, q_heads, shape, accumulate).bytes;
  return TGB_STATUS_OK;
}

int32_t tgb_cache_attend(const tgb_paged_cache *cache, const void *query, int64_t query_token_stride,
                         int64_t query_head_stride, void *out, int32_t q_heads, float scale, int32_t accumulate,
                         void *scratch, uint64_t scratch_bytes, uint64_t stream) {
  const int32_t status = tgb::check_heads(cache, q_heads, accumulate);
  if (status) return status;
  tgb::Shape shape;
  tgb::shape_of(*cache, q_heads, accumulate, shape);
  if (!cache->sequences) return TGB_STATUS_OK;
  if (!query || !out) TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "null query or out");
  if (reinterpret_cast<uintptr_t>(query) % 4 || query_token_stride % 2 || query_head_stride % 2)
    TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "query heads must be 4-byte aligned");
  const tgb::Scratch r = tgb::scratch_of(*cache, q_heads, shape, accumulate);
  if (r.bytes && (!scratch || scratch_bytes < r.bytes || reinterpret_cast<uintptr_t>(scratch) % 256))
    TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "attention needs %llu bytes of 256-byte aligned scratch", (unsigned long long)r.bytes);
  if ((int64_t)cache->sequences * cache->heads * shape.head_tiles > 0x7fffffff)
    TGB_FAIL(TGB_STATUS_UNSUPPORTED, "too many sequences and heads");
  unsigned char *base = static_cast<unsigned char *>(scratch);
  tgb::DecodeArgs a;
  a.cache = *cache;
  a.query = query;
  a.query_token_stride = query_token_stride, a.query_head_stride = query_head_stride;
  a.out = out;
  a.q_heads = q_heads, a.group = q_heads / cache->heads, a.head_tiles = shape.head_tiles;
  a.accumulate = accumulate ? 1 : 0;
  a.scale = scale * tgb::kLog2e;
  a.first_unit = reinterpret_cast<int64_t *>(base + r.first_unit);
  a.cuts = reinterpret_cast<int4 *>(base + r.cuts);
  a.part_state = reinterpret_cast<float2 *>(base + r.part_state);
  a.part_sum = reinterpret_cast<float *>(base + r.part_sum);
  a.state = reinterpret_cast<float2 *>(base + r.state);
  a.scores = reinterpret_cast<float *>(base + r.scores);
  a.blocks = shape.blocks, a.runs = shape.runs;
  // with 2^log >= page_size: factor = 2^(30 + log) / page_size rounded up is below 2^31 + 1 and too large by less than
  // 2^log / 2^(30 + log), so t * factor stays below the next multiple for t < 2^30
  uint32_t log = 0;
  while ((1ll << log) < cache->page_size) ++log;
  a.page_shift = 30 + log;
  a.page_factor = (uint32_t)(((1ull << a.page_shift) + cache->page_size - 1) / cache->page_size);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return cache->dtype == TGB_DTYPE_BF16 ? tgb::dispatch<__nv_bfloat16>(a, shape, s) : tgb::dispatch<__half>(a, shape, s);
}

}  // extern "C"
