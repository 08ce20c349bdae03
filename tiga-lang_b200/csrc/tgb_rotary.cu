// Root-mean-square norm of every query and key head and the rotation of its
// pairs by the token's position, in one pass, with the gradients.
//
//   n = x * r * w,  r = 1 / sqrt(mean(x^2) + eps)           (per head, over D values)
//   angle[j] = sum_a position[a] * frequency[a, j]          (one or more axes)
//   y_a = n_a cos - n_b sin,  y_b = n_b cos + n_a sin       (pair j = (a, b))
//
// Every output value is r * (x * c1 + x' * c2) with x' the pair's other value,
// c1 = w cos, c2 = -+ w' sin: the coefficients are per token, so a head costs two
// multiply-adds a value next to its sum of squares.  Backward with dn = R^T dy:
//   dw = sum dn x r,   g = dn w,   dx = r (g - x r * mean(g x) * r).
//
// Bandwidth bound: one read and one write of every head (the backward reads two).
// 16384 tokens of 32 + 8 heads of 128 bf16: 59 to 62 us, 5.4 to 5.7 TB/s (a plain copy of
// as many bytes: 57 us); gradients of 8192 tokens of 16 + 16 heads: 46 us, 4.4 TB/s, bound by
// instruction issue.
// Angles are formed and reduced to [-pi, pi] in 64 bits (position * frequency
// reaches 10^5 and more, where float32 is off by 1/128), then sine and cosine are
// taken in 32 bits of an angle rounded to 32 bits (off by 2^-22 at most, next to output
// types of 2^-24, 2^-11 and 2^-8: enough but for float32, whose tests allow for it);
// a warp computes a token's table once and walks its heads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tgb_cache.cuh"

namespace tgb {
namespace {

constexpr int kWarps = 8;

// two float32 values that are worked on by one instruction
struct Two {
  unsigned long long bits;
};
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.bits) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split(Two v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v.bits));
  return r;
}
__device__ __forceinline__ Two mul(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
  return r;
}
__device__ __forceinline__ float sum(Two v) {
  const float2 f = split(v);
  return f.x + f.y;
}

// V values of T (4 or 8) as they lie in memory, two at a time as float32
template <typename T> __device__ __forceinline__ Two widen(uint32_t v);
template <> __device__ __forceinline__ Two widen<__nv_bfloat16>(uint32_t v) {
  return two(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <> __device__ __forceinline__ Two widen<__half>(uint32_t v) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&v));
  return two(f.x, f.y);
}
template <typename T> __device__ __forceinline__ uint32_t narrow(Two v);
template <> __device__ __forceinline__ uint32_t narrow<__nv_bfloat16>(Two v) {
  const float2 f = split(v);
  const __nv_bfloat162 r = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t *>(&r);
}
template <> __device__ __forceinline__ uint32_t narrow<__half>(Two v) {
  const float2 f = split(v);
  const __half2 r = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t *>(&r);
}

template <typename T, int V> struct alignas(V * sizeof(T)) Piece {
  uint32_t w[V / 2];
  __device__ __forceinline__ Two get(int i) const { return widen<T>(w[i]); }
  __device__ __forceinline__ void set(int i, Two v) { w[i] = narrow<T>(v); }
};
template <int V> struct alignas(16) Piece<float, V> {
  float w[V];
  __device__ __forceinline__ Two get(int i) const { return two(w[2 * i], w[2 * i + 1]); }
  __device__ __forceinline__ void set(int i, Two v) {
    const float2 f = split(v);
    w[2 * i] = f.x, w[2 * i + 1] = f.y;
  }
};

template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t to, const void *from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ float load_scalar(const float *p) { return *p; }
__device__ __forceinline__ float load_scalar(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ float load_scalar(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_scalar(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_scalar(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_scalar(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float load_as(const void *p, int dtype, int64_t at) {
  if (dtype == TGB_DTYPE_F32) return static_cast<const float *>(p)[at];
  if (dtype == TGB_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[at]);
  return __half2float(static_cast<const __half *>(p)[at]);
}

// cosine and sine of one pair's angle at one token, the angle in half turns reduced to [-1, 1]
__device__ __forceinline__ float2 turn_of(const tgb_norm_rotary &a, int64_t token, int pair) {
  double angle = 0.0;
  for (int axis = 0; axis < a.axes; ++axis) {
    const int64_t at = token * a.axes + axis;
    const double position = a.position_bits == 64 ? (double)static_cast<const int64_t *>(a.positions)[at]
                                                  : (double)static_cast<const int32_t *>(a.positions)[at];
    angle = __fma_rn(position, (double)a.frequencies[axis * a.pairs + pair], angle);
  }
  angle *= 0.31830988618379067153776752674503;
  angle = __fma_rn(-2.0, rint(0.5 * angle), angle);
  float s, c;
  sincospif((float)angle, &s, &c);
  return make_float2(c, s);
}

template <int LPR> __device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int step = LPR / 2; step; step >>= 1) v += __shfl_xor_sync(0xffffffffu, v, step);
  return v;
}

// The part of a list of `rows` heads of one token that a warp walks.  A token is cut into `parts` so that a
// few tokens still fill the machine.
struct Item {
  int64_t token;
  int first, last;
};
__device__ __forceinline__ Item item_of(int64_t id, int parts, int rows) {
  const int64_t token = id / parts;
  const int part = (int)(id - token * parts);
  return {token, (int)((int64_t)rows * part / parts), (int)((int64_t)rows * (part + 1) / parts)};
}

// ALL_TURN: the pairs cover the head (the test for values that do not turn costs the forward 7 % where it is never true).
//
// One head lies on LPR lanes, two pieces of V values each, so that both values of a pair are in one lane: the
// pieces are R/2 apart (half-split; the values behind the turned ones are paired the same way, with a
// cosine of 1), or next to each other (interleaved).
//
// Instruction issue is what a head costs next to its bytes, so values are worked on two at a time (f32x2), pieces
// are of 8 values where types and sizes allow it, and coefficients are formed once per token and side.  The loads run
// ahead of the arithmetic through a ring of cp.async stages per warp, over heads, sides and tokens alike: a lane
// reads back only what it copied itself, so there is nothing to synchronise, and the angles of the next token
// do not stop the stream.
//
// The forward walks query and key heads of a token with one table.  The backward walks all tokens' query heads,
// then all tokens' key heads: one set of sums for the weights' gradient is live at a time.
template <typename T, int LPR, int V, bool BACKWARD> struct Plan {
  static constexpr int kRows = 32 / LPR;                                  // heads a warp holds at once: a group
  static constexpr int kStages = 4;
  static constexpr int kPieces = BACKWARD ? 4 : 2;
  static constexpr int kPieceBytes = sizeof(Piece<T, V>);
  static constexpr int kStageBytes = kPieces * 32 * kPieceBytes;          // of a warp
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kTable = kWarps * LPR * V * (int)sizeof(float2);
  static constexpr int kWeights = 2 * LPR * 2 * V * 4;
  static constexpr int kShared = kRing + kTable + kWeights + (BACKWARD ? 2 * kWarps * LPR * 2 * V * 4 : 0);
  // resident on an SM, by registers
  static constexpr int kBlocks = V == 8 || sizeof(T) == 4 ? 2 : BACKWARD ? 3 : 4;
};

// All tokens' groups of ROWS heads (a forward pass has both sides, a backward pass one), token after token, are cut
// into equal shares, one per warp; a share is walked in runs of groups of one side of one token.
template <int ROWS, bool BACKWARD> struct Runs {
  int next_token, next_group, left;          // of the share
  int token, side, first, count;             // the run; count is 0 when nothing is left
  __device__ __forceinline__ int groups(const tgb_norm_rotary &a, int pass, int side_) const {
    return BACKWARD && side_ != pass ? 0 : (a.heads[side_] + ROWS - 1) / ROWS;
  }
  __device__ __forceinline__ void begin(const tgb_norm_rotary &a, int pass) {
    const int per_token = groups(a, pass, 0) + groups(a, pass, 1);
    const int64_t all = a.tokens * per_token, warps = (int64_t)gridDim.x * kWarps;
    const int64_t warp = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
    const int64_t from = all * warp / warps;
    left = (int)(all * (warp + 1) / warps - from);
    next_token = per_token ? (int)(from / per_token) : 0, next_group = (int)(from - (int64_t)next_token * per_token);
    next(a, pass);
  }
  __device__ __forceinline__ void next(const tgb_norm_rotary &a, int pass) {
    const int groups0 = groups(a, pass, 0), all = groups0 + groups(a, pass, 1);
    token = next_token, side = next_group >= groups0, first = side ? next_group - groups0 : next_group;
    count = min((side ? all : groups0) - next_group, left);
    left -= count, next_group += count;
    if (next_group == all) next_group = 0, ++next_token;
  }
};

template <typename T, int LPR, int V, bool INTERLEAVED, bool ALL_TURN, bool BACKWARD>
__global__ void __launch_bounds__(kWarps * 32, Plan<T, LPR, V, BACKWARD>::kBlocks)
k_norm_rotary(const __grid_constant__ tgb_norm_rotary a, float *__restrict__ partial) {
  using P = Plan<T, LPR, V, BACKWARD>;
  constexpr int kTwos = V / 2;                       // of a piece
  extern __shared__ __align__(16) unsigned char shared[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int D = a.dim, half = a.pairs;
  unsigned char *ring = shared + warp * P::kStages * P::kStageBytes + lane * P::kPieceBytes;
  const uint32_t ring_address = (uint32_t)__cvta_generic_to_shared(ring);
  float2 *table = reinterpret_cast<float2 *>(shared + P::kRing) + warp * LPR * V;
  float *weights = reinterpret_cast<float *>(shared + P::kRing + P::kTable);
  float *sums = reinterpret_cast<float *>(shared + P::kRing + P::kTable + P::kWeights);
  const int row_in_group = lane / LPR, lane_in_row = lane % LPR, first_pair = lane_in_row * V;
  const bool inside = first_pair < D / 2;
  // where the first (i < V) or second value of one of a lane's V pairs is in the head
  auto value_at = [&](int lane_of_row, int i) {
    const int pair = lane_of_row * V + i % V, second = i / V;
    if (INTERLEAVED) return 2 * pair + second;
    return pair < half ? pair + second * half : pair + (second ? D / 2 : half);
  };
  const int at0 = value_at(lane_in_row, 0), at1 = INTERLEAVED ? at0 + V : value_at(lane_in_row, V);
  const float inverse_dim = 1.f / D;
  wait_for_previous();

  // weights as float32, two of a lane's next to each other and the row's lanes in order, so that a warp reads no bank twice
  for (int i = threadIdx.x; i < 2 * LPR * 2 * V; i += kWarps * 32) {
    const int side = i / (LPR * 2 * V), lane_of_row = i / 2 % LPR, e = value_at(lane_of_row, i / (2 * LPR) % V * 2 + i % 2);
    weights[i] = a.weight[side] && e < D ? load_as(a.weight[side], a.weight_dtype, e) : 1.f;
  }
  if (!inside)                                         // these lanes never copy: they add zeros to their row's sums
    for (int i = 0; i < P::kStages * P::kPieces; ++i) *reinterpret_cast<Piece<T, V> *>(ring + i * 32 * P::kPieceBytes) = {};
  __syncthreads();

#pragma unroll 1
  for (int pass = 0; pass < (BACKWARD ? 2 : 1); ++pass) {
    Two dw[2 * kTwos];                                 // of the pairs' first values, then of their second ones
#pragma unroll
    for (int i = 0; i < 2 * kTwos; ++i) dw[i] = two(0.f, 0.f);
    Runs<P::kRows, BACKWARD> now;
    now.begin(a, pass);
    Runs<P::kRows, BACKWARD> ahead = now;

    // the producer: this lane's head in the group to be fetched next
    const T *px = nullptr, *pdy = nullptr;
    int64_t x_step = 0, dy_step = 0;
    int heads_left = 0, groups_left = 0;               // heads_left > 0: the lane has a head to copy
    auto enter_ahead = [&]() {
      groups_left = ahead.count;
      const int head = ahead.first * P::kRows + row_in_group, side = ahead.side;
      heads_left = inside ? a.heads[side] - head : 0;
      x_step = a.x_head_stride[side] * P::kRows;
      px = static_cast<const T *>(a.x[side]) + ahead.token * a.x_token_stride[side] + head * a.x_head_stride[side] + at0;
      if (BACKWARD) {
        dy_step = a.dy_head_stride[side] * P::kRows;
        pdy = static_cast<const T *>(a.dy[side]) + ahead.token * a.dy_token_stride[side] + head * a.dy_head_stride[side] + at0;
      }
    };
    enter_ahead();
    auto fetch = [&](int stage) {
      if (groups_left) {
        if (heads_left > 0) {                          // a head that does not exist keeps what is there: it is not stored
          const uint32_t to = ring_address + stage * P::kStageBytes;
          copy_async<P::kPieceBytes>(to, px);
          copy_async<P::kPieceBytes>(to + 32 * P::kPieceBytes, px + (at1 - at0));
          if (BACKWARD) {
            copy_async<P::kPieceBytes>(to + 64 * P::kPieceBytes, pdy);
            copy_async<P::kPieceBytes>(to + 96 * P::kPieceBytes, pdy + (at1 - at0));
          }
        }
        heads_left -= P::kRows, px += x_step, pdy += dy_step;
        if (--groups_left == 0) {
          ahead.next(a, pass);
          if (ahead.count > 0) enter_ahead();
        }
      }
      commit_copies();
    };
#pragma unroll
    for (int s = 0; s < P::kStages - 1; ++s) fetch(s);

    int stage = 0, table_of = -1;
    while (now.count > 0) {
      if (table_of != now.token) {
        table_of = now.token;
        __syncwarp();
#pragma unroll 1
        for (int pair = lane; pair < LPR * V; pair += 32)
          table[(pair % V / 2 * LPR + pair / V) * 2 + pair % 2] =      // two of a lane's pairs, the row's lanes in order
              pair < half ? turn_of(a, now.token, pair) : make_float2(1.f, 0.f);
        __syncwarp();
      }
      const int side = now.side;
      // forward, per two pairs: ya from a, ya from b, yb from b, yb from a; backward: cos and sin, the weights are read
      // again for every group
      Two c[(BACKWARD ? 2 : 4) * kTwos];
      const float2 *own_weights = reinterpret_cast<const float2 *>(weights) + side * LPR * V + lane_in_row;
#pragma unroll
      for (int i = 0; i < kTwos; ++i) {
        const float4 t = *reinterpret_cast<const float4 *>(table + (i * LPR + lane_in_row) * 2);
        const Two cosine = two(t.x, t.z), sine = two(t.y, t.w);
        if constexpr (BACKWARD) {
          c[2 * i] = cosine, c[2 * i + 1] = sine;
        } else {
          const float2 w0 = own_weights[i * LPR], w1 = own_weights[(kTwos + i) * LPR];
          const Two wa = two(w0.x, w0.y), wb = two(w1.x, w1.y);
          c[4 * i] = mul(wa, cosine), c[4 * i + 1] = mul(mul(wb, two(-1.f, -1.f)), sine);
          c[4 * i + 2] = mul(wb, cosine), c[4 * i + 3] = mul(wa, sine);
        }
      }
      int head = now.first * P::kRows + row_in_group;
      const int heads = inside ? a.heads[side] : 0;
      T *out = static_cast<T *>(a.out[side]) + ((int64_t)now.token * a.heads[side] + head) * D + at0;
#pragma unroll 1
      for (int left = now.count; left; --left) {
        wait_copies<P::kStages - 2>();
        fetch((stage + P::kStages - 1) % P::kStages);           // into the stage that the last round read
        // pairs (a, b): first[i] has the first values of pairs 2i and 2i + 1
        auto read = [&](int piece, Two (&first)[kTwos], Two (&second)[kTwos]) {
          const unsigned char *from = ring + stage * P::kStageBytes + piece * 32 * P::kPieceBytes;
          const Piece<T, V> p0 = *reinterpret_cast<const Piece<T, V> *>(from);
          const Piece<T, V> p1 = *reinterpret_cast<const Piece<T, V> *>(from + 32 * P::kPieceBytes);
#pragma unroll
          for (int i = 0; i < kTwos; ++i) {
            if (INTERLEAVED) {
              const Piece<T, V> &p = 2 * i < kTwos ? p0 : p1;
              const float2 f = split(p.get(2 * i % kTwos)), g = split(p.get(2 * i % kTwos + 1));
              first[i] = two(f.x, g.x), second[i] = two(f.y, g.y);
            } else {
              first[i] = p0.get(i), second[i] = p1.get(i);
            }
          }
        };
        // values that belong to no pair keep what they were: the other value times 0 could be an infinity times 0
        auto restore = [&](Two &v, Two kept, int i) {
          const float2 turned = split(v), plain = split(kept);
          v = two(first_pair + 2 * i < half ? turned.x : plain.x, first_pair + 2 * i + 1 < half ? turned.y : plain.y);
        };
        Two x0[kTwos], x1[kTwos], y0[kTwos], y1[kTwos];
        read(0, x0, x1);
        Two square = mul(x0[0], x0[0]);
#pragma unroll
        for (int i = 1; i < kTwos; ++i) square = fma(x0[i], x0[i], square);
#pragma unroll
        for (int i = 0; i < kTwos; ++i) square = fma(x1[i], x1[i], square);
        if constexpr (!BACKWARD) {
          const float r = a.normalise ? rsqrtf(fmaf(row_sum<LPR>(sum(square)), inverse_dim, a.eps)) : 1.f;
          const Two rr = two(r, r);
#pragma unroll
          for (int i = 0; i < kTwos; ++i) {
            y0[i] = mul(rr, fma(x0[i], c[4 * i], mul(x1[i], c[4 * i + 1])));
            y1[i] = mul(rr, fma(x1[i], c[4 * i + 2], mul(x0[i], c[4 * i + 3])));
          }
          if constexpr (!ALL_TURN) {
#pragma unroll
            for (int i = 0; i < kTwos; ++i)
              restore(y0[i], mul(rr, mul(x0[i], c[4 * i])), i), restore(y1[i], mul(rr, mul(x1[i], c[4 * i + 2])), i);
          }
        } else {
          Two g0[kTwos], g1[kTwos];                            // dn: dy turned the other way
          read(2, y0, y1);
          const Two minus = two(-1.f, -1.f);
#pragma unroll
          for (int i = 0; i < kTwos; ++i) {
            g0[i] = fma(y0[i], c[2 * i], mul(y1[i], c[2 * i + 1]));
            g1[i] = fma(y1[i], c[2 * i], mul(mul(y0[i], minus), c[2 * i + 1]));
          }
          if constexpr (!ALL_TURN) {
#pragma unroll
            for (int i = 0; i < kTwos; ++i) restore(g0[i], y0[i], i), restore(g1[i], y1[i], i);
          }
          if (a.normalise) {
            Two wa[kTwos], wb[kTwos];
#pragma unroll
            for (int i = 0; i < kTwos; ++i) {
              const float2 w0 = own_weights[i * LPR], w1 = own_weights[(kTwos + i) * LPR];
              wa[i] = two(w0.x, w0.y), wb[i] = two(w1.x, w1.y);
            }
            Two dot = two(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < kTwos; ++i) {
              dot = fma(mul(g0[i], wa[i]), x0[i], dot);
              dot = fma(mul(g1[i], wb[i]), x1[i], dot);
            }
            const float r = rsqrtf(fmaf(row_sum<LPR>(sum(square)), inverse_dim, a.eps));
            const float mean = row_sum<LPR>(sum(dot)) * r * inverse_dim;   // of g times the unit vector
            const Two rr = two(r, r), back = two(-mean, -mean);
#pragma unroll
            for (int i = 0; i < kTwos; ++i) {
              const Two unit0 = mul(x0[i], rr), unit1 = mul(x1[i], rr);
              if (head < heads) dw[i] = fma(g0[i], unit0, dw[i]), dw[kTwos + i] = fma(g1[i], unit1, dw[kTwos + i]);
              y0[i] = mul(rr, fma(unit0, back, mul(g0[i], wa[i])));
              y1[i] = mul(rr, fma(unit1, back, mul(g1[i], wb[i])));
            }
          } else {
#pragma unroll
            for (int i = 0; i < kTwos; ++i) y0[i] = g0[i], y1[i] = g1[i];
          }
        }
        if (head < heads) {
          Piece<T, V> p0, p1;
#pragma unroll
          for (int i = 0; i < kTwos; ++i) {
            if (INTERLEAVED) {
              Piece<T, V> &p = 2 * i < kTwos ? p0 : p1;
              const float2 f = split(y0[i]), g = split(y1[i]);
              p.set(2 * i % kTwos, two(f.x, g.x)), p.set(2 * i % kTwos + 1, two(f.y, g.y));
            } else {
              p0.set(i, y0[i]), p1.set(i, y1[i]);
            }
          }
          *reinterpret_cast<Piece<T, V> *>(out) = p0;
          *reinterpret_cast<Piece<T, V> *>(out + (at1 - at0)) = p1;
        }
        head += P::kRows, out += P::kRows * D;
        stage = (stage + 1) % P::kStages;
      }
      now.next(a, pass);
    }
    wait_copies<0>();
    if constexpr (BACKWARD) {
      // a row of partial sums per block, added in a fixed order: heads of a warp, warps, then blocks
#pragma unroll
      for (int i = 0; i < 2 * kTwos; ++i) {
        const float2 f = split(dw[i]);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          float v = n ? f.y : f.x;
#pragma unroll
          for (int step = LPR; step < 32; step <<= 1) v += __shfl_xor_sync(0xffffffffu, v, step);
          const int e = value_at(lane_in_row, 2 * i + n);
          if (row_in_group == 0 && inside) sums[(warp * 2 + pass) * LPR * 2 * V + e] = v;
        }
      }
    }
  }

  if constexpr (BACKWARD) {
    if (!partial) return;
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += kWarps * 32) {
      const int side = i / D, d = i - side * D;
      float v = 0.f;
      for (int k = 0; k < kWarps; ++k) v += sums[(k * 2 + side) * LPR * 2 * V + d];
      partial[(int64_t)blockIdx.x * 2 * D + i] = v;
    }
  }
}

// Any head size up to 1024, any alignment: a warp stages one head in shared memory, a value per lane and load. 8192
// tokens of 16 + 8 heads of 320 bf16: 179 us, 1.4 TB/s; their gradients 510 us, 0.7 TB/s. Bound by the wait for loads that
// nothing runs ahead of (6 and 12 clocks an instruction, 52 % and 34 % of issue slots); it is for heads above 256
// values, odd sizes and rotations, and rows off their alignment.
template <typename T, bool BACKWARD>
__global__ void __launch_bounds__(kWarps * 32)
k_norm_rotary_any(const __grid_constant__ tgb_norm_rotary a, int parts, int64_t items, float *__restrict__ partial) {
  extern __shared__ __align__(16) unsigned char shared[];
  float *staged = reinterpret_cast<float *>(shared);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int D = a.dim, pairs = a.pairs;
  float2 *table = reinterpret_cast<float2 *>(staged) + warp * pairs;
  float *row = staged + kWarps * 2 * pairs + warp * D;       // x w (forward) or dn (backward)
  float *dw = staged + kWarps * (2 * pairs + D) + warp * 2 * D;
  if constexpr (BACKWARD)
    for (int c = lane; c < 2 * D; c += 32) dw[c] = 0.f;
  wait_for_previous();
  for (int64_t id = (int64_t)blockIdx.x * kWarps + warp; id < items; id += (int64_t)gridDim.x * kWarps) {
    const Item item = item_of(id, parts, a.heads[0] + a.heads[1]);
    __syncwarp();
    for (int pair = lane; pair < pairs; pair += 32) table[pair] = turn_of(a, item.token, pair);
    __syncwarp();
    for (int r0 = item.first; r0 < item.last; ++r0) {
      const int side = r0 >= a.heads[0], h = side ? r0 - a.heads[0] : r0;
      const T *x = static_cast<const T *>(a.x[side]) + item.token * a.x_token_stride[side] + h * a.x_head_stride[side];
      T *out = static_cast<T *>(a.out[side]) + (item.token * a.heads[side] + h) * (int64_t)D;
      float square = 0.f;
      for (int d = lane; d < D; d += 32) {
        const float v = load_scalar(x + d);
        square = fmaf(v, v, square);
      }
      const float r = a.normalise ? rsqrtf(row_sum<32>(square) / D + a.eps) : 1.f;
      const T *in = BACKWARD ? static_cast<const T *>(a.dy[side]) + item.token * a.dy_token_stride[side] +
                                   h * a.dy_head_stride[side]
                             : x;
      __syncwarp();
      for (int d = lane; d < D; d += 32) {
        const float w = !BACKWARD && a.weight[side] ? load_as(a.weight[side], a.weight_dtype, d) : 1.f;
        row[d] = load_scalar(in + d) * w;
      }
      __syncwarp();
      // every pair is turned by one lane, in place; the backward turns the other way
      for (int pair = lane; pair < pairs; pair += 32) {
        const int p = a.interleaved ? 2 * pair : pair, q = a.interleaved ? 2 * pair + 1 : pair + pairs;
        const float c = table[pair].x, s = BACKWARD ? -table[pair].y : table[pair].y;
        const float va = row[p], vb = row[q];
        row[p] = va * c - vb * s, row[q] = vb * c + va * s;
      }
      __syncwarp();
      if constexpr (!BACKWARD) {
        for (int d = lane; d < D; d += 32) store_scalar(out + d, r * row[d]);
      } else if (!a.normalise) {
        for (int d = lane; d < D; d += 32) store_scalar(out + d, row[d]);
      } else {
        float dot = 0.f;
        for (int d = lane; d < D; d += 32) {
          const float w = a.weight[side] ? load_as(a.weight[side], a.weight_dtype, d) : 1.f;
          dot = fmaf(row[d] * w, load_scalar(x + d), dot);
        }
        const float mean = row_sum<32>(dot) * r / D;
        for (int d = lane; d < D; d += 32) {
          const float w = a.weight[side] ? load_as(a.weight[side], a.weight_dtype, d) : 1.f;
          const float unit = load_scalar(x + d) * r;
          dw[side * D + d] = fmaf(row[d], unit, dw[side * D + d]);
          store_scalar(out + d, r * (row[d] * w - unit * mean));
        }
      }
    }
  }
  if constexpr (BACKWARD) {
    if (!partial) return;
    __syncthreads();
    const float *all = staged + kWarps * (2 * pairs + D);
    for (int c = threadIdx.x; c < 2 * D; c += kWarps * 32) {
      float v = 0.f;
      for (int k = 0; k < kWarps; ++k) v += all[k * 2 * D + c];
      partial[(int64_t)blockIdx.x * 2 * D + c] = v;
    }
  }
}

// dw[c] = sum over the blocks' rows of partial sums: 32 columns a block, each column's rows dealt to 32 warps
__global__ void __launch_bounds__(1024)
k_weight_grad(const float *partial, int rows, int D, void *dq, void *dk, int dtype) {
  __shared__ float sums[32][33];
  const int column = blockIdx.x * 32 + threadIdx.x;
  wait_for_previous();
  float v = 0.f;
  if (column < 2 * D)
    for (int r = threadIdx.y; r < rows; r += 32) v += partial[(int64_t)r * 2 * D + column];
  sums[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y || column >= 2 * D) return;
  v = 0.f;
#pragma unroll
  for (int k = 0; k < 32; ++k) v += sums[k][threadIdx.x];
  void *out = column < D ? dq : dk;
  const int d = column < D ? column : column - D;
  if (!out) return;
  if (dtype == TGB_DTYPE_F32) static_cast<float *>(out)[d] = v;
  else if (dtype == TGB_DTYPE_BF16) static_cast<__nv_bfloat16 *>(out)[d] = __float2bfloat16_rn(v);
  else static_cast<__half *>(out)[d] = __float2half_rn(v);
}

constexpr int kMaxDim = 1024;            // of a head
constexpr int kMaxBlocks = 148 * 4;      // of the backward: rows of partial sums

// values of a piece (8, 4; 0: the any-size kernel): heads are read in aligned pieces with both values of every pair in
// one lane. Pieces of 8 hold twice the heads in a warp (8192 tokens of 16 + 16 heads of 128: gradient and forward 53 + 28
// us with 4, 46 + 24 with 8), which pays unless that leaves a quarter more heads missing from the last groups (12 + 4 heads
// of 64: 63 us with 4, 66 with 8; 9 + 9 heads of 128: 113 and 105); float32 has registers for 4
int piece_values(const tgb_norm_rotary &a, bool backward) {
  const int size = a.dtype == TGB_DTYPE_F32 ? 4 : 2;
  for (int v = size == 4 ? 4 : 8; v >= 4; v /= 2) {
    if (a.dim % (2 * v) || a.dim > 256 || (!a.interleaved && a.pairs % v) || (v == 8 && 2 * a.pairs != a.dim)) continue;
    bool fits = true;
    int64_t with8 = 0, with4 = 0;            // heads that the warps' groups have room for
    for (int side = 0; side < 2; ++side) {
      if (!a.heads[side]) continue;
      auto aligned = [&](const void *p, int64_t token, int64_t head) {
        return reinterpret_cast<uintptr_t>(p) % (v * size) == 0 && token % v == 0 && head % v == 0;
      };
      fits = fits && aligned(a.x[side], a.x_token_stride[side], a.x_head_stride[side]) && aligned(a.out[side], 0, 0) &&
             (!backward || aligned(a.dy[side], a.dy_token_stride[side], a.dy_head_stride[side]));
      const int rows = a.dim <= 64 ? 4 : a.dim <= 128 ? 2 : 1;
      with4 += ceil_div(a.heads[side], rows) * rows, with8 += ceil_div(a.heads[side], 2 * rows) * 2 * rows;
    }
    if (fits && (v == 4 || 4 * with8 <= 5 * with4)) return v;
  }
  return 0;
}

template <typename T, int LPR, int V, bool INTERLEAVED, bool ALL_TURN, bool BACKWARD>
int32_t launch_pieces(const tgb_norm_rotary &a, float *partial, cudaStream_t stream, int &blocks) {
  using P = Plan<T, LPR, V, BACKWARD>;
  auto groups = [&](int side) { return ceil_div(a.heads[side], P::kRows); };
  const int64_t all = a.tokens * (BACKWARD ? (groups(0) > groups(1) ? groups(0) : groups(1)) : groups(0) + groups(1));
  // one round of resident blocks, but no warp with less than two groups: it forms a table of sines first
  const int64_t limit = (int64_t)148 * P::kBlocks, full = ceil_div(all, 2 * kWarps);
  blocks = (int)(full < limit ? full : limit);
  auto kernel = k_norm_rotary<T, LPR, V, INTERLEAVED, ALL_TURN, BACKWARD>;
  static std::atomic<uint64_t> asked{0};
  TGB_CUDA(allow_shared(kernel, P::kShared, asked));
  TGB_CUDA(launch_dependent(kernel, dim3(blocks), dim3(kWarps * 32), P::kShared, stream, a, partial));
  return TGB_STATUS_OK;
}

template <typename T, int V, bool INTERLEAVED, bool ALL_TURN, bool BACKWARD>
int32_t launch_lanes(const tgb_norm_rotary &a, float *partial, cudaStream_t stream, int &blocks) {
  if (a.dim <= 64) return launch_pieces<T, 32 / V, V, INTERLEAVED, ALL_TURN, BACKWARD>(a, partial, stream, blocks);
  if (a.dim <= 128) return launch_pieces<T, 64 / V, V, INTERLEAVED, ALL_TURN, BACKWARD>(a, partial, stream, blocks);
  return launch_pieces<T, 128 / V, V, INTERLEAVED, ALL_TURN, BACKWARD>(a, partial, stream, blocks);
}

template <typename T, bool BACKWARD>
int32_t launch(const tgb_norm_rotary &a, float *partial, cudaStream_t stream, int &blocks) {
  const int v = piece_values(a, BACKWARD);
  if constexpr (sizeof(T) == 2) {
    if (v == 8)
      return a.interleaved ? launch_lanes<T, 8, true, true, BACKWARD>(a, partial, stream, blocks)
                           : launch_lanes<T, 8, false, true, BACKWARD>(a, partial, stream, blocks);
  }
  if (v) {
    const bool all = 2 * a.pairs == a.dim;
    if (a.interleaved)
      return all ? launch_lanes<T, 4, true, true, BACKWARD>(a, partial, stream, blocks)
                 : launch_lanes<T, 4, true, false, BACKWARD>(a, partial, stream, blocks);
    return all ? launch_lanes<T, 4, false, true, BACKWARD>(a, partial, stream, blocks)
               : launch_lanes<T, 4, false, false, BACKWARD>(a, partial, stream, blocks);
  }
  const int rows = a.heads[0] + a.heads[1];
  const int64_t wanted = ceil_div(148 * 4 * kWarps, a.tokens);
  const int parts = (int)(wanted < rows ? wanted : rows);
  const int64_t items = a.tokens * parts, full = ceil_div(items, kWarps);
  blocks = (int)(full < kMaxBlocks ? full : kMaxBlocks);
  constexpr int kMost = sizeof(float) * kWarps * (BACKWARD ? 4 : 2) * kMaxDim;
  const size_t bytes = sizeof(float) * kWarps * (2 * a.pairs + a.dim + (BACKWARD ? 2 * a.dim : 0));
  static std::atomic<uint64_t> asked{0};
  TGB_CUDA(allow_shared(k_norm_rotary_any<T, BACKWARD>, kMost, asked));
  TGB_CUDA(launch_dependent(k_norm_rotary_any<T, BACKWARD>, dim3(blocks), dim3(kWarps * 32), bytes, stream, a, parts, items,
                            partial));
  return TGB_STATUS_OK;
}

template <bool BACKWARD>
int32_t dispatch(const tgb_norm_rotary &a, float *partial, cudaStream_t stream, int &blocks) {
  if (a.dtype == TGB_DTYPE_BF16) return launch<__nv_bfloat16, BACKWARD>(a, partial, stream, blocks);
  if (a.dtype == TGB_DTYPE_F16) return launch<__half, BACKWARD>(a, partial, stream, blocks);
  return launch<float, BACKWARD>(a, partial, stream, blocks);
}

bool is_float(int dtype) { return dtype == TGB_DTYPE_F32 || dtype == TGB_DTYPE_BF16 || dtype == TGB_DTYPE_F16; }

int32_t check(const tgb_norm_rotary *a, bool backward) {
  if (!a) TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "null arguments");
  if (!is_float(a->dtype) || !is_float(a->weight_dtype)) TGB_FAIL(TGB_STATUS_UNSUPPORTED, "dtype must be float32, bfloat16 or float16");
  if (a->tokens > (1 << 30)) TGB_FAIL(TGB_STATUS_UNSUPPORTED, "at most 2^30 tokens");
  if (a->tokens < 0 || a->heads[0] < 0 || a->heads[1] < 0 || a->heads[0] > (1 << 20) || a->heads[1] > (1 << 20))
    TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "tokens and heads must be non-negative, heads at most 2^20");
  if (a->dim < 1 || a->dim > kMaxDim) TGB_FAIL(TGB_STATUS_UNSUPPORTED, "head size must be in [1, %d], got %d", kMaxDim, a->dim);
  if (a->pairs < 0 || 2 * a->pairs > a->dim) TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "2 * pairs must be at most the head size");
  if (a->axes < 1 || a->axes > 8) TGB_FAIL(TGB_STATUS_UNSUPPORTED, "1 to 8 position axes, got %d", a->axes);
  if (a->position_bits != 32 && a->position_bits != 64) TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "position_bits must be 32 or 64");
  if (!a->tokens) return TGB_STATUS_OK;
  if (a->pairs && (!a->positions || !a->frequencies)) TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "null positions or frequencies");
  for (int side = 0; side < 2; ++side)
    if (a->heads[side] && (!a->x[side] || !a->out[side] || (backward && !a->dy[side])))
      TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "null field pointer");
  return TGB_STATUS_OK;
}

}  // namespace
}  // namespace tgb

extern "C" {

int32_t tgb_norm_rotary_fwd(const tgb_norm_rotary *arguments, uint64_t stream) {
  const int32_t status = tgb::check(arguments, false);
  if (status) return status;
  if (!arguments->tokens || !(arguments->heads[0] + arguments->heads[1])) return TGB_STATUS_OK;
  int blocks;
  return tgb::dispatch<false>(*arguments, nullptr, reinterpret_cast<cudaStream_t>(stream), blocks);
}

uint64_t tgb_norm_rotary_scratch_bytes(int32_t dim) {
  return dim < 1 ? 0 : (uint64_t)tgb::kMaxBlocks * 2 * dim * sizeof(float);
}

int32_t tgb_norm_rotary_bwd(const tgb_norm_rotary *arguments, void *query_weight_grad, void *key_weight_grad,
                            void *scratch, uint64_t scratch_bytes, uint64_t stream_handle) {
  const int32_t status = tgb::check(arguments, true);
  if (status) return status;
  const tgb_norm_rotary &a = *arguments;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
  const bool weights = query_weight_grad || key_weight_grad;
  if (weights && !a.normalise) TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "weights without the norm have no gradient");
  if (weights && (!scratch || scratch_bytes < tgb_norm_rotary_scratch_bytes(a.dim)))
    TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "weight gradients need %llu bytes of scratch",
             (unsigned long long)tgb_norm_rotary_scratch_bytes(a.dim));
  int blocks = 0;                     // no tokens: the weights' gradients are sums of nothing
  if (a.tokens && a.heads[0] + a.heads[1]) {
    const int32_t launched = tgb::dispatch<true>(a, weights ? static_cast<float *>(scratch) : nullptr, stream, blocks);
    if (launched) return launched;
  }
  if (weights) {
    TGB_CUDA(tgb::launch_dependent(tgb::k_weight_grad, dim3((2 * a.dim + 31) / 32), dim3(32, 32), 0, stream,
                                   static_cast<const float *>(scratch), blocks, a.dim, query_weight_grad, key_weight_grad,
                                   a.weight_dtype));
  }
  return TGB_STATUS_OK;
}

}  // extern "C"
