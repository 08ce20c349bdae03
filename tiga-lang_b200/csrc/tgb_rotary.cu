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
// Angles are formed and reduced to [-pi, pi] in 64 bits (position * frequency
// reaches 10^5 and more, where float32 is off by 1/128), then sine and cosine are
// taken in 32 bits; a warp computes a token's table once and walks its heads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tgb_common.cuh"

namespace tgb {
namespace {

constexpr int kWarps = 8;

template <typename T> struct Packed;            // V values of T as 32-bit words
template <> struct Packed<__nv_bfloat16> { static constexpr int per_word = 2; };
template <> struct Packed<__half> { static constexpr int per_word = 2; };
template <> struct Packed<float> { static constexpr int per_word = 1; };

template <typename T> __device__ __forceinline__ float2 unpack(uint32_t w);
template <> __device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

template <typename T> __device__ __forceinline__ uint32_t pack(float a, float b);
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}

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

// V consecutive values as words, and as floats
template <typename T, int V> struct Chunk {
  static constexpr int words = V / Packed<T>::per_word;
  uint32_t w[words];

  __device__ __forceinline__ void load(const T *p) {
    if constexpr (words % 4 == 0) {
#pragma unroll
      for (int i = 0; i < words; i += 4) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(p) + i / 4);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    } else {
      const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(p));
      w[0] = v.x, w[1] = v.y;
    }
  }
  __device__ __forceinline__ void store(T *p) const {
    if constexpr (words % 4 == 0) {
#pragma unroll
      for (int i = 0; i < words; i += 4)
        *(reinterpret_cast<uint4 *>(p) + i / 4) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    } else {
      *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < words; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void floats(float (&f)[V]) const {
    if constexpr (Packed<T>::per_word == 1) {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < words; ++i) {
        const float2 v = unpack<T>(w[i]);
        f[2 * i] = v.x, f[2 * i + 1] = v.y;
      }
    }
  }
  __device__ __forceinline__ void from(const float (&f)[V]) {
    if constexpr (Packed<T>::per_word == 1) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < words; ++i) w[i] = pack<T>(f[2 * i], f[2 * i + 1]);
    }
  }
  // the pair's other values: of lane `partner`, or the neighbours inside the chunk; 0 for the values
  // from `turned` on, which belong to no pair (an infinity there must not meet the zero sine)
  __device__ __forceinline__ void other(int partner, bool interleaved, int turned, float (&f)[V]) const {
    if (interleaved) {
      float own[V];
      floats(own);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = own[i ^ 1];
    } else {
      Chunk<T, V> c;
#pragma unroll
      for (int i = 0; i < words; ++i) c.w[i] = __shfl_sync(0xffffffffu, w[i], partner);
      c.floats(f);
    }
    if (turned < V) {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = i < turned ? f[i] : 0.f;
    }
  }
};

// cosine and sine of one pair's angle at one token
__device__ __forceinline__ float2 turn_of(const tgb_norm_rotary &a, int64_t token, int pair) {
  double angle = 0.0;
  for (int axis = 0; axis < a.axes; ++axis) {
    const int64_t at = token * a.axes + axis;
    const double position = a.position_bits == 64 ? (double)static_cast<const int64_t *>(a.positions)[at]
                                                  : (double)static_cast<const int32_t *>(a.positions)[at];
    angle += position * (double)a.frequencies[(int64_t)axis * a.pairs + pair];
  }
  constexpr double kTurn = 6.283185307179586476925286766559;
  angle -= kTurn * rint(angle / kTurn);
  float s, c;
  sincosf((float)angle, &s, &c);
  return make_float2(c, s);
}

template <int LPR> __device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int step = LPR / 2; step; step >>= 1) v += __shfl_xor_sync(0xffffffffu, v, step);
  return v;
}

// The part of the combined list of a token's query and key heads that a warp walks.
// A token is cut into `parts` so that a few tokens still fill the machine.
struct Item {
  int64_t token;
  int first, last;   // of heads[0] + heads[1] rows
};
__device__ __forceinline__ Item item_of(const tgb_norm_rotary &a, int64_t id, int parts) {
  const int rows = a.heads[0] + a.heads[1];
  const int64_t token = id / parts;
  const int part = (int)(id - token * parts);
  return {token, (int)((int64_t)rows * part / parts), (int)((int64_t)rows * (part + 1) / parts)};
}

// LPR lanes hold one head, V values each.  In the half-split layout a pair's values
// lie R/2 apart, which is a whole number of lanes: the other value comes by shuffle,
// still packed in its own type.
template <typename T, int LPR, int V, bool BACKWARD>
__global__ void __launch_bounds__(kWarps * 32)
k_norm_rotary(const __grid_constant__ tgb_norm_rotary a, int parts, int64_t items, float *__restrict__ partial) {
  constexpr int kRows = 32 / LPR;                    // heads a warp holds at once
  constexpr int kUnroll = BACKWARD ? 2 : 4;          // their loads are issued together
  __shared__ float2 table[kWarps][LPR * V / 2];
  __shared__ float sums[BACKWARD ? 2 * kWarps * LPR * V : 1];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int group = lane / LPR, at = (lane % LPR) * V;   // first value of this lane
  const int D = a.dim, half = a.pairs;
  const bool inside = at < D;
  const bool interleaved = a.interleaved;
  int partner = lane;
  if (!interleaved && at < 2 * half) partner = at < half ? lane + half / V : lane - half / V;

  float dw[2][V];
  if constexpr (BACKWARD) {
#pragma unroll
    for (int i = 0; i < V; ++i) dw[0][i] = dw[1][i] = 0.f;
  }

  for (int64_t id = (int64_t)blockIdx.x * kWarps + warp; id < items; id += (int64_t)gridDim.x * kWarps) {
    const Item item = item_of(a, id, parts);
    __syncwarp();
    for (int pair = lane; pair < LPR * V / 2; pair += 32)
      table[warp][pair] = pair < half ? turn_of(a, item.token, pair) : make_float2(1.f, 0.f);
    __syncwarp();
    float cosine[V], sine[V];                          // sine with the sign that y takes it with
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = at + i;
      if (interleaved) {
        const float2 t = table[warp][e / 2];
        cosine[i] = t.x, sine[i] = (e & 1) ? t.y : -t.y;
      } else {
        const float2 t = e < 2 * half ? table[warp][e < half ? e : e - half] : make_float2(1.f, 0.f);
        cosine[i] = t.x, sine[i] = e < half ? -t.y : t.y;
      }
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int base = side ? a.heads[0] : 0;
      const int first = max(item.first, base) - base, last = min(item.last, base + a.heads[side]) - base;
      if (first >= last) continue;
      float w[V], c1[V], c2[V];
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = a.weight[side] && inside ? load_as(a.weight[side], a.weight_dtype, at + i) : 1.f;
      if constexpr (BACKWARD) {                        // dn = dy cos + dy' (the other sign) sin
#pragma unroll
        for (int i = 0; i < V; ++i) c1[i] = cosine[i], c2[i] = -sine[i];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float v = interleaved ? w[i ^ 1] : __shfl_sync(0xffffffffu, w[i], partner);
          c1[i] = w[i] * cosine[i], c2[i] = v * sine[i];
        }
      }
      const T *x = static_cast<const T *>(a.x[side]) + item.token * a.x_token_stride[side] + at;
      const T *dy = BACKWARD ? static_cast<const T *>(a.dy[side]) + item.token * a.dy_token_stride[side] + at : nullptr;
      T *out = static_cast<T *>(a.out[side]) + item.token * a.heads[side] * (int64_t)D + at;
      for (int row = first; row < last; row += kRows * kUnroll) {
        Chunk<T, V> in[kUnroll], up[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int h = row + u * kRows + group;
          in[u].zero();
          if constexpr (BACKWARD) up[u].zero();
          if (inside && h < last) {
            in[u].load(x + h * a.x_head_stride[side]);
            if constexpr (BACKWARD) up[u].load(dy + h * a.dy_head_stride[side]);
          }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          if (row + u * kRows >= last) break;          // the same for all lanes
          const int h = row + u * kRows + group;
          float v[V], square = 0.f;
          in[u].floats(v);
#pragma unroll
          for (int i = 0; i < V; ++i) square = fmaf(v[i], v[i], square);
          if constexpr (!BACKWARD) {
            float other[V];
            in[u].other(partner, interleaved, 2 * half - at, other);
            const float r = a.normalise ? rsqrtf(row_sum<LPR>(square) / D + a.eps) : 1.f;
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = r * fmaf(v[i], c1[i], other[i] * c2[i]);
          } else {
            float dn[V], other[V], dot = 0.f;
            up[u].floats(dn);
            up[u].other(partner, interleaved, 2 * half - at, other);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              dn[i] = fmaf(dn[i], c1[i], other[i] * c2[i]);
              dot = fmaf(dn[i] * w[i], v[i], dot);
            }
            if (a.normalise) {
              const float r = rsqrtf(row_sum<LPR>(square) / D + a.eps);
              const float mean = row_sum<LPR>(dot) * r / D;       // of g times the unit vector
#pragma unroll
              for (int i = 0; i < V; ++i) {
                const float unit = v[i] * r;
                dw[side][i] = fmaf(dn[i], unit, dw[side][i]);
                v[i] = r * (dn[i] * w[i] - unit * mean);
              }
            } else {
#pragma unroll
              for (int i = 0; i < V; ++i) v[i] = dn[i];
            }
          }
          if (inside && h < last) {
            Chunk<T, V> c;
            c.from(v);
            c.store(out + h * (int64_t)D);
          }
        }
      }
    }
  }

  if constexpr (BACKWARD) {
    if (!partial) return;
    // one row of partial sums per block, added in a fixed order: heads of a warp, warps, then blocks
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float v = dw[side][i];
#pragma unroll
        for (int step = LPR; step < 32; step <<= 1) v += __shfl_xor_sync(0xffffffffu, v, step);
        if (group == 0) sums[(warp * 2 + side) * LPR * V + at + i] = v;
      }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * D; c += kWarps * 32) {
      const int side = c / D, d = c - side * D;
      float v = 0.f;
      for (int k = 0; k < kWarps; ++k) v += sums[(k * 2 + side) * LPR * V + d];
      partial[(int64_t)blockIdx.x * 2 * D + c] = v;
    }
  }
}

// Any head size up to 1024, any alignment: a warp stages one head in shared memory.
template <typename T, bool BACKWARD>
__global__ void __launch_bounds__(kWarps * 32)
k_norm_rotary_any(const __grid_constant__ tgb_norm_rotary a, int parts, int64_t items, float *__restrict__ partial) {
  extern __shared__ float shared[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int D = a.dim, pairs = a.pairs;
  float2 *table = reinterpret_cast<float2 *>(shared) + warp * pairs;
  float *row = shared + kWarps * 2 * pairs + warp * D;       // x w (forward) or dn (backward)
  float *dw = shared + kWarps * (2 * pairs + D) + warp * 2 * D;
  if constexpr (BACKWARD)
    for (int c = lane; c < 2 * D; c += 32) dw[c] = 0.f;
  for (int64_t id = (int64_t)blockIdx.x * kWarps + warp; id < items; id += (int64_t)gridDim.x * kWarps) {
    const Item item = item_of(a, id, parts);
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
    const float *all = shared + kWarps * (2 * pairs + D);
    for (int c = threadIdx.x; c < 2 * D; c += kWarps * 32) {
      float v = 0.f;
      for (int k = 0; k < kWarps; ++k) v += all[k * 2 * D + c];
      partial[(int64_t)blockIdx.x * 2 * D + c] = v;
    }
  }
}

// dw[c] = sum over the blocks' rows of partial sums: 32 columns a block, each column's rows dealt to 32 warps
__global__ void __launch_bounds__(1024)
k_weight_grad(const float *__restrict__ partial, int rows, int D, void *dq, void *dk, int dtype) {
  __shared__ float sums[32][33];
  const int column = blockIdx.x * 32 + threadIdx.x;
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

constexpr int kMaxBlocks = 148 * 4;      // of the backward: rows of partial sums

// values per lane: the widest that keeps a pair's halves whole lanes apart and every access aligned
int lane_values(const tgb_norm_rotary &a, bool backward) {
  const int size = a.dtype == TGB_DTYPE_F32 ? 4 : 2;
  for (int v = 8; v >= 4; v /= 2) {
    if (a.dim % v || a.dim > 32 * v || (!a.interleaved && a.pairs % v)) continue;
    const int bytes = v * size < 16 ? v * size : 16;
    bool aligned = true;
    for (int side = 0; side < 2; ++side) {
      if (!a.heads[side]) continue;
      auto fits = [&](const void *p, int64_t token, int64_t head) {
        return reinterpret_cast<uintptr_t>(p) % bytes == 0 && token * size % bytes == 0 && head * size % bytes == 0;
      };
      aligned = aligned && fits(a.x[side], a.x_token_stride[side], a.x_head_stride[side]) &&
                fits(a.out[side], a.dim, a.dim) &&
                (!backward || fits(a.dy[side], a.dy_token_stride[side], a.dy_head_stride[side]));
    }
    if (aligned) return v;
  }
  return 0;
}

template <typename T, bool BACKWARD>
int32_t launch(const tgb_norm_rotary &a, float *partial, cudaStream_t stream, int &blocks) {
  const int rows = a.heads[0] + a.heads[1];
  const int v = lane_values(a, BACKWARD);
  const int lanes = v ? (a.dim <= 8 * v ? 8 : a.dim <= 16 * v ? 16 : 32) : 32;
  // parts of a token: enough warps for every SM, no part below what a warp holds at once
  const int at_once = (32 / lanes) * (v ? (BACKWARD ? 2 : 4) : 1);
  const int most = rows / at_once > 1 ? rows / at_once : 1;
  const int64_t wanted = ceil_div(148 * 4 * kWarps, a.tokens);
  const int parts = (int)(wanted < most ? wanted : most);
  const int64_t items = a.tokens * parts;
  const int64_t full = ceil_div(items, kWarps);
  const int64_t limit = BACKWARD ? kMaxBlocks : 148 * 8;
  blocks = (int)(full < limit ? full : limit);
  if (!v) {
    const size_t bytes = sizeof(float) * kWarps * (2 * a.pairs + a.dim + (BACKWARD ? 2 * a.dim : 0));
    TGB_CUDA(cudaFuncSetAttribute(k_norm_rotary_any<T, BACKWARD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    k_norm_rotary_any<T, BACKWARD><<<blocks, kWarps * 32, bytes, stream>>>(a, parts, items, partial);
  } else if (v == 8) {
    if (lanes == 8) k_norm_rotary<T, 8, 8, BACKWARD><<<blocks, kWarps * 32, 0, stream>>>(a, parts, items, partial);
    else if (lanes == 16) k_norm_rotary<T, 16, 8, BACKWARD><<<blocks, kWarps * 32, 0, stream>>>(a, parts, items, partial);
    else k_norm_rotary<T, 32, 8, BACKWARD><<<blocks, kWarps * 32, 0, stream>>>(a, parts, items, partial);
  } else {
    if (lanes == 8) k_norm_rotary<T, 8, 4, BACKWARD><<<blocks, kWarps * 32, 0, stream>>>(a, parts, items, partial);
    else if (lanes == 16) k_norm_rotary<T, 16, 4, BACKWARD><<<blocks, kWarps * 32, 0, stream>>>(a, parts, items, partial);
    else k_norm_rotary<T, 32, 4, BACKWARD><<<blocks, kWarps * 32, 0, stream>>>(a, parts, items, partial);
  }
  TGB_LAUNCHED();
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
  if (a->tokens < 0 || a->heads[0] < 0 || a->heads[1] < 0 || a->heads[0] > (1 << 20) || a->heads[1] > (1 << 20))
    TGB_FAIL(TGB_STATUS_INVALID_ARGUMENT, "tokens and heads must be non-negative, heads at most 2^20");
  if (a->dim < 1 || a->dim > 1024) TGB_FAIL(TGB_STATUS_UNSUPPORTED, "head size must be in [1, 1024], got %d", a->dim);
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
    tgb::k_weight_grad<<<(2 * a.dim + 31) / 32, dim3(32, 32), 0, stream>>>(
        static_cast<const float *>(scratch), blocks, a.dim, query_weight_grad, key_weight_grad, a.weight_dtype);
    TGB_LAUNCHED();
  }
  return TGB_STATUS_OK;
}

}  // extern "C"
