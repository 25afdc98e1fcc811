// What the kernels of attention over a window share: arguments, visibility, the bias by buckets, tiles of rows in LDS and their
// products.
//
// All products run on 32 x 32 tiles of (rows in LDS) x (rows that a lane holds in registers), so that a lane keeps one query (or, in
// the gradients of keys and values, one key) and the softmax needs no exchange but that between the two half-waves:
//   scores   z[r][i] = sum_d X[r][d] own_i[d]        X: 32 rows in LDS, A operands as they lie; own: B operands
//   outcome  o[d][i] = sum_r X[r][d] w[r][i]         w: the weights of the tile, packed where they were formed (a C tile is a pair
//                                                    of B operands in the order rowmap); X transposed: bf16 by the transposing LDS
//                                                    read, float32 element by element (lanes run along d: no conflicts)
// bf16 rows go through v_mfma_f32_32x32x16_bf16, and so do float32 rows to widths of 64 in the kernels over windows, three bf16 values each (Split);
// wider ones and the steps, which are bound by memory, through v_mfma_f32_32x32x2_f32.
#pragma once

#include "pa_common.h"
#include "pa_host.h"
#include "pa_mfma_ops.h"

namespace pa {
namespace window {

using mfma::f32x16;
using mfma::half_max;
using mfma::half_sum;
using mfma::rowmap;
using mfma::u32x2;
using mfma::u32x4;

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kNoBound = 1 << 30;  // past every distance: positions stay below 2^29

// ---- arguments ----
struct View {
  const void *data;
  int64_t batch, row, head;
  bool plain;  // see Stage
};
struct BiasArgs {
  const float *table;  // (buckets, Hq)
  int buckets, side, exact, distance;  // buckets of a side (j <= i, or j > i); of them one distance each; beyond `distance` nothing changes
  bool both;
  int borders[PA_MAX_BUCKETS / 2];  // least distance of bucket exact + 1, exact + 2, ...
};
struct Args {
  View q, k, v, dy;
  int N, Hq, Hk, D, B;
  int left, right, sinks;
  float c;      // scale log2(e)
  float scale;
  const int32_t *lengths;
  BiasArgs bias;
  void *y;
  float *stats;  // forward: written
  // backward
  const void *saved_y;
  const float *saved_stats;
  void *dq, *dk, *dv;
  float *delta, *bias_parts, *sink_parts;
  int blocks;       // query (key) blocks of a sequence
  int sink_chunks;  // parts of the queries of the key tiles with sinks
  int sink_rows;    // rows of those tiles
};

__device__ __forceinline__ int length_of(const Args &a, int b) {
  if (!a.lengths) return a.N;
  const int n = __builtin_amdgcn_readfirstlane(a.lengths[b]);
  return n < 0 ? 0 : n > a.N ? a.N : n;
}
// whether it is so in some lane: a branch on this is one of the whole wave, and known as such (branches that are taken for divergent cost copies
// of all sums that they change)
__device__ __forceinline__ bool some_lane(bool v) { return __builtin_amdgcn_ballot_w64(v) != 0; }

// Workgroup -> work: consecutive work on one XCD (workgroups go round them), whose L2 then holds what neighbours share
__device__ __forceinline__ uint32_t own_work() {
  const uint32_t n = gridDim.x, id = blockIdx.x, per = n / 8, rest = n % 8, xcd = id % 8, slot = id / 8;
  return xcd * per + (xcd < rest ? xcd : rest) + slot;
}

// ---- bias ----
__device__ __forceinline__ int bucket_of(const BiasArgs &b, int d) {  // d >= 0
  if (d < b.exact) return d;
  int lo = 0, hi = b.side - b.exact - 1;  // borders passed: the first of [lo, hi] that d has not reached
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (d >= b.borders[mid]) lo = mid + 1;
    else hi = mid;
  }
  return b.exact + lo;
}
__device__ __forceinline__ int bucket_of_offset(const BiasArgs &b, int off) {  // off = j - i
  const int d = off < 0 ? -off : off;
  return bucket_of(b, d < b.distance ? d : b.distance) + (off > 0 && b.both ? b.side : 0);
}
// Offsets j - i of a table in LDS: -(distance + kPad) .. (distance or 0) + kPad.  A tile that comes within `distance` of the diagonal
// stays inside, so that its lookups need no bounds.
constexpr int kPad = 64;
__host__ __device__ inline int table_low(const BiasArgs &b) { return b.distance + kPad; }
__host__ __device__ inline int table_size(const BiasArgs &b) { return b.distance + 2 * kPad + 1 + (b.both ? b.distance : 0); }
// A bias as the products start from it, in units of q . k: z = q . k + bias / scale, and a weight is exp2(c z - ..).  Biases of -2^16 and less
// hide as -inf does, and none is above 2^16: a float32 score keeps nothing of q . k beside larger ones, nor does the sum that the backward
// pass reads, the logarithm of the denominator with the reference.
__device__ __forceinline__ float bias_start(float v, float c) {
  return v <= -65536.f ? -INFINITY : (v > 65536.f ? 65536.f : v) * (kLog2e / c);
}
__device__ __forceinline__ void fill_bias_table(const Args &a, int head, float *lds) {
  const int low = table_low(a.bias), n = table_size(a.bias);
  for (int u = threadIdx.x; u < n; u += blockDim.x)
    lds[u] = bias_start(a.bias.table[(int64_t)bucket_of_offset(a.bias, u - low) * a.Hq + head], a.c);
}
// where a 32 x 32 tile's offsets lie, least and most of them
enum Reach { kNear, kFarBehind, kFarAhead };
__device__ __forceinline__ Reach reach_of(const BiasArgs &b, int least, int most) {
  if (most <= -b.distance) return kFarBehind;
  if (b.both && least >= b.distance) return kFarAhead;
  return kNear;
}

// ---- which tiles of 32 rows from r0 on a wave's 32 own rows see: some of it, or all.  Formed once, so that a tile costs a few scalar
// comparisons (formed for each tile anew it cost 90 scalar instructions and a third of the time) ----
struct Sights {
  int low, high, first, full;  // some: low .. high or below `first`; all: full .. full + span
  uint32_t span;
  __device__ __forceinline__ bool none(int r0) const { return r0 > high || (r0 < low && r0 >= first); }
  __device__ __forceinline__ bool all(int r0) const { return (uint32_t)(r0 - full) < span; }
  __device__ __forceinline__ void set_full(int from, int to) {  // to: the last first row
    full = from, span = to < from ? 0u : (uint32_t)(to - from) + 1u;
  }
};
// keys for the queries from q0
__device__ __forceinline__ Sights sights_of_queries(const Args &a, int len, int q0) {
  Sights s;
  const int last = q0 + 31 + a.right < len - 1 ? q0 + 31 + a.right : len - 1;
  s.low = q0 - a.left - 31, s.high = q0 < len ? last : -1, s.first = q0 < len ? a.sinks : 0;
  const int least = q0 + a.right < len - 1 ? q0 + a.right : len - 1;  // what the first of them sees
  s.set_full(q0 + 31 - a.left > 0 ? q0 + 31 - a.left : 0, q0 + 31 < len ? least - 31 : -1);
  return s;
}
// queries for the keys from k0
__device__ __forceinline__ Sights sights_of_keys(const Args &a, int len, int k0) {
  Sights s;
  s.low = k0 - a.right - 31, s.first = 0;
  s.high = k0 >= len ? -1 : k0 >= a.sinks && k0 + 31 + a.left < len - 1 ? k0 + 31 + a.left : len - 1;
  const int least = k0 + 31 >= a.sinks && k0 + a.left < len - 1 ? k0 + a.left : len - 1;
  s.set_full(k0 + 31 - a.right > 0 ? k0 + 31 - a.right : 0, k0 + 31 < len ? least - 31 : -1);
  return s;
}
// The rows that lie in a lane's sight: low .. high, and those below `first`
struct Span {
  int low, high, first;
  __device__ __forceinline__ bool sees(int r) const { return (r >= low && r <= high) || r < first; }
};
// what query i sees
__device__ __forceinline__ Span keys_of(const Args &a, int len, int i) {
  Span s;
  s.high = i + a.right < len - 1 ? i + a.right : len - 1;
  if (i < 0 || i >= len) s.high = -1;
  s.low = i - a.left > 0 ? i - a.left : 0;
  s.first = a.sinks < s.high + 1 ? a.sinks : s.high + 1;
  return s;
}
// the queries that see key j; of a sink all from low on
__device__ __forceinline__ Span queries_of(const Args &a, int len, int j) {
  Span s;
  s.low = j - a.right > 0 ? j - a.right : 0;
  s.high = j + a.left < len - 1 && j >= a.sinks ? j + a.left : len - 1;
  if (j >= len) s.high = -1;
  s.first = 0;
  return s;
}
// z <- instead where the row of a tile is out of sight; FIRST: some of its rows may be seen as first ones
template <bool FIRST>
__device__ __forceinline__ void hide_low(f32x16 &z, const Span &span, int r0, int g, float instead) {
  const int lo = span.low - r0 - 4 * g, of_first = span.first - r0 - 4 * g;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int n = 8 * (r >> 2) + (r & 3);
    z[r] = n >= lo || (FIRST && n < of_first) ? z[r] : instead;
  }
}
__device__ __forceinline__ void hide_high(f32x16 &z, const Span &span, int r0, int g, float instead) {
  const int hi = span.high - r0 - 4 * g;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 8 * (r >> 2) + (r & 3) <= hi ? z[r] : instead;
}
__device__ __forceinline__ void hide(f32x16 &z, const Span &span, int r0, int g, float instead) {
  if (some_lane(span.first > r0)) hide_low<true>(z, span, r0, g, instead);
  else if (some_lane(span.low > r0)) hide_low<false>(z, span, r0, g, instead);
  if (some_lane(span.high < r0 + 31)) hide_high(z, span, r0, g, instead);
}

// The key tiles of kt rows that queries from q0 to q1 of a sequence see: those of the sinks, then those of the window
struct Tiles {
  int sinks, first, count;
  __device__ __forceinline__ Tiles(const Args &a, int len, int q0, int q1, int kt) {
    const int lo = q0 - a.left > 0 ? q0 - a.left : 0;
    int hi = q1 + a.right;
    if (hi > len - 1) hi = len - 1;
    first = lo / kt;
    const int of_sinks = (a.sinks + kt - 1) / kt;
    sinks = of_sinks < first ? of_sinks : first;
    count = hi < lo ? 0 : sinks + hi / kt - first + 1;
  }
  __device__ __forceinline__ int operator[](int n) const { return n < sinks ? n : first + n - sinks; }
};

// ---- rows and their products ----
typedef short s16x4 __attribute__((ext_vector_type(4)));

// eight (bf16) or four (float32) neighbouring channels of a row, zeros from D on; rows may start on any element
typedef u32x4 unit_at4 __attribute__((aligned(4)));
typedef u32x4 unit_at2 __attribute__((aligned(2)));
template <class T>
using Piece = typename std::conditional<sizeof(T) == 4, unit_at4, unit_at2>::type;
template <class T>
__device__ __forceinline__ u32x4 load_piece(const T *row, int col, int D) {
  constexpr int V = 16 / sizeof(T);
  u32x4 w = {0u, 0u, 0u, 0u};
  if (col + V <= D) {
    w = *reinterpret_cast<const Piece<T> *>(row + col);
  } else if (col < D) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (sizeof(T) == 2) w[j / 2] |= (col + j < D ? (uint32_t)row[col + j].bits : 0u) << (16 * (j & 1));
      else w[j] = col + j < D ? __float_as_uint(row[col + j]) : 0u;
    }
  }
  return w;
}
// the same without a branch where D is whole pieces (PLAIN); zeros where not `there`: the row itself has to be readable all the same
template <bool PLAIN, class T>
__device__ __forceinline__ u32x4 load_some(const T *row, int col, int D, bool there) {
  u32x4 w;
  if constexpr (PLAIN) w = *reinterpret_cast<const Piece<T> *>(row + (col < D ? col : 0));
  else w = load_piece(row, col, D);
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = there && col < D ? w[k] : 0u;
  return w;
}
template <class T>
__device__ __forceinline__ void store_piece(T *row, int col, int D, const u32x4 &w) {
  constexpr int V = 16 / sizeof(T);
  if (col + V <= D) {
    *reinterpret_cast<Piece<T> *>(row + col) = w;
  } else if (col < D) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (col + j >= D) continue;
      if constexpr (sizeof(T) == 2) row[col + j].bits = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
      else row[col + j] = __uint_as_float(w[j]);
    }
  }
}

__device__ __forceinline__ float sum_of(const f32x16 &v) {
  float s[2] = {};
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r & 1] += v[r];
  return s[0] + s[1];
}

template <class T, int DP>
struct Ops;

template <int DP>
struct Ops<bf16, DP> {
  static constexpr int kStride = DP + 8;  // of a row in LDS, elements: 16-byte reads of neighbouring rows share no bank
  struct Rows {
    u32x4 v[DP / 16];
  };
  using Raw = Rows;  // as loaded
  struct Weights {
    u32x4 v[2];
  };
  // row n of a head's 0 .. limit - 1, zeros where not `there` (and from channel D on)
  template <bool PLAIN>
  static __device__ __forceinline__ Rows rows(const bf16 *head, int64_t stride, int n, int limit, bool there, int D, int g) {
    const bf16 *const row = head + (n < 0 ? 0 : n < limit ? n : limit - 1) * stride;
    Rows r;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) r.v[kk] = load_some<PLAIN>(row, 16 * kk + 8 * g, D, there);
    return r;
  }
  // Waits for the rows here: left to their first use, inside the loop, the wait would be for the next tile's loads, too
  static __device__ __forceinline__ Rows settle(Raw r) {
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) asm volatile("" : "+v"(r.v[kk]));
    return r;
  }
  static __device__ __forceinline__ float dot(const Rows &x, const Raw &y) {  // of this lane's channels
    float s = 0.f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t a = x.v[kk][w], b = y.v[kk][w];
        s = fmaf(__uint_as_float(a << 16), __uint_as_float(b << 16), s);
        s = fmaf(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u), s);
      }
    return s;
  }
  // acc[row of lds][lane's row] += product over the channels
  static __device__ __forceinline__ f32x16 scores(const bf16 *lds, const Rows &own, int i, int g, f32x16 acc, int) {
    const u32x4 *p = reinterpret_cast<const u32x4 *>(lds + i * kStride + 8 * g);
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) acc = mfma::mma(p[2 * kk], own.v[kk], acc);
    return acc;
  }
  static __device__ __forceinline__ f32x16 scores(const Rows &x, const Rows &own, f32x16 acc) {  // both in registers
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) acc = mfma::mma(x.v[kk], own.v[kk], acc);
    return acc;
  }
  static __device__ __forceinline__ Weights pack(const f32x16 &v) { return {{mfma::pack_half<0>(v), mfma::pack_half<1>(v)}}; }
  // sum of this lane's weights as they are multiplied
  static __device__ __forceinline__ float sum(const Weights &w, const f32x16 &) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 ones = {(__bf16)1.f, (__bf16)1.f};
    float s[2] = {};
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t word = w.v[q][k];
        s[q] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, word), ones, s[q], false);
      }
    return s[0] + s[1];
  }
  static __device__ __forceinline__ void put(bf16 *row, int col, const u32x4 &w) { *reinterpret_cast<u32x4 *>(row + col) = w; }
  // acc[channel][column] += sum over the 32 rows of lds.  The transposing read: in a group of 16 lanes, lane l addresses four
  // channels 4 (l % 4) .. of row l / 4 and receives channel l of the four rows.
  static __device__ __forceinline__ void outcome(const bf16 *lds, const Weights &w, int lane, f32x16 (&acc)[DP / 32]) {
    const int l = lane & 15, h = (lane >> 4) & 1, g = lane >> 5;
    const bf16 *p = lds + (4 * g + (l >> 2)) * kStride + 16 * h + 4 * (l & 3);
    typedef __attribute__((address_space(3))) s16x4 lds_piece;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        union {
          s16x4 h[2];
          u32x4 v;
        } x;
        x.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_piece *)(p + (16 * q) * kStride + 32 * db));
        x.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_piece *)(p + (16 * q + 8) * kStride + 32 * db));
        acc[db] = mfma::mma(x.v, w.v[q], acc[db]);
      }
  }
  // the same good to 2^-8 of the weights and the rows
  static __device__ __forceinline__ void outcome_coarse(const bf16 *lds, const f32x16 &v, int lane, f32x16 (&acc)[DP / 32]) { outcome(lds, pack(v), lane, acc); }
};

template <int DP>
struct Ops<float, DP> {
  static constexpr int kStride = DP + 4;
  struct Rows {
    float v[DP / 2];  // channels g DP / 2 ..
  };
  using Raw = Rows;
  struct Weights {
    f32x16 v;
  };
  template <bool PLAIN>
  static __device__ __forceinline__ Rows rows(const float *head, int64_t stride, int n, int limit, bool there, int D, int g) {
    const float *const row = head + (n < 0 ? 0 : n < limit ? n : limit - 1) * stride;
    Rows r;
#pragma unroll
    for (int k = 0; k < DP / 8; ++k) {
      const u32x4 w = load_some<PLAIN>(row, g * (DP / 2) + 4 * k, D, there);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t b = w[j];
        r.v[4 * k + j] = __uint_as_float(b);
      }
    }
    return r;
  }
  static __device__ __forceinline__ Rows settle(Raw r) {
#pragma unroll
    for (int k = 0; k < DP / 2; ++k) asm volatile("" : "+v"(r.v[k]));
    return r;
  }
  static __device__ __forceinline__ float dot(const Rows &x, const Rows &y) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < DP / 2; ++k) s = fmaf(x.v[k], y.v[k], s);
    return s;
  }
  static __device__ __forceinline__ f32x16 scores(const float *lds, const Rows &own, int i, int g, f32x16 acc, int) {
    const f32x4 *p = reinterpret_cast<const f32x4 *>(lds + i * kStride + g * (DP / 2));
#pragma unroll
    for (int k = 0; k < DP / 8; ++k) {
      const f32x4 x = p[k];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], own.v[4 * k + j], acc, 0, 0, 0);
    }
    return acc;
  }
  static __device__ __forceinline__ f32x16 scores(const Rows &x, const Rows &own, f32x16 acc) {
#pragma unroll
    for (int k = 0; k < DP / 2; ++k) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x.v[k], own.v[k], acc, 0, 0, 0);
    return acc;
  }
  static __device__ __forceinline__ Weights pack(const f32x16 &v) { return {v}; }
  static __device__ __forceinline__ float sum(const Weights &, const f32x16 &v) { return sum_of(v); }
  static __device__ __forceinline__ void put(float *row, int col, const u32x4 &w) { *reinterpret_cast<u32x4 *>(row + col) = w; }
  static __device__ __forceinline__ void outcome(const float *lds, const Weights &w, int lane, f32x16 (&acc)[DP / 32]) {
    const float *p = lds + 4 * (lane >> 5) * kStride + (lane & 31);
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(p[(8 * (r >> 2) + (r & 3)) * kStride + 32 * db], w.v[r], acc[db], 0, 0, 0);
  }
  static __device__ __forceinline__ void outcome_coarse(const float *lds, const f32x16 &v, int lane, f32x16 (&acc)[DP / 32]) { outcome(lds, pack(v), lane, acc); }
};

// Float32 rows for the bf16 matrix instructions: a value is three bf16 values, each the rounding of what the ones before leave over, which
// together hold all of its 24 bits; a . b is a1 b1 + a1 b2 + a2 b1 + a2 b2 + a1 b3 + a3 b1, and what is dropped is below 2^-24 |a| |b|.  A
// product of 32 x 32 over 16 takes 48 passes of the matrix unit against 128 by v_mfma_f32_32x32x2_f32, and a width of 16 one step of 16 (4 x 7 225 x 8 x 16,
// 171 keys, when it was taken: forward 92 -> 66 us, queries 123 -> 78, keys 156 -> 101, today 67, 91, 108; 20 000 x 4 x 64, 401 keys: 140 -> 98, 197 -> 131,
// 269 -> 175, today 93, 161, 184).
struct Thirds {
  uint32_t w[3];  // of two neighbouring values
};
// INNER: what is known to be finite.  Otherwise an infinity or NaN is in the first alone, so that the others give it back.
template <bool INNER>
__device__ __forceinline__ Thirds thirds_of(float x, float y) {
  Thirds t;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    t.w[k] = mfma::pack2(x, y);
    if (k == 2) break;
    x -= __uint_as_float(t.w[k] << 16);
    y -= __uint_as_float(t.w[k] & 0xffff0000u);
    if (!INNER) x = x == x ? x : 0.f, y = y == y ? y : 0.f;
  }
  return t;
}

template <int DP>
struct Split {
  static constexpr int kPlane = DP + 8, kStride = 3 * kPlane / 2;  // of a row's third in LDS in bf16, of the row in floats
  using Raw = struct {
    u32x4 v[DP / 8];  // channels 16 k + 8 g .. + 3 and + 4 .. + 7
  };
  struct Rows {
    u32x4 v[3][DP / 16];
  };
  struct Weights {
    u32x4 v[3][2];
  };
  template <bool PLAIN>
  static __device__ __forceinline__ Raw rows(const float *head, int64_t stride, int n, int limit, bool there, int D, int g) {
    const float *const row = head + (n < 0 ? 0 : n < limit ? n : limit - 1) * stride;
    Raw r;
#pragma unroll
    for (int k = 0; k < DP / 8; ++k) r.v[k] = load_some<PLAIN>(row, 16 * (k >> 1) + 8 * g + 4 * (k & 1), D, there);
    return r;
  }
  static __device__ __forceinline__ Rows settle(const Raw &r) {
    Rows s;
#pragma unroll
    for (int k = 0; k < DP / 8; ++k)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t x = r.v[k][2 * w], y = r.v[k][2 * w + 1];
        const Thirds t = thirds_of<false>(__uint_as_float(x), __uint_as_float(y));
#pragma unroll
        for (int p = 0; p < 3; ++p) s.v[p][k >> 1][2 * (k & 1) + w] = t.w[p];
      }
#pragma unroll
    for (int p = 0; p < 3; ++p)
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) asm volatile("" : "+v"(s.v[p][kk]));
    return s;
  }
  static __device__ __forceinline__ float dot(const Rows &x, const Raw &y) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < DP / 8; ++k)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float v = 0.f;
#pragma unroll
        for (int p = 2; p >= 0; --p) {  // exact in this order
          const uint32_t two = x.v[p][k >> 1][2 * (k & 1) + (w >> 1)];
          v += __uint_as_float(w & 1 ? two & 0xffff0000u : two << 16);
        }
        const uint32_t b = y.v[k][w];
        s = fmaf(v, __uint_as_float(b), s);
      }
    return s;
  }
  // the small ones first
  static __device__ __forceinline__ f32x16 products(const u32x4 (&a)[3], const u32x4 &b0, const u32x4 &b1, const u32x4 &b2, f32x16 acc) {
    acc = mfma::mma(a[2], b0, acc);
    acc = mfma::mma(a[0], b2, acc);
    acc = mfma::mma(a[1], b1, acc);
    acc = mfma::mma(a[1], b0, acc);
    acc = mfma::mma(a[0], b1, acc);
    return mfma::mma(a[0], b0, acc);
  }
  static __device__ __forceinline__ f32x16 scores(const float *lds, const Rows &own, int i, int g, f32x16 acc, int D) {
    const uint16_t *const p = reinterpret_cast<const uint16_t *>(lds + i * kStride) + 8 * g;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      if (kk % 2 == 1 && 16 * kk >= D) break;  // the upper half of 32 channels is empty
      u32x4 a[3];
#pragma unroll
      for (int q = 0; q < 3; ++q) a[q] = *reinterpret_cast<const u32x4 *>(p + q * kPlane + 16 * kk);
      acc = products(a, own.v[0][kk], own.v[1][kk], own.v[2][kk], acc);
    }
    return acc;
  }
  static __device__ __forceinline__ Weights pack(const f32x16 &v) {
    Weights w;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const Thirds t = thirds_of<true>(v[2 * k], v[2 * k + 1]);
#pragma unroll
      for (int p = 0; p < 3; ++p) w.v[p][k >> 2][k & 3] = t.w[p];
    }
    return w;
  }
  static __device__ __forceinline__ float sum(const Weights &, const f32x16 &v) { return sum_of(v); }
  static __device__ __forceinline__ void put(float *row, int col, const u32x4 &w) {
    const uint32_t x0 = w[0], x1 = w[1], x2 = w[2], x3 = w[3];
    const Thirds t = thirds_of<false>(__uint_as_float(x0), __uint_as_float(x1)), u = thirds_of<false>(__uint_as_float(x2), __uint_as_float(x3));
#pragma unroll
    for (int p = 0; p < 3; ++p) *reinterpret_cast<mfma::u32x2 *>(reinterpret_cast<uint16_t *>(row) + p * kPlane + col) = mfma::u32x2{t.w[p], u.w[p]};
  }
  static __device__ __forceinline__ void outcome(const float *lds, const Weights &w, int lane, f32x16 (&acc)[DP / 32]) {
    const int l = lane & 15, h = (lane >> 4) & 1, g = lane >> 5;
    const uint16_t *const p = reinterpret_cast<const uint16_t *>(lds + (4 * g + (l >> 2)) * kStride) + 16 * h + 4 * (l & 3);
    typedef __attribute__((address_space(3))) s16x4 lds_piece;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        u32x4 a[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          union {
            s16x4 h[2];
            u32x4 v;
          } x;
          x.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_piece *)(p + (16 * q) * 2 * kStride + k * kPlane + 32 * db));
          x.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_piece *)(p + (16 * q + 8) * 2 * kStride + k * kPlane + 32 * db));
          a[k] = x.v;
        }
        acc[db] = products(a, w.v[0][q], w.v[1][q], w.v[2][q], acc[db]);
      }
  }
  // of the first parts alone
  static __device__ __forceinline__ void outcome_coarse(const float *lds, const f32x16 &v, int lane, f32x16 (&acc)[DP / 32]) {
    const int l = lane & 15, h = (lane >> 4) & 1, g = lane >> 5;
    const uint16_t *const p = reinterpret_cast<const uint16_t *>(lds + (4 * g + (l >> 2)) * kStride) + 16 * h + 4 * (l & 3);
    const u32x4 w[2] = {mfma::pack_half<0>(v), mfma::pack_half<1>(v)};
    typedef __attribute__((address_space(3))) s16x4 lds_piece;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        union {
          s16x4 h[2];
          u32x4 v;
        } x;
        x.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_piece *)(p + (16 * q) * 2 * kStride + 32 * db));
        x.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_piece *)(p + (16 * q + 8) * 2 * kStride + 32 * db));
        acc[db] = mfma::mma(x.v, w[q], acc[db]);
      }
  }
};
// what the kernels over windows multiply with: float32 rows of 128 channels leave no room for thirds beside the bias tables
template <class T, int DP>
using WindowOps = typename std::conditional<sizeof(T) == 4 && DP <= 64, Split<(DP <= 64 ? DP : 64)>, Ops<T, DP>>::type;

// ROWS rows of DP channels on their way from memory to LDS by THREADS threads: loaded into registers, written later.  PLAIN rows come by
// buffer loads: a lane's offsets in a tile never change, the tile's place is in scalar registers, and what lies outside reads as zero without a
// comparison.  All of an offset is in the vector register: the scalar one takes no part in the comparison with the buffer's size.  Others by
// element where a piece is not whole.
template <class O, class T, int DP, bool PLAIN, int ROWS, int THREADS>
struct Stage {
  static constexpr int V = 16 / sizeof(T), PER_ROW = DP / V, UNITS = ROWS * PER_ROW / THREADS;
  static_assert(ROWS * PER_ROW % THREADS == 0 && THREADS % PER_ROW == 0, "whole units a thread");
  u32x4 w[UNITS];
  // rows first .. first + ROWS - 1 of a head, of which 0 .. limit - 1 are there
  __device__ __forceinline__ void load(const View &view, const T *head, int first, int limit, int D, int tid) {
    if constexpr (PLAIN) {
      const int left = limit - first, bytes = (int)view.row * (int)sizeof(T), col = tid % PER_ROW * V;
      const __amdgpu_buffer_rsrc_t src = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<T *>(head + first * view.row), 0, left <= 0 ? 0 : (left < ROWS ? left : ROWS) * bytes, 0x00027000);
      // rows are below 2^22 bytes (make_view) and at most 64: what starts at 2^31 - 16 stays outside for every unit
      uint32_t at = col < D ? (uint32_t)(tid / PER_ROW * bytes + col * (int)sizeof(T)) : 0x7ffffff0u;
      asm volatile("" : "+v"(at));  // the units' offsets are formed here, not kept in a register each around the loop
#pragma unroll
      for (int u = 0; u < UNITS; ++u) w[u] = __builtin_amdgcn_raw_buffer_load_b128(src, at + (uint32_t)(u * (THREADS / PER_ROW) * bytes), 0, 0);
    } else {
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int at = tid + u * THREADS, row = first + at / PER_ROW, col = at % PER_ROW * V;
        w[u] = u32x4{0u, 0u, 0u, 0u};
        if (row < limit) w[u] = load_piece(head + row * view.row, col, D);
      }
    }
  }
  __device__ __forceinline__ void store(T *lds, int tid) const {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int at = tid + u * THREADS;
      O::put(lds + at / PER_ROW * O::kStride, at % PER_ROW * V, w[u]);
    }
  }
};

template <class T>
__device__ __forceinline__ const T *head_of(const View &v, int b, int h) {
  return static_cast<const T *>(v.data) + b * v.batch + h * v.head;
}

// acc[channel][lane's row] to the row, scaled; zeros where not `some`
template <class T, int DP>
__device__ __forceinline__ void store_rows(f32x16 (&acc)[DP / 32], float scale, bool some, T *row, bool there, int D, int g) {
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) {
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] = some ? acc[db][r] * scale : 0.f;
    if constexpr (sizeof(T) == 2) {
      u32x4 s0, s1;
      mfma::tile_natural(acc[db], s0, s1);
      if (there) store_piece(row, 32 * db + 16 * g, D, s0), store_piece(row, 32 * db + 16 * g + 8, D, s1);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(acc[db][4 * q + j]);
        if (there) store_piece(row, 32 * db + 8 * q + 4 * g, D, w);
      }
    }
  }
}

// What a lane's row does not see has no part in its sum, but a product multiplies it by zero: an infinity or NaN leaves NaN.  Sums that are not
// finite are formed again from what is seen alone, row by row, which costs its time only where there are such.
template <int N>
__device__ __forceinline__ bool not_finite(const f32x16 (&acc)[N]) {
  float s = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) s = fmaf(acc[n][r], 0.f, s);
  return s != s;
}
// acc += weight(n, seen) row n of a head, for rows first .. last, in the lanes that see it and are `bad`; on(): whether a lane goes on with sums that are all NaN
struct Nothing {
  __device__ __forceinline__ bool operator()() const { return false; }
};
template <class T, int DP, class F, class W = Nothing>
__device__ __forceinline__ void add_rows(const T *head, int64_t stride, int first, int last, int D, int g, bool bad, f32x16 (&acc)[DP / 32], F &&weight,
                                         W &&on = W()) {
#pragma unroll 1
  for (int n = first; n <= last; ++n) {
    bool seen;
    const float w = weight(n, seen);
    const T *const row = head + n * stride;
    bool open = on();  // or some of the lane's sums are not NaN
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int col = 32 * db + rowmap(r, g);
        const float x = col < D ? load_as_f32(row + col) : 0.f;
        acc[db][r] = bad && seen ? fmaf(w, x, acc[db][r]) : acc[db][r];
        open |= col < D && acc[db][r] == acc[db][r];
        if (r % 4 == 3) asm volatile("" ::: "memory");  // few loads at a time, to cost the paths beside it fewer registers
      }
    if (!some_lane(bad && open)) return;  // NaN whatever follows: an input full of them takes no longer for it
  }
}
__device__ __forceinline__ float bias_at(const BiasArgs &b, const float *table, int off) {
  const int low = table_low(b), at = off + low, n = table_size(b);
  return table[at < 0 ? 0 : at < n ? at : n - 1];
}

template <int N>
__device__ __forceinline__ void zero(f32x16 (&acc)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[n][r] = 0.f;
}

// rows of a tile in LDS at a time, in sub-tiles of 32: two buffers of two tensors leave room for two workgroups a CU (float32 rows of 128
// channels: for one)
template <class T, int DP>
constexpr int tile_rows() {
  return sizeof(T) == 4 ? 32 : 64;
}

// f(std::integral_constant<int, DP>{}, std::bool_constant<PLAIN>{}) for the padded width of D channels
template <class F>
int by_width(int D, bool plain, F &&f) {
  auto with = [&](auto dp) { return plain ? f(dp, std::true_type{}) : f(dp, std::false_type{}); };
  if (D <= 32) return with(std::integral_constant<int, 32>{});
  if (D <= 64) return with(std::integral_constant<int, 64>{});
  return with(std::integral_constant<int, 128>{});
}

// host
Args make_args(const pa_window_params &p);
// rows that the buffer loads take: whole 16-byte pieces on 4-byte boundaries, rows apart and no further than 2^31 bytes a tile
inline View make_view(const pa_heads &h, int64_t D, int64_t elem) {
  const bool plain = D * elem % 16 == 0 && reinterpret_cast<uintptr_t>(h.data) % 4 == 0 && h.batch * elem % 4 == 0 && h.row * elem % 4 == 0 &&
                     h.head * elem % 4 == 0 && h.row >= D && h.row <= (1 << 20);
  return {h.data, h.batch, h.row, h.head, plain};
}

}  // namespace window
}  // namespace pa
