// What the kernels of attention over a window share: arguments, visibility, the bias by buckets, tiles of rows in LDS and their
// products.
//
// All products run on 32 x 32 tiles of (rows in LDS) x (rows that a lane holds in registers), so that a lane keeps one query (or, in
// the gradients of keys and values, one key) and the softmax needs no exchange but that between the two half-waves:
//   scores   z[r][i] = sum_d X[r][d] own_i[d]        X: 32 rows in LDS, A operands as they lie; own: B operands
//   outcome  o[d][i] = sum_r X[r][d] w[r][i]         w: the weights of the tile, packed where they were formed (a C tile is a pair
//                                                    of B operands in the order rowmap); X transposed: bf16 by the transposing LDS
//                                                    read, float32 element by element (lanes run along d: no conflicts)
// bf16 rows go through v_mfma_f32_32x32x16_bf16, float32 rows through v_mfma_f32_32x32x2_f32.
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
  bool units;  // every row of a head is whole 16-byte units on 16-byte boundaries
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
  int sink_chunks;  // parts of the queries of a key block with sinks
  bool out_units;   // rows of the results are whole 16-byte units
};

__device__ __forceinline__ int length_of(const Args &a, int b) {
  if (!a.lengths) return a.N;
  const int n = a.lengths[b];
  return n < 0 ? 0 : n > a.N ? a.N : n;
}

// Workgroup -> work: consecutive work on one XCD (workgroups go round them), whose L2 then holds what neighbours share
__device__ __forceinline__ int64_t own_work() {
  const int64_t n = gridDim.x, id = blockIdx.x, per = n / 8, rest = n % 8, xcd = id % 8, slot = id / 8;
  return xcd < rest ? xcd * (per + 1) + slot : rest * (per + 1) + (xcd - rest) * per + slot;
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
// to log2 units; finite values stay finite, so that a bias of the lowest float leaves what the softmax of such scores is
__device__ __forceinline__ float bias_log2(float v) {
  const float s = v * kLog2e;
  return fabsf(v) < INFINITY ? fminf(fmaxf(s, -3.0e38f), 3.0e38f) : s;
}
__device__ __forceinline__ void fill_bias_table(const Args &a, int head, float *lds) {
  const int low = table_low(a.bias), n = table_size(a.bias);
  for (int u = threadIdx.x; u < n; u += blockDim.x)
    lds[u] = bias_log2(a.bias.table[(int64_t)bucket_of_offset(a.bias, u - low) * a.Hq + head]);
}
// where a 32 x 32 tile's offsets lie, least and most of them
enum Reach { kNear, kFarBehind, kFarAhead };
__device__ __forceinline__ Reach reach_of(const BiasArgs &b, int least, int most) {
  if (most <= -b.distance) return kFarBehind;
  if (b.both && least >= b.distance) return kFarAhead;
  return kNear;
}

// ---- visibility of 32 keys from k0 for 32 queries from q0 ----
enum Sight { kNone, kSome, kAll };
__device__ __forceinline__ Sight sight_of(const Args &a, int len, int q0, int k0) {
  if (k0 >= len || q0 >= len || k0 > q0 + 31 + a.right || (k0 + 31 < q0 - a.left && k0 >= a.sinks)) return kNone;
  if (k0 + 31 < len && q0 + 31 < len && k0 + 31 <= q0 + a.right && (k0 >= q0 + 31 - a.left || k0 + 31 < a.sinks)) return kAll;
  return kSome;
}
__device__ __forceinline__ bool sees(const Args &a, int len, int i, int j) {
  return j < len && i < len && j <= i + a.right && (j >= i - a.left || j < a.sinks);
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

// eight (bf16) or four (float32) neighbouring channels of a row, zeros from D on
template <class T>
__device__ __forceinline__ u32x4 load_piece(const T *row, int col, int D, bool units) {
  constexpr int V = 16 / sizeof(T);
  u32x4 w = {0u, 0u, 0u, 0u};
  if (units) {
    if (col < D) w = *reinterpret_cast<const u32x4 *>(row + col);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (sizeof(T) == 2) w[j / 2] |= (col + j < D ? (uint32_t)row[col + j].bits : 0u) << (16 * (j & 1));
      else w[j] = col + j < D ? __float_as_uint(row[col + j]) : 0u;
    }
  }
  return w;
}

template <class T, int DP>
struct Ops;

template <int DP>
struct Ops<bf16, DP> {
  static constexpr int kStride = DP + 8;  // of a row in LDS, elements: 16-byte reads of neighbouring rows share no bank
  struct Rows {
    u32x4 v[DP / 16];
  };
  struct Weights {
    u32x4 v[2];
  };
  static __device__ __forceinline__ Rows rows(const bf16 *row, bool there, int D, bool units, int g) {
    Rows r;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      r.v[kk] = u32x4{0u, 0u, 0u, 0u};
      if (there) r.v[kk] = load_piece(row, 16 * kk + 8 * g, D, units);
    }
    return r;
  }
  static __device__ __forceinline__ float dot(const Rows &x, const Rows &y) {  // of this lane's channels
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
  static __device__ __forceinline__ f32x16 scores(const bf16 *lds, const Rows &own, int i, int g, f32x16 acc) {
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
};

template <int DP>
struct Ops<float, DP> {
  static constexpr int kStride = DP + 4;
  struct Rows {
    float v[DP / 2];  // channels g DP / 2 ..
  };
  struct Weights {
    f32x16 v;
  };
  static __device__ __forceinline__ Rows rows(const float *row, bool there, int D, bool units, int g) {
    Rows r;
#pragma unroll
    for (int k = 0; k < DP / 8; ++k) {
      u32x4 w = {0u, 0u, 0u, 0u};
      if (there) w = load_piece(row, g * (DP / 2) + 4 * k, D, units);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t b = w[j];
        r.v[4 * k + j] = __uint_as_float(b);
      }
    }
    return r;
  }
  static __device__ __forceinline__ float dot(const Rows &x, const Rows &y) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < DP / 2; ++k) s = fmaf(x.v[k], y.v[k], s);
    return s;
  }
  static __device__ __forceinline__ f32x16 scores(const float *lds, const Rows &own, int i, int g, f32x16 acc) {
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
  static __device__ __forceinline__ void outcome(const float *lds, const Weights &w, int lane, f32x16 (&acc)[DP / 32]) {
    const float *p = lds + 4 * (lane >> 5) * kStride + (lane & 31);
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(p[(8 * (r >> 2) + (r & 3)) * kStride + 32 * db], w.v[r], acc[db], 0, 0, 0);
  }
};

// ROWS rows of DP channels on their way from memory to LDS by THREADS threads: loaded into registers, written later
template <class T, int DP, int ROWS, int THREADS>
struct Stage {
  static constexpr int V = 16 / sizeof(T), PER_ROW = DP / V, UNITS = ROWS * PER_ROW / THREADS;
  static_assert(ROWS * PER_ROW % THREADS == 0, "whole units a thread");
  u32x4 w[UNITS];
  // rows first .. first + ROWS - 1 of a head; zeros outside 0 .. limit - 1
  __device__ __forceinline__ void load(const View &view, const T *head, int first, int limit, int D, int tid) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int at = tid + u * THREADS, row = first + at / PER_ROW, col = at % PER_ROW * V;
      w[u] = u32x4{0u, 0u, 0u, 0u};
      if (row >= 0 && row < limit) w[u] = load_piece(head + row * view.row, col, D, view.units);
    }
  }
  __device__ __forceinline__ void store(T *lds, int tid) const {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int at = tid + u * THREADS;
      *reinterpret_cast<u32x4 *>(lds + at / PER_ROW * Ops<T, DP>::kStride + at % PER_ROW * V) = w[u];
    }
  }
};

template <class T>
__device__ __forceinline__ const T *head_of(const View &v, int b, int h) {
  return static_cast<const T *>(v.data) + b * v.batch + h * v.head;
}

// acc[channel][lane's row] to the row, scaled; zeros where not `some`
template <class T, int DP>
__device__ __forceinline__ void store_rows(f32x16 (&acc)[DP / 32], float scale, bool some, T *row, bool there, int D, bool units, int g) {
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) {
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] = some ? acc[db][r] * scale : 0.f;
    if constexpr (sizeof(T) == 2) {
      if (units) {
        u32x4 s0, s1;
        mfma::tile_natural(acc[db], s0, s1);
        const int col = 32 * db + 16 * g;
        uint16_t *out = reinterpret_cast<uint16_t *>(row);
        if (there && col < D) *reinterpret_cast<u32x4 *>(out + col) = s0;
        if (there && col + 8 < D) *reinterpret_cast<u32x4 *>(out + col + 8) = s1;
        continue;
      }
    } else {
      if (units) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int col = 32 * db + 8 * q + 4 * g;
          if (there && col < D) *reinterpret_cast<f32x4 *>(row + col) = f32x4{acc[db][4 * q], acc[db][4 * q + 1], acc[db][4 * q + 2], acc[db][4 * q + 3]};
        }
        continue;
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int col = 32 * db + rowmap(r, g);
      if (there && col < D) store_from_f32(row + col, acc[db][r]);
    }
  }
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
  return sizeof(T) == 4 && DP == 128 ? 32 : 64;
}

// f(std::integral_constant<int, DP>{}) for the padded width of D channels
template <class F>
int by_width(int D, F &&f) {
  if (D <= 32) return f(std::integral_constant<int, 32>{});
  if (D <= 64) return f(std::integral_constant<int, 64>{});
  return f(std::integral_constant<int, 128>{});
}

// host
Args make_args(int dtype, const pa_window_params &p);
View make_view(int dtype, const pa_heads &h, int64_t D);

}  // namespace window
}  // namespace pa
