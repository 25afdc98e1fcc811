// Dropout, residual add and LayerNorm of rows in one pass, forward and backward, with a mask that is formed from a counter on
// both ways and never stored:
//   y = residual + keep x / (1 - p),  n = (y - mean) rstd gamma + beta
//   ds = dy + rstd (t - mean_c(t) - xh mean_c(t xh)),  t = dn gamma,  xh = (s - mean) rstd,  s the sum before its rounding to y
//   d residual = ds,  dx = keep ds / (1 - p),  d gamma = sum_rows dn xh,  d beta = sum_rows dn
// keep(r, c): word c % 4 of Philox4x32-10 (J. K. Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", SC 2011) of the
// counter (c / 4, r mod 2^32, r / 2^32, offset) under the 64-bit seed is at least p 2^32.  It depends on the element's place
// alone, not on types, alignment or launches.  Seed and offset are read from device memory, so that a captured graph draws a
// new mask on every replay when the offset is advanced in it.
//
// Sums, statistics and all arithmetic are float32.  n is formed from the sum before its rounding to y, and the backward pass forms
// that sum again from x and the residual, which costs one read more than y and keeps d gamma as exact as float32 sums are (from
// the rounded y: 2e-3 off).
#include "pa_common.h"
#include "pa_host.h"
#include "pa_mfma_ops.h"

namespace pa {
namespace dropout {

using mfma::u32x2;
using mfma::u32x4;

struct Words {
  uint32_t w[4];
};
__device__ __forceinline__ Words philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

struct Mask {
  const int64_t *rng;  // seed, offset
  uint32_t threshold;  // kept: word >= threshold
  bool none;           // p = 1: nothing is kept
  bool all;            // p = 0
  float scale;
};
struct Stream {
  uint32_t k0, k1, offset;
};
__device__ __forceinline__ Stream stream_of(const Mask &m) {
  const uint64_t seed = (uint64_t)m.rng[0];
  return {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)m.rng[1]};
}
// which of the VEC columns from col (a multiple of 4) of a row are kept, a bit each
template <int VEC>
__device__ __forceinline__ uint32_t kept(const Mask &m, const Stream &s, int64_t row, int col) {
  if (m.all) return 0xffu;
  if (m.none) return 0u;
  uint32_t bits = 0;
#pragma unroll
  for (int q = 0; q < VEC / 4; ++q) {
    const Words w = philox((uint32_t)(col >> 2) + q, (uint32_t)row, (uint32_t)((uint64_t)row >> 32), s.offset, s.k0, s.k1);
#pragma unroll
    for (int j = 0; j < 4; ++j) bits |= w.w[j] >= m.threshold ? 1u << (4 * q + j) : 0u;
  }
  return bits;
}
// v[j] <- keep ? v[j] * scale : 0
template <int VEC>
__device__ __forceinline__ void apply(uint32_t bits, float scale, float (&v)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) v[j] = bits >> j & 1u ? v[j] * scale : 0.f;
}

// ---- VEC neighbouring elements of a row, 16 bytes; UNITS: rows are whole 16-byte units.  Rows that are not start on any
// element: the same 16-byte accesses without that alignment, element by element at a row's end ----
typedef u32x4 unit_at4 __attribute__((aligned(4)));
typedef u32x4 unit_at2 __attribute__((aligned(2)));
template <class T, bool UNITS>
using UnitAt = typename std::conditional<UNITS, u32x4, typename std::conditional<sizeof(T) == 4, unit_at4, unit_at2>::type>::type;

template <class T, int VEC, bool UNITS>
__device__ __forceinline__ void load(const T *row, int col, int C, float (&v)[VEC]) {
  static_assert(VEC * sizeof(T) == 16, "one access");
  typedef UnitAt<T, UNITS> unit_at;
  u32x4 w = {0u, 0u, 0u, 0u};
  if (UNITS ? col < C : col + VEC <= C) {
    w = __builtin_nontemporal_load(reinterpret_cast<const unit_at *>(row + col));
  } else if (!UNITS && col < C) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if constexpr (sizeof(T) == 2) w[j / 2] |= (col + j < C ? (uint32_t)row[col + j].bits : 0u) << (16 * (j & 1));
      else w[j] = col + j < C ? __float_as_uint(row[col + j]) : 0u;
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    if constexpr (sizeof(T) == 2) {
      const uint32_t b = w[j / 2];
      v[j] = __uint_as_float(j & 1 ? b & 0xffff0000u : b << 16);
    } else {
      const uint32_t b = w[j];
      v[j] = __uint_as_float(b);
    }
  }
}
template <class T, int VEC, bool UNITS>
__device__ __forceinline__ void store(T *row, int col, int C, const float (&v)[VEC]) {
  typedef UnitAt<T, UNITS> unit_at;
  if (UNITS ? col < C : col + VEC <= C) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 2) w[j] = mfma::pack2(v[2 * j], v[2 * j + 1]);
      else w[j] = __float_as_uint(v[j]);
    }
    __builtin_nontemporal_store(w, reinterpret_cast<unit_at *>(row + col));
  } else if (!UNITS) {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (col + j < C) store_from_f32(row + col + j, v[j]);
  }
}

// sum over groups of LANES neighbouring lanes, in every lane
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  auto step = [](float x, auto ctrl) {
    constexpr int c = decltype(ctrl)::value;
    return x + __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(x), c, 0xf, 0xf, true));
  };
  if constexpr (LANES >= 2) v = step(v, std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  if constexpr (LANES >= 4) v = step(v, std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  if constexpr (LANES >= 8) v = step(v, std::integral_constant<int, 0x141>{});  // row_half_mirror
  if constexpr (LANES >= 16) v = step(v, std::integral_constant<int, 0x140>{}); // row_mirror
  if constexpr (LANES >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (LANES >= 64) v = mfma::half_sum(v);
  return v;
}

// the same over the 256 lanes of a workgroup, through four floats of LDS; all of it calls this
template <int LANES>
__device__ __forceinline__ float group_sum(float v, float *red) {
  if constexpr (LANES <= 64) return lanes_sum<LANES>(v);
  v = lanes_sum<64>(v);
  __syncthreads();  // the sum before has been read
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

struct Args {
  const void *x, *residual, *dy, *dn;
  void *out_y, *out_n, *dx, *d_residual;
  const float *gamma, *beta;
  float *stats;     // (M, 2): mean, rstd
  float *partials;  // [workgroup][2][C]
  float eps;
  int64_t M;
  int C;
  Mask mask;
};

// ---------------------------------------------------------------------------------------------------------------
// rows_forward_kernel, rows_backward_kernel.  LANES lanes (256: the workgroup) share a row, each NCH pieces of VEC neighbouring columns, so that a row
// is read once and stays in registers; a workgroup of four waves walks the rows.  In the backward pass a lane adds d gamma and d beta
// of its columns up over all its rows; the workgroup's sums become one partial result, added up in a fixed order by one more
// small launch.  Bound by HBM: (3 + norm) element reads and writes forward, 6 backward; the generator's twenty 32 x 32 bit
// products per four elements run behind them.
// ---------------------------------------------------------------------------------------------------------------
template <class T, int VEC, bool UNITS, int LANES, int NCH, bool NORM>
__global__ __launch_bounds__(256) void rows_forward_kernel(Args a) {
  __shared__ float wide[4];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  constexpr int ROWS = 256 / LANES;
  const int C = a.C;
  const float inv = 1.f / (float)C;
  const Stream rng = stream_of(a.mask);
  float gamma[NCH][VEC], beta[NCH][VEC];
  if constexpr (NORM) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int col = (k * LANES + lane) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        gamma[k][j] = col + j < C ? a.gamma[col + j] : 0.f;
        beta[k][j] = col + j < C ? a.beta[col + j] : 0.f;
      }
    }
  }
  for (int64_t row = (int64_t)blockIdx.x * ROWS + group; row < a.M; row += (int64_t)gridDim.x * ROWS) {
    const int64_t at = row * C;
    float s[NCH][VEC];
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int col = (k * LANES + lane) * VEC;
      float r[VEC];
      load<T, VEC, UNITS>(static_cast<const T *>(a.x) + at, col, C, s[k]);
      if (a.residual) load<T, VEC, UNITS>(static_cast<const T *>(a.residual) + at, col, C, r);
      apply(kept<VEC>(a.mask, rng, row, col), a.mask.scale, s[k]);
      if (a.residual) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[k][j] += r[j];
      }
      store<T, VEC, UNITS>(static_cast<T *>(a.out_y) + at, col, C, s[k]);
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum += s[k][j];
    }
    if constexpr (NORM) {
      const float mean = group_sum<LANES>(sum, wide) * inv;
      float sq = 0.f;
#pragma unroll
      for (int k = 0; k < NCH; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = (k * LANES + lane) * VEC + j < C ? s[k][j] - mean : 0.f;
          sq = fmaf(d, d, sq);
        }
      const float rstd = 1.f / sqrtf(group_sum<LANES>(sq, wide) * inv + a.eps);
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        float n[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) n[j] = fmaf((s[k][j] - mean) * rstd, gamma[k][j], beta[k][j]);
        store<T, VEC, UNITS>(static_cast<T *>(a.out_n) + at, (k * LANES + lane) * VEC, C, n);
      }
      if (a.stats && lane == 0) a.stats[2 * row] = mean, a.stats[2 * row + 1] = rstd;
    }
  }
}

template <class T, int VEC, bool UNITS, int LANES, int NCH, bool NORM>
__global__ __launch_bounds__(256) void rows_backward_kernel(Args a) {
  constexpr int ROWS = 256 / LANES, WIDE = LANES * NCH * VEC;
  __shared__ float red[NORM && LANES <= 64 ? 4 * WIDE : 4];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int C = a.C;
  const float inv = 1.f / (float)C;
  const Stream rng = stream_of(a.mask);
  float gamma[NCH][VEC], dg[NCH][VEC], db[NCH][VEC];
  if constexpr (NORM) {
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int col = (k * LANES + lane) * VEC + j;
        gamma[k][j] = col < C ? a.gamma[col] : 0.f;
        dg[k][j] = db[k][j] = 0.f;
      }
  }
  for (int64_t row = (int64_t)blockIdx.x * ROWS + group; row < a.M; row += (int64_t)gridDim.x * ROWS) {
    const int64_t at = row * C;
    float ds[NCH][VEC];
    uint32_t bits[NCH];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int col = (k * LANES + lane) * VEC;
      if (a.dy) {
        load<T, VEC, UNITS>(static_cast<const T *>(a.dy) + at, col, C, ds[k]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) ds[k][j] = 0.f;
      }
    }
    if constexpr (NORM) {
      float t[NCH][VEC], xh[NCH][VEC];
      const float mean = a.stats[2 * row], rstd = a.stats[2 * row + 1];
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        const int col = (k * LANES + lane) * VEC;
        float r[VEC];
        load<T, VEC, UNITS>(static_cast<const T *>(a.x) + at, col, C, xh[k]);
        load<T, VEC, UNITS>(static_cast<const T *>(a.dn) + at, col, C, t[k]);
        if (a.residual) load<T, VEC, UNITS>(static_cast<const T *>(a.residual) + at, col, C, r);
        bits[k] = kept<VEC>(a.mask, rng, row, col);
        apply(bits[k], a.mask.scale, xh[k]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          xh[k][j] = ((a.residual ? xh[k][j] + r[j] : xh[k][j]) - mean) * rstd;
          dg[k][j] = fmaf(t[k][j], xh[k][j], dg[k][j]);
          db[k][j] += t[k][j];
          t[k][j] *= gamma[k][j];  // 0 past the last column
          s1 += t[k][j];
          s2 = fmaf(t[k][j], xh[k][j], s2);
        }
      }
      s1 = group_sum<LANES>(s1, red) * inv;
      s2 = group_sum<LANES>(s2, red) * inv;
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) ds[k][j] = fmaf(rstd, t[k][j] - s1 - xh[k][j] * s2, ds[k][j]);
        if (a.d_residual) store<T, VEC, UNITS>(static_cast<T *>(a.d_residual) + at, (k * LANES + lane) * VEC, C, ds[k]);
      }
    }
    if (a.dx) {
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        const int col = (k * LANES + lane) * VEC;
        if constexpr (!NORM) bits[k] = kept<VEC>(a.mask, rng, row, col);
        apply(bits[k], a.mask.scale, ds[k]);
        store<T, VEC, UNITS>(static_cast<T *>(a.dx) + at, col, C, ds[k]);
      }
    }
  }
  if constexpr (NORM) {
    if (!a.partials) return;
    if constexpr (LANES > 64) {  // a column is one lane's
#pragma unroll
      for (int k = 0; k < NCH; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int c = (k * LANES + lane) * VEC + j;
          if (c < C) a.partials[(int64_t)blockIdx.x * 2 * C + c] = dg[k][j], a.partials[((int64_t)blockIdx.x * 2 + 1) * C + c] = db[k][j];
        }
      return;
    }
    const int wave = threadIdx.x >> 6;
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NCH; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float v = which ? db[k][j] : dg[k][j];
#pragma unroll
          for (int off = LANES; off < 64; off *= 2) v += __shfl_xor(v, off, 64);
          if ((threadIdx.x & 63) < LANES) red[wave * WIDE + (k * LANES + lane) * VEC + j] = v;
        }
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += 256)
        a.partials[((int64_t)blockIdx.x * 2 + which) * C + c] = (red[c] + red[WIDE + c]) + (red[2 * WIDE + c] + red[3 * WIDE + c]);
    }
  }
}

// ---- rows that do not fit the registers: a workgroup per row, the row read again for every pass over it ----
constexpr int kWideThreads = 1024;

__device__ __forceinline__ float block_sum(float v, float *red) {
  v = lanes_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < kWideThreads / 64; ++k) s += red[k];
  return s;
}

template <class T, int VEC, bool UNITS, bool NORM>
__global__ __launch_bounds__(kWideThreads) void long_rows_forward_kernel(Args a) {
  __shared__ float red[kWideThreads / 64];
  const int C = a.C;
  const float inv = 1.f / (float)C;
  const Stream rng = stream_of(a.mask);
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const int64_t at = row * C;
    auto sums = [&](int col, float (&s)[VEC]) {
      float r[VEC];
      load<T, VEC, UNITS>(static_cast<const T *>(a.x) + at, col, C, s);
      apply(kept<VEC>(a.mask, rng, row, col), a.mask.scale, s);
      if (!a.residual) return;
      load<T, VEC, UNITS>(static_cast<const T *>(a.residual) + at, col, C, r);
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[j] += r[j];
    };
    float sum = 0.f, s[VEC];
    if constexpr (NORM) {
      for (int col = threadIdx.x * VEC; col < C; col += kWideThreads * VEC) {
        sums(col, s);
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum += s[j];
      }
      const float mean = block_sum(sum, red) * inv;
      float sq = 0.f;
      for (int col = threadIdx.x * VEC; col < C; col += kWideThreads * VEC) {
        sums(col, s);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = col + j < C ? s[j] - mean : 0.f;
          sq = fmaf(d, d, sq);
        }
      }
      const float rstd = 1.f / sqrtf(block_sum(sq, red) * inv + a.eps);
      for (int col = threadIdx.x * VEC; col < C; col += kWideThreads * VEC) {
        sums(col, s);
        float n[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) n[j] = col + j < C ? fmaf((s[j] - mean) * rstd, a.gamma[col + j], a.beta[col + j]) : 0.f;
        store<T, VEC, UNITS>(static_cast<T *>(a.out_y) + at, col, C, s);
        store<T, VEC, UNITS>(static_cast<T *>(a.out_n) + at, col, C, n);
      }
      if (a.stats && threadIdx.x == 0) a.stats[2 * row] = mean, a.stats[2 * row + 1] = rstd;
    } else {
      for (int col = threadIdx.x * VEC; col < C; col += kWideThreads * VEC) {
        sums(col, s);
        store<T, VEC, UNITS>(static_cast<T *>(a.out_y) + at, col, C, s);
      }
    }
  }
}

template <class T, int VEC, bool UNITS, bool NORM>
__global__ __launch_bounds__(kWideThreads) void long_rows_backward_kernel(Args a) {
  __shared__ float red[kWideThreads / 64];
  const int C = a.C;
  const float inv = 1.f / (float)C;
  const Stream rng = stream_of(a.mask);
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const int64_t at = row * C;
    float mean = 0.f, rstd = 0.f, s1 = 0.f, s2 = 0.f;
    auto parts = [&](int col, float (&t)[VEC], float (&xh)[VEC]) {  // returns which columns are kept
      float r[VEC];
      load<T, VEC, UNITS>(static_cast<const T *>(a.x) + at, col, C, xh);
      load<T, VEC, UNITS>(static_cast<const T *>(a.dn) + at, col, C, t);
      if (a.residual) load<T, VEC, UNITS>(static_cast<const T *>(a.residual) + at, col, C, r);
      const uint32_t bits = kept<VEC>(a.mask, rng, row, col);
      apply(bits, a.mask.scale, xh);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        xh[j] = ((a.residual ? xh[j] + r[j] : xh[j]) - mean) * rstd;
        t[j] *= col + j < C ? a.gamma[col + j] : 0.f;
      }
      return bits;
    };
    float t[VEC], xh[VEC];
    if constexpr (NORM) {
      mean = a.stats[2 * row], rstd = a.stats[2 * row + 1];
      for (int col = threadIdx.x * VEC; col < C; col += kWideThreads * VEC) {
        parts(col, t, xh);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s1 += t[j], s2 = fmaf(t[j], xh[j], s2);
      }
      s1 = block_sum(s1, red) * inv;
      s2 = block_sum(s2, red) * inv;
    }
    for (int col = threadIdx.x * VEC; col < C; col += kWideThreads * VEC) {
      float ds[VEC];
      uint32_t bits = 0;
      if (a.dy) {
        load<T, VEC, UNITS>(static_cast<const T *>(a.dy) + at, col, C, ds);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) ds[j] = 0.f;
      }
      if constexpr (NORM) {
        bits = parts(col, t, xh);
#pragma unroll
        for (int j = 0; j < VEC; ++j) ds[j] = fmaf(rstd, t[j] - s1 - xh[j] * s2, ds[j]);
        if (a.d_residual) store<T, VEC, UNITS>(static_cast<T *>(a.d_residual) + at, col, C, ds);
      }
      if (a.dx) {
        if constexpr (!NORM) bits = kept<VEC>(a.mask, rng, row, col);
        apply(bits, a.mask.scale, ds);
        store<T, VEC, UNITS>(static_cast<T *>(a.dx) + at, col, C, ds);
      }
    }
  }
}

// d gamma and d beta of such rows: a thread per column, a chunk of rows per workgroup
template <class T>
__global__ __launch_bounds__(256) void long_rows_grads_kernel(Args a, int64_t per) {
  const int c = blockIdx.y * 256 + threadIdx.x;
  if (c >= a.C) return;
  const int64_t r0 = (int64_t)blockIdx.x * per, r1 = r0 + per < a.M ? r0 + per : a.M;
  const Stream rng = stream_of(a.mask);
  float dg = 0.f, db = 0.f;
  for (int64_t r = r0; r < r1; ++r) {
    const float t = load_as_f32(static_cast<const T *>(a.dn) + r * a.C + c);
    const bool keep = kept<4>(a.mask, rng, r, c & ~3) >> (c & 3) & 1u;
    const float s = (keep ? load_as_f32(static_cast<const T *>(a.x) + r * a.C + c) * a.mask.scale : 0.f) +
                    (a.residual ? load_as_f32(static_cast<const T *>(a.residual) + r * a.C + c) : 0.f);
    const float xh = (s - a.stats[2 * r]) * a.stats[2 * r + 1];
    dg = fmaf(t, xh, dg);
    db += t;
  }
  a.partials[((int64_t)blockIdx.x * 2 + 0) * a.C + c] = dg;
  a.partials[((int64_t)blockIdx.x * 2 + 1) * a.C + c] = db;
}

__global__ void advance_kernel(int64_t *state, int64_t *taken) {
  taken[0] = state[0];
  taken[1] = state[1];
  state[1] = (int64_t)((uint64_t)state[1] + 1);
}

// ================================================================================================
// host side
// ================================================================================================
static Mask mask_of(double p, const int64_t *rng) {
  Mask m{};
  const double t = p * 4294967296.0;
  const uint64_t threshold = (uint64_t)(t + 0.5);
  m.rng = rng;
  m.none = threshold >= 4294967296ull;
  m.all = threshold == 0;
  m.threshold = m.none ? 0xffffffffu : (uint32_t)threshold;
  m.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
  return m;
}

// How a row lies over lanes: the fewest lanes that hold it in one piece each, then more pieces; 0 lanes: rows that do not fit.
struct Shape {
  int vec, lanes, pieces;
  bool units;
};
static Shape shape_of(int dtype, int64_t C, bool aligned) {
  Shape s{};
  const int per = dtype == PA_F32 ? 4 : 8;
  s.units = aligned && C % per == 0;
  s.vec = per;
  const int64_t q = (C + s.vec - 1) / s.vec;
  if (q <= 64) {
    s.pieces = 1;
    for (s.lanes = 8; s.lanes < q; s.lanes *= 2) {}
  } else if (q <= 1024) {
    s.lanes = q <= 256 ? 64 : 256;
    s.pieces = q <= 128 || (q > 256 && q <= 512) ? 2 : 4;
  }
  return s;
}

static int64_t groups_of(const Shape &s, int64_t M, int per_cu, int num_cu) {
  const int64_t rows = s.lanes ? 256 / s.lanes : 1, blocks = (M + rows - 1) / rows, most = (int64_t)num_cu * per_cu;
  return blocks < most ? blocks : most;
}

static constexpr int kForwardPerCu = 8, kBackwardPerCu = 4;

// partial results of d gamma and d beta; those of long rows are a kernel of their own and kept below 256 MB
static int64_t partials_of(const Shape &s, int64_t M, int64_t C, int num_cu) {
  const int64_t g = groups_of(s, M, kBackwardPerCu, num_cu), most = ((int64_t)1 << 25) / C;
  return s.lanes || g <= most ? g : most < 1 ? 1 : most;
}

template <class T, int VEC, bool UNITS, int LANES, int NCH>
static void launch_rows(const Args &a, bool forward, bool norm, int64_t grid, hipStream_t st) {
  const dim3 g((unsigned)grid), b(256);
  if (forward && norm) hipLaunchKernelGGL((rows_forward_kernel<T, VEC, UNITS, LANES, NCH, true>), g, b, 0, st, a);
  else if (forward) hipLaunchKernelGGL((rows_forward_kernel<T, VEC, UNITS, LANES, NCH, false>), g, b, 0, st, a);
  else if (norm) hipLaunchKernelGGL((rows_backward_kernel<T, VEC, UNITS, LANES, NCH, true>), g, b, 0, st, a);
  else hipLaunchKernelGGL((rows_backward_kernel<T, VEC, UNITS, LANES, NCH, false>), g, b, 0, st, a);
}

template <class T, int VEC, bool UNITS>
static int launch(const Args &a, const Shape &s, bool forward, bool norm, int num_cu, hipStream_t st) {
  const int64_t grid = groups_of(s, a.M, forward ? kForwardPerCu : kBackwardPerCu, num_cu);
  if (s.lanes == 8) launch_rows<T, VEC, UNITS, 8, 1>(a, forward, norm, grid, st);
  else if (s.lanes == 16) launch_rows<T, VEC, UNITS, 16, 1>(a, forward, norm, grid, st);
  else if (s.lanes == 32) launch_rows<T, VEC, UNITS, 32, 1>(a, forward, norm, grid, st);
  else if (s.lanes == 64 && s.pieces == 1) launch_rows<T, VEC, UNITS, 64, 1>(a, forward, norm, grid, st);
  else if (s.lanes == 64 && s.pieces == 2) launch_rows<T, VEC, UNITS, 64, 2>(a, forward, norm, grid, st);
  else if (s.lanes == 64 && s.pieces == 4) launch_rows<T, VEC, UNITS, 64, 4>(a, forward, norm, grid, st);
  else if (s.lanes == 256 && s.pieces == 2) launch_rows<T, VEC, UNITS, 256, 2>(a, forward, norm, grid, st);
  else if (s.lanes == 256) launch_rows<T, VEC, UNITS, 256, 4>(a, forward, norm, grid, st);
  else {
    const dim3 g((unsigned)grid), b(kWideThreads);
    if (forward && norm) hipLaunchKernelGGL((long_rows_forward_kernel<T, VEC, UNITS, true>), g, b, 0, st, a);
    else if (forward) hipLaunchKernelGGL((long_rows_forward_kernel<T, VEC, UNITS, false>), g, b, 0, st, a);
    else if (norm) hipLaunchKernelGGL((long_rows_backward_kernel<T, VEC, UNITS, true>), g, b, 0, st, a);
    else hipLaunchKernelGGL((long_rows_backward_kernel<T, VEC, UNITS, false>), g, b, 0, st, a);
    if (!forward && norm && a.partials) {
      const int64_t parts = partials_of(s, a.M, a.C, num_cu), per = (a.M + parts - 1) / parts;
      hipLaunchKernelGGL((long_rows_grads_kernel<T>), dim3((unsigned)parts, (unsigned)((a.C + 255) / 256)), dim3(256), 0, st, a, per);
    }
  }
  return launch_status();
}

static int launch(int dtype, const Args &a, const Shape &s, bool forward, bool norm, int num_cu, hipStream_t st) {
  if (dtype == PA_F32) return s.units ? launch<float, 4, true>(a, s, forward, norm, num_cu, st) : launch<float, 4, false>(a, s, forward, norm, num_cu, st);
  return s.units ? launch<bf16, 8, true>(a, s, forward, norm, num_cu, st) : launch<bf16, 8, false>(a, s, forward, norm, num_cu, st);
}

int advance(int64_t *state, int64_t *taken, hipStream_t st) {
  hipLaunchKernelGGL(advance_kernel, dim3(1), dim3(1), 0, st, state, taken);
  return launch_status();
}

int forward(int dtype, int64_t M, int64_t C, const void *x, const void *residual, double p, const int64_t *rng, void *y,
            const float *gamma, const float *beta, float eps, void *normed, float *stats, int num_cu, hipStream_t st) {
  Args a{};
  a.x = x, a.residual = residual, a.out_y = y, a.out_n = normed;
  a.gamma = gamma, a.beta = beta, a.stats = stats, a.eps = eps;
  a.M = M, a.C = (int)C, a.mask = mask_of(p, rng);
  const bool aligned = aligned16(x) && aligned16(residual) && aligned16(y) && aligned16(normed);
  return launch(dtype, a, shape_of(dtype, C, aligned), true, normed != nullptr, num_cu, st);
}

// the plan does not know the pointers: the larger of the two shapes' needs
int64_t backward_workspace_bytes(int dtype, int64_t M, int64_t C, int num_cu) {
  int64_t most = 0;
  for (int k = 0; k < 2; ++k) {
    const int64_t g = partials_of(shape_of(dtype, C, k == 0), M, C, num_cu);
    if (g > most) most = g;
  }
  return most * 2 * C * 4;
}

int backward(int dtype, int64_t M, int64_t C, const void *dy, const void *d_normed, const void *x, const void *residual,
             const float *stats, const float *gamma, double p, const int64_t *rng, void *dx, void *d_residual, float *grads, void *workspace, int num_cu,
             hipStream_t st) {
  Args a{};
  a.dy = dy, a.dn = d_normed, a.x = x, a.residual = residual, a.dx = dx, a.d_residual = d_residual;
  a.gamma = gamma, a.stats = const_cast<float *>(stats);
  a.partials = grads ? static_cast<float *>(workspace) : nullptr;
  a.M = M, a.C = (int)C, a.mask = mask_of(p, rng);
  const bool aligned = aligned16(dy) && aligned16(d_normed) && aligned16(x) && aligned16(residual) && aligned16(dx) && aligned16(d_residual);
  const Shape s = shape_of(dtype, C, aligned);
  int rc = launch(dtype, a, s, false, d_normed != nullptr, num_cu, st);
  if (!rc && grads && d_normed) rc = wgrad::sum_rows(a.partials, partials_of(s, M, C, num_cu), 2 * C, grads, st);
  return rc;
}

}  // namespace dropout
}  // namespace pa
