// Products of activation rows with weight rows, out[m][n] = sum_k X[m][k] W[n][k], on gfx950 matrix instructions, with the
// work that follows them in their registers: the core under the gated feed-forward block (pa_gated.hip) and the 8-bit
// Linears (pa_int8.hip).
//
// Element types differ only in the matrix instruction: an operand is the 16 bytes ("unit") of one row that a lane holds, and
// lane half g takes unit 2 k + g of a row's units 0 .. 7 of a stage.  bf16 32x32x16: 8 elements; int8 32x32x32: 16; float32:
// 4, one per 32x32x2 instruction, so that the reduction runs in an order that both operands share.
//
// W is the first operand and X the second, so that a lane ends with one row of X and, per four registers, four neighbouring
// columns: C/D register r of lane (i, g) is row i, column rowmap(r, g) (pa_mfma_ops.h).
#pragma once

#include "pa_host.h"
#include "pa_mfma_ops.h"

namespace pa {
namespace tile {

using mfma::f32x16;
using mfma::load_unit_to_lds;
using mfma::pack2;
using mfma::rowmap;
using mfma::u32x2;
using mfma::u32x4;

typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Bf16 {
  using Acc = f32x16;
  static constexpr int kBytes = 2;
  static __device__ __forceinline__ Acc mma(u32x4 a, u32x4 b, Acc c) { return mfma::mma(a, b, c); }
};
// float32 as sums of three bf16 values (8 + 8 + 8 bits), six products of them: hi hi + hi mid + mid hi + hi lo + lo hi + mid mid.
// The first part is cut off, not rounded, so that the second is up to 2^-7 of the value and the third 2^-16: what is left out is
// up to 2^-22 of a product (8 % of products of operands just above a power of two pass 2^-24, a float32 product's own error).
// Parts of an infinity are not numbers, nor is their product with a part that is zero: a sum that holds one is NaN.  Against
// float32 matrix instructions: 192 cycles per 32 x 32 x 16 instead of 512, and 44 vector instructions per operand.
struct F32 {
  using Acc = f32x16;
  static constexpr int kBytes = 4;
  struct Parts {
    u32x4 hi, mid, lo;
  };
  static __device__ __forceinline__ Parts split(u32x4 a, u32x4 b) {  // eight elements
    Parts r;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const u32x4 &s = k < 2 ? a : b;
      const uint32_t w0 = s[(2 * k) & 3], w1 = s[(2 * k + 1) & 3];
      // the upper 16 bits as they are: no value rounds up to infinity
      r.hi[k] = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
      const float r0 = __uint_as_float(w0) - __uint_as_float(w0 & 0xffff0000u), r1 = __uint_as_float(w1) - __uint_as_float(w1 & 0xffff0000u);
      const uint32_t m = pack2(r0, r1);
      r.mid[k] = m;
      r.lo[k] = pack2(r0 - __uint_as_float(m << 16), r1 - __uint_as_float(m & 0xffff0000u));
    }
    return r;
  }
  static __device__ __forceinline__ Acc mma(const Parts &a, const Parts &b, Acc c) {
    c = mfma::mma(a.mid, b.mid, c);
    c = mfma::mma(a.lo, b.hi, c);
    c = mfma::mma(a.hi, b.lo, c);
    c = mfma::mma(a.mid, b.hi, c);
    c = mfma::mma(a.hi, b.mid, c);
    return mfma::mma(a.hi, b.hi, c);
  }
};
struct I8 {
  using Acc = i32x16;
  static constexpr int kBytes = 1;
  static __device__ __forceinline__ Acc mma(u32x4 a, u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
  }
};

// ---- activations: PA_ACT_* ----
enum Act { kNone = 0, kGelu = 1, kRelu = 2, kSilu = 3, kSigmoid = 4, kTanh = 5 };

__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * v)); }

template <bool SHORT, class V>  // SHORT: rounded to bf16 next
__device__ __forceinline__ void act_values(int act, V &v) {
  constexpr int N = sizeof(V) / 4;
  switch (act) {
    case kGelu:
#pragma unroll
      for (int r = 0; r < N; ++r) v[r] = SHORT ? gelu_short(v[r]) : gelu_full(v[r]);
      break;
    case kRelu:  // NaN passes, as torch's does
#pragma unroll
      for (int r = 0; r < N; ++r) v[r] = v[r] < 0.f ? 0.f : v[r];
      break;
    case kSilu:
#pragma unroll
      for (int r = 0; r < N; ++r) v[r] *= sigmoid(v[r]);
      break;
    case kSigmoid:
#pragma unroll
      for (int r = 0; r < N; ++r) v[r] = sigmoid(v[r]);
      break;
    case kTanh:
#pragma unroll
      for (int r = 0; r < N; ++r) v[r] = tanhf(v[r]);
      break;
    default: break;
  }
}

// v <- act(v), slope <- act'(v)
template <bool SHORT>
__device__ __forceinline__ void act_slopes(int act, f32x16 &v, f32x16 &slope) {
  switch (act) {
    case kGelu:
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float d;
        v[r] = SHORT ? gelu_short_slope(v[r], d) : gelu_full_slope(v[r], d);
        slope[r] = d;
      }
      break;
    case kRelu:
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        slope[r] = v[r] > 0.f ? 1.f : 0.f;
        v[r] = v[r] < 0.f ? 0.f : v[r];
      }
      break;
    case kSilu:
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = v[r], s = sigmoid(x);
        v[r] = x * s;
        slope[r] = fmaf(v[r], 1.f - s, s);
      }
      break;
    case kSigmoid:
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float s = sigmoid(v[r]);
        v[r] = s;
        slope[r] = s * (1.f - s);
      }
      break;
    case kTanh:
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float t = tanhf(v[r]);
        v[r] = t;
        slope[r] = fmaf(-t, t, 1.f);
      }
      break;
    default:
#pragma unroll
      for (int r = 0; r < 16; ++r) slope[r] = 1.f;
  }
}

// What the product's registers become.
enum Kind {
  kPlain,  // out = act(X W0^T + b0) + residual
  kGated,  // out = act(X W0^T + b0) * (X W1^T + b1)
  kBack,   // the gated block's hidden layer again, g = X W0^T + b0, u = X W1^T + b1, and d = X2 W2^T:
           // out[:, :ldh] = d u act'(g), out[:, ldh:] = d act(g), out2 = act(g) u
  kPeak,   // int8: peak[m] = max over n of |act(X W0^T + b0) * (X W1^T + b1)|, as bits
  kCodes,  // the same products again, out = rint(127 of them / peak) as int8 in column groups, row_scale = peak / 127
};

// The hidden layer's matrices are written and read by kernels of this library alone, and lie in groups of 32 bytes of columns where
// the type is bf16: [32 rows][column group][row][32 bytes].  A wave's 32 x 32 tile is then 2 KB in one piece; as rows it
// is 32 pieces of 64 bytes, kilobytes apart, which memory takes at half the rate (131 072 rows of 3 x 1 024 values: 476 us as
// rows, 326 in groups).
template <class T>
constexpr bool kGrouped = sizeof(T) == 2;
constexpr int64_t kGroupRows = 32;

struct Args {
  const void *X, *X2;            // rows of activations; a row is `units` units of 16 bytes, ldx / ldx2 bytes apart
  const void *W[3];              // rows of weights, ldw / ldw2 (W[2]) bytes apart
  int64_t ldx, ldx2, ldw, ldw2;
  int units, units2;             // of the reduction over X, over X2
  int64_t M;
  int N, limit;                  // columns; columns N .. limit - 1 are written as zeros (limit: a multiple of a unit's elements, or N)
  const float *bias[2];          // or NULL
  const float *sx, *sw[2];       // int8: scale per row of X, per row of W
  uint32_t *peak;                // kPeak, kCodes
  float *row_scale;              // kCodes
  const void *residual;          // (M, N), kPlain, or NULL
  float *sums;                   // kBack, bf16: per 32 rows the column sums of dg and du before their rounding, (2 ldh), or NULL
  void *out, *out2;
  int64_t ldo, ldh;              // elements between rows of out (residual alike); of out2, and from dg to du
  int act;
  bool x_groups;                 // X lies in column groups
  bool vec;                      // out and residual start on 16 bytes and their rows are whole units apart
  int mt, nt;                    // tiles
};

typedef __amdgpu_buffer_rsrc_t Buffer;
constexpr unsigned kNowhere = 0x80000000u;  // an offset past every buffer below: loads give zero, stores are dropped

// 16-byte stores of a 32 x 32 tile: this lane's row at byte offset `at`, columns col .. col + 31 below limit.  Neighbouring
// columns of a row come from both halves of the wave: a lane's 16 bytes lie beside its partner's.  GROUPS: `at` is the row's place in
// its column groups.
template <bool GROUPS = false>
__device__ __forceinline__ void store_tile(const f32x16 &v, const Buffer &out, unsigned at, int col, int limit, int g, const bf16 *) {
  uint32_t p[4][2];
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int w = 0; w < 2; ++w) p[q][w] = pack2(v[4 * q + 2 * w], v[4 * q + 2 * w + 1]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    u32x4 s;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const auto r = __builtin_amdgcn_permlane32_swap(p[2 * h][w], p[2 * h + 1][w], false, false);
      s[w] = r[0], s[2 + w] = r[1];
    }
    const int c = col + 16 * h + 8 * g;
    const unsigned place = GROUPS ? at + 64 * (col + 16 * h) + 16 * g : at + 2 * c;
    __builtin_amdgcn_raw_buffer_store_b128(s, out, c < limit ? place : kNowhere, 0, 0);
  }
}
template <bool GROUPS = false>
__device__ __forceinline__ void store_tile(const f32x16 &v, const Buffer &out, unsigned at, int col, int limit, int g, const float *) {
  static_assert(!GROUPS, "float32 lies as rows");
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int c = col + 8 * q + 4 * g;
    u32x4 s;
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = __float_as_uint(v[4 * q + j]);
    __builtin_amdgcn_raw_buffer_store_b128(s, out, c < limit ? at + 4 * c : kNowhere, 0, 0);
  }
}
// ---- sums over the 32 rows (lanes) of two 32 x 32 tiles of the same 32 columns (16 registers and both halves of the wave) ----
// First pairs of registers in exchange for pairs of lanes, then the two tiles, then over the lanes that are left: 3 instructions per
// pair of values where adding each over the lanes takes 10.  In the end lane (i, g) holds columns 8 q + 4 g .. + 3, q = i % 4, of the
// second tile where bit 2 of i is set.
template <int BIT>  // 0 .. 2, of the lane
__device__ __forceinline__ float exchange_add(float even, float odd, int lane) {
  constexpr int CTRL = BIT == 0 ? 0xB1 : BIT == 1 ? 0x4E : 0x124;  // quad_perm [1,0,3,2], [2,3,0,1], row_ror 4
  const bool upper = lane >> BIT & 1;
  const float keep = upper ? odd : even, send = upper ? even : odd;
  return keep + __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(send), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float both_add(float first, float second, int lane) {
  float v = exchange_add<2>(first, second, lane);
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), 0x128, 0xf, 0xf, true));  // row_ror 8
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ f32x4 column_sums(const f32x16 &v, const f32x16 &w, int lane) {
  f32x4 s;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    auto four = [&](const f32x16 &x) {
      return exchange_add<1>(exchange_add<0>(x[j], x[4 + j], lane), exchange_add<0>(x[8 + j], x[12 + j], lane), lane);
    };
    s[j] = both_add(four(v), four(w), lane);
  }
  return s;
}

template <class T>
constexpr int kTileStores = sizeof(T) == 2 ? 2 : 4;

// four neighbouring elements of a row of the residual, as they lie and as float32
template <class T>
struct Quad;
template <>
struct Quad<bf16> {
  u32x2 w;
  __device__ __forceinline__ void load(const Buffer &in, unsigned at) { w = __builtin_amdgcn_raw_buffer_load_b64(in, at, 0, 0); }
  __device__ __forceinline__ float operator[](int j) const {
    const uint32_t b = w[j >> 1];
    return __uint_as_float(j & 1 ? b & 0xffff0000u : b << 16);
  }
};
template <>
struct Quad<float> {
  u32x4 w;
  __device__ __forceinline__ void load(const Buffer &in, unsigned at) { w = __builtin_amdgcn_raw_buffer_load_b128(in, at, 0, 0); }
  __device__ __forceinline__ float operator[](int j) const {
    const uint32_t b = w[j];
    return __uint_as_float(b);
  }
};

// ---- rows that are not whole units: the same 16-byte accesses wherever they start, element by element where a row ends.  (Stored
// element by element throughout, the 32 rows of an instruction are 64 pieces of 2 bytes: gated block with residual, 60 000 x 257,
// F = 1 028: 266 us, this way 223.) ----
typedef u32x2 loose2 __attribute__((aligned(2)));
typedef u32x4 loose4 __attribute__((aligned(2)));
typedef f32x4 loose4f __attribute__((aligned(4)));
__device__ __forceinline__ void add_quad(const bf16 *p, int left, float (&v)[4]) {  // left: elements of the row from p on
  if (left >= 4) {
    const u32x2 w = *reinterpret_cast<const loose2 *>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t b = w[j >> 1];
      v[j] += __uint_as_float(j & 1 ? b & 0xffff0000u : b << 16);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j) v[j] += j < left ? load_as_f32(p + j) : 0.f;
  }
}
__device__ __forceinline__ void add_quad(const float *p, int left, float (&v)[4]) {
  if (left >= 4) {
    const f32x4 w = *reinterpret_cast<const loose4f *>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += w[j];
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j) v[j] += j < left ? p[j] : 0.f;
  }
}
// a 32 x 32 tile from column col on; this lane's row, of N columns, lies `at` bytes behind the base, which is the same for all
__device__ __forceinline__ void store_tile_loose(const f32x16 &v, char *base, unsigned at, bool there, int col, int N, int g, const bf16 *) {
  uint32_t p[4][2];
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int w = 0; w < 2; ++w) p[q][w] = pack2(v[4 * q + 2 * w], v[4 * q + 2 * w + 1]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    u32x4 s;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const auto r = __builtin_amdgcn_permlane32_swap(p[2 * h][w], p[2 * h + 1][w], false, false);
      s[w] = r[0], s[2 + w] = r[1];
    }
    const int c = col + 16 * h + 8 * g;
    if (there && c + 8 <= N) {
      *reinterpret_cast<loose4 *>(base + (at + 2 * c)) = s;
    } else if (there) {
#pragma unroll
      for (int j = 0; j < 7; ++j) {
        const uint32_t b = s[j / 2];
        if (c + j < N) *reinterpret_cast<uint16_t *>(base + (at + 2 * (c + j))) = (uint16_t)(j & 1 ? b >> 16 : b);
      }
    }
  }
}
__device__ __forceinline__ void store_tile_loose(const f32x16 &v, char *base, unsigned at, bool there, int col, int N, int g, const float *) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int c = col + 8 * q + 4 * g;
    if (there && c + 4 <= N) {
      *reinterpret_cast<loose4f *>(base + (at + 4 * c)) = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
    } else if (there) {
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (c + j < N) *reinterpret_cast<float *>(base + (at + 4 * (c + j))) = v[4 * q + j];
    }
  }
}

// one float per lane, to dst + 4 lane
__device__ __forceinline__ void load_word_to_lds(const float *p, unsigned dst) {
  asm volatile(
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dword %0, off" ::"v"(p), "s"(dst)
      : "memory");
}

// accumulators to float32: int8 sums take their scales; then the bias.  `side` points at the tile's 32 biases, `scale` at its
// 32 scales.
template <class E>
__device__ __forceinline__ f32x16 values_of(const typename E::Acc &acc, const float *side, const float *scale, int g, float sx) {
  f32x16 v;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const f32x4 b = *reinterpret_cast<const f32x4 *>(side + 8 * q + 4 * g);
    f32x4 s = {1.f, 1.f, 1.f, 1.f};
    if constexpr (E::kBytes == 1) s = *reinterpret_cast<const f32x4 *>(scale + 8 * q + 4 * g) * sx;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (E::kBytes == 1) v[4 * q + j] = fmaf((float)acc[4 * q + j], s[j], b[j]);
      else v[4 * q + j] = acc[4 * q + j] + b[j];
    }
  }
  return v;
}

// ---------------------------------------------------------------------------------------------------------------
// rows_tile_kernel.  A workgroup of WM x WN waves owns tiles of BM rows x BN weight rows; a wave's part is TM x TN tiles of
// 32 x 32.  kGated and kBack take 32 rows of W0 and the 32 rows of W1 in turn, so that a wave holds both factors of its
// hidden units.  Stages of UPS units of every row pass through a ring of RING LDS buffers, filled RING - 1 stages ahead by
// direct global -> LDS loads, one barrier per stage; the stages of a workgroup's tiles form one sequence, so that the
// first stages of a tile arrive behind the last products and the stores of the one before.
// Position p of row r holds the row's unit p ^ (r / 4 % 4) (UPS = 4) or p ^ (r / 2 % 8) (UPS = 8): the 16 lanes of an access
// phase fall on all 64 banks.
// Units past a row's last one repeat it and are left out of the products; rows past the last row repeat it and are not stored.
// What the epilogue needs besides (biases; int8: both scales) arrives in LDS with a tile's first stage, a buffer per tile.
// Loads and stores are counted in order: the stores of a tile leave behind the first AHEAD stages of the next one and must not be
// waited for with those, so the vector paths issue every store, with an offset past the buffer where there is nothing to
// store, and the waits of a tile's first stages leave that many operations more in flight.
// Tiles are dealt out to the XCDs (= workgroup id mod 8) in eight equal runs with the columns running fastest, so that the
// workgroups of an L2 share rows of X and W.
// ---------------------------------------------------------------------------------------------------------------
template <int WM_, int WN_, int TM_, int TN_, int UPS_, int RING_, int OCC_>
struct Config {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, UPS = UPS_, RING = RING_, OCC = OCC_;  // OCC: waves per SIMD
  static constexpr int WAVES = WM * WN, BM = WM * TM * 32, BN = WN * TN * 32;
  static constexpr int STAGE = (BM + BN) * 16 * UPS;
  // floats: biases; int8: scales of W, of X; kCodes: peaks
  static constexpr int side(int bytes, Kind kind) { return BN + (bytes == 1 ? BN + BM : 0) + (kind == kCodes ? BM : 0); }
  static constexpr int lds(int bytes, Kind kind) { return RING * (STAGE + 4 * side(bytes, kind)); }
};

template <class E, class TO, Kind KIND, class CFG>
__global__ __launch_bounds__(64 * CFG::WAVES, CFG::OCC) void rows_tile_kernel(Args a) {
  constexpr int WM = CFG::WM, TM = CFG::TM, TN = CFG::TN, WAVES = CFG::WAVES, BM = CFG::BM, BN = CFG::BN, UPS = CFG::UPS;
  constexpr int RING = CFG::RING, AHEAD = RING - 1, GROUP = 64 / UPS;  // rows of one load
  constexpr bool DUAL = KIND != kPlain;
  constexpr int NX = BM / GROUP / WAVES, NW = BN / GROUP / WAVES, TN2 = TN / 2;  // loads a wave issues
  static_assert(BM % (GROUP * WAVES) == 0 && BN % (GROUP * WAVES) == 0, "whole groups");
  static_assert(!DUAL || TN % 2 == 0, "pairs of tiles");
  constexpr unsigned STAGE = CFG::STAGE, SIDE = CFG::side(E::kBytes, KIND);
  static_assert(BM % 64 == 0 && BN % 64 == 0, "whole loads of 64 floats");
  // stores a wave leaves behind a tile
  constexpr int STORES = KIND == kPeak ? 0 : KIND == kCodes ? TM * TN2 : kTileStores<TO> * TM * (KIND == kPlain ? TN : KIND == kGated ? TN2 : 3 * TN2);
  constexpr int YOUNGER = (AHEAD - 1) * (NX + NW);
  constexpr int LEFT = YOUNGER + STORES < 63 ? YOUNGER + STORES : 63;
  using Acc = typename E::Acc;
  extern __shared__ u32x4 smem[];
  const int lane = threadIdx.x & 63, i = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  constexpr int CN = DUAL ? BN / 2 : BN;  // output columns of a tile

  const int total = a.mt * a.nt, xcd = blockIdx.x & 7, step = gridDim.x >> 3;
  const int last = (int)((int64_t)total * (xcd + 1) / 8);
  int t = (int)((int64_t)total * xcd / 8) + (blockIdx.x >> 3);
  if (t >= last) return;

  const int nk1 = (a.units + UPS - 1) / UPS, nk = nk1 + (KIND == kBack ? (a.units2 + UPS - 1) / UPS : 0);

  // ---- the loads run RING - 1 stages ahead of the products ----
  int lt = t, lk = 0;  // tile and stage that are fetched next
  unsigned buf = 0;    // where they go
  int sbuf = 0;        // and the side data
  int left = 0;        // units of its rows from its first on
  unsigned offx[NX], offw[NW];
  const char *xs = nullptr, *ws0 = nullptr, *ws1 = nullptr;
  const int64_t xstep = KIND == kPlain && a.x_groups ? 512 * UPS : 16 * UPS;
  const int frow = lane / UPS, fpos = lane % UPS;
  auto uniform = [](const char *p) {  // what is the same for every lane, in scalar registers
    const uint64_t v = (uint64_t)(uintptr_t)p;
    return reinterpret_cast<const char *>((uintptr_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
                                                      (uint32_t)__builtin_amdgcn_readfirstlane((int)v)));
  };
  auto swizzle = [](int row) { return UPS == 8 ? (row >> 1) & 7 : (row >> 2) & 3; };
  auto place = [&](bool second) {  // offsets of tile lt: rows of X and W (second: of X2 and W[2])
    const int tm = lt / a.nt, tn = lt - tm * a.nt;
    const int64_t m0 = (int64_t)tm * BM, ldx = second ? a.ldx2 : a.ldx, ldw = second ? a.ldw2 : a.ldw;
    const int have = (int)(a.M - m0 < BM ? a.M - m0 : BM), n0 = tn * CN, haven = a.N - n0;
    left = second ? a.units2 : a.units;
    xs = uniform(static_cast<const char *>(second ? a.X2 : a.X) + m0 * ldx);
    ws0 = uniform(static_cast<const char *>(second ? a.W[2] : a.W[0]) + n0 * ldw);
    if constexpr (DUAL) ws1 = uniform(static_cast<const char *>(a.W[1]) + n0 * ldw);
#pragma unroll
    for (int q = 0; q < NX; ++q) {
      const int row = (wave * NX + q) * GROUP + frow, r = row < have ? row : have - 1;
      const int unit = fpos ^ swizzle(row);
      offx[q] = KIND == kPlain && a.x_groups ? (unsigned)((r & ~31) * ldx + (r & 31) * 32 + (unit >> 1) * 1024 + (unit & 1) * 16)
                                             : (unsigned)(r * ldx) + 16 * unit;
    }
#pragma unroll
    for (int q = 0; q < NW; ++q) {
      const int row = (wave * NW + q) * GROUP + frow;
      const int col = DUAL && !second ? (row >> 6) * 32 + (row & 31) : row, c = col < haven ? col : haven - 1;
      offw[q] = (unsigned)(c * ldw) + 16 * (fpos ^ swizzle(row));
    }
  };
  auto fetch = [&]() {
    const bool none = lt >= last;  // past the last tile: the last stage again, so that every stage counts the same loads
    const bool second = KIND == kBack && (none ? nk1 < nk : lk >= nk1);
    if (!none && (lk == 0 || (KIND == kBack && lk == nk1))) place(second);
    else if (!none) left -= UPS, xs += xstep, ws0 += 16 * UPS, ws1 += DUAL ? 16 * UPS : 0;
    const unsigned dst = (unsigned)(uintptr_t)smem + buf;
    if (!none && lk == 0) {
      const int n0 = (lt % a.nt) * CN;
      const int64_t m0 = (int64_t)(lt / a.nt) * BM;
      for (int k = wave; k < (int)SIDE / 64; k += WAVES) {
        const int at = 64 * k + lane;
        const float *p;
        if (64 * k < 2 * BN) {
          const int v = 64 * k < BN ? at : at - BN, which = DUAL ? (v >> 5) & 1 : 0, col = n0 + (DUAL ? (v >> 6) * 32 + (v & 31) : v);
          const float *from = 64 * k < BN ? a.bias[which] : a.sw[which];
          p = from ? from + (col < a.N ? col : a.N - 1) : reinterpret_cast<const float *>(&mfma::kZeroUnit);
        } else {
          const bool peaks = KIND == kCodes && 64 * k >= 2 * BN + BM;
          const int64_t m = m0 + at - 2 * BN - (peaks ? BM : 0);
          p = (peaks ? reinterpret_cast<const float *>(a.peak) : a.sx) + (m < a.M ? m : a.M - 1);
        }
        load_word_to_lds(p, (unsigned)(uintptr_t)smem + RING * STAGE + 4 * (sbuf * SIDE + 64 * k));
      }
      sbuf = sbuf + 1 == RING ? 0 : sbuf + 1;
    }
    auto load = [&](auto x_off, auto w_off) {
#pragma unroll
      for (int q = 0; q < NX; ++q) {
        const int grp = wave * NX + q;
        load_unit_to_lds(xs, (int)x_off(offx[q], grp), dst + grp * 1024);
      }
#pragma unroll
      for (int q = 0; q < NW; ++q) {
        const int grp = wave * NW + q;
        // second: half as many rows; in a longer ring the other loads are made all the same, so that every stage counts as many
        if (AHEAD == 1 && second && grp * GROUP >= BN / 2) continue;
        load_unit_to_lds(DUAL && !second && (grp & (32 / GROUP)) ? ws1 : ws0, (int)w_off(offw[q], grp), dst + BM * 16 * UPS + grp * 1024);
      }
    };
    if (left >= UPS) {
      auto as_it_is = [](unsigned off, int) { return off; };
      load(as_it_is, as_it_is);
    } else {  // units past the row's last one: that one again; the products leave them out
      const int unit[2] = {fpos ^ swizzle(frow), fpos ^ swizzle(frow + GROUP)};
      auto w_off = [&](unsigned off, int grp) {
        const int u = unit[grp & 1];
        return off - 16u * (unsigned)(u >= left ? u - left + 1 : 0);
      };
      auto x_off = [&](unsigned off, int grp) {
        const int u = unit[grp & 1], to = u >= left ? left - 1 : u;
        return KIND == kPlain && a.x_groups ? off - (unsigned)(((u >> 1) - (to >> 1)) * 1024 + ((u & 1) - (to & 1)) * 16) : w_off(off, grp);
      };
      load(x_off, w_off);
    }
    buf = buf + STAGE == RING * STAGE ? 0 : buf + STAGE;
    if (!none && ++lk == nk) lk = 0, lt += step;
  };

#pragma unroll
  for (int k = 0; k < AHEAD; ++k) fetch();
  unsigned cur = 0;
  int cside = 0;
  bool stored = false;  // the tile before left exactly STORES stores
  for (; t < last; t += step) {
    Acc acc[TM][TN], acc2[KIND == kBack ? TM : 1][KIND == kBack ? TN2 : 1];
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
      for (int n = 0; n < TN; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[m][n][r] = 0;
    if constexpr (KIND == kBack) {
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN2; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc2[m][n][r] = 0;
    }
    const int swz = swizzle(i);
    int at_stage = 0;
    auto next_stage = [&]() {
      // this wave's share of the stage has landed; the younger stages and, at first, the stores of the tile before stay in flight
      if (stored && at_stage < AHEAD) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
      else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(YOUNGER) : "memory");
      ++at_stage;
      __syncthreads();  // everyone's; and everyone is past the stage before
      fetch();
    };
    auto multiply = [&](auto &to, auto tn_, auto whole_, int left, int wrow) {  // left: units of the stage, UPS where `whole`
      constexpr int T = decltype(tn_)::value;
      constexpr bool WHOLE = decltype(whole_)::value;
      const u32x4 *xs = smem + cur / 16 + (wm * TM * 32 + i) * UPS;
      const u32x4 *ws = smem + cur / 16 + (BM + wrow + i) * UPS;
      if constexpr (E::kBytes == 4) {  // two units make an operand
#pragma unroll
        for (int ks = 0; ks < UPS / 2; ks += 2) {
          if (!WHOLE && 2 * ks >= left) break;
          auto operand = [&](const u32x4 *row) {
            u32x4 v[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              v[h] = row[(2 * (ks + h) + g) ^ swz];
              if (!WHOLE && 2 * (ks + h) + g >= left) v[h] = u32x4{0u, 0u, 0u, 0u};
            }
            return E::split(v[0], v[1]);
          };
          typename E::Parts w[T];
#pragma unroll
          for (int n = 0; n < T; ++n) w[n] = operand(ws + n * 32 * UPS);
#pragma unroll
          for (int m = 0; m < TM; ++m) {
            const typename E::Parts x = operand(xs + m * 32 * UPS);
#pragma unroll
            for (int n = 0; n < T; ++n) to[m][n] = E::mma(w[n], x, to[m][n]);
          }
        }
      } else {
#pragma unroll
      for (int ks = 0; ks < UPS / 2; ++ks) {
        if (!WHOLE && 2 * ks >= left) break;
        const int at = (2 * ks + g) ^ swz;
        u32x4 w[T], x[TM];
#pragma unroll
        for (int n = 0; n < T; ++n) w[n] = ws[n * 32 * UPS + at];
#pragma unroll
        for (int m = 0; m < TM; ++m) x[m] = xs[m * 32 * UPS + at];
        if (!WHOLE && 2 * ks + 1 >= left && g == 1) {
#pragma unroll
          for (int n = 0; n < T; ++n) w[n] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
          for (int m = 0; m < TM; ++m) x[m] = u32x4{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int m = 0; m < TM; ++m)
#pragma unroll
          for (int n = 0; n < T; ++n) to[m][n] = E::mma(w[n], x[m], to[m][n]);
      }
      }
      cur = cur + STAGE == RING * STAGE ? 0 : cur + STAGE;
    };
    auto reduce = [&](auto &to, auto tn_, int units, int wrow) {
#pragma clang loop unroll(disable)
      for (; units >= UPS; units -= UPS) {
        next_stage();
        multiply(to, tn_, std::true_type{}, UPS, wrow);
      }
      if (units > 0) {
        next_stage();
        multiply(to, tn_, std::false_type{}, units, wrow);
      }
    };
    reduce(acc, std::integral_constant<int, TN>{}, a.units, wn * TN * 32);
    if constexpr (KIND == kBack) reduce(acc2, std::integral_constant<int, TN2>{}, a.units2, wn * TN2 * 32);

    // ---- what follows the product, in registers ----
    const int tm = t / a.nt, tn = t - tm * a.nt;
    const float *side = reinterpret_cast<const float *>(smem) + RING * STAGE / 4 + cside * SIDE;
    cside = cside + 1 == RING ? 0 : cside + 1;
    const int64_t m0 = (int64_t)tm * BM;
    const int have = (int)(a.M - m0 < BM ? a.M - m0 : BM);
    auto rows_at = [&](const void *p, int64_t ld) {  // the tile's rows of an output; past them loads give zero, stores are dropped
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(uniform(static_cast<const char *>(p) + m0 * ld * sizeof(TO))), 0,
                                               (int)(have * ld * sizeof(TO)), 0x00027000);
    };
    const TO *type = nullptr;
    auto bias_of = [&](int n) { return side + (wn * TN + n) * 32; };  // of the wave's n-th tile of weight rows
    auto scale_of = [&](int n) { return side + BN + (wn * TN + n) * 32; };
    // kPeak leaves none; row_scale's stores of kCodes come on top
    stored = KIND == kGated || KIND == kBack || KIND == kCodes || (KIND == kPlain && a.vec);
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      const int rl = (wm * TM + m) * 32 + i;  // row of the tile
      const float sx = E::kBytes == 1 ? side[2 * BN + rl] : 1.f;
      const unsigned at = (unsigned)(rl * a.ldo * sizeof(TO));
      if constexpr (KIND == kPlain) {
        if (a.vec) {
          const Buffer out = rows_at(a.out, a.ldo);
          // the residual's loads run one tile ahead
          Quad<TO> add[2][4];
          const Buffer res = rows_at(a.residual ? a.residual : a.out, a.ldo);
          auto ask = [&](int n) {
            if (a.residual) {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int c = tn * CN + (wn * TN + n) * 32 + 8 * q + 4 * g;
                add[n & 1][q].load(res, c < a.N ? at + (unsigned)sizeof(TO) * c : kNowhere);
              }
            }
          };
          ask(0);
#pragma unroll
          for (int n = 0; n < TN; ++n) {
            if (n + 1 < TN) ask(n + 1);
            f32x16 v = values_of<E>(acc[m][n], bias_of(n), scale_of(n), g, sx);
            act_values<sizeof(TO) == 2>(a.act, v);
            if (a.residual) {
#pragma unroll
              for (int r = 0; r < 16; ++r) v[r] += add[n & 1][r / 4][r % 4];
            }
            store_tile(v, out, at, tn * CN + (wn * TN + n) * 32, a.N, g, type);
          }
        } else {  // rows that are not whole units
          const int64_t first = m0 * a.ldo * (int64_t)sizeof(TO);
          char *to = const_cast<char *>(uniform(static_cast<const char *>(a.out) + first));
          const char *from = uniform(static_cast<const char *>(a.residual ? a.residual : a.out) + first);
#pragma unroll
          for (int n = 0; n < TN; ++n) {
            const int col = tn * CN + (wn * TN + n) * 32;
            f32x16 v = values_of<E>(acc[m][n], bias_of(n), scale_of(n), g, sx);
            act_values<sizeof(TO) == 2>(a.act, v);
            if (a.residual && rl < have) {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int c = col + 8 * q + 4 * g;
                float four[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
                if (c < a.N) add_quad(reinterpret_cast<const TO *>(from + (at + (unsigned)sizeof(TO) * c)), a.N - c, four);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * q + j] = four[j];
                __builtin_amdgcn_sched_barrier(0);  // few registers are left beside the accumulators
              }
            }
            store_tile_loose(v, to, at, rl < have, col, a.N, g, type);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      } else if constexpr (KIND == kPeak || KIND == kCodes) {
        // both passes run the same operations on the same sums: no code passes 127
        const uint32_t top_bits = KIND == kCodes ? __float_as_uint(side[2 * BN + BM + rl]) : 0u;
        const float top = __uint_as_float(top_bits);
        const bool finite = top_bits < 0x7f800000u;
        const float by = finite && top >= 0x1p-100f ? 127.f / top : 0.f;  // a smaller layer counts as zero
        uint32_t most = 0;
        const Buffer out = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char *>(uniform(static_cast<const char *>(a.out) + m0 * a.ldo)), 0, (int)(((have + 31) & ~31) * a.ldo), 0x00027000);
#pragma unroll
        for (int n = 0; n < TN2; ++n) {
          const int col = tn * CN + (wn * TN2 + n) * 32;
          f32x16 h = values_of<E>(acc[m][2 * n], bias_of(2 * n), scale_of(2 * n), g, sx);
          const f32x16 up = values_of<E>(acc[m][2 * n + 1], bias_of(2 * n + 1), scale_of(2 * n + 1), g, sx);
          act_values<sizeof(TO) == 2>(a.act, h);
#pragma unroll
          for (int r = 0; r < 16; ++r) h[r] *= up[r];
          if (col + 32 > a.N) {
#pragma unroll
            for (int r = 0; r < 16; ++r) h[r] = col + rowmap(r, g) < a.N ? h[r] : 0.f;
          }
          if constexpr (KIND == kPeak) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const uint32_t b = __float_as_uint(h[r]) & 0x7fffffffu;
              most = b > most ? b : most;
            }
          } else {
            uint32_t w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              int c[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) c[j] = (int)rintf(h[4 * q + j] * by);
              const uint32_t lo = __builtin_amdgcn_perm((uint32_t)c[1], (uint32_t)c[0], 0x0c0c0400u);
              w[q] = __builtin_amdgcn_perm((uint32_t)c[3], (uint32_t)c[2], 0x04000c0cu) | lo;
            }
            const auto r0 = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
            const auto r1 = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
            const u32x4 s = {r0[0], r0[1], r1[0], r1[1]};
            const unsigned place = (unsigned)((rl & ~31) * a.ldo + (rl & 31) * 32 + 32 * col + 16 * g);
            __builtin_amdgcn_raw_buffer_store_b128(s, out, col + 16 * g < a.limit ? place : kNowhere, 0, 0);
          }
        }
        if constexpr (KIND == kPeak) {
          const auto r = __builtin_amdgcn_permlane32_swap(most, most, false, false);
          most = r[0] > r[1] ? r[0] : r[1];
          if (g == 0 && rl < have) atomicMax(a.peak + m0 + rl, most);  // a maximum: the order does not matter
        } else if (tn == 0 && wn == 0 && g == 0 && rl < have) {
          a.row_scale[m0 + rl] = finite ? top / 127.f : __uint_as_float(0x7fc00000u);
        }
      } else {
        constexpr bool GROUPS = kGrouped<TO> && E::kBytes == 2;
        auto rows_or_blocks_at = [&](const void *p, int64_t ld) {  // whole blocks of 32 rows: what lies past the last row is never read as a value
          const int rows = GROUPS ? (have + 31) & ~31 : have;
          return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(uniform(static_cast<const char *>(p) + m0 * ld * sizeof(TO))), 0,
                                                   (int)(rows * ld * sizeof(TO)), 0x00027000);
        };
        auto place_of = [&](int64_t ld) {  // of this lane's row
          return GROUPS ? (unsigned)((rl & ~31) * ld * sizeof(TO) + (rl & 31) * 32) : (unsigned)(rl * ld * sizeof(TO));
        };
        const Buffer out = rows_or_blocks_at(a.out, a.ldo);
        const unsigned at_out = place_of(a.ldo);
#pragma unroll
        for (int n = 0; n < TN2; ++n) {
          const int col = tn * CN + (wn * TN2 + n) * 32;
          f32x16 gate = values_of<E>(acc[m][2 * n], bias_of(2 * n), scale_of(2 * n), g, sx);
          f32x16 up = values_of<E>(acc[m][2 * n + 1], bias_of(2 * n + 1), scale_of(2 * n + 1), g, sx);
          const bool whole = col + 32 <= a.N;
          auto cut = [&](f32x16 &v) {  // weight rows past the last one were repeated
            if (!whole) {
#pragma unroll
              for (int r = 0; r < 16; ++r) v[r] = col + rowmap(r, g) < a.N ? v[r] : 0.f;
            }
          };
          if constexpr (KIND == kGated) {
            act_values<sizeof(TO) == 2>(a.act, gate);
#pragma unroll
            for (int r = 0; r < 16; ++r) gate[r] *= up[r];
            cut(gate);
            store_tile<GROUPS>(gate, out, at_out, col, a.limit, g, type);
          } else {
            const Buffer hidden = rows_or_blocks_at(a.out2, a.ldh);
            f32x16 slope, d = acc2[m][n];
            act_slopes<sizeof(TO) == 2>(a.act, gate, slope);
            f32x16 h;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              h[r] = gate[r] * up[r];
              slope[r] *= d[r] * up[r];
              gate[r] *= d[r];
            }
            cut(h), cut(slope), cut(gate);
            if (E::kBytes == 2 && a.sums) {
              if (rl >= have) {  // a repeated row
#pragma unroll
                for (int r = 0; r < 16; ++r) slope[r] = gate[r] = 0.f;
              }
              const f32x4 s = column_sums(slope, gate, lane);
              const int c = col + 8 * (lane & 3) + 4 * g;
              if (i < 8 && c < a.limit && (wm * TM + m) * 32 < have)
                *reinterpret_cast<f32x4 *>(a.sums + (m0 / 32 + wm * TM + m) * 2 * a.ldh + (i & 4 ? a.ldh : 0) + c) = s;
            }
            store_tile<GROUPS>(slope, out, at_out, col, a.limit, g, type);
            store_tile<GROUPS>(gate, out, at_out + (unsigned)(a.ldh * sizeof(TO)) * (GROUPS ? 32 : 1), col, a.limit, g, type);
            store_tile<GROUPS>(h, hidden, place_of(a.ldh), col, a.limit, g, type);
          }
        }
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing is landing in LDS when the workgroup ends
}

template <class E, class TO, Kind KIND, class CFG>
int launch_tiles(Args a, int num_cu, hipStream_t st) {
  constexpr int CN = KIND == kPlain ? CFG::BN : CFG::BN / 2;
  constexpr size_t lds = CFG::lds(E::kBytes, KIND);
  static_assert(lds <= kMaxLdsBytes, "the ring fits a workgroup");
  const int64_t mt = (a.M + CFG::BM - 1) / CFG::BM, nt = (a.N + CN - 1) / CN;
  if (mt * nt > (int64_t)1 << 30) return PA_ERR_UNSUPPORTED;
  a.mt = (int)mt, a.nt = (int)nt;
  constexpr int by_lds = (int)(kMaxLdsBytes / lds), by_waves = CFG::OCC * 4 / CFG::WAVES, per_cu = by_lds < by_waves ? by_lds : by_waves;
  int64_t grid = (int64_t)num_cu * (per_cu < 1 ? 1 : per_cu);
  if (grid > mt * nt) grid = mt * nt;
  grid = (grid + 7) / 8 * 8;  // every XCD the same number
  auto kernel = rows_tile_kernel<E, TO, KIND, CFG>;
  if (int rc = allow_dynamic_lds(kernel, lds)) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * CFG::WAVES), lds, st, a);
  return launch_status();
}

// ---------------------------------------------------------------------------------------------------------------
// few_rows_kernel.  Products of so few rows that tiles of them leave most CUs idle while each works through the whole reduction,
// a stage behind the other.  A workgroup of eight waves forms 32 rows x 32 columns (kGated: both factors of them); each wave takes an
// eighth of the reduction, operands straight from memory to registers, CHUNK steps of loads in flight and no barrier; the eight
// sums meet in LDS and are added in the order of the waves.  Tiles are dealt out to the XCDs in eight equal runs with the rows running
// fastest, so that the workgroups of an L2 share columns of W.
// ---------------------------------------------------------------------------------------------------------------
template <class E, class TO, Kind KIND>
__global__ __launch_bounds__(512) void few_rows_kernel(Args a) {
  constexpr int UNITS = E::kBytes == 4 ? 4 : 2, HALVES = UNITS / 2, PAIR = KIND == kGated ? 2 : 1;  // units of a step; products
  constexpr int CHUNK = (E::kBytes == 4 ? 8 : 16) / PAIR;
  using Acc = typename E::Acc;
  extern __shared__ u32x4 smem[];  // [wave][product][q][lane]
  const int lane = threadIdx.x & 63, i = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8, tn = tile / a.mt, tm = tile - tn * a.mt;
  if (tn >= a.nt) return;
  const int64_t m = (int64_t)tm * 32 + i;
  const int n = tn * 32 + i < a.N ? tn * 32 + i : a.N - 1;
  const char *xp = static_cast<const char *>(a.X) + (a.x_groups ? (int64_t)tm * 32 * a.ldx + i * 32 : (m < a.M ? m : a.M - 1) * a.ldx);
  const char *wp[PAIR];
#pragma unroll
  for (int k = 0; k < PAIR; ++k) wp[k] = static_cast<const char *>(a.W[k]) + n * a.ldw;
  const int steps = (a.units + UNITS - 1) / UNITS, per = (steps + 7) / 8, first = wave * per, last = first + per < steps ? first + per : steps;
  Acc acc[PAIR];
#pragma unroll
  for (int k = 0; k < PAIR; ++k)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[k][r] = 0;
#pragma clang loop unroll(disable)
  for (int s = first; s < last; s += CHUNK) {
    u32x4 x[CHUNK][HALVES], w[PAIR][CHUNK][HALVES];
#pragma unroll
    for (int c = 0; c < CHUNK; ++c) {
      if (s + c >= last) break;
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        const int want = UNITS * (s + c) + 2 * h + g, u = want < a.units ? want : a.units - 1;
        x[c][h] = *reinterpret_cast<const u32x4 *>(xp + (a.x_groups ? u / 2 * 1024 + u % 2 * 16 : u * 16));
#pragma unroll
        for (int k = 0; k < PAIR; ++k) w[k][c][h] = *reinterpret_cast<const u32x4 *>(wp[k] + u * 16);
      }
    }
#pragma unroll
    for (int c = 0; c < CHUNK; ++c) {
      if (s + c >= last) break;
      if (UNITS * (s + c + 1) > a.units) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
          if (UNITS * (s + c) + 2 * h + g >= a.units) {
            x[c][h] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int k = 0; k < PAIR; ++k) w[k][c][h] = u32x4{0u, 0u, 0u, 0u};
          }
      }
      if constexpr (E::kBytes == 4) {
        const typename E::Parts xs = E::split(x[c][0], x[c][1]);
#pragma unroll
        for (int k = 0; k < PAIR; ++k) acc[k] = E::mma(E::split(w[k][c][0], w[k][c][1]), xs, acc[k]);
      } else {
#pragma unroll
        for (int k = 0; k < PAIR; ++k) acc[k] = E::mma(w[k][c][0], x[c][0], acc[k]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < PAIR; ++k)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const auto r = acc[k][4 * q + j];
        v[j] = __builtin_bit_cast(uint32_t, r);
      }
      smem[((wave * PAIR + k) * 4 + q) * 64 + lane] = v;
    }
  __syncthreads();
  if (wave >= 4) return;
  const int q = wave, col = tn * 32 + 8 * q + 4 * g;
  const float sx = E::kBytes == 1 && m < a.M ? a.sx[m] : 1.f;
  f32x4 v[PAIR];
#pragma unroll
  for (int k = 0; k < PAIR; ++k) {
    using Sum = typename std::conditional<E::kBytes == 1, int, float>::type;
    Sum sum[4] = {};
#pragma unroll
    for (int from = 0; from < 8; ++from) {
      const u32x4 t = smem[((from * PAIR + k) * 4 + q) * 64 + lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t bits = t[j];
        sum[j] += __builtin_bit_cast(Sum, bits);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = col + j < a.N;
      const float bias = a.bias[k] && in ? a.bias[k][col + j] : 0.f;
      if constexpr (E::kBytes == 1) v[k][j] = fmaf((float)sum[j], (in ? a.sw[k][col + j] : 0.f) * sx, bias);
      else v[k][j] = sum[j] + bias;
    }
  }
  act_values<sizeof(TO) == 2>(a.act, v[0]);
  if (m >= a.M) return;
  if constexpr (KIND == kGated) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[0][j] = col + j < a.N ? v[0][j] * v[1][j] : 0.f;
    if (col >= a.limit) return;
    char *to = static_cast<char *>(a.out) + (kGrouped<TO> ? m / 32 * 32 * a.ldo * 2 + col / 16 * 1024 + m % 32 * 32 + col % 16 * 2
                                                           : (m * a.ldo + col) * (int64_t)sizeof(TO));
    if constexpr (sizeof(TO) == 2) *reinterpret_cast<u32x2 *>(to) = u32x2{pack2(v[0][0], v[0][1]), pack2(v[0][2], v[0][3])};
    else *reinterpret_cast<f32x4 *>(to) = v[0];
  } else {
    TO *to = static_cast<TO *>(a.out) + m * a.ldo + col;
    const TO *add = a.residual ? static_cast<const TO *>(a.residual) + m * a.ldo + col : nullptr;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (add && col + j < a.N) v[0][j] += load_as_f32(add + j);
    if (a.vec) {  // whole units: four columns or none
      if (col >= a.N) return;
      if constexpr (sizeof(TO) == 2) *reinterpret_cast<u32x2 *>(to) = u32x2{pack2(v[0][0], v[0][1]), pack2(v[0][2], v[0][3])};
      else *reinterpret_cast<f32x4 *>(to) = v[0];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < a.N) store_from_f32(to + j, v[0][j]);
    }
  }
}

// Whether it is the shorter way, in us behind the launch: what a wave works through one after the other, its eighth of the reduction
// for every round of workgroups over the CUs, against all stages of a 64 x 64 tile, as long as those are one round.  Measured, tiles
// / few rows:
// bf16 2 048 -> 512, 64 rows 17.9 / 8.8, 1 000 (two rounds) 18.0 / 17.1, 1 500 17.8 / 25.0; 512 -> 2 x 2 048, 64 rows 6.5 / 6.9;
// float32 2 048 -> 512, 64 rows 75.6 / 21.9, 1 500 77.6 / 68.5, 2 000 77.9 / 89.3, 512 -> 2 x 2 048, 64 rows 21.6 / 10.1, 400 32.7 /
// 36.4; int8 512 -> 2 048, 64 rows 6.0 / 4.3, 400 6.3 / 9.5, 2 048 -> 512, 64 rows 11.0 / 7.6, 600 11.3 / 12.3.  The 8-bit gated pair has
// no such form: its codes need the largest value of a whole row first.
inline bool few_rows_worth(int bytes, Kind kind, int64_t M, int64_t N, int64_t row_units, int64_t stages, int num_cu) {
  if (kind != kPlain && !(kind == kGated && bytes != 1)) return false;
  const double step = bytes == 4 ? 1.2 : 0.4;  // of a tile's stage and of a wave's step alike
  const int64_t units = bytes == 4 ? 4 : 2, per = ((row_units + units - 1) / units + 7) / 8;
  const int64_t groups = ((M + 31) / 32) * ((N + 31) / 32), columns = kind == kGated ? 32 : 64;
  const int64_t tiles = ((M + 63) / 64) * ((N + columns - 1) / columns);
  const int64_t rounds = (groups + num_cu - 1) / num_cu;
  return tiles <= num_cu && rounds * (1.5 + step * per * (kind == kGated ? 2 : 1)) <= 1.5 + step * stages;
}

template <class E, class TO, Kind KIND>
int launch_few_rows(Args a, hipStream_t st) {
  constexpr size_t lds = 8 * (KIND == kGated ? 2 : 1) * 4 * 1024;
  a.mt = (int)((a.M + 31) / 32), a.nt = (a.N + 31) / 32;
  auto kernel = few_rows_kernel<E, TO, KIND>;
  if (int rc = allow_dynamic_lds(kernel, lds)) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(((int64_t)a.nt * a.mt + 7) / 8 * 8)), dim3(512), lds, st, a);
  return launch_status();
}

// Tiles of 256 x 256 (kBack: 128 x 256) for large products, 128 x 128 and two workgroups per CU where those leave CUs idle, 64 x 64
// where the product is small.  Taken by the weight rows and rows that the busiest CU has to work off, smaller tiles counted
// dearer for the operands they fetch again.  Measured at 256 / 128 (us): 131 072 rows, 1 024 -> 256 bf16 107 / 117, 2 048 -> 256
// 162 / 189, 256 -> 2 x 1 024 201 / 227; int8 131 072 rows 2 048 -> 512 144 / 193; float32 28 900 rows, 512 -> 128 126 / 43.
// Rows past whole rounds of large tiles go to a launch of smaller ones where that is the shorter way: 100 003 rows, 1 368 -> 512,
// three rounds and 1 699 rows: 254 -> 214 us.
struct Plan {
  int64_t rows;  // on tiles of `size`; the rest on tiles of their own
  int size;      // 0 large, 1 medium, 2 small
  double cost;   // in stages of a large tile
};
inline Plan plan_of(int64_t M, int64_t N, int64_t stages, bool back, bool pairs, int num_cu, bool split) {
  const double launch = 2.5;  // of one more launch: about 8 us
  auto cost = [&](int64_t rows, int64_t bm, int64_t bn, double dearer) {
    const int64_t cn = pairs ? bn / 2 : bn, tiles = ((rows + bm - 1) / bm) * ((N + cn - 1) / cn);
    return (double)((tiles + num_cu - 1) / num_cu) * bm * bn * dearer * stages / 65536;
  };
  const int64_t bm = back ? 128 : 256;
  const double of[3] = {cost(M, bm, 256, 1.0), cost(M, 128, 128, 1.13), cost(M, 64, 64, 1.5)};
  Plan p{M, of[0] <= of[1] && of[0] <= of[2] ? 0 : of[1] <= of[2] ? 1 : 2, 0.0};
  p.cost = of[p.size];
  if (split) {
    const int64_t cn = pairs ? 128 : 256, nt = (N + cn - 1) / cn, rounds = (M / bm) * nt / num_cu, rows = rounds * num_cu / nt * bm;
    if (rounds > 0 && rows < M) {
      const double c = cost(rows, bm, 256, 1.0) + launch + plan_of(M - rows, N, stages, back, pairs, num_cu, false).cost;
      if (c < p.cost) return Plan{rows, 0, c};
    }
  }
  return p;
}

// The launches of a product: on tiles of `size` (3: few_rows_kernel) the first rows[0] rows, the rest on tiles of their own.
struct Launches {
  int64_t rows[2];
  int size[2];
};
inline Launches launches_of(int bytes, Kind kind, int64_t M, int64_t N, int64_t units, int64_t units2, int num_cu) {
  const bool back = kind == kBack, pairs = kind != kPlain;
  const int64_t stages = (units + 7) / 8 + (back ? (units2 + 7) / 8 : 0);
  if (few_rows_worth(bytes, kind, M, N, units, stages, num_cu)) return {{M, 0}, {3, 0}};
  const Plan p = plan_of(M, N, stages, back, pairs, num_cu, true);
  if (p.rows == M) return {{M, 0}, {p.size, 0}};
  return {{p.rows, M - p.rows}, {p.size, plan_of(M - p.rows, N, stages, back, pairs, num_cu, false).size}};
}

template <class E, class TO, Kind KIND>
int launch(Args a, int num_cu, hipStream_t st) {
  using Large = typename std::conditional<KIND == kBack, Config<2, 4, 2, 2, 8, 3, 2>, Config<4, 2, 2, 4, 8, 2, 2>>::type;
  using Medium = Config<2, 2, 2, 2, 8, 2, 2>;
  using Small = Config<2, 1, 1, 2, 8, 3, 2>;
  const Launches l = launches_of(E::kBytes, KIND, a.M, a.N, a.units, a.units2, num_cu);
  if constexpr (KIND == kPlain || (KIND == kGated && E::kBytes != 1))
    if (l.size[0] == 3) return launch_few_rows<E, TO, KIND>(a, st);
  auto run = [&](const Args &t, int size) {
    if (size == 0) return launch_tiles<E, TO, KIND, Large>(t, num_cu, st);
    if (size == 1) return launch_tiles<E, TO, KIND, Medium>(t, num_cu, st);
    return launch_tiles<E, TO, KIND, Small>(t, num_cu, st);
  };
  Args rest = a;
  a.M = l.rows[0];
  int rc = run(a, l.size[0]);
  if (rc || l.rows[1] == 0) return rc;
  auto past = [&](const void *q, int64_t row) { return q ? const_cast<char *>(static_cast<const char *>(q)) + l.rows[0] * row : nullptr; };
  rest.M = l.rows[1];
  rest.X = past(a.X, a.ldx), rest.X2 = past(a.X2, a.ldx2);
  rest.sx = a.sx ? a.sx + l.rows[0] : nullptr;
  rest.sums = a.sums ? a.sums + l.rows[0] / 32 * 2 * a.ldh : nullptr;
  rest.peak = a.peak ? a.peak + l.rows[0] : nullptr, rest.row_scale = a.row_scale ? a.row_scale + l.rows[0] : nullptr;
  rest.residual = past(a.residual, a.ldo * (int64_t)sizeof(TO));
  rest.out = past(a.out, a.ldo * (int64_t)(KIND == kCodes ? 1 : sizeof(TO))), rest.out2 = past(a.out2, a.ldh * (int64_t)sizeof(TO));
  return run(rest, l.size[1]);
}

// ---- host side of the calls that use the products ----
inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

struct Space {  // workspace carved in order; without a base it only counts
  char *base;
  int64_t used = 0;
  void *take(int64_t bytes) {
    void *p = base ? base + used : nullptr;
    used += up(bytes, 256);
    return p;
  }
};

inline bool whole_rows(const void *p, int64_t width, int64_t elem) { return aligned16(p) && width * elem % 16 == 0; }

// Matrices to be copied into padded rows or transposed, in one launch.
struct Layout {
  static constexpr int kMost = 8;
  struct One {
    const void *src;
    void *dst;
    int64_t rows, first;  // of dst; the launch's first workgroup for it
    int cols, width;      // of dst: columns with values; columns that are written, zeros from `cols` on
    int64_t ld, src_ld;   // elements between rows
    bool turned;          // dst[r][c] = src[c][r]
  } m[kMost];
  int count = 0;
  int64_t blocks = 0;
  void add(const void *src, int64_t src_ld, void *dst, int64_t rows, int64_t cols, int64_t width, int64_t ld, bool turned) {
    m[count++] = One{src, dst, rows, blocks, (int)cols, (int)width, ld, src_ld, turned};
    blocks += (rows + 63) / 64 * ((width + 63) / 64);
  }
};
int lay_out(const Layout &a, size_t elem_bytes, hipStream_t st);

}  // namespace tile
}  // namespace pa
