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
struct F32 {
  using Acc = f32x16;
  static constexpr int kBytes = 4;
  static __device__ __forceinline__ Acc mma(u32x4 a, u32x4 b, Acc c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = a[j], y = b[j];
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(x), __uint_as_float(y), c, 0, 0, 0);
    }
    return c;
  }
};
struct I8 {
  using Acc = i32x16;
  static constexpr int kBytes = 1;
  static __device__ __forceinline__ Acc mma(u32x4 a, u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
  }
};

// ---- activations of the library's Mlp (see pa_gated_act_code) ----
enum Act { kNone = 0, kGelu = 1, kRelu = 2, kSilu = 3, kSigmoid = 4, kTanh = 5, kActs = 6 };

__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * v)); }

__device__ __forceinline__ void act_values(int act, f32x16 &v) {
  switch (act) {
    case kGelu:
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] = gelu_fit(v[r]);
      break;
    case kRelu:  // NaN passes, as torch's does
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] = v[r] < 0.f ? 0.f : v[r];
      break;
    case kSilu:
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] *= sigmoid(v[r]);
      break;
    case kSigmoid:
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] = sigmoid(v[r]);
      break;
    case kTanh:
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] = tanhf(v[r]);
      break;
    default: break;
  }
}

// v <- act(v), slope <- act'(v)
__device__ __forceinline__ void act_slopes(int act, f32x16 &v, f32x16 &slope) {
  switch (act) {
    case kGelu:
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = v[r];
        const GeluParts p = gelu_parts(x);
        slope[r] = gelu_grad(x, p);
        v[r] = x * p.phi;
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
};

struct Args {
  const void *X, *X2;            // rows of activations; a row is `units` units of 16 bytes, ldx / ldx2 bytes apart
  const void *W[3];              // rows of weights, ldw / ldw2 (W[2]) bytes apart
  int64_t ldx, ldx2, ldw, ldw2;
  int units, units2;             // of the reduction over X, over X2
  int64_t M;
  int N, limit;                  // columns; columns N .. limit - 1 are written as zeros (limit: a multiple of a unit's elements, or N)
  const float *bias[2];          // or NULL
  const float *sx, *sw[2];       // int8: scale per row of X, per row of W
  const void *residual;          // (M, N), kPlain, or NULL
  void *out, *out2;
  int64_t ldo, ldh;              // elements between rows of out (residual alike); of out2, and from dg to du
  int act;
  bool vec;                      // out and residual start on 16 bytes and their rows are whole units apart
  int mt, nt;                    // tiles
};

// four neighbouring floats (p on any float); past the last of n that one again
__device__ __forceinline__ f32x4 quad_at(const float *p, int col, int n, bool whole) {
  typedef float f32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
  if (whole) return *reinterpret_cast<const f32x4_at4 *>(p + col);
  f32x4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = p[col + j < n ? col + j : n - 1];
  return v;
}

__device__ __forceinline__ f32x4 widen4(const float *p) { return *reinterpret_cast<const f32x4 *>(p); }
__device__ __forceinline__ f32x4 widen4(const bf16 *p) {
  const u32x2 w = *reinterpret_cast<const u32x2 *>(p);
  const uint32_t a = w[0], b = w[1];
  return f32x4{__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u), __uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u)};
}

// columns col .. col + 31 (below limit) of this lane's row; row points at the row's column 0
template <bool VEC>
__device__ __forceinline__ void store_tile(const f32x16 &v, bf16 *row, int col, int limit, int g, bool ok) {
  if constexpr (VEC) {
    u32x4 s0, s1;
    mfma::tile_natural(v, s0, s1);
    const int c = col + 16 * g;
    if (ok && c < limit) *reinterpret_cast<u32x4 *>(row + c) = s0;
    if (ok && c + 8 < limit) *reinterpret_cast<u32x4 *>(row + c + 8) = s1;
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int c = col + rowmap(r, g);
      if (ok && c < limit) row[c].bits = mfma::to_bf16_bits(v[r]);
    }
  }
}
template <bool VEC>
__device__ __forceinline__ void store_tile(const f32x16 &v, float *row, int col, int limit, int g, bool ok) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int c = col + 8 * q + 4 * g;
    if constexpr (VEC) {
      if (ok && c < limit) *reinterpret_cast<f32x4 *>(row + c) = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (ok && c + j < limit) row[c + j] = v[4 * q + j];
    }
  }
}

// accumulators to float32: int8 sums take their scales; then the bias.  Columns past N hold something of column N - 1.
template <class E>
__device__ __forceinline__ f32x16 values_of(const typename E::Acc &acc, const Args &a, int which, int col, int g, float sx) {
  f32x16 v;
  const bool whole = col + 32 <= a.N;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int c = col + 8 * q + 4 * g;
    f32x4 b = {0.f, 0.f, 0.f, 0.f}, s = b;
    if (a.bias[which]) b = quad_at(a.bias[which], c, a.N, whole);
    if constexpr (E::kBytes == 1) s = quad_at(a.sw[which], c, a.N, whole) * sx;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (E::kBytes == 1) v[4 * q + j] = (float)acc[4 * q + j] * s[j] + b[j];
      else v[4 * q + j] = acc[4 * q + j] + b[j];
    }
  }
  return v;
}

// ---------------------------------------------------------------------------------------------------------------
// rows_tile_kernel.  A workgroup of WM x WN waves owns tiles of BM rows x BN weight rows; a wave's part is TM x TN tiles of
// 32 x 32.  kGated and kBack take 32 rows of W0 and the 32 rows of W1 in turn, so that a wave holds both factors of its
// hidden units.  Stages of 128 bytes of every row pass through two LDS buffers, filled by direct global -> LDS loads while
// the stage before is multiplied, one barrier per stage; the stages of a workgroup's tiles form one sequence, so that the
// first stage of a tile arrives behind the last products and the stores of the one before.
// Position p of row r holds the row's unit p ^ (r / 2 % 8): the 16 lanes of an access phase fall on all 64 banks.
// Units past a row's last one repeat it and are left out of the products; rows past the last row repeat it and are not stored.
// Tiles are dealt out to the XCDs (= workgroup id mod 8) in eight equal runs with the columns running fastest, so that the
// workgroups of an L2 share rows of X and W.
// ---------------------------------------------------------------------------------------------------------------
template <class E, class TO, Kind KIND, int WM, int WN, int TM, int TN, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void rows_tile_kernel(Args a) {
  constexpr int WAVES = WM * WN, BM = WM * TM * 32, BN = WN * TN * 32;
  constexpr bool DUAL = KIND != kPlain;
  constexpr int NX = BM / 8 / WAVES, NW = BN / 8 / WAVES, TN2 = TN / 2;  // groups of 8 rows a wave fetches
  static_assert(BM % (8 * WAVES) == 0 && BN % (16 * WAVES) == 0, "whole groups");
  static_assert(!DUAL || TN % 2 == 0, "pairs of tiles");
  constexpr unsigned STAGE = (BM + BN) * 128;
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

  const int nk1 = (a.units + 7) / 8, nk = nk1 + (KIND == kBack ? (a.units2 + 7) / 8 : 0);

  // ---- the loads run one stage ahead of the products ----
  int lt = t, lk = 0;       // tile and stage that are fetched next
  unsigned buf = 0;         // where they go
  unsigned offx[NX], offw[NW];
  const char *xbase = nullptr, *wbase[2] = {nullptr, nullptr};
  const int frow = lane >> 3;
  auto uniform = [](const char *p) {  // what is the same for every lane, in scalar registers
    const uint64_t v = (uint64_t)(uintptr_t)p;
    return reinterpret_cast<const char *>((uintptr_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
                                                      (uint32_t)__builtin_amdgcn_readfirstlane((int)v)));
  };
  auto unit_of = [&](int row) { return (lane & 7) ^ ((row >> 1) & 7); };
  auto place = [&](bool second) {  // offsets of tile lt: rows of X and W (second: of X2 and W[2])
    const int tm = lt / a.nt, tn = lt - tm * a.nt;
    const int64_t m0 = (int64_t)tm * BM, ldx = second ? a.ldx2 : a.ldx, ldw = second ? a.ldw2 : a.ldw;
    const int have = (int)(a.M - m0 < BM ? a.M - m0 : BM), n0 = tn * CN, haven = a.N - n0;
    xbase = static_cast<const char *>(second ? a.X2 : a.X) + m0 * ldx;
    wbase[0] = static_cast<const char *>(second ? a.W[2] : a.W[0]) + n0 * ldw;
    if constexpr (DUAL) wbase[1] = static_cast<const char *>(a.W[1]) + n0 * ldw;
#pragma unroll
    for (int q = 0; q < NX; ++q) {
      const int row = (wave * NX + q) * 8 + frow, r = row < have ? row : have - 1;
      offx[q] = (unsigned)(r * ldx) + 16 * unit_of(row);
    }
#pragma unroll
    for (int q = 0; q < NW; ++q) {
      const int row = second ? (wave * (NW / 2) + (q < NW / 2 ? q : 0)) * 8 + frow : (wave * NW + q) * 8 + frow;
      const int col = DUAL && !second ? (row >> 6) * 32 + (row & 31) : row, c = col < haven ? col : haven - 1;
      offw[q] = (unsigned)(c * ldw) + 16 * unit_of(row);
    }
  };
  auto fetch = [&]() {
    if (lt >= last) return;
    const bool second = KIND == kBack && lk >= nk1;
    if (lk == 0 || (KIND == kBack && lk == nk1)) place(second);
    const int kb = second ? lk - nk1 : lk, left = (second ? a.units2 : a.units) - 8 * kb;
    const unsigned dst = (unsigned)(uintptr_t)smem + buf;
    // units past the row's last one: that one again; the products leave them out
    auto past = [&](int unit) { return 16u * (unsigned)(unit >= left ? unit - left + 1 : 0); };
    const unsigned past_even = past((lane & 7) ^ (frow >> 1)), past_odd = past((lane & 7) ^ (frow >> 1) ^ 4);
    auto off_of = [&](unsigned off, int grp) { return (int)(off - (grp & 1 ? past_odd : past_even)); };
    const char *xs = uniform(xbase + (int64_t)kb * 128);
#pragma unroll
    for (int q = 0; q < NX; ++q) {
      const int grp = wave * NX + q;
      load_unit_to_lds(xs, off_of(offx[q], grp), dst + grp * 1024);
    }
    const char *ws0 = uniform(wbase[0] + (int64_t)kb * 128), *ws1 = DUAL ? uniform(wbase[1] + (int64_t)kb * 128) : ws0;
#pragma unroll
    for (int q = 0; q < NW; ++q) {
      if (second && q >= NW / 2) break;
      const int grp = second ? wave * (NW / 2) + q : wave * NW + q;
      load_unit_to_lds(DUAL && !second && (grp & 4) ? ws1 : ws0, off_of(offw[q], grp), dst + BM * 128 + grp * 1024);
    }
    buf ^= STAGE;
    if (++lk == nk) lk = 0, lt += step;
  };

  fetch();
  unsigned cur = 0;
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
    const int swz = (i >> 1) & 7;
    auto next_stage = [&]() {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's share of the stage has landed
      __syncthreads();                                  // everyone's; and everyone is past the stage before
      fetch();
    };
    auto multiply = [&](auto &to, auto tn_, auto whole_, int left, int wrow) {  // left: units of the stage, 8 where `whole`
      constexpr int T = decltype(tn_)::value;
      constexpr bool WHOLE = decltype(whole_)::value;
      const u32x4 *xs = smem + cur / 16 + (wm * TM * 32 + i) * 8;
      const u32x4 *ws = smem + cur / 16 + (BM + wrow + i) * 8;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        if (!WHOLE && 2 * ks >= left) break;
        const int at = (2 * ks + g) ^ swz;
        u32x4 w[T], x[TM];
#pragma unroll
        for (int n = 0; n < T; ++n) w[n] = ws[n * 256 + at];
#pragma unroll
        for (int m = 0; m < TM; ++m) x[m] = xs[m * 256 + at];
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
      cur ^= STAGE;
    };
    auto reduce = [&](auto &to, auto tn_, int units, int wrow) {
#pragma clang loop unroll(disable)
      for (; units >= 8; units -= 8) {
        next_stage();
        multiply(to, tn_, std::true_type{}, 8, wrow);
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
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      const int64_t row = (int64_t)tm * BM + (wm * TM + m) * 32 + i;
      const bool ok = row < a.M;
      const float sx = E::kBytes == 1 ? a.sx[ok ? row : a.M - 1] : 1.f;
      if constexpr (KIND == kPlain) {
#pragma unroll
        for (int n = 0; n < TN; ++n) {
          const int col = tn * CN + (wn * TN + n) * 32;
          f32x16 v = values_of<E>(acc[m][n], a, 0, col, g, sx);
          act_values(a.act, v);
          TO *out = static_cast<TO *>(a.out) + row * a.ldo;
          if (a.residual) {
            const TO *res = static_cast<const TO *>(a.residual) + row * a.ldo;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int c = col + 8 * q + 4 * g;
              f32x4 add = {0.f, 0.f, 0.f, 0.f};
              if (a.vec) {
                if (ok && c < a.N) add = widen4(res + c);
              } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  if (ok && c + j < a.N) add[j] = load_as_f32(res + c + j);
              }
#pragma unroll
              for (int j = 0; j < 4; ++j) v[4 * q + j] += add[j];
            }
          }
          if (a.vec) store_tile<true>(v, out, col, a.N, g, ok);
          else store_tile<false>(v, out, col, a.N, g, ok);
        }
      } else {
#pragma unroll
        for (int n = 0; n < TN2; ++n) {
          const int col = tn * CN + (wn * TN2 + n) * 32;
          f32x16 gate = values_of<E>(acc[m][2 * n], a, 0, col, g, sx);
          f32x16 up = values_of<E>(acc[m][2 * n + 1], a, 1, col, g, sx);
          const bool whole = col + 32 <= a.N;
          auto cut = [&](f32x16 &v) {  // weight rows past the last one were repeated
            if (!whole) {
#pragma unroll
              for (int r = 0; r < 16; ++r) v[r] = col + rowmap(r, g) < a.N ? v[r] : 0.f;
            }
          };
          if constexpr (KIND == kGated) {
            act_values(a.act, gate);
#pragma unroll
            for (int r = 0; r < 16; ++r) gate[r] *= up[r];
            cut(gate);
            store_tile<true>(gate, static_cast<TO *>(a.out) + row * a.ldo, col, a.limit, g, ok);
          } else {
            f32x16 slope, d = acc2[m][n];
            act_slopes(a.act, gate, slope);
            f32x16 h;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              h[r] = gate[r] * up[r];
              slope[r] *= d[r] * up[r];
              gate[r] *= d[r];
            }
            cut(h), cut(slope), cut(gate);
            TO *out = static_cast<TO *>(a.out) + row * a.ldo;
            store_tile<true>(slope, out, col, a.limit, g, ok);
            store_tile<true>(gate, out + a.ldh, col, a.limit, g, ok);
            store_tile<true>(h, static_cast<TO *>(a.out2) + row * a.ldh, col, a.limit, g, ok);
          }
        }
      }
    }
  }
}

template <class E, class TO, Kind KIND, int WM, int WN, int TM, int TN, int OCC>
int launch_tiles(Args a, int num_cu, hipStream_t st) {
  constexpr int BM = WM * TM * 32, BN = WN * TN * 32, CN = KIND == kPlain ? BN : BN / 2;
  constexpr size_t lds = 2 * (BM + BN) * 128;
  const int64_t mt = (a.M + BM - 1) / BM, nt = (a.N + CN - 1) / CN;
  if (mt * nt > (int64_t)1 << 30) return PA_ERR_UNSUPPORTED;
  a.mt = (int)mt, a.nt = (int)nt;
  const int per_cu = (int)(kMaxLdsBytes / lds) < OCC * 4 / (WM * WN) ? (int)(kMaxLdsBytes / lds) : OCC * 4 / (WM * WN);
  int64_t grid = (int64_t)num_cu * (per_cu < 1 ? 1 : per_cu);
  if (grid > mt * nt) grid = mt * nt;
  grid = (grid + 7) / 8 * 8;  // every XCD the same number
  auto kernel = rows_tile_kernel<E, TO, KIND, WM, WN, TM, TN, OCC>;
  if (int rc = allow_dynamic_lds(kernel, lds)) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * WM * WN), lds, st, a);
  return launch_status();
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
