// The gated feed-forward block with the hidden layer on chip, bf16 rows of up to 256 channels (see pa_gated.hip for the formulas):
// a wave owns 32 rows and all their channels, the weights stream past it in slots of 32 hidden units.  x is read once and y
// written once, where the two products of the tile kernel pass 4 F bytes per row through memory.
#include "pa_common.h"
#include "pa_host.h"
#include "pa_tile.h"

namespace pa {
namespace gated {

using mfma::f32x16;
using mfma::load_unit_to_lds;
using mfma::mma;
using mfma::pack2;
using mfma::rowmap;
using mfma::static_for;
using mfma::u32x4;
using tile::Buffer;

__host__ __device__ __forceinline__ int chunks_of(int F) { return (F + 63) / 64 * 2; }

// ---------------------------------------------------------------------------------------------------------------
// rows_pack_kernel: slot c = 0 .. NCH of the weight stream (NCH: chunks of 32 hidden units, an even number), (6 CT + 1) KB: for every k-step the fragments of W_up's and W_gate's
// rows 32 c .. + 31; then W_down's columns 32 (c - 1) .. + 31, k half major, its reduction index in the order in which the
// hidden layer leaves the accumulators (kperm); then 32 biases of each of the two.  What lies outside the matrices is zero.
// ---------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void rows_pack_kernel(const uint16_t *__restrict__ wg, const uint16_t *__restrict__ wu,
                                                        const uint16_t *__restrict__ wd, const float *__restrict__ bg,
                                                        const float *__restrict__ bu, u32x4 *__restrict__ blob, int C, int F, int CT) {
  const int KS = 2 * CT, SU = (6 * CT + 1) * 64, NCH = chunks_of(F);
  const int64_t total = (int64_t)(NCH + 1) * SU;
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < total; u += (int64_t)gridDim.x * 256) {
    const int c = (int)(u / SU), r = (int)(u - (int64_t)c * SU), frag = r >> 6, lane = r & 63, i = lane & 31, g = lane >> 5;
    u32x4 e = {0u, 0u, 0u, 0u};
    if (frag < 2 * KS) {
      const uint16_t *w = frag & 1 ? wg : wu;
      const int row = 32 * c + i, col = 16 * (frag >> 1) + 8 * g;
      if (row < F) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col + j < C) e[j / 2] |= (uint32_t)w[(int64_t)row * C + col + j] << (16 * (j & 1));
      }
    } else if (frag < 2 * KS + 2 * CT) {
      const int t = frag - 2 * KS, kk = t / CT, row = 32 * (t % CT) + i;
      if (c > 0 && row < C) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int col = 32 * (c - 1) + mfma::kperm(kk, g, j);
          if (col < F) e[j / 2] |= (uint32_t)wd[(int64_t)row * F + col] << (16 * (j & 1));
        }
      }
    } else if (lane < 16) {
      const float *b = lane < 8 ? bu : bg;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = 32 * c + 4 * (lane & 7) + j;
        if (b && at < F) e[j] = __float_as_uint(b[at]);
      }
    }
    blob[u] = e;
  }
}

struct RowsArgs {
  const u32x4 *blob;
  const uint16_t *x, *residual;
  const float *b_down;
  uint16_t *y;
  int64_t M, nblocks;
  int C, F, act;
};

// ---------------------------------------------------------------------------------------------------------------
// rows_forward_kernel<CT>: rows of up to 32 CT channels.  Per slot c a wave runs
//   u(c)^T = W_up[chunk c] x^T + b_up and g(c)^T = W_gate[chunk c] x^T + b_gate, in turn          4 CT MFMAs
//     with h(c - 1) = act(g) u of the chunk before formed behind them, 16 values in 32 pieces; two sets of accumulators take turns
//   y^T += W_down[:, chunk c - 1] h(c - 1)^T                                                      2 CT MFMAs
// CT = 8: one wave per SIMD with 512 registers (y 128, x 64, two sets of g and u 64); narrower rows: two.  One barrier per slot:
// two waves per SIMD meet at its beginning and cover each other (two LDS buffers); a wave alone has the next slot's data a
// slot earlier (three) and its first fragments and biases in registers, and meets the others behind its first products
// (262 144 x 256, F = 1 024, GELU of degree 5: 549 -> 517 us; meeting behind step 10 of 48 530; with two waves per SIMD the registers that this takes cost more than it gives,
// 262 144 x 128, F = 512, backward 197 -> 245).
// ---------------------------------------------------------------------------------------------------------------
// Twenty ticks of vector work spread evenly behind the first 5 CT matrix instructions of a slot: those behind step S.
template <int S, int CT, class F>
__device__ __forceinline__ void ticks_behind(F &&tick) {
  constexpr int first = (4 * S + CT - 1) / CT, end = (4 * (S + 1) + CT - 1) / CT;
  static_for<end - first>([&](auto p_) { tick(std::integral_constant<int, first + decltype(p_)::value>{}); });
}

// One value of h in four pieces, so that what a piece depends on lies a step of the matrix instructions behind it.
template <int ACT>
struct Gate {
  float x, t, q;
  __device__ __forceinline__ void piece0(float v) {
    x = v;
    if constexpr (ACT == tile::kSilu) {
      t = -kLog2e * v;
    } else if constexpr (ACT == tile::kGelu) {
      t = fabsf(v);
      q = gelu_short_upper_terms(t);
    }
  }
  __device__ __forceinline__ void piece1() {
    if constexpr (ACT == tile::kSilu) t = __builtin_amdgcn_exp2f(t);
    else if constexpr (ACT == tile::kGelu) q = __builtin_amdgcn_exp2f(gelu_short_lower_terms(t, q));
  }
  __device__ __forceinline__ void piece2() {
    if constexpr (ACT == tile::kSilu) t = __builtin_amdgcn_rcpf(1.f + t);
    else if constexpr (ACT == tile::kGelu) x = gelu_from_tail(x, q);
  }
  __device__ __forceinline__ float piece3(float up, int act) const {
    if constexpr (ACT == tile::kSilu) return x * t * up;
    else if constexpr (ACT == tile::kGelu) return x * up;
    switch (act) {
      case tile::kRelu: return (x < 0.f ? 0.f : x) * up;
      case tile::kSigmoid: return tile::sigmoid(x) * up;
      case tile::kTanh: return tanhf(x) * up;
      default: return x * up;
    }
  }
};

template <int CT, int ACT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(WAVES / 4, WAVES / 4))) void rows_forward_kernel(RowsArgs a) {
  constexpr int KS = 2 * CT, SU = (6 * CT + 1) * 64, NF = 6 * CT, ROWS = 32 * WAVES;
  constexpr bool ALONE = WAVES == 4;  // one wave per SIMD
  constexpr int BUFFERS = ALONE ? 3 : 2, AHEAD = 4, RING = ALONE ? 6 : AHEAD + 1, MEET = 1;
  static_assert(!ALONE || NF % RING == 0, "a slot's fragments begin where the last one's end");
  extern __shared__ u32x4 smem[];
  const int lane = threadIdx.x & 63, i = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int NCH = chunks_of(a.F), C = a.C;
  float *bd = reinterpret_cast<float *>(smem + BUFFERS * SU);  // b_down
  for (int k = threadIdx.x; k < 32 * CT; k += 64 * WAVES) bd[k] = a.b_down && k < C ? a.b_down[k] : 0.f;
  __syncthreads();
  auto fetch = [&](int buf, int c) {  // this wave's share of slot c, 1 KB at a time
    const u32x4 *src = a.blob + (int64_t)c * SU;
    const unsigned dst = (unsigned)(uintptr_t)(smem + buf * SU);
#pragma unroll
    for (int k = 0; k < (NF + 1 + WAVES - 1) / WAVES; ++k) {
      const int part = k * WAVES + wave;
      if (part < NF + 1) load_unit_to_lds(src + part * 64, lane * 16, dst + part * 1024);
    }
  };
  u32x4 xb[KS];
  auto load_rows = [&](int64_t mb) {
    int64_t r = mb * ROWS + wave * 32 + i;
    if (r >= a.M) r = a.M - 1;
    const uint16_t *src = a.x + r * C;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int col = 16 * ks + 8 * g;
      xb[ks] = *reinterpret_cast<const u32x4 *>(src + (col < C ? col : 0));  // past the last channel: W's columns are zero there
      if (32 * CT > C && col >= C) xb[ks] = u32x4{0u, 0u, 0u, 0u};
    }
  };
  auto next_of = [](int b) { return b + 1 == BUFFERS ? 0 : b + 1; };
  int buf = 0;
  u32x4 fr[RING];
  f32x16 ga[2], ua[2];
  auto biases = [&](int b, auto set_) {  // of the slot in buffer b, to accumulators SET
    constexpr int set = decltype(set_)::value;
    const float *bias = reinterpret_cast<const float *>(smem + b * SU + NF * 64);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const tile::f32x4 bu = *reinterpret_cast<const tile::f32x4 *>(bias + 8 * q + 4 * g);
      const tile::f32x4 bg = *reinterpret_cast<const tile::f32x4 *>(bias + 32 + 8 * q + 4 * g);
#pragma unroll
      for (int j = 0; j < 4; ++j) ua[set][4 * q + j] = bu[j], ga[set][4 * q + j] = bg[j];
    }
  };
  auto begin = [&](int b, auto set_) {
    static_for<AHEAD>([&](auto q) { fr[decltype(q)::value] = smem[b * SU + decltype(q)::value * 64 + lane]; });
    biases(b, set_);
  };
  fetch(0, 0);
  if (ALONE) fetch(1, 1);
  load_rows(blockIdx.x);
  if (ALONE) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    begin(0, std::integral_constant<int, 0>{});
  }
  for (int64_t mb = blockIdx.x; mb < a.nblocks; mb += gridDim.x) {
    f32x16 yacc[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const tile::f32x4 b = *reinterpret_cast<const tile::f32x4 *>(bd + 32 * ct + 8 * q + 4 * g);
#pragma unroll
        for (int j = 0; j < 4; ++j) yacc[ct][4 * q + j] = b[j];
      }
#pragma unroll
    for (int r = 0; r < 16; ++r) ga[1][r] = ua[1][r] = 0.f;  // no chunk before the first: act(0) 0 = 0
    auto slot = [&](int c, auto set_) {
      constexpr int now = decltype(set_)::value, old = 1 - now;
      if constexpr (!ALONE) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's share of the slot has landed
        __syncthreads();                                  // everyone's, and the other buffer is free
        begin(buf, set_);
      }
      const u32x4 *wb = smem + buf * SU + lane;
      u32x4 hop[2];
      Gate<ACT> gate[4];
      float even = 0.f;
      auto tick = [&](auto t_) {  // pieces of values T, T - 1, T - 2, T - 3
        constexpr int T = decltype(t_)::value;
        if constexpr (T >= 3 && T < 19) {
          constexpr int J = T - 3;
          const float h = gate[J % 4].piece3(ua[old][J], a.act);
          if constexpr (J % 2 == 0) even = h;
          else hop[J / 8][J / 2 % 4] = pack2(even, h);
        }
        if constexpr (T >= 2 && T < 18) gate[(T - 2) % 4].piece2();
        if constexpr (T >= 1 && T < 17) gate[(T - 1) % 4].piece1();
        if constexpr (T < 16) gate[T % 4].piece0(ga[old][T]);
      };
      // the 19 ticks are done before step 5 CT, which reads the upper half of h; the lower half, ready at tick 11, is read from step 4 CT on
      auto behind = [&](auto s_) {
        constexpr int S = decltype(s_)::value;
        ticks_behind<S, CT>(tick);
      };
      static_for<NF>([&](auto s_) {
        constexpr int S = decltype(s_)::value;
        if constexpr (S + AHEAD < NF) fr[(S + AHEAD) % RING] = wb[(S + AHEAD) * 64];
        else if constexpr (ALONE) fr[(S + AHEAD) % RING] = smem[next_of(buf) * SU + (S + AHEAD - NF) * 64 + lane];
        if constexpr (S >= 2 * KS) {
          constexpr int t = S - 2 * KS;
          yacc[t % CT] = mma(fr[S % RING], hop[t / CT], yacc[t % CT]);
        } else if constexpr (S % 2 == 0) {
          ua[now] = mma(fr[S % RING], xb[S / 2], ua[now]);
        } else {
          ga[now] = mma(fr[S % RING], xb[S / 2], ga[now]);
        }
        __builtin_amdgcn_sched_barrier(0);
        behind(s_);
        if constexpr (!ALONE && S == 1) fetch(buf ^ 1, c + 1);
        if constexpr (ALONE && S == MEET) {
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's share of the next slot has landed
          __syncthreads();                                  // everyone's, and the buffer of the slot before is free
          fetch(next_of(next_of(buf)), c + 2 <= NCH ? c + 2 : c + 1 - NCH);
        }
        if constexpr (ALONE && S == NF - AHEAD) biases(next_of(buf), std::integral_constant<int, old>{});
        __builtin_amdgcn_sched_barrier(0);
      });
      buf = next_of(buf);
    };
#pragma clang loop unroll(disable)
    for (int c = 0; c < NCH; c += 2) {
      slot(c, std::integral_constant<int, 0>{});
      slot(c + 1, std::integral_constant<int, 1>{});
    }
    {  // the last chunk's share of y
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      const u32x4 *wb = smem + buf * SU + 2 * KS * 64 + lane;
      if (ALONE) fetch(next_of(next_of(buf)), 1);
      else fetch(buf ^ 1, 0);  // the first slot of the next block
      u32x4 hop[2];
      auto value = [&](int j) {
        Gate<ACT> v;
        v.piece0(ga[1][j]);
        v.piece1();
        v.piece2();
        return v.piece3(ua[1][j], a.act);
      };
#pragma unroll
      for (int j = 0; j < 16; j += 2) hop[j / 8][j / 2 % 4] = pack2(value(j), value(j + 1));
#pragma unroll
      for (int t = 0; t < 2 * CT; ++t) yacc[t % CT] = mma(wb[t * 64], hop[t / CT], yacc[t % CT]);
      buf = next_of(buf);
      if (ALONE) begin(buf, std::integral_constant<int, 0>{});
    }

    const int64_t row0 = mb * ROWS + wave * 32;
    const int64_t next = mb + gridDim.x;
    load_rows(next < a.nblocks ? next : mb);
    const int have = (int)(a.M - row0 < 32 ? (a.M > row0 ? a.M - row0 : 0) : 32);
    auto rows_at = [&](const uint16_t *p) {
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(p) + row0 * C, 0, have * C * 2, 0x00027000);
    };
    const Buffer out = rows_at(a.y), res = rows_at(a.residual ? a.residual : a.y);
    tile::Quad<bf16> add[2][4];
    auto ask = [&](int ct) {
      if (a.residual) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int col = 32 * ct + 8 * q + 4 * g;
          add[ct & 1][q].load(res, col < C ? (unsigned)(i * C + col) * 2 : tile::kNowhere);
        }
      }
    };
    ask(0);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      if (ct + 1 < CT) ask(ct + 1);
      f32x16 v = yacc[ct];
      if (a.residual) {
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] += add[ct & 1][r / 4][r % 4];
      }
      tile::store_tile(v, out, (unsigned)(i * C) * 2, 32 * ct, C, g, static_cast<const bf16 *>(nullptr));
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing is landing in LDS when the workgroup ends
}

// ---------------------------------------------------------------------------------------------------------------
// hidden_pack_kernel: slot c = 0 .. NCH - 1 of the backward's weight stream, (6 CT + 1) KB: for every k-step the fragments of
// W_up's and W_gate's rows 32 c .. + 31 and of W_down's columns 32 c .. + 31 (reduction over its rows); 32 biases of W_up and W_gate.
// ---------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void hidden_pack_kernel(const uint16_t *__restrict__ wg, const uint16_t *__restrict__ wu,
                                                          const uint16_t *__restrict__ wd, const float *__restrict__ bg,
                                                          const float *__restrict__ bu, u32x4 *__restrict__ blob, int C, int F, int CT) {
  const int SU = (6 * CT + 1) * 64, NCH = chunks_of(F);
  const int64_t total = (int64_t)NCH * SU;
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < total; u += (int64_t)gridDim.x * 256) {
    const int c = (int)(u / SU), r = (int)(u - (int64_t)c * SU), frag = r >> 6, lane = r & 63, i = lane & 31, g = lane >> 5;
    u32x4 e = {0u, 0u, 0u, 0u};
    if (frag < 6 * CT) {
      const int which = frag % 3, row = 32 * c + i, col = 16 * (frag / 3) + 8 * g;
      if (row < F) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col + j < C) {
            const uint16_t v = which == 2 ? wd[(int64_t)(col + j) * F + row] : (which ? wg : wu)[(int64_t)row * C + col + j];
            e[j / 2] |= (uint32_t)v << (16 * (j & 1));
          }
      }
    } else if (lane < 16) {
      const float *b = lane < 8 ? bu : bg;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = 32 * c + 4 * (lane & 7) + j;
        if (b && at < F) e[j] = __float_as_uint(b[at]);
      }
    }
    blob[u] = e;
  }
}

struct HiddenArgs {
  const u32x4 *blob;
  const uint16_t *x, *dy;
  uint16_t *dgu, *h;  // (M, 2 Fp): dg, du; (M, Fp); in column groups (pa_tile.h), whole blocks of 32 rows
  float *sums;        // per 32 rows the column sums of dg and du before their rounding, (2 Fp)
  int64_t M, nblocks;
  int C, F, Fp, act;
};

// One hidden unit of a row in five pieces: h = act(g) u, dg = d u act'(g), du = d act(g).
template <int ACT>
struct Slope {
  float x, a, s, t;
  __device__ __forceinline__ void piece0(float v) {
    x = v;
    if constexpr (ACT == tile::kSilu) {
      t = -kLog2e * v;
    } else if constexpr (ACT == tile::kGelu) {
      a = fabsf(v);
      s = gelu_short_upper_terms(a);
    }
  }
  __device__ __forceinline__ void piece1() {
    if constexpr (ACT == tile::kSilu) {
      t = __builtin_amdgcn_exp2f(t);
    } else if constexpr (ACT == tile::kGelu) {
      s = gelu_short_lower_terms(a, s);
      t = a * a * (-0.5f * kLog2e);
    }
  }
  __device__ __forceinline__ void piece2() {
    if constexpr (ACT == tile::kSilu) {
      s = __builtin_amdgcn_rcpf(1.f + t);
    } else if constexpr (ACT == tile::kGelu) {
      s = __builtin_amdgcn_exp2f(s);
      t = __builtin_amdgcn_exp2f(t);
    }
  }
  __device__ __forceinline__ void piece3(int act) {  // a <- act(g), s and t what the derivative needs besides
    if constexpr (ACT == tile::kSilu) {
      a = x * s;
      t = 1.f - s;
    } else if constexpr (ACT == tile::kGelu) {
      a = gelu_from_tail(x, s);
      s = gelu_slope_from_tail(x, s, t);
    } else {
      switch (act) {
        case tile::kRelu: a = x < 0.f ? 0.f : x, s = x > 0.f ? 1.f : 0.f; break;
        case tile::kSigmoid: a = tile::sigmoid(x), s = a * (1.f - a); break;
        case tile::kTanh: a = tanhf(x), s = fmaf(-a, a, 1.f); break;
        default: a = x, s = 1.f;
      }
    }
  }
  __device__ __forceinline__ void piece4(float up, float d, float &h, float &dg, float &du) const {
    float slope = s;
    if constexpr (ACT == tile::kSilu) slope = fmaf(a, t, s);
    h = a * up;
    dg = d * up * slope;
    du = d * a;
  }
};

// ---------------------------------------------------------------------------------------------------------------
// rows_hidden_backward_kernel<CT>: the hidden layer of the backward pass for rows of up to 32 CT channels.  Per slot c a wave runs
//   u(c)^T = W_up[chunk c] x^T + b_up, g(c)^T = W_gate[chunk c] x^T + b_gate, d(c)^T = W_down[:, chunk c]^T dy^T     6 CT MFMAs
// in turn, with h, dg and du of the chunk before formed behind them, 16 values in five pieces each; two sets of accumulators take
// turns.  A chunk's results leave 2 KB in one piece each (pa_tile.h); the column sums of dg and du, for the bias gradients, are
// formed before their rounding.  Buffers and barriers as in rows_forward_kernel.  131 072 x 256, F = 1 024: 362 us for 940 MB and 206
// GFLOP; vector instructions 38 %, matrix pipes 28 % of the time, waits 21 %.
// ---------------------------------------------------------------------------------------------------------------
__host__ __device__ constexpr int value_at(int t) { return t / 2 % 4 * 4 + t / 8 * 2 + t % 2; }
template <int CT, int ACT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(WAVES / 4, WAVES / 4))) void rows_hidden_backward_kernel(
    HiddenArgs a) {
  constexpr int KS = 2 * CT, SU = (6 * CT + 1) * 64, NF = 6 * CT, ROWS = 32 * WAVES;
  constexpr int STORES = 6 + 1;  // of a chunk
  constexpr bool ALONE = WAVES == 4;
  constexpr int BUFFERS = ALONE ? 3 : 2, AHEAD = 4, RING = ALONE ? 6 : AHEAD + 1, MEET = 1;
  static_assert(!ALONE || NF % RING == 0, "a slot's fragments begin where the last one's end");
  extern __shared__ u32x4 smem[];
  const int lane = threadIdx.x & 63, i = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int NCH = chunks_of(a.F), C = a.C;
  auto fetch = [&](int buf, int c) {  // this wave's share of slot c, 1 KB at a time
    const u32x4 *src = a.blob + (int64_t)c * SU;
    const unsigned dst = (unsigned)(uintptr_t)(smem + buf * SU);
#pragma unroll
    for (int k = 0; k < (NF + 1 + WAVES - 1) / WAVES; ++k) {
      const int part = k * WAVES + wave;
      if (part < NF + 1) load_unit_to_lds(src + part * 64, lane * 16, dst + part * 1024);
    }
  };
  u32x4 xb[KS], db[KS];
  auto load_rows = [&](int64_t mb) {
    int64_t r = mb * ROWS + wave * 32 + i;
    if (r >= a.M) r = a.M - 1;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int col = 16 * ks + 8 * g, at = col < C ? col : 0;
      xb[ks] = *reinterpret_cast<const u32x4 *>(a.x + r * C + at);
      db[ks] = *reinterpret_cast<const u32x4 *>(a.dy + r * C + at);
      if (32 * CT > C && col >= C) xb[ks] = db[ks] = u32x4{0u, 0u, 0u, 0u};
      if (mb * ROWS + wave * 32 + i >= a.M) xb[ks] = db[ks] = u32x4{0u, 0u, 0u, 0u};  // a repeated row: of no gradient
    }
  };
  auto next_of = [](int b) { return b + 1 == BUFFERS ? 0 : b + 1; };
  int buf = 0;
  u32x4 fr[RING];
  f32x16 ga[2], ua[2], da[2];
  auto biases = [&](int b, auto set_) {
    constexpr int set = decltype(set_)::value;
    const float *bias = reinterpret_cast<const float *>(smem + b * SU + NF * 64);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const tile::f32x4 bu = *reinterpret_cast<const tile::f32x4 *>(bias + 8 * q + 4 * g);
      const tile::f32x4 bg = *reinterpret_cast<const tile::f32x4 *>(bias + 32 + 8 * q + 4 * g);
#pragma unroll
      for (int j = 0; j < 4; ++j) ua[set][4 * q + j] = bu[j], ga[set][4 * q + j] = bg[j], da[set][4 * q + j] = 0.f;
    }
  };
  auto begin = [&](int b, auto set_) {
    static_for<AHEAD>([&](auto q) { fr[decltype(q)::value] = smem[b * SU + decltype(q)::value * 64 + lane]; });
    biases(b, set_);
  };
  fetch(0, 0);
  if (ALONE) fetch(1, 1);
  load_rows(blockIdx.x);
  if (ALONE) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    begin(0, std::integral_constant<int, 0>{});
  }
  for (int64_t mb = blockIdx.x; mb < a.nblocks; mb += gridDim.x) {
    const int64_t row0 = mb * ROWS + wave * 32;
    const int have = (int)(a.M - row0 < 32 ? (a.M > row0 ? a.M - row0 : 0) : 32);
    const Buffer out = __builtin_amdgcn_make_buffer_rsrc(a.dgu + row0 * 2 * a.Fp, 0, have > 0 ? 32 * 2 * a.Fp * 2 : 0, 0x00027000);
    const Buffer hidden = __builtin_amdgcn_make_buffer_rsrc(a.h + row0 * a.Fp, 0, have > 0 ? 32 * a.Fp * 2 : 0, 0x00027000);
#pragma unroll
    for (int r = 0; r < 16; ++r) ga[1][r] = ua[1][r] = da[1][r] = 0.f;
    uint32_t packed[3][8];  // of a chunk: dg, du, h
    auto store_chunk = [&](int c) {
#pragma unroll
      for (int which = 0; which < 3; ++which)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          u32x4 s;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const auto r = __builtin_amdgcn_permlane32_swap(packed[which][4 * half + w], packed[which][4 * half + 2 + w], false, false);
            s[w] = r[0], s[2 + w] = r[1];
          }
          const int col = 32 * c + 16 * half + 8 * g;
          const unsigned at = (unsigned)(((which == 1 ? a.Fp : 0) + 32 * c + 16 * half) * 64 + i * 32 + g * 16);
          __builtin_amdgcn_raw_buffer_store_b128(s, which < 2 ? out : hidden, col < a.Fp ? at : tile::kNowhere, 0, 0);
        }
    };
    // Column sums on their way (tile::column_sums).  Values are taken in an order that keeps few of them: the four q of columns
    // j = 0, 1, then of 2, 3.
    float held[2][2], half[2][2];
    tile::f32x4 total;
    auto add_up = [&](auto j_, float dg, float du) {  // value J of the chunk's 16 in this lane
      constexpr int q = decltype(j_)::value / 4, j = decltype(j_)::value % 4;
      if constexpr (q % 2 == 0) {
        held[0][j % 2] = dg, held[1][j % 2] = du;
      } else {
        const float s0 = tile::exchange_add<0>(held[0][j % 2], dg, lane), s1 = tile::exchange_add<0>(held[1][j % 2], du, lane);
        if constexpr (q == 1) half[0][j % 2] = s0, half[1][j % 2] = s1;
        else
          total[j] = tile::both_add(tile::exchange_add<1>(half[0][j % 2], s0, lane), tile::exchange_add<1>(half[1][j % 2], s1, lane), lane);
      }
    };
    const Buffer sums = __builtin_amdgcn_make_buffer_rsrc(a.sums + row0 / 32 * 2 * a.Fp, 0, have > 0 ? 2 * a.Fp * 4 : 0, 0x00027000);
    auto store_sums = [&](int c) {
      const int col = 32 * c + 8 * (lane & 3) + 4 * g;
      const unsigned at = (unsigned)((i & 4 ? a.Fp : 0) + col) * 4;
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, total), sums, i < 8 && col < a.Fp ? at : tile::kNowhere, 0, 0);
    };
    auto slot = [&](int c, auto set_) {
      constexpr int now = decltype(set_)::value, old = 1 - now;
      // this wave's share of the slot has landed; the stores that left behind it stay in flight
      if constexpr (!ALONE) {
        if (c > 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(STORES) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // everyone's, and the other buffer is free
        begin(buf, set_);
      }
      const u32x4 *wb = smem + buf * SU + lane;
      Slope<ACT> v[5];
      float even[3];
      auto tick = [&](auto t_) {  // pieces of values T .. T - 4
        constexpr int T = decltype(t_)::value;
        if constexpr (T >= 4 && T < 20) {
          constexpr int J = value_at(T - 4);
          float h, dg, du;
          v[(T - 4) % 5].piece4(ua[old][J], da[old][J], h, dg, du);
          add_up(std::integral_constant<int, J>{}, dg, du);
          if constexpr (J % 2 == 0) {
            even[0] = dg, even[1] = du, even[2] = h;
          } else {
            packed[0][J / 2] = pack2(even[0], dg);
            packed[1][J / 2] = pack2(even[1], du);
            packed[2][J / 2] = pack2(even[2], h);
          }
        }
        if constexpr (T >= 3 && T < 19) v[(T - 3) % 5].piece3(a.act);
        if constexpr (T >= 2 && T < 18) v[(T - 2) % 5].piece2();
        if constexpr (T >= 1 && T < 17) v[(T - 1) % 5].piece1();
        if constexpr (T < 16) v[T % 5].piece0(ga[old][value_at(T)]);
      };
      static_for<NF>([&](auto s_) {
        constexpr int S = decltype(s_)::value;
        if constexpr (S + AHEAD < NF) fr[(S + AHEAD) % RING] = wb[(S + AHEAD) * 64];
        else if constexpr (ALONE) fr[(S + AHEAD) % RING] = smem[next_of(buf) * SU + (S + AHEAD - NF) * 64 + lane];
        if constexpr (S % 3 == 0) ua[now] = mma(fr[S % RING], xb[S / 3], ua[now]);
        else if constexpr (S % 3 == 1) ga[now] = mma(fr[S % RING], xb[S / 3], ga[now]);
        else da[now] = mma(fr[S % RING], db[S / 3], da[now]);
        __builtin_amdgcn_sched_barrier(0);
        ticks_behind<S, CT>(tick);
        if constexpr (!ALONE && S == 1) fetch(buf ^ 1, c + 1 < NCH ? c + 1 : 0);  // past the last slot: the first of the next block
        if constexpr (ALONE && S == MEET) {
          // this wave's share of the next slot has landed; no stores came behind it in slot 0
          if (c == 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(STORES) : "memory");
          __syncthreads();  // everyone's, and the buffer of the slot before is free
          fetch(next_of(next_of(buf)), c + 2 < NCH ? c + 2 : c + 2 - NCH);
        }
        if constexpr (ALONE && S == NF - AHEAD) biases(next_of(buf), std::integral_constant<int, old>{});
        __builtin_amdgcn_sched_barrier(0);
      });
      if (now == 1 || c > 0) store_sums(c - 1), store_chunk(c - 1);
      buf = next_of(buf);
    };
#pragma clang loop unroll(disable)
    for (int c = 0; c < NCH; c += 2) {
      slot(c, std::integral_constant<int, 0>{});
      slot(c + 1, std::integral_constant<int, 1>{});
    }
    const int64_t next = mb + gridDim.x;
    load_rows(next < a.nblocks ? next : mb);
    float even[3];
    static_for<16>([&](auto j_) {  // the last chunk
      constexpr int J = value_at(decltype(j_)::value);
      float h, dg, du;
      Slope<ACT> v;
      v.piece0(ga[1][J]);
      v.piece1();
      v.piece2();
      v.piece3(a.act);
      v.piece4(ua[1][J], da[1][J], h, dg, du);
      add_up(std::integral_constant<int, J>{}, dg, du);
      if constexpr (J % 2 == 0) {
        even[0] = dg, even[1] = du, even[2] = h;
      } else {
        packed[0][J / 2] = pack2(even[0], dg);
        packed[1][J / 2] = pack2(even[1], du);
        packed[2][J / 2] = pack2(even[2], h);
      }
    });
    store_sums(NCH - 1), store_chunk(NCH - 1);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing is landing in LDS when the workgroup ends
}

// ================================================================================================
// host side
// ================================================================================================
static int channel_tiles(int64_t C) { return (int)((C + 31) / 32); }
static int waves_of(int64_t C) { return C <= 128 ? 8 : 4; }

bool rows_supported(int64_t C, int64_t F) { return C <= 256 && F <= 1 << 18; }

// How many of M rows these kernels take.  A round is one block of 32 rows per wave on every CU; part of one costs as much, and the
// tile kernels then have the smaller pieces.  Wide rows take long for a block, so that they need most of a round; rows of up to 64
// channels are worth it always.  Forward, rows + 4 us for the weights / tiles (us): C = 256, F = 1024: 16 384 rows 59 / 45,
// 32 768 71 / 78, 262 144 474 / 582; C = 200, F = 800: 32 768 43 / 60; C = 128, F = 512: 16 384 28 / 21, 32 768 28 / 34, 262 144
// 124 / 225; C = 64, F = 256: 2 000 13 / 19, 32 768 13 / 20.  Forward and the hidden layer's backward together: C = 160, F = 640:
// 20 480 rows 104 / 101, 24 576 108 / 113; C = 192, F = 768: 20 480 125 / 117, 24 576 132 / 132, 28 672 139 / 152.  (Run as seven
// tiles, 262 144 rows of these two widths take 225 and 272 forward instead of 181 and 244.)  Rows past the whole rounds go to the tile kernels where they are less
// than half a round.
int64_t rows_worth(int64_t M, int64_t C, int num_cu) {
  static const int least[9] = {0, 0, 0, 25, 45, 65, 75, 75, 85};  // per cent of a round, by channel tiles
  const int64_t block = 32 * waves_of(C), blocks = (M + block - 1) / block, rounds = blocks / num_cu, over = blocks - rounds * num_cu;
  if (rounds == 0 ? 100 * over >= least[channel_tiles(C)] * num_cu : 2 * over >= num_cu) return M;
  const int64_t rows = rounds * num_cu * block;
  return rows < M ? rows : M;
}
int64_t rows_blob_bytes(int64_t C, int64_t F) { return (int64_t)(chunks_of((int)F) + 1) * (6 * channel_tiles(C) + 1) * 1024; }

template <int CT, int ACT, int WAVES>
static int launch_rows(const RowsArgs &a, int num_cu, hipStream_t st) {
  constexpr size_t lds = (WAVES == 4 ? 3 : 2) * (6 * CT + 1) * 1024 + 32 * CT * 4;
  auto kernel = rows_forward_kernel<CT, ACT, WAVES>;
  if (int rc = allow_dynamic_lds(kernel, lds)) return rc;
  const int64_t grid = a.nblocks < num_cu ? a.nblocks : num_cu;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * WAVES), lds, st, a);
  return launch_status();
}
template <int CT, int WAVES>
static int launch_rows(const RowsArgs &a, int num_cu, hipStream_t st) {
  if (a.act == tile::kSilu) return launch_rows<CT, tile::kSilu, WAVES>(a, num_cu, st);
  if (a.act == tile::kGelu) return launch_rows<CT, tile::kGelu, WAVES>(a, num_cu, st);
  return launch_rows<CT, -1, WAVES>(a, num_cu, st);
}

int rows_pack(int64_t C, int64_t F, const pa_gated_params &p, void *blob, hipStream_t st) {
  const int64_t units = rows_blob_bytes(C, F) / 16;
  const int64_t blocks = (units + 255) / 256 < 4096 ? (units + 255) / 256 : 4096;
  hipLaunchKernelGGL(rows_pack_kernel, dim3((unsigned)blocks), dim3(256), 0, st, static_cast<const uint16_t *>(p.w_gate),
                     static_cast<const uint16_t *>(p.w_up), static_cast<const uint16_t *>(p.w_down), p.b_gate, p.b_up,
                     static_cast<u32x4 *>(blob), (int)C, (int)F, channel_tiles(C));
  return launch_status();
}

// rows 0 .. M - 1 on the weights of rows_pack
int rows_forward(int64_t M, int64_t C, int64_t F, const void *blob, const float *b_down, int act, const void *x, const void *residual,
                 void *y, int num_cu, hipStream_t st) {
  RowsArgs a{};
  a.blob = static_cast<const u32x4 *>(blob);
  a.x = static_cast<const uint16_t *>(x), a.residual = static_cast<const uint16_t *>(residual), a.y = static_cast<uint16_t *>(y);
  a.b_down = b_down;
  a.M = M, a.nblocks = (M + 32 * waves_of(C) - 1) / (32 * waves_of(C));
  a.C = (int)C, a.F = (int)F, a.act = act;
  switch (channel_tiles(C)) {
    case 1: return launch_rows<1, 8>(a, num_cu, st);
    case 2: return launch_rows<2, 8>(a, num_cu, st);
    case 3: return launch_rows<3, 8>(a, num_cu, st);
    case 4: return launch_rows<4, 8>(a, num_cu, st);
    case 5: return launch_rows<5, 4>(a, num_cu, st);
    case 6: return launch_rows<6, 4>(a, num_cu, st);
    case 7: return launch_rows<7, 4>(a, num_cu, st);
    default: return launch_rows<8, 4>(a, num_cu, st);
  }
}

// ---- the backward's hidden layer ----
int64_t hidden_blob_bytes(int64_t C, int64_t F) { return (int64_t)chunks_of((int)F) * (6 * channel_tiles(C) + 1) * 1024; }

template <int CT, int ACT, int WAVES>
static int launch_hidden(const HiddenArgs &a, int num_cu, hipStream_t st) {
  constexpr size_t lds = (WAVES == 4 ? 3 : 2) * (6 * CT + 1) * 1024;
  auto kernel = rows_hidden_backward_kernel<CT, ACT, WAVES>;
  if (int rc = allow_dynamic_lds(kernel, lds)) return rc;
  const int64_t grid = a.nblocks < num_cu ? a.nblocks : num_cu;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * WAVES), lds, st, a);
  return launch_status();
}
template <int CT, int WAVES>
static int launch_hidden(const HiddenArgs &a, int num_cu, hipStream_t st) {
  if (a.act == tile::kSilu) return launch_hidden<CT, tile::kSilu, WAVES>(a, num_cu, st);
  if (a.act == tile::kGelu) return launch_hidden<CT, tile::kGelu, WAVES>(a, num_cu, st);
  return launch_hidden<CT, -1, WAVES>(a, num_cu, st);
}

int hidden_pack(int64_t C, int64_t F, const pa_gated_params &p, void *blob, hipStream_t st) {
  const int64_t units = hidden_blob_bytes(C, F) / 16;
  const int64_t blocks = (units + 255) / 256 < 4096 ? (units + 255) / 256 : 4096;
  hipLaunchKernelGGL(hidden_pack_kernel, dim3((unsigned)blocks), dim3(256), 0, st, static_cast<const uint16_t *>(p.w_gate),
                     static_cast<const uint16_t *>(p.w_up), static_cast<const uint16_t *>(p.w_down), p.b_gate, p.b_up,
                     static_cast<u32x4 *>(blob), (int)C, (int)F, channel_tiles(C));
  return launch_status();
}

int rows_hidden_backward(int64_t M, int64_t C, int64_t F, int64_t Fp, const void *blob, int act, const void *x, const void *dy, void *dgu,
                         void *h, float *sums, int num_cu, hipStream_t st) {
  HiddenArgs a{};
  a.sums = sums;
  a.blob = static_cast<const u32x4 *>(blob);
  a.x = static_cast<const uint16_t *>(x), a.dy = static_cast<const uint16_t *>(dy);
  a.dgu = static_cast<uint16_t *>(dgu), a.h = static_cast<uint16_t *>(h);
  a.M = M, a.nblocks = (M + 32 * waves_of(C) - 1) / (32 * waves_of(C));
  a.C = (int)C, a.F = (int)F, a.Fp = (int)Fp, a.act = act;
  switch (channel_tiles(C)) {
    case 1: return launch_hidden<1, 8>(a, num_cu, st);
    case 2: return launch_hidden<2, 8>(a, num_cu, st);
    case 3: return launch_hidden<3, 8>(a, num_cu, st);
    case 4: return launch_hidden<4, 8>(a, num_cu, st);
    case 5: return launch_hidden<5, 4>(a, num_cu, st);
    case 6: return launch_hidden<6, 4>(a, num_cu, st);
    case 7: return launch_hidden<7, 4>(a, num_cu, st);
    default: return launch_hidden<8, 4>(a, num_cu, st);
  }
}

}  // namespace gated
}  // namespace pa
