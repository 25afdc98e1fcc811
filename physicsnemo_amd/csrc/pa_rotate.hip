// Queries and keys of attention heads normalised and turned by the angles of their positions, in one pass, forward and backward:
//   u = x r w,  r = (mean_d x^2 + eps)^(-1/2);  y = T u, T turning pair p of the channels by t_p = sum_a pos_a f_{a,p}
//   g = T^-1 dy;  dw = sum g x r;  dx = r (t - xh mean_d(t xh)),  t = g w,  xh = x r
// Angles of far positions: t / (2 pi) is formed as a product of two doubles with the rounding of the first one carried along, and
// only what is left of it after whole quarter turns is rounded to float32, so that cos and sin are good to 2.4e-7 (4 u) while every pos_a f_{a,p} is
// within 2^78 (error of the turn: 2^-107 of the product, 4e-8 at 2^79 in all) and whole positions within 2^53.  What lies further out is NaN.  Sums,
// norms and the turn are float32; a result is rounded once.
//
// Bound by HBM: two element accesses forward, three backward.  A workgroup forms cos and sin of its points once, in LDS, for all heads
// (a double-precision product and two polynomials per angle, for Hq + Hk rows of use); a lane holds eight channels of a row, its pairs
// whole, so that the turn needs no neighbour and the norm three or four lane exchanges (halves that are no multiple of four go through LDS).
//
// What it takes: 131 072 x 16 rows of 32 bf16, 30 channels turned: 85 us (0.27 GB: 49; 230 vector instructions a row of four lanes and the angles in
// double precision, 68 % of the issue slots); 4 x 7 225 x 16 x 16 float32, all turned: 15 forward, 21 backward (11 and 17 at the copy's rate).  The next row
// loaded ahead gives 4 us of the 85 for eight registers; a point's heads one after the other by the same lanes, its turns in registers, 7, but
// one point costs 5.1 instead of 4.3 and the backward pass 21.2 instead of 20.8: neither is kept.
#include "pa_common.h"
#include "pa_host.h"
#include "pa_mfma_ops.h"

namespace pa {
namespace rotate {

using mfma::u32x2;
using mfma::u32x4;

struct Side {
  const void *x, *dy;  // dy: backward
  int64_t batch, row, head, dy_batch, dy_row, dy_head;
  void *out;  // y, or dx
  const float *weight;
};
struct Args {
  Side q, k;
  const void *positions;
  const float *frequencies;
  float *partials;  // backward: [workgroup][2][D]
  int64_t points, N, position_batch;
  int Hq, Hk, D, half, axes, position_type, interleaved, norm, per_block;  // half: pairs that are turned
  uint32_t by_heads, by_half;  // 2^32 over Hq + Hk and over half, rounded up
  float eps;
};

// where point first + n lies, first being row r0 of sequence b0: 64-bit divisions once a workgroup's pass, not once a row
struct Spot {
  int64_t b, r;
};
__device__ __forceinline__ Spot spot_of(const Args &a, const Spot &first, int n) {
  Spot s = {first.b, first.r + n};
  if (a.N >= a.per_block) {
    const bool over = s.r >= a.N;
    s.b += over, s.r -= over ? a.N : 0;
  } else {  // N < 32
    const uint32_t r = (uint32_t)s.r, whole = r / (uint32_t)a.N;
    s.b += whole, s.r = r - whole * (uint32_t)a.N;
  }
  return s;
}
// n / d for n < 2^18, d <= 2^13, by = ceil(2^32 / d)
__device__ __forceinline__ int quotient(int n, uint32_t by, int d) { return d == 1 ? n : (int)__umulhi((uint32_t)n, by); }

// ---- cos and sin of a point's angle ----
constexpr int64_t kMostWhole = 1ll << 53;
constexpr double kMostAngle = 0x1p78;
__device__ __forceinline__ double position(const Args &a, int64_t at) {
  if (a.position_type == PA_POS_F32) return (double)static_cast<const float *>(a.positions)[at];
  if (a.position_type == PA_POS_I64) {
    const int64_t n = static_cast<const int64_t *>(a.positions)[at];
    return n <= kMostWhole && n >= -kMostWhole ? (double)n : __builtin_nan("");
  }
  return (double)static_cast<const int32_t *>(a.positions)[at];
}
// pos f in turns, less whole turns
__device__ __forceinline__ double turns(double pos, double f) {
#pragma clang fp contract(off)  // u is its rounded value wherever it stands: `rest` is what it lacks
  constexpr double hi = 0x1.45f306dc9c883p-3, lo = -0x1.6b01ec5417056p-57;  // 1 / (2 pi)
  const double t = pos * f, t_rest = fma(pos, f, -t);
  const double u = t * hi, rest = fma(t, hi, -u) + fma(t, lo, t_rest * hi);
  return fabs(t) <= kMostAngle ? (u - rint(u)) + rest : __builtin_nan("");
}
__device__ __forceinline__ float2 cos_sin(const Args &a, const Spot &spot, int p) {
  const int64_t at = spot.b * a.position_batch + spot.r * a.axes;
  double turn = 0;
  for (int x = 0; x < a.axes; ++x) turn += turns(position(a, at + x), (double)a.frequencies[x * a.half + p]);
  const double quarters = turn * 4, whole = rint(quarters);
  const float rest = (float)(quarters - whole);
  float s, c;
  sincospif(0.5f * rest, &s, &c);
  const int k = (int)whole & 3;  // NaN and infinite positions: rest is NaN
  if (k & 1) {
    const float t = c;
    c = -s;
    s = t;
  }
  return (k & 2) ? make_float2(-c, -s) : make_float2(c, s);
}

// ---- a lane's eight channels ----
// kNeighbours: pairs (2 p, 2 p + 1), eight channels in a row, whole pairs.  kQuarters: pairs (p, p + half) of whole fours: four channels of the first
// half and theirs of the second (behind the halves eight in a row).  kApart: pairs (p, p + half) of any half: eight channels in a row, their
// partners' values through LDS.
enum Pairs { kNeighbours, kQuarters, kApart };
typedef u32x4 unit_at4 __attribute__((aligned(4)));
typedef u32x4 unit_at2 __attribute__((aligned(2)));
typedef u32x2 half_at2 __attribute__((aligned(2)));
__device__ __forceinline__ void load4(const float *p, float *v) {
  const u32x4 w = *reinterpret_cast<const unit_at4 *>(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b = w[j];
    v[j] = __uint_as_float(b);
  }
}
__device__ __forceinline__ void load4(const bf16 *p, float *v) {
  const u32x2 w = *reinterpret_cast<const half_at2 *>(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b = w[j / 2];
    v[j] = __uint_as_float(j & 1 ? b & 0xffff0000u : b << 16);
  }
}
__device__ __forceinline__ void load8(const float *p, float *v) { load4(p, v), load4(p + 4, v + 4); }
__device__ __forceinline__ void load8(const bf16 *p, float *v) {
  const u32x4 w = *reinterpret_cast<const unit_at2 *>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t b = w[j / 2];
    v[j] = __uint_as_float(j & 1 ? b & 0xffff0000u : b << 16);
  }
}
__device__ __forceinline__ void store4(float *p, const float *v) {
  u32x4 w;
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(v[j]);
  *reinterpret_cast<unit_at4 *>(p) = w;
}
__device__ __forceinline__ void store4(bf16 *p, const float *v) {
  u32x2 w;
  w[0] = mfma::pack2(v[0], v[1]);
  w[1] = mfma::pack2(v[2], v[3]);
  *reinterpret_cast<half_at2 *>(p) = w;
}
__device__ __forceinline__ void store8(float *p, const float *v) { store4(p, v), store4(p + 4, v + 4); }
__device__ __forceinline__ void store8(bf16 *p, const float *v) {
  u32x4 w;
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = mfma::pack2(v[2 * j], v[2 * j + 1]);
  *reinterpret_cast<unit_at2 *>(p) = w;
}

// where the two fours of a lane's channels start
struct Place {
  int at0, at1;
};
template <Pairs PAIRS>
__device__ __forceinline__ Place place_of(int half, int slot) {
  if (PAIRS == kQuarters && 4 * slot < half) return {4 * slot, 4 * slot + half};
  return {8 * slot, 8 * slot + 4};
}
template <class T, Pairs PAIRS>
__device__ __forceinline__ void load_row(const T *row, const Place &p, int D, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.f;
  if constexpr (PAIRS == kQuarters) {  // D is whole eights
    if (p.at0 < D) load4(row + p.at0, v), load4(row + p.at1, v + 4);
  } else if (p.at0 + 8 <= D) {
    load8(row + p.at0, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (p.at0 + j < D) v[j] = load_as_f32(row + p.at0 + j);
  }
}
template <class T, Pairs PAIRS>
__device__ __forceinline__ void store_row(T *row, const Place &p, int D, const float (&v)[8]) {
  if constexpr (PAIRS == kQuarters) {
    if (p.at0 < D) store4(row + p.at0, v), store4(row + p.at1, v + 4);
  } else if (p.at0 + 8 <= D) {
    store8(row + p.at0, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (p.at0 + j < D) store_from_f32(row + p.at0 + j, v[j]);
  }
}

// kApart: where each of a lane's channels finds its partner in the exchange and its pair in the point's turns, and which way its partner's part goes
struct Partners {
  int other[8], pair[8];
  float sign[8];
};
__device__ __forceinline__ int spread(int c) { return c + (c >> 3); }  // a gap every eight floats spreads lanes over the banks
constexpr int kNone = 8;  // the first gap: -0, what a channel that is not turned takes from its partner, so that it stays as it is, infinite or not
template <int LANES>
__device__ __forceinline__ Partners partners_of(int half, int slot) {
  Partners p;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = 8 * slot + j;
    const bool lower = c < half, turned = c < 2 * half;
    p.other[j] = !turned ? kNone : spread(lower ? c + half : c - half);
    p.pair[j] = !turned ? half : lower ? c : c - half;  // behind the pairs: one that turns nothing
    p.sign[j] = lower ? -1.f : 1.f;
  }
  return p;
}

// v <- v turned by the point's angles (cs: cos and sin of its pairs), backwards with sign = -1
template <Pairs PAIRS, int LANES>
__device__ __forceinline__ void turn(float (&v)[8], const float2 *cs, int half, int slot, float sign, float *exchange, const Partners &p) {
  if constexpr (PAIRS != kApart) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int a = PAIRS == kNeighbours ? 2 * j : j, b = PAIRS == kNeighbours ? 2 * j + 1 : j + 4, pair = 4 * slot + j;
      const bool turned = pair < half;  // others stay as they are: a product with a sine of zero would make an infinity in one NaN in both
      const float2 t = cs[turned ? pair : half];
      const float x = v[a], y = v[b];
      v[a] = turned ? x * t.x - sign * y * t.y : x;
      v[b] = turned ? sign * x * t.y + y * t.x : y;
    }
  } else {
    // the lanes of a row are lanes of one wave, whose LDS accesses happen in order
    float *const mine = exchange + threadIdx.x / LANES * (9 * LANES + 1);
#pragma unroll
    for (int j = 0; j < 8; ++j) mine[9 * slot + j] = v[j];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 t = cs[p.pair[j]];
      v[j] = fmaf(v[j], t.x, mine[p.other[j]] * (sign * p.sign[j] * t.y));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
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
  return v;
}

// cos and sin of the points from `first` on, [point][pair], and behind a point's pairs one that turns nothing
__device__ __forceinline__ void fill_turns(const Args &a, const Spot &first, int points, float2 *cs) {
  for (int u = threadIdx.x; u < points * a.half; u += blockDim.x) {
    const int n = quotient(u, a.by_half, a.half), p = u - n * a.half;
    cs[n * (a.half + 1) + p] = cos_sin(a, spot_of(a, first, n), p);
  }
  if ((int)threadIdx.x < points) cs[threadIdx.x * (a.half + 1) + a.half] = make_float2(1.f, 0.f);
}

// LANES lanes a row; a workgroup takes per_block points at a time, their rows (heads of q, then of k) one after the other
template <class T, Pairs PAIRS, int LANES, bool BACK>
__global__ __launch_bounds__(256) void rows_kernel(Args a) {
  extern __shared__ float2 cs[];
  float *const exchange = reinterpret_cast<float *>(cs + a.per_block * (a.half + 1));
  const int slot = threadIdx.x % LANES, group = threadIdx.x / LANES;
  constexpr int GROUPS = 256 / LANES;
  const int H = a.Hq + a.Hk, D = a.D;
  const Place place = place_of<PAIRS>(a.half, slot);
  auto channel = [&](int j) { return j < 4 ? place.at0 + j : place.at1 + j - 4; };
  const Partners partners = partners_of<LANES>(a.half, slot);
  if (PAIRS == kApart && slot == 0) exchange[group * (9 * LANES + 1) + kNone] = -0.f;
  const float inv = 1.f / (float)D;
  float wq[8], wk[8], sq[8] = {}, sk[8] = {};  // weights, sums of their gradients
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    wq[j] = a.norm && a.q.weight && channel(j) < D ? a.q.weight[channel(j)] : 1.f;
    wk[j] = a.norm && a.k.weight && channel(j) < D ? a.k.weight[channel(j)] : 1.f;
  }
  for (int64_t first = (int64_t)blockIdx.x * a.per_block; first < a.points; first += (int64_t)gridDim.x * a.per_block) {
    const int points = (int)(a.points - first < a.per_block ? a.points - first : a.per_block);
    __syncthreads();  // the pass before has read its turns
    const Spot start = {first / a.N, first % a.N};
    fill_turns(a, start, points, cs);
    __syncthreads();
    const int rows = points * H;
    for (int row = group; row < (rows + GROUPS - 1) / GROUPS * GROUPS; row += GROUPS) {  // all lanes: the sums exchange
      const bool live = row < rows;
      const int n = live ? quotient(row, a.by_heads, H) : 0, h = live ? row - n * H : 0;
      const bool key = h >= a.Hq;
      const Side &s = key ? a.k : a.q;
      const Spot spot = spot_of(a, start, n);
      const int head = key ? h - a.Hq : h;
      const T *x = static_cast<const T *>(s.x) + spot.b * s.batch + spot.r * s.row + head * s.head;
      T *out = static_cast<T *>(s.out) + ((first + n) * (key ? a.Hk : a.Hq) + head) * D;
      float v[8], g[8];
      load_row<T, PAIRS>(x, place, live ? D : 0, v);
      if constexpr (BACK) load_row<T, PAIRS>(static_cast<const T *>(s.dy) + spot.b * s.dy_batch + spot.r * s.dy_row + head * s.dy_head, place, live ? D : 0, g);
      float rstd = 1.f;
      if (a.norm) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(v[j], v[j], sum);
        rstd = __builtin_amdgcn_rsqf(fmaf(lanes_sum<LANES>(sum), inv, a.eps));
        if (BACK && !live) rstd = 1.f;  // with eps = 0 a row of zeros is NaN: not in lanes that hold no row, which add to the weights' sums, too
      }
      if constexpr (!BACK) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] * rstd * (key ? wk[j] : wq[j]);
        turn<PAIRS, LANES>(v, cs + n * (a.half + 1), a.half, slot, 1.f, exchange, partners);
      } else {
        turn<PAIRS, LANES>(g, cs + n * (a.half + 1), a.half, slot, -1.f, exchange, partners);
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] *= rstd;
          sq[j] += key ? 0.f : g[j] * v[j], sk[j] += key ? g[j] * v[j] : 0.f;
          g[j] *= key ? wk[j] : wq[j];
          dot = fmaf(g[j], v[j], dot);
        }
        const float mean = a.norm ? lanes_sum<LANES>(dot) * inv : 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = a.norm ? rstd * (g[j] - v[j] * mean) : g[j];  // without the norm x has no part in it, infinite or not
      }
      if (s.out) store_row<T, PAIRS>(out, place, live ? D : 0, v);
    }
  }
  if constexpr (BACK) {
    if (!a.partials) return;
    // the workgroup's sums over its rows: groups' shares side by side in LDS, added up in order
    float *share = reinterpret_cast<float *>(cs);  // [GROUPS][LANES * 8]
    for (int side = 0; side < 2; ++side) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) share[threadIdx.x * 8 + j] = side ? sk[j] : sq[j];
      __syncthreads();
      if ((int)threadIdx.x < LANES * 8) {
        float sum = 0.f;
        for (int k = 0; k < GROUPS; ++k) sum += share[k * LANES * 8 + threadIdx.x];
        const Place mine = place_of<PAIRS>(a.half, threadIdx.x / 8);
        const int j = threadIdx.x & 7, c = j < 4 ? mine.at0 + j : mine.at1 + j - 4;
        if (c < D) a.partials[((int64_t)blockIdx.x * 2 + side) * D + c] = sum;
      }
    }
  }
}

template <class T, Pairs PAIRS, bool BACK>
int launch_lanes(const Args &a, int64_t blocks, hipStream_t st) {
  const int slots = (a.D + 7) / 8;
  auto go = [&](auto lanes) {
    constexpr int LANES = decltype(lanes)::value;
    const size_t turns = (size_t)a.per_block * (a.half + 1) * sizeof(float2) + (PAIRS == kApart ? 256 / LANES * (9 * LANES + 1) * sizeof(float) : 0);
    const size_t shares = BACK ? 256 * 8 * sizeof(float) : 0;
    rows_kernel<T, PAIRS, LANES, BACK><<<(unsigned)blocks, 256, turns > shares ? turns : shares, st>>>(a);
    return launch_status();
  };
  if (slots <= 1) return go(std::integral_constant<int, 1>{});
  if (slots <= 2) return go(std::integral_constant<int, 2>{});
  if (slots <= 4) return go(std::integral_constant<int, 4>{});
  if (slots <= 8) return go(std::integral_constant<int, 8>{});
  return go(std::integral_constant<int, 16>{});
}
template <class T, bool BACK>
int launch_type(const Args &a, int64_t blocks, hipStream_t st) {
  if (a.interleaved || a.half == 0) return launch_lanes<T, kNeighbours, BACK>(a, blocks, st);
  if (a.half % 4 == 0 && a.D % 8 == 0) return launch_lanes<T, kQuarters, BACK>(a, blocks, st);
  return launch_lanes<T, kApart, BACK>(a, blocks, st);
}

// totals of the workgroups' sums: 4 columns a workgroup, their rows in 64 parts that are joined in order
__global__ __launch_bounds__(256) void weight_sums_kernel(const float *partials, int64_t rows, int D, float *d_q, float *d_k) {
  __shared__ float part[64][4];
  const int col = threadIdx.x & 3, p = threadIdx.x >> 2, c = blockIdx.x * 4 + col;
  float sum = 0.f;
  if (c < 2 * D) {
#pragma unroll 4
    for (int64_t r = p; r < rows; r += 64) sum += partials[r * 2 * D + c];
  }
  part[p][col] = sum;
  for (int n = 32; n > 0; n >>= 1) {
    __syncthreads();
    if (p < n) part[p][col] += part[p + n][col];
  }
  if (p != 0 || c >= 2 * D) return;
  float *out = c < D ? d_q : d_k;
  if (out) out[c < D ? c : c - D] = part[0][col];
}

struct Plan {
  int per_block;
  int64_t blocks;
};
// Points a workgroup takes at a time: enough rows to keep its lanes busy and its angles worth their barrier, but few enough that
// the workgroups fill the chip.
static Plan plan_of(int64_t points, int num_cu) {
  int per = 1;
  while (per < 32 && points > (int64_t)per * 4 * num_cu) per *= 2;
  const int64_t wanted = (points + per - 1) / per, most = (int64_t)num_cu * 8;
  return {per, wanted < most ? wanted : most};
}
static Args args_of(const pa_rotate_params &p, const pa_heads &q, const pa_heads &k) {
  Args a = {};
  a.q.x = q.data, a.q.batch = q.batch, a.q.row = q.row, a.q.head = q.head, a.q.weight = p.q_weight;
  a.k.x = k.data, a.k.batch = k.batch, a.k.row = k.row, a.k.head = k.head, a.k.weight = p.k_weight;
  a.positions = p.positions, a.frequencies = p.frequencies;
  a.points = p.B * p.N, a.N = p.N, a.position_batch = p.position_batch;
  a.Hq = (int)p.Hq, a.Hk = (int)p.Hk, a.D = (int)p.D, a.half = (int)(p.rotated / 2), a.axes = (int)p.axes;
  a.by_heads = (uint32_t)(((1ull << 32) + a.Hq + a.Hk - 1) / (a.Hq + a.Hk));
  a.by_half = a.half ? (uint32_t)(((1ull << 32) + a.half - 1) / a.half) : 0;
  a.position_type = p.position_type, a.interleaved = p.interleaved, a.norm = p.norm, a.eps = (float)p.eps;
  return a;
}
int forward(int dtype, const pa_rotate_params &p, const pa_heads &q, const pa_heads &k, void *q_out, void *k_out, int num_cu, hipStream_t st) {
  Args a = args_of(p, q, k);
  a.q.out = q_out, a.k.out = k_out;
  const Plan plan = plan_of(a.points, num_cu);
  a.per_block = plan.per_block;
  return dtype == PA_F32 ? launch_type<float, false>(a, plan.blocks, st) : launch_type<bf16, false>(a, plan.blocks, st);
}

int64_t backward_workspace_bytes(const pa_rotate_params &p, int num_cu) {
  return plan_of(p.B * p.N, num_cu).blocks * 2 * p.D * (int64_t)sizeof(float);
}
int backward(int dtype, const pa_rotate_params &p, const pa_heads &q, const pa_heads &k, const pa_heads &d_q, const pa_heads &d_k, void *dq,
             void *dk, float *d_q_weight, float *d_k_weight, float *workspace, int num_cu, hipStream_t st) {
  Args a = args_of(p, q, k);
  a.q.out = dq, a.k.out = dk;
  a.q.dy = d_q.data, a.q.dy_batch = d_q.batch, a.q.dy_row = d_q.row, a.q.dy_head = d_q.head;
  a.k.dy = d_k.data, a.k.dy_batch = d_k.batch, a.k.dy_row = d_k.row, a.k.dy_head = d_k.head;
  const Plan plan = plan_of(a.points, num_cu);
  a.per_block = plan.per_block;
  a.partials = d_q_weight || d_k_weight ? workspace : nullptr;
  const int rc = dtype == PA_F32 ? launch_type<float, true>(a, plan.blocks, st) : launch_type<bf16, true>(a, plan.blocks, st);
  if (rc || !a.partials) return rc;
  weight_sums_kernel<<<(unsigned)((2 * p.D + 3) / 4), 256, 0, st>>>(workspace, plan.blocks, (int)p.D, d_q_weight, d_k_weight);
  return launch_status();
}

}  // namespace rotate
}  // namespace pa
