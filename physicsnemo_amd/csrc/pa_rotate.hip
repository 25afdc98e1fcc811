// Queries and keys of attention heads normalised and turned by the angles of their positions, in one pass, forward and backward:
//   u = x r w,  r = (mean_d x^2 + eps)^(-1/2);  y = T u, T turning pair p of the channels by t_p = sum_a pos_a f_{a,p}
//   g = T^-1 dy;  dw = sum g x r;  dx = r (t - xh mean_d(t xh)),  t = g w,  xh = x r
// Angles of far positions: t / (2 pi) is formed as a product of two doubles with the rounding of the first one carried along, and
// only what is left of it after whole quarter turns is rounded to float32, so that cos and sin are good to 2e-7 for every position
// that a float32 or a 53-bit integer holds.  Sums, norms and the turn are float32; a result is rounded once.
//
// Bound by HBM: two element accesses forward, three backward.  A workgroup forms cos and sin of its points once, in LDS, for all heads
// (a double-precision product and two polynomials per angle, for Hq + Hk rows of use); a lane holds eight channels of a row, its pairs
// whole, so that the turn needs no neighbour and the norm three or four lane exchanges.
#include "pa_common.h"
#include "pa_host.h"
#include "pa_mfma_ops.h"

namespace pa {
namespace rotate {

using mfma::u32x2;

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
  float eps;
};

// ---- cos and sin of a point's angle ----
__device__ __forceinline__ double position(const Args &a, int64_t at) {
  if (a.position_type == PA_POS_F32) return (double)static_cast<const float *>(a.positions)[at];
  if (a.position_type == PA_POS_I64) return (double)static_cast<const int64_t *>(a.positions)[at];
  return (double)static_cast<const int32_t *>(a.positions)[at];
}
// pos f in turns, less whole turns
__device__ __forceinline__ double turns(double pos, double f) {
#pragma clang fp contract(off)  // u is its rounded value wherever it stands: `rest` is what it lacks
  constexpr double hi = 0x1.45f306dc9c883p-3, lo = -0x1.6b01ec5417056p-57;  // 1 / (2 pi)
  const double t = pos * f, t_rest = fma(pos, f, -t);
  const double u = t * hi, rest = fma(t, hi, -u) + fma(t, lo, t_rest * hi);
  return (u - rint(u)) + rest;
}
__device__ __forceinline__ float2 cos_sin(const Args &a, int64_t point, int p) {
  const int64_t b = point / a.N, n = point - b * a.N, at = b * a.position_batch + n * a.axes;
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

// ---- a lane's eight channels: pairs j of (first(j), second(j)) ----
struct Place {
  int a[4], b[4];  // channels of the pairs, in the order the registers hold them
  int at0, at1;    // UNITS: where the two pieces of four start
  bool turned[4];
};
template <bool INTERLEAVED>
__device__ __forceinline__ Place place_of(const Args &a, int slot, bool units) {
  Place p;
  p.at0 = 8 * slot, p.at1 = 8 * slot + 4;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int pair = 4 * slot + j;
    p.turned[j] = pair < a.half;
    if (INTERLEAVED || !p.turned[j]) {
      p.a[j] = 2 * pair, p.b[j] = 2 * pair + 1;
      if (!INTERLEAVED && units) p.a[j] = 8 * slot + j, p.b[j] = 8 * slot + 4 + j;  // no pairs there: any will do
    } else {
      p.a[j] = pair, p.b[j] = pair + a.half;
      p.at0 = 4 * slot, p.at1 = 4 * slot + a.half;
    }
  }
  return p;
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load4(const float *p, float (&v)[4]) {
  const f32x4 w = *reinterpret_cast<const f32x4 *>(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = w[j];
}
__device__ __forceinline__ void load4(const bf16 *p, float (&v)[4]) {
  const u32x2 w = *reinterpret_cast<const u32x2 *>(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b = w[j / 2];
    v[j] = __uint_as_float(j & 1 ? b & 0xffff0000u : b << 16);
  }
}
__device__ __forceinline__ void store4(float *p, const float (&v)[4]) {
  f32x4 w;
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = v[j];
  *reinterpret_cast<f32x4 *>(p) = w;
}
__device__ __forceinline__ void store4(bf16 *p, const float (&v)[4]) {
  u32x2 w;
  w[0] = mfma::pack2(v[0], v[1]);
  w[1] = mfma::pack2(v[2], v[3]);
  *reinterpret_cast<u32x2 *>(p) = w;
}
// UNITS: heads are whole pieces of eight channels on boundaries of four, and so are the turned halves
template <class T, bool UNITS, bool INTERLEAVED>
__device__ __forceinline__ void load_row(const T *row, const Place &p, int D, float (&a)[4], float (&b)[4]) {
  if constexpr (UNITS) {
    float lo[4] = {}, hi[4] = {};
    if (p.a[0] < D) load4(row + p.at0, lo), load4(row + p.at1, hi);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (INTERLEAVED) {
        a[j] = j < 2 ? lo[2 * j] : hi[2 * j - 4];
        b[j] = j < 2 ? lo[2 * j + 1] : hi[2 * j - 3];
      } else {
        a[j] = lo[j], b[j] = hi[j];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = p.a[j] < D ? load_as_f32(row + p.a[j]) : 0.f;
      b[j] = p.b[j] < D ? load_as_f32(row + p.b[j]) : 0.f;
    }
  }
}
template <class T, bool UNITS, bool INTERLEAVED>
__device__ __forceinline__ void store_row(T *row, const Place &p, int D, const float (&a)[4], const float (&b)[4]) {
  if constexpr (UNITS) {
    float lo[4], hi[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (INTERLEAVED) {
        lo[j] = j & 1 ? b[j / 2] : a[j / 2];
        hi[j] = j & 1 ? b[2 + j / 2] : a[2 + j / 2];
      } else {
        lo[j] = a[j], hi[j] = b[j];
      }
    }
    if (p.a[0] < D) store4(row + p.at0, lo), store4(row + p.at1, hi);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (p.a[j] < D) store_from_f32(row + p.a[j], a[j]);
      if (p.b[j] < D) store_from_f32(row + p.b[j], b[j]);
    }
  }
}

template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int off = 1; off < LANES; off <<= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// cos and sin of per_block points from `first` on, [point][pair]
__device__ __forceinline__ void fill_turns(const Args &a, int64_t first, int points, float2 *cs) {
  for (int u = threadIdx.x; u < points * a.half; u += blockDim.x) {
    const int n = u / a.half;
    cs[u] = cos_sin(a, first + n, u - n * a.half);
  }
}

// LANES lanes a row; a workgroup takes per_block points at a time, their rows (heads of q, then of k) one after the other
template <class T, bool UNITS, bool INTERLEAVED, int LANES, bool BACK>
__global__ __launch_bounds__(256) void rows_kernel(Args a) {
  extern __shared__ float2 cs[];
  const int slot = threadIdx.x % LANES, group = threadIdx.x / LANES;
  constexpr int GROUPS = 256 / LANES;
  const int H = a.Hq + a.Hk, D = a.D;
  const Place at = place_of<INTERLEAVED>(a, slot, UNITS);
  const float inv = 1.f / (float)D;
  float wq[2][4], wk[2][4], sq[2][4] = {}, sk[2][4] = {};  // weights, sums of their gradients: first, second of the pairs
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    wq[0][j] = a.norm && a.q.weight && at.a[j] < D ? a.q.weight[at.a[j]] : 1.f;
    wq[1][j] = a.norm && a.q.weight && at.b[j] < D ? a.q.weight[at.b[j]] : 1.f;
    wk[0][j] = a.norm && a.k.weight && at.a[j] < D ? a.k.weight[at.a[j]] : 1.f;
    wk[1][j] = a.norm && a.k.weight && at.b[j] < D ? a.k.weight[at.b[j]] : 1.f;
  }
  for (int64_t first = (int64_t)blockIdx.x * a.per_block; first < a.points; first += (int64_t)gridDim.x * a.per_block) {
    const int points = (int)(a.points - first < a.per_block ? a.points - first : a.per_block);
    __syncthreads();  // the pass before has read its turns
    fill_turns(a, first, points, cs);
    __syncthreads();
    for (int row = group; row < (points * H + GROUPS - 1) / GROUPS * GROUPS; row += GROUPS) {  // all lanes: the sums exchange
      const int n = row / H, h = row - n * H;
      const bool live = n < points, key = h >= a.Hq;
      const Side &s = key ? a.k : a.q;
      const int64_t point = first + (live ? n : 0), b = point / a.N, r = point - b * a.N;
      const int head = key ? h - a.Hq : h;
      const T *x = static_cast<const T *>(s.x) + b * s.batch + r * s.row + head * s.head;
      T *out = static_cast<T *>(s.out) + ((point * (key ? a.Hk : a.Hq)) + head) * D;
      float xa[4], xb[4];
      load_row<T, UNITS, INTERLEAVED>(x, at, live ? D : 0, xa, xb);
      float2 turn[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) turn[j] = at.turned[j] && live ? cs[n * a.half + 4 * slot + j] : make_float2(1.f, 0.f);
      float rstd = 1.f;
      if (a.norm) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) sum = fmaf(xa[j], xa[j], fmaf(xb[j], xb[j], sum));
        rstd = 1.f / sqrtf(fmaf(lanes_sum<LANES>(sum), inv, a.eps));
      }
      float ya[4], yb[4];
      if constexpr (!BACK) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float u = xa[j] * rstd * (key ? wk[0][j] : wq[0][j]), v = xb[j] * rstd * (key ? wk[1][j] : wq[1][j]);
          ya[j] = u * turn[j].x - v * turn[j].y;
          yb[j] = u * turn[j].y + v * turn[j].x;
        }
      } else {
        const T *dy = static_cast<const T *>(s.dy) + b * s.dy_batch + r * s.dy_row + head * s.dy_head;
        float ga[4], gb[4];
        load_row<T, UNITS, INTERLEAVED>(dy, at, live ? D : 0, ga, gb);
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float u = ga[j] * turn[j].x + gb[j] * turn[j].y, v = gb[j] * turn[j].x - ga[j] * turn[j].y;
          xa[j] *= rstd, xb[j] *= rstd;
          sq[0][j] += key ? 0.f : u * xa[j], sq[1][j] += key ? 0.f : v * xb[j];
          sk[0][j] += key ? u * xa[j] : 0.f, sk[1][j] += key ? v * xb[j] : 0.f;
          ga[j] = u * (key ? wk[0][j] : wq[0][j]), gb[j] = v * (key ? wk[1][j] : wq[1][j]);
          dot = fmaf(ga[j], xa[j], fmaf(gb[j], xb[j], dot));
        }
        const float mean = a.norm ? lanes_sum<LANES>(dot) * inv : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) ya[j] = rstd * (ga[j] - xa[j] * mean), yb[j] = rstd * (gb[j] - xb[j] * mean);
      }
      if (s.out) store_row<T, UNITS, INTERLEAVED>(out, at, live ? D : 0, ya, yb);
    }
  }
  if constexpr (BACK) {
    if (!a.partials) return;
    // the workgroup's sums over its rows: groups' shares side by side in LDS, added up in order
    float *share = reinterpret_cast<float *>(cs);  // [GROUPS][LANES * 8]
    for (int side = 0; side < 2; ++side) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        share[threadIdx.x * 8 + j] = side ? sk[0][j] : sq[0][j];
        share[threadIdx.x * 8 + 4 + j] = side ? sk[1][j] : sq[1][j];
      }
      __syncthreads();
      if ((int)threadIdx.x < LANES * 8) {
        float sum = 0.f;
        for (int g = 0; g < GROUPS; ++g) sum += share[g * LANES * 8 + threadIdx.x];
        const Place mine = place_of<INTERLEAVED>(a, threadIdx.x / 8, UNITS);
        int channel = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if ((threadIdx.x & 7) == j) channel = mine.a[j];
          if ((threadIdx.x & 7) == 4 + j) channel = mine.b[j];
        }
        if (channel < D) a.partials[((int64_t)blockIdx.x * 2 + side) * D + channel] = sum;
      }
    }
  }
}

template <class T, bool UNITS, bool INTERLEAVED, bool BACK>
int launch_lanes(const Args &a, int64_t blocks, size_t lds, hipStream_t st) {
  const int slots = (a.D + 7) / 8;
  auto go = [&](auto lanes) {
    rows_kernel<T, UNITS, INTERLEAVED, decltype(lanes)::value, BACK><<<(unsigned)blocks, 256, lds, st>>>(a);
    return launch_status();
  };
  if (slots <= 1) return go(std::integral_constant<int, 1>{});
  if (slots <= 2) return go(std::integral_constant<int, 2>{});
  if (slots <= 4) return go(std::integral_constant<int, 4>{});
  if (slots <= 8) return go(std::integral_constant<int, 8>{});
  return go(std::integral_constant<int, 16>{});
}
template <class T, bool BACK>
int launch_type(const Args &a, bool units, int64_t blocks, size_t lds, hipStream_t st) {
  if (units) return a.interleaved ? launch_lanes<T, true, true, BACK>(a, blocks, lds, st) : launch_lanes<T, true, false, BACK>(a, blocks, lds, st);
  return a.interleaved ? launch_lanes<T, false, true, BACK>(a, blocks, lds, st) : launch_lanes<T, false, false, BACK>(a, blocks, lds, st);
}

// totals of the workgroups' sums: 16 columns a workgroup, their rows in 16 parts that are added up in order
__global__ __launch_bounds__(256) void weight_sums_kernel(const float *partials, int64_t rows, int D, float *d_q, float *d_k) {
  __shared__ float part[16][17];
  const int col = threadIdx.x & 15, p = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
  float sum = 0.f;
  if (c < 2 * D)
    for (int64_t r = p; r < rows; r += 16) sum += partials[r * 2 * D + c];
  part[p][col] = sum;
  __syncthreads();
  if (p != 0 || c >= 2 * D) return;
  for (int k = 1; k < 16; ++k) sum += part[k][col];
  float *out = c < D ? d_q : d_k;
  if (out) out[c < D ? c : c - D] = sum;
}

static bool on_fours(const pa_heads &h, size_t elem) {
  return reinterpret_cast<uintptr_t>(h.data) % (4 * elem) == 0 && h.batch % 4 == 0 && h.row % 4 == 0 && h.head % 4 == 0;
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
static size_t lds_of(const Plan &plan, int half, bool back) {
  const size_t turns = (size_t)plan.per_block * half * sizeof(float2), shares = back ? 256 * 8 * sizeof(float) : 0;
  return turns > shares ? turns : shares;
}

static Args args_of(const pa_rotate_params &p, const pa_heads &q, const pa_heads &k) {
  Args a = {};
  a.q.x = q.data, a.q.batch = q.batch, a.q.row = q.row, a.q.head = q.head, a.q.weight = p.q_weight;
  a.k.x = k.data, a.k.batch = k.batch, a.k.row = k.row, a.k.head = k.head, a.k.weight = p.k_weight;
  a.positions = p.positions, a.frequencies = p.frequencies;
  a.points = p.B * p.N, a.N = p.N, a.position_batch = p.position_batch;
  a.Hq = (int)p.Hq, a.Hk = (int)p.Hk, a.D = (int)p.D, a.half = (int)(p.rotated / 2), a.axes = (int)p.axes;
  a.position_type = p.position_type, a.interleaved = p.interleaved, a.norm = p.norm, a.eps = (float)p.eps;
  return a;
}
static bool units_of(const Args &a, size_t elem) {
  return a.D % 8 == 0 && (a.interleaved || a.half % 4 == 0) && reinterpret_cast<uintptr_t>(a.q.out) % (4 * elem) == 0 &&
         reinterpret_cast<uintptr_t>(a.k.out) % (4 * elem) == 0;
}

int forward(int dtype, const pa_rotate_params &p, const pa_heads &q, const pa_heads &k, void *q_out, void *k_out, int num_cu, hipStream_t st) {
  const size_t elem = dtype == PA_F32 ? 4 : 2;
  Args a = args_of(p, q, k);
  a.q.out = q_out, a.k.out = k_out;
  const Plan plan = plan_of(a.points, num_cu);
  a.per_block = plan.per_block;
  const bool units = units_of(a, elem) && on_fours(q, elem) && on_fours(k, elem);
  const size_t lds = lds_of(plan, a.half, false);
  return dtype == PA_F32 ? launch_type<float, false>(a, units, plan.blocks, lds, st) : launch_type<bf16, false>(a, units, plan.blocks, lds, st);
}

int64_t backward_workspace_bytes(const pa_rotate_params &p, int num_cu) {
  return plan_of(p.B * p.N, num_cu).blocks * 2 * p.D * (int64_t)sizeof(float);
}
int backward(int dtype, const pa_rotate_params &p, const pa_heads &q, const pa_heads &k, const pa_heads &d_q, const pa_heads &d_k, void *dq,
             void *dk, float *d_q_weight, float *d_k_weight, float *workspace, int num_cu, hipStream_t st) {
  const size_t elem = dtype == PA_F32 ? 4 : 2;
  Args a = args_of(p, q, k);
  a.q.out = dq, a.k.out = dk;
  a.q.dy = d_q.data, a.q.dy_batch = d_q.batch, a.q.dy_row = d_q.row, a.q.dy_head = d_q.head;
  a.k.dy = d_k.data, a.k.dy_batch = d_k.batch, a.k.dy_row = d_k.row, a.k.dy_head = d_k.head;
  const Plan plan = plan_of(a.points, num_cu);
  a.per_block = plan.per_block;
  a.partials = d_q_weight || d_k_weight ? workspace : nullptr;
  const bool units = units_of(a, elem) && on_fours(q, elem) && on_fours(k, elem) && on_fours(d_q, elem) && on_fours(d_k, elem);
  const size_t lds = lds_of(plan, a.half, true);
  int rc = dtype == PA_F32 ? launch_type<float, true>(a, units, plan.blocks, lds, st) : launch_type<bf16, true>(a, units, plan.blocks, lds, st);
  if (rc || !a.partials) return rc;
  weight_sums_kernel<<<(unsigned)((2 * p.D + 15) / 16), 256, 0, st>>>(workspace, plan.blocks, (int)p.D, d_q_weight, d_k_weight);
  return launch_status();
}

}  // namespace rotate
}  // namespace pa
