// Products of 8-bit integers with one float32 scale per token (row of activations) and per output channel (row of weights):
//   q = rint(x (127 / max |x|)) per row, s = max |x| / 127;  y = act(s s_w (q . q_w) + b) + residual
// Both quotients are rounded to float32: of a value half a step between two codes (max |x| / 2, say) either may be taken.
// The sums of whole numbers are exact in 32 bits up to 131 072 terms of 127 x 127.  int8 matrix instructions have twice the
// rate of bf16 ones and the operands half the bytes, so the products run on the tile kernel of pa_tile.h with stages of 128
// elements.
#include "pa_common.h"
#include "pa_host.h"
#include "pa_tile.h"

namespace pa {
namespace int8 {

using tile::Args;
using tile::Layout;
using tile::Space;
using tile::u32x2;
using tile::u32x4;
using tile::up;
using tile::whole_rows;

// eight neighbouring elements as float32, zeros past `left`
template <bool VEC>
__device__ __forceinline__ void load8(const bf16 *p, int64_t left, float (&v)[8]) {
  if (VEC && left >= 8) {
    const u32x4 w = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t b = w[j];
      v[2 * j] = __uint_as_float(b << 16), v[2 * j + 1] = __uint_as_float(b & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? load_as_f32(p + j) : 0.f;
  }
}
template <bool VEC>
__device__ __forceinline__ void load8(const float *p, int64_t left, float (&v)[8]) {
  if (VEC && left >= 8) {
    const tile::f32x4 a = *reinterpret_cast<const tile::f32x4 *>(p), b = *reinterpret_cast<const tile::f32x4 *>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : 0.f;
  }
}

// largest value over groups of LANES neighbouring lanes, in every lane
template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  auto larger = [](uint32_t x, uint32_t y) { return x > y ? x : y; };
  auto step = [&](uint32_t x, auto ctrl) {
    constexpr int c = decltype(ctrl)::value;
    return larger(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, c, 0xf, 0xf, true));
  };
  v = step(v, std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  v = step(v, std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  v = step(v, std::integral_constant<int, 0x141>{});  // row_half_mirror
  v = step(v, std::integral_constant<int, 0x140>{});  // row_mirror
  if constexpr (LANES >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = larger(r[0], r[1]);
  }
  if constexpr (LANES >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = larger(r[0], r[1]);
  }
  return v;
}

// ---------------------------------------------------------------------------------------------------------------
// quantize_rows_kernel: LANES lanes per row, eight elements per lane and step; rows of up to 8 LANES NCH elements stay in
// registers between the maximum and the rounding, longer ones are read again.  A wave has ROWS sets of rows in flight.  The
// maximum runs over the bits of |x|, in which NaN lies above infinity above the numbers: a row with one of them gets scale NaN,
// which is what a product with it would be.  Bound by HBM.
// ---------------------------------------------------------------------------------------------------------------
struct Quantize {
  const void *x;
  int64_t M, K, ldx, ldq;  // elements; bytes
  uint8_t *q;
  float *scale;
  uint32_t *clear;  // (M) set to zero, or NULL
};

template <class T, int LANES, int NCH, int ROWS, bool VEC>
__global__ __launch_bounds__(256) void quantize_rows_kernel(Quantize a) {
  constexpr int SPAN = LANES * 8, PER = 256 / LANES;  // elements of a step; rows of a workgroup
  const int lane = threadIdx.x % LANES, first = threadIdx.x / LANES;
  const T *x = static_cast<const T *>(a.x);
  const int64_t stride = (int64_t)gridDim.x * PER;
  for (int64_t base = (int64_t)blockIdx.x * PER + first; base < a.M; base += ROWS * stride) {
    float v[ROWS][NCH][8];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int64_t row = base + r * stride;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int64_t k = c * SPAN + lane * 8;
        load8<VEC>(x + row * a.ldx + k, row < a.M ? a.K - k : 0, v[r][c]);
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int64_t row = base + r * stride;
      if (row >= a.M) break;
      uint32_t most = 0;
      auto larger = [&](const float (&w)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t b = __float_as_uint(w[j]) & 0x7fffffffu;
          most = b > most ? b : most;
        }
      };
#pragma unroll
      for (int c = 0; c < NCH; ++c) larger(v[r][c]);
      for (int64_t k = NCH * SPAN + lane * 8; k < a.K; k += SPAN) {
        float w[8];
        load8<VEC>(x + row * a.ldx + k, a.K - k, w);
        larger(w);
      }
      most = lanes_max<LANES>(most);
      const bool finite = most < 0x7f800000u;
      const float top = __uint_as_float(most);
      const float lift = top < 0x1p-100f ? 0x1p100f : 1.f;  // 127 / top stays finite
      const float inv = finite && most > 0 ? 127.f / (top * lift) : 0.f;
      auto store = [&](int64_t k, const float (&w)[8]) {
        if (k >= a.ldq) return;
        u32x2 out = {0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float r = fminf(fmaxf(rintf(w[j] * lift * inv), -127.f), 127.f);
          const uint32_t code = finite ? (uint32_t)((int)r & 0xff) : 0u;
          if (j < 4) out[0] |= code << (8 * j);
          else out[1] |= code << (8 * (j - 4));
        }
        *reinterpret_cast<u32x2 *>(a.q + row * a.ldq + k) = out;
      };
#pragma unroll
      for (int c = 0; c < NCH; ++c) store(c * SPAN + lane * 8, v[r][c]);
      for (int64_t k = NCH * SPAN + lane * 8; k < a.ldq; k += SPAN) {
        float w[8];
        load8<VEC>(x + row * a.ldx + k, a.K - k, w);
        store(k, w);
      }
      if (lane == 0) a.scale[row] = finite ? top / 127.f : __uint_as_float(0x7fc00000u);
      if (lane == 0 && a.clear) a.clear[row] = 0u;
    }
  }
}

static constexpr int64_t kMaxTerms = 131072;  // 127 x 127 of them stay below 2^31

bool supported(int dtype, int64_t M, int64_t K, int64_t N) {
  return (dtype == PA_F32 || dtype == PA_BF16) && M > 0 && K > 0 && N > 0 && M <= (int64_t)1 << 32 && K <= kMaxTerms && N <= 1 << 18;
}

template <class T, bool VEC>
static int quantize(const Quantize &a, int num_cu, hipStream_t st) {
  auto go = [&](auto kernel, int64_t per) {
    int64_t grid = (a.M + per - 1) / per;
    if (grid > 8 * (int64_t)num_cu) grid = 8 * (int64_t)num_cu;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, st, a);
    return launch_status();
  };
  const int64_t w = a.ldq;  // zeros behind the last element are written by the lanes that would hold them
  if (w <= 128) return go(quantize_rows_kernel<T, 16, 1, 4, VEC>, 16);
  if (w <= 256) return go(quantize_rows_kernel<T, 32, 1, 4, VEC>, 8);
  if (w <= 512) return go(quantize_rows_kernel<T, 64, 1, 4, VEC>, 4);
  return go(quantize_rows_kernel<T, 64, 4, 1, VEC>, 4);
}

static int quantize(int dtype, const Quantize &a, int num_cu, hipStream_t st) {
  const bool vec = whole_rows(a.x, a.ldx, dtype == PA_F32 ? 4 : 2);
  if (dtype == PA_F32) return vec ? quantize<float, true>(a, num_cu, st) : quantize<float, false>(a, num_cu, st);
  return vec ? quantize<bf16, true>(a, num_cu, st) : quantize<bf16, false>(a, num_cu, st);
}

int quantize_rows(int dtype, int64_t M, int64_t K, const void *x, int64_t ldx, void *q, int64_t ldq, float *scale, int num_cu,
                  hipStream_t st) {
  return quantize(dtype, Quantize{x, M, K, ldx, ldq, static_cast<uint8_t *>(q), scale, nullptr}, num_cu, st);
}

template <class TO, tile::Kind KIND>
static int product(const Args &a, int num_cu, hipStream_t st) {
  return tile::launch<tile::I8, TO, KIND>(a, num_cu, st);
}

// codes of a weight (rows, width) as the tile kernel reads them: as they lie, or copied to rows of whole units
static const void *codes_of(const void *w, int64_t rows, int64_t width, bool plan, Space &ws, Layout &lay) {
  if (!plan && whole_rows(w, width, 1)) return w;
  void *dst = ws.take(rows * up(width, 16));
  lay.add(w, width, dst, rows, width, up(width, 16), up(width, 16), false);
  return dst;
}

struct Tokens {
  uint8_t *q;
  float *scale;
};
static Tokens tokens(int64_t M, int64_t K, Space &ws) {
  return {static_cast<uint8_t *>(ws.take(M * up(K, 16))), static_cast<float *>(ws.take(M * 4))};
}

template <class TO>
static int linear(int dtype, int64_t M, int64_t K, int64_t N, const void *w, const float *w_scale, const float *bias, int act,
                  const void *x, const void *residual, void *y, char *workspace, int64_t *bytes, int num_cu, hipStream_t st) {
  Space ws{workspace};
  Layout lay;
  const Tokens q = tokens(M, K, ws);
  const void *codes = codes_of(w, N, K, bytes != nullptr, ws, lay);
  if (bytes) return *bytes = ws.used, PA_OK;
  int rc = tile::lay_out(lay, 1, st);
  if (!rc) rc = quantize_rows(dtype, M, K, x, K, q.q, up(K, 16), q.scale, num_cu, st);
  if (rc) return rc;
  Args a{};
  a.X = q.q, a.ldx = a.ldw = up(K, 16), a.units = (int)(up(K, 16) / 16);
  a.W[0] = codes;
  a.M = M, a.N = a.limit = (int)N;
  a.bias[0] = bias, a.sx = q.scale, a.sw[0] = w_scale;
  a.residual = residual, a.out = y, a.ldo = N, a.act = act;
  a.vec = whole_rows(y, N, sizeof(TO)) && (!residual || aligned16(residual));
  return product<TO, tile::kPlain>(a, num_cu, st);
}

int64_t linear_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  int64_t bytes = 0;
  linear<float>(PA_F32, M, K, N, nullptr, nullptr, nullptr, 0, nullptr, nullptr, nullptr, nullptr, &bytes, 0, nullptr);
  return bytes;
}

int linear(int dtype, int64_t M, int64_t K, int64_t N, const void *w, const float *w_scale, const float *bias, int act, const void *x,
           const void *residual, void *y, void *workspace, int num_cu, hipStream_t st) {
  char *ws = static_cast<char *>(workspace);
  if (dtype == PA_F32) return linear<float>(dtype, M, K, N, w, w_scale, bias, act, x, residual, y, ws, nullptr, num_cu, st);
  return linear<bf16>(dtype, M, K, N, w, w_scale, bias, act, x, residual, y, ws, nullptr, num_cu, st);
}

// The gated block: x's codes against W_gate and W_up in one product, the hidden layer's codes against W_down.  A row's scale is known
// when the row is complete, and the product is formed twice, first for the largest value of each row and then for the codes: the
// hidden layer is in memory as codes alone.  Kept in bf16 between one product and its quantisation it would be rounded twice,
// which moves the output by 0.9 % of itself (the codes' own rounding: 0.3); in float32 its 8 F bytes per row
// cost as much as the second product.
template <class TO>
static int gated(int dtype, int64_t M, int64_t C, int64_t F, const pa_int8_gated_params &p, int act, const void *x,
                 const void *residual, void *y, char *workspace, int64_t *bytes, int num_cu, hipStream_t st) {
  Space ws{workspace};
  Layout lay;
  const bool plan = bytes != nullptr;
  const int64_t Kc = up(C, 16), Kf = up(F, 16), Fp = up(F, 32), Mp = up(M, tile::kGroupRows);
  const Tokens qx = tokens(M, C, ws), qh = tokens(Mp, Fp, ws);
  uint32_t *peak = static_cast<uint32_t *>(ws.take(M * 4));
  const void *gate = codes_of(p.w_gate, F, C, plan, ws, lay), *upw = codes_of(p.w_up, F, C, plan, ws, lay),
             *down = codes_of(p.w_down, C, F, plan, ws, lay);
  if (plan) return *bytes = ws.used, PA_OK;
  int rc = tile::lay_out(lay, 1, st);
  if (!rc) rc = quantize(dtype, Quantize{x, M, C, C, Kc, qx.q, qx.scale, peak}, num_cu, st);
  if (rc) return rc;
  Args a{};
  a.X = qx.q, a.ldx = a.ldw = Kc, a.units = (int)(Kc / 16);
  a.W[0] = gate, a.W[1] = upw;
  a.M = M, a.N = (int)F, a.limit = (int)Fp;
  a.bias[0] = p.b_gate, a.bias[1] = p.b_up;
  a.sx = qx.scale, a.sw[0] = p.s_gate, a.sw[1] = p.s_up;
  a.act = act, a.peak = peak;
  if ((rc = product<TO, tile::kPeak>(a, num_cu, st))) return rc;
  a.out = qh.q, a.ldo = Fp, a.row_scale = qh.scale;
  if ((rc = product<TO, tile::kCodes>(a, num_cu, st))) return rc;
  Args d{};
  d.X = qh.q, d.ldx = Fp, d.ldw = Kf, d.units = (int)(Kf / 16), d.x_groups = true;
  d.W[0] = down;
  d.M = M, d.N = d.limit = (int)C;
  d.bias[0] = p.b_down, d.sx = qh.scale, d.sw[0] = p.s_down;
  d.residual = residual, d.out = y, d.ldo = C;
  d.vec = whole_rows(y, C, sizeof(TO)) && (!residual || aligned16(residual));
  return product<TO, tile::kPlain>(d, num_cu, st);
}

int64_t gated_workspace_bytes(int dtype, int64_t M, int64_t C, int64_t F) {
  int64_t bytes = 0;
  const pa_int8_gated_params p{};
  if (dtype == PA_F32) gated<float>(dtype, M, C, F, p, 0, nullptr, nullptr, nullptr, nullptr, &bytes, 0, nullptr);
  else gated<bf16>(dtype, M, C, F, p, 0, nullptr, nullptr, nullptr, nullptr, &bytes, 0, nullptr);
  return bytes;
}

int gated(int dtype, int64_t M, int64_t C, int64_t F, const pa_int8_gated_params &p, int act, const void *x, const void *residual,
          void *y, void *workspace, int num_cu, hipStream_t st) {
  char *ws = static_cast<char *>(workspace);
  if (dtype == PA_F32) return gated<float>(dtype, M, C, F, p, act, x, residual, y, ws, nullptr, num_cu, st);
  return gated<bf16>(dtype, M, C, F, p, act, x, residual, y, ws, nullptr, num_cu, st);
}

}  // namespace int8
}  // namespace pa
