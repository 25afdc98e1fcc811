// Gated feed-forward block, y = residual + W_down (act(W_gate x + b_gate) * (W_up x + b_up)) + b_down, and its backward pass:
//   h  = act(g) u                     g = W_gate x + b_gate,  u = W_up x + b_up
//   dh = W_down^T dy                  dg = dh u act'(g),      du = dh act(g)
//   dx = W_gate^T dg + W_up^T du,     d W_gate = dg^T x, d W_up = du^T x, d W_down = dy^T h, d b = column sums
// Both input products, the activation and the factor are one kernel (kGated); for many bf16 rows of up to 256 channels all three
// products are (pa_gated_rows.hip).  The backward forms g and u again beside dh
// (kBack: 4 C F operations per row more, against 4 F elements per row written by the forward and read back), so the forward
// leaves nothing behind.  Sums and all that happens between two products are float32; h, dg and du are rounded once, to the
// activations' type, as operands of the next product.
//
// Operands whose rows are not whole 16-byte units (odd widths, views off a boundary) are copied to padded rows first, with the
// transposed weights of the backward pass in the same launch.
#include <algorithm>

#include "pa_common.h"
#include "pa_host.h"
#include "pa_tile.h"

namespace pa {
namespace gated {

using tile::Args;
using tile::Layout;
using tile::Space;
using tile::up;
using tile::whole_rows;

// ---------------------------------------------------------------------------------------------------------------
// lay_out_kernel: up to eight matrices copied into rows of whole units, zeros behind their last column, or transposed.  A
// workgroup moves 64 x 64 elements; transposed ones turn in LDS.
// ---------------------------------------------------------------------------------------------------------------
template <class U>  // unsigned integer of the elements' size
__global__ __launch_bounds__(256) void lay_out_kernel(Layout a) {
  __shared__ U turn[64][65];
  Layout::One o = a.m[0];
#pragma unroll
  for (int k = 1; k < Layout::kMost; ++k)
    if (k < a.count && (int64_t)blockIdx.x >= a.m[k].first) o = a.m[k];
  const int64_t block = (int64_t)blockIdx.x - o.first;
  const int across = (o.width + 63) / 64, c0 = (int)(block % across) * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const int64_t r0 = block / across * 64;
  const U *src = static_cast<const U *>(o.src);
  U *dst = static_cast<U *>(o.dst);
  U v[16];  // all of a thread's loads before its first store: places outside are read at the nearest inside
  if (!o.turned) {
    const int c = c0 + x < o.cols ? c0 + x : o.cols - 1;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int64_t r = r0 + y + 4 * k;
      v[k] = src[(r < o.rows ? r : o.rows - 1) * o.src_ld + c];
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int64_t r = r0 + y + 4 * k;
      if (r < o.rows && c0 + x < o.width) dst[r * o.ld + c0 + x] = c0 + x < o.cols ? v[k] : U(0);
    }
    return;
  }
  const int64_t r = r0 + x < o.rows ? r0 + x : o.rows - 1;
#pragma unroll
  for (int k = 0; k < 16; ++k) {  // row c of src is column c of dst
    const int c = c0 + y + 4 * k;
    v[k] = src[(int64_t)(c < o.cols ? c : o.cols - 1) * o.src_ld + r];
  }
#pragma unroll
  for (int k = 0; k < 16; ++k) turn[y + 4 * k][x] = c0 + y + 4 * k < o.cols ? v[k] : U(0);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 16; ++k)
    if (r0 + y + 4 * k < o.rows && c0 + x < o.width) dst[(r0 + y + 4 * k) * o.ld + c0 + x] = turn[x][y + 4 * k];
}

}  // namespace gated

namespace tile {
int lay_out(const Layout &a, size_t elem, hipStream_t st) {
  using gated::lay_out_kernel;
  if (a.count == 0) return PA_OK;
  if (a.blocks > 0x7fffffff) return PA_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)a.blocks);
  if (elem == 1) hipLaunchKernelGGL(lay_out_kernel<uint8_t>, grid, dim3(256), 0, st, a);
  else if (elem == 2) hipLaunchKernelGGL(lay_out_kernel<uint16_t>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(lay_out_kernel<uint32_t>, grid, dim3(256), 0, st, a);
  return launch_status();
}

bool launches_query(int bytes, int kind, int64_t M, int64_t N, int64_t units, int64_t units2, int num_cu, int64_t out[4]) {
  if ((bytes != 1 && bytes != 2 && bytes != 4) || kind < kPlain || kind > kCodes) return false;
  if ((bytes == 1 && (kind == kGated || kind == kBack)) || (bytes != 1 && kind >= kPeak)) return false;
  const Launches l = launches_of(bytes, (Kind)kind, M, N, units, units2, num_cu);
  for (int k = 0; k < 2; ++k) out[2 * k] = l.rows[k], out[2 * k + 1] = l.size[k];
  return true;
}

}  // namespace tile

namespace gated {

// ---------------------------------------------------------------------------------------------------------------
// totals_kernel: partial products of the row-axis kernels added up in a fixed order, cropped to the parameter's size and
// rounded to its type, all gradients in one launch.  A workgroup takes 256 neighbouring elements of a partial's rows, every
// fourth partial per wave, four elements per lane.
// ---------------------------------------------------------------------------------------------------------------
struct Totals {
  static constexpr int kMost = 6;
  struct One {
    const float *src;  // [G][..][ld], stride elements between partials
    void *dst;         // (rows, cols)
    int64_t stride, n, first;
    int G, cols, ld, bytes;
  } r[kMost];
  int count = 0;
  int64_t blocks = 0;
  void add(const float *src, int64_t G, int64_t stride, int64_t ld, void *dst, int64_t rows, int64_t cols, int bytes) {
    if (!dst) return;
    r[count++] = One{src, dst, stride, rows * ld, blocks, (int)G, (int)cols, (int)ld, bytes};
    blocks += (rows * ld + 255) / 256;
  }
};

__global__ __launch_bounds__(256) void totals_kernel(Totals a) {
  __shared__ float part[4][256];
  Totals::One o = a.r[0];
#pragma unroll
  for (int k = 1; k < Totals::kMost; ++k)
    if (k < a.count && (int64_t)blockIdx.x >= a.r[k].first) o = a.r[k];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t e0 = ((int64_t)blockIdx.x - o.first) * 256;
  float s[4] = {};  // of elements e0 + 64 j + lane: whole lines, whatever the alignment; past the end the last one again
  const float *p[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) p[j] = o.src + (e0 + 64 * j + lane < o.n ? e0 + 64 * j + lane : o.n - 1);
  int g = wave;
  for (; g + 4 < o.G; g += 8) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[j & 3][(g + (j & 4)) * o.stride];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] += v[j] + v[4 + j];
  }
  if (g < o.G)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] += p[j][g * o.stride];
#pragma unroll
  for (int j = 0; j < 4; ++j) part[wave][64 * j + lane] = s[j];
  __syncthreads();
  const int64_t e = e0 + threadIdx.x;
  if (e >= o.n) return;
  const int64_t row = e / o.ld;
  const int col = (int)(e - row * o.ld);
  if (col >= o.cols) return;
  const float v = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
  if (o.bytes == 2) static_cast<uint16_t *>(o.dst)[row * o.cols + col] = f32_to_bf16_bits(v);
  else static_cast<float *>(o.dst)[row * o.cols + col] = v;
}

// ---------------------------------------------------------------------------------------------------------------
// tile_sums_kernel: the column sums that the hidden layer's kernels leave per 32 rows, [tiles][n], to [gridDim.y][n].
// ---------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void tile_sums_kernel(const float *__restrict__ src, float *__restrict__ dst, int64_t tiles, int n) {
  const int e = blockIdx.x * 256 + threadIdx.x;
  if (e >= n) return;
  const int64_t per = (tiles + gridDim.y - 1) / gridDim.y, t0 = blockIdx.y * per, t1 = t0 + per < tiles ? t0 + per : tiles;
  float s[8] = {};
  int64_t t = t0;
  for (; t + 8 <= t1; t += 8)
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] += src[(t + k) * n + e];
  for (; t < t1; ++t) s[0] += src[t * n + e];
  dst[(int64_t)blockIdx.y * n + e] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
}

// ================================================================================================
// host side
// ================================================================================================
// rows of `width` elements as the tile kernels read them: as they lie, or a padded copy queued in `lay`
struct Rows {
  const void *p;
  int64_t ld;  // bytes
  int units;
};
static Rows rows_of(const void *p, int64_t rows, int64_t width, int64_t elem, bool copy, Space &ws, Layout *lay) {
  const int64_t padded = up(width, 16 / elem);
  Rows r{p, padded * elem, (int)(padded * elem / 16)};
  if (copy) {
    void *dst = ws.take(rows * padded * elem);
    if (lay) lay->add(p, width, dst, rows, width, padded, padded, false);
    r.p = dst;
  }
  return r;
}

// pa_gated_rows.hip
bool rows_supported(int64_t C, int64_t F);
int64_t rows_worth(int64_t M, int64_t C, int num_cu);
int64_t rows_blob_bytes(int64_t C, int64_t F);
int rows_pack(int64_t C, int64_t F, const pa_gated_params &p, void *blob, hipStream_t st);
int rows_forward(int64_t M, int64_t C, int64_t F, const void *blob, const float *b_down, int act, const void *x, const void *residual,
                 void *y, int num_cu, hipStream_t st);
int64_t hidden_blob_bytes(int64_t C, int64_t F);
int hidden_pack(int64_t C, int64_t F, const pa_gated_params &p, void *blob, hipStream_t st);
int rows_hidden_backward(int64_t M, int64_t C, int64_t F, int64_t Fp, const void *blob, int act, const void *x, const void *dy, void *dgu,
                         void *h, float *sums, int num_cu, hipStream_t st);

template <class E, class TO, tile::Kind KIND>
static int product(const Args &a, int num_cu, hipStream_t st) {
  return tile::launch<E, TO, KIND>(a, num_cu, st);
}

// The forward's workspace: packed weights of the kernel that keeps the hidden layer on chip, h of the rows that the tile kernels
// take, and padded copies of what is not laid out in whole units.  The query does not know the pointers.  Rows whose width is
// whole units are off a boundary only as views are, and then run in pieces, so that no call has to bring room for copies of all
// rows, or for the hidden layer of rows that have it on chip: of kLooseRows rows for widths that keep it there (262 144 x 256, F = 1 024,
// bf16: 87 MB instead of 674; off a boundary 627 -> 676 us), else of the multiple of it whose copies and hidden layer fit what all
// rows' hidden layer takes (100 003 x 512, F = 1 365, bf16: 279 MB instead of 382; 550 -> 547 us; in equal halves 611).
static constexpr int64_t kLooseRows = 32768;

template <class E, class TO>
static int forward(int64_t M, int64_t C, int64_t F, const pa_gated_params &p, int act, const void *x, const void *residual, void *y,
                   char *workspace, int64_t *bytes, int num_cu, hipStream_t st) {
  constexpr int64_t e = E::kBytes;
  const bool plan = bytes != nullptr, whole = C * e % 16 == 0, on_chip = e == 2 && whole && rows_supported(C, F);
  const bool loose = whole && !plan && !(aligned16(x) && aligned16(y) && aligned16(residual));
  const bool copy_x = plan ? !whole : !whole_rows(x, C, e);
  Space ws{workspace};
  Layout lay;
  const int64_t Fp = up(F, 32 / e), Cp = up(C, 16 / e);  // the hidden layer's columns: whole 32-byte groups
  void *blob = on_chip ? ws.take(rows_blob_bytes(C, F)) : nullptr;
  const int64_t done = on_chip && !loose ? rows_worth(M, C, num_cu) : 0;
  if (done > 0 && !plan) {
    int rc = rows_pack(C, F, p, blob, st);
    if (!rc) rc = rows_forward(done, C, F, blob, p.b_down, act, x, residual, y, num_cu, st);
    if (rc || done == M) return rc;
  }
  auto room = [&](Space &s, int64_t rows, bool copies, void *&h, void *&copy) {
    h = s.take(up(rows, tile::kGroupRows) * Fp * e);
    copy = copies ? s.take(rows * Cp * e) : nullptr;
  };
  const int64_t piece = M <= kLooseRows ? M : std::max<int64_t>(on_chip ? 1 : M * Fp / (Fp + Cp) / kLooseRows, 1) * kLooseRows;
  const int64_t per = loose && (on_chip || copy_x) ? piece : M - done;
  void *h, *copy;
  if (plan) {
    Space pieces = ws;
    room(ws, per, copy_x, h, copy);
    if (whole) room(pieces, piece, true, h, copy);
    if (pieces.used > ws.used) ws.used = pieces.used;
  } else {
    room(ws, per, copy_x, h, copy);
  }
  auto weight = [&](const void *w, int64_t rows, int64_t width) { return rows_of(w, rows, width, e, plan || !whole_rows(w, width, e), ws, &lay); };
  const Rows wg = weight(p.w_gate, F, C), wu = weight(p.w_up, F, C), wd = weight(p.w_down, C, F);
  if (plan) return *bytes = ws.used, PA_OK;
  for (int64_t r0 = done; r0 < M; r0 += per) {
    const int64_t rows = M - r0 < per ? M - r0 : per;
    auto from = [&](const void *q) { return q ? static_cast<const char *>(q) + r0 * C * e : nullptr; };
    if (copy_x) lay.add(from(x), C, copy, rows, C, Cp, Cp, false);
    if (int rc = tile::lay_out(lay, e, st)) return rc;
    lay = Layout{};  // the weights with the first piece
    Args a{};
    a.X = copy_x ? copy : from(x), a.ldx = Cp * e, a.units = (int)(Cp * e / 16);
    a.W[0] = wg.p, a.W[1] = wu.p, a.ldw = wg.ld;
    a.M = rows, a.N = (int)F, a.limit = (int)Fp;
    a.bias[0] = p.b_gate, a.bias[1] = p.b_up;
    a.out = h, a.ldo = Fp, a.act = act;
    if (int rc = product<E, TO, tile::kGated>(a, num_cu, st)) return rc;
    Args d{};
    d.X = h, d.ldx = Fp * e, d.units = wd.units, d.x_groups = tile::kGrouped<TO>;
    d.W[0] = wd.p, d.ldw = wd.ld;
    d.M = rows, d.N = d.limit = (int)C;
    d.bias[0] = p.b_down;
    d.residual = from(residual), d.out = const_cast<char *>(from(y)), d.ldo = C;
    d.vec = whole_rows(d.out, C, e) && (!residual || aligned16(d.residual));
    if (int rc = product<E, TO, tile::kPlain>(d, num_cu, st)) return rc;
  }
  return PA_OK;
}

static constexpr int64_t kMaxWidth = 1 << 18;  // 256 rows of two hidden layers of it stay below 2^31 bytes

bool supported(int dtype, int64_t M, int64_t C, int64_t F) {
  return (dtype == PA_F32 || dtype == PA_BF16) && M > 0 && C > 0 && F > 0 && M <= PA_MAX_ROWS && C <= kMaxWidth && F <= kMaxWidth &&
         M <= ((int64_t)1 << 60) / (16 * (C > F ? C : F));
}

int64_t forward_workspace_bytes(int dtype, int64_t M, int64_t C, int64_t F, int num_cu) {
  int64_t bytes = 0;
  const pa_gated_params p{};
  if (dtype == PA_F32) forward<tile::F32, float>(M, C, F, p, 0, nullptr, nullptr, nullptr, nullptr, &bytes, num_cu, nullptr);
  else forward<tile::Bf16, bf16>(M, C, F, p, 0, nullptr, nullptr, nullptr, nullptr, &bytes, num_cu, nullptr);
  return bytes;
}

int forward(int dtype, int64_t M, int64_t C, int64_t F, const pa_gated_params &p, int act, const void *x, const void *residual, void *y,
            void *workspace, int num_cu, hipStream_t st) {
  char *ws = static_cast<char *>(workspace);
  if (dtype == PA_F32) return forward<tile::F32, float>(M, C, F, p, act, x, residual, y, ws, nullptr, num_cu, st);
  return forward<tile::Bf16, bf16>(M, C, F, p, act, x, residual, y, ws, nullptr, num_cu, st);
}

// partial results of a row-axis product of `oa` by `ob` columns, and of the column sums of its first operand
template <class E>
static int64_t chunks_of(int64_t rows, int64_t oa, int64_t ob, int num_cu) {
  if (E::kBytes == 4) return gemm::cols_gemm_f32_chunks(rows, oa, ob, num_cu);
  return wgrad::chunks_for(rows, ((oa + 255) / 256) * ((ob + 255) / 256), oa * ob, num_cu);
}
struct Partials {
  int64_t G = 0, oa = 0, ob = 0;  // G: how many there are so far
  float *product = nullptr, *sums = nullptr;
};
template <class E>
static Partials partials_of(int64_t M, int64_t rows, int64_t oa, int64_t ob, int num_cu, Space &ws) {
  const int64_t before = (M - 1) / rows;  // pieces before the last one
  const int64_t most = (before > 0 ? before * chunks_of<E>(rows, oa, ob, num_cu) : 0) + chunks_of<E>(M - before * rows, oa, ob, num_cu);
  Partials r;
  r.oa = oa, r.ob = ob;
  r.product = static_cast<float *>(ws.take(most * oa * ob * 4));
  r.sums = static_cast<float *>(ws.take(most * oa * 4));
  return r;
}
template <class E>
static int rows_product(Partials &r, const void *A, const void *B, int64_t rows, int groups, int num_cu,
                        hipStream_t st) {  // groups: 1 if A, 2 if B is a matrix of the hidden layer
  float *product = r.product + r.G * r.oa * r.ob, *sums = r.sums + r.G * r.oa;
  const int64_t G = chunks_of<E>(rows, r.oa, r.ob, num_cu);
  r.G += G;
  if (E::kBytes == 2) return wgrad::launch_wide(A, r.oa, r.oa, B, r.ob, r.ob, rows, G, nullptr, product, groups == 1 ? nullptr : sums, st, groups);
  return gemm::cols_gemm_f32(A, r.oa, r.oa, B, r.ob, r.ob, rows, nullptr, product, sums, num_cu, st);
}

// The backward's workspace: dg and du, h, transposed weights, partial weight gradients, and copies of what is not laid out in whole
// units.  As in the forward, x and dy off a boundary run in pieces, as few as leave room for their copies beside a piece's
// hidden layer, and for partial gradients of their own, in what a call on boundaries needs (131 072 x 256, F = 1 024, bf16: 978 MB
// instead of 1 112; 1 048 576 x 256, F = 256: 1 814 instead of 2 887; off a boundary 262 144 x 256, F = 1 024: 1 690 -> 1 787 us).
struct BackwardRoom {
  void *dgu, *h, *x, *dy;
  Partials in, down;
};
template <class E>
static BackwardRoom backward_room(int64_t M, int64_t rows, int64_t Cp, int64_t Fp, bool copy_x, bool copy_dy, int num_cu, Space &ws) {
  constexpr int64_t e = E::kBytes;
  const int64_t whole = up(rows, tile::kGroupRows);
  BackwardRoom r;
  r.dgu = ws.take(whole * 2 * Fp * e), r.h = ws.take(whole * Fp * e);
  r.x = copy_x ? ws.take(rows * Cp * e) : nullptr, r.dy = copy_dy ? ws.take(rows * Cp * e) : nullptr;
  r.in = partials_of<E>(M, rows, 2 * Fp, Cp, num_cu, ws), r.down = partials_of<E>(M, rows, Cp, Fp, num_cu, ws);
  return r;
}

template <class E, class TO>
static int backward(int64_t M, int64_t C, int64_t F, const pa_gated_params &p, int act, const void *x, const void *dy, void *dx,
                    const pa_gated_grads &out, char *workspace, int64_t *bytes, int num_cu, hipStream_t st) {
  constexpr int64_t e = E::kBytes, U = 16 / e, LEAST = e == 4 ? 16 : 8;  // narrowest operand of the row-axis kernels
  const bool plan = bytes != nullptr;
  Space ws{workspace};
  Layout lay;
  const int64_t Cp = up(C < LEAST ? LEAST : C, U), Fp = up(F < LEAST ? LEAST : F, 32 / e);
  const bool whole = C == Cp, copy_x = !whole || !aligned16(x), copy_dy = !whole || !aligned16(dy);
  auto need = [&](int64_t rows, bool copies) {
    Space s{nullptr};
    backward_room<E>(M, rows, Cp, Fp, copies, copies, num_cu, s);
    return s.used;
  };
  int64_t per = M;  // rows of a piece: all of them, or of x and dy off a boundary
  if (whole && (plan || copy_x || copy_dy) && M > kLooseRows) {
    const int64_t most = need(M, false);
    for (int64_t n = 2; n == 2 || (per > kLooseRows && need(per, true) > most); n += n / 2) per = up((M + n - 1) / n, kLooseRows);
  }
  Space aligned = ws;
  BackwardRoom room = backward_room<E>(M, per, Cp, Fp, whole && plan ? true : copy_x, whole && plan ? true : copy_dy, num_cu, ws);
  if (plan) {
    backward_room<E>(M, M, Cp, Fp, copy_x, copy_dy, num_cu, aligned);
    if (aligned.used > ws.used) ws.used = aligned.used;
  }
  // rows of the kernel that owns them, which has the weights in an order of its own
  const bool by_rows = e == 2 && rows_supported(Cp, F);
  auto rows_done = [&](int64_t rows) { return by_rows && !plan ? rows_worth(rows, Cp, num_cu) : 0; };
  const bool tiles_too = per < M || rows_done(M) < M;  // some rows may be the tile kernels'
  void *blob = by_rows ? ws.take(hidden_blob_bytes(C, F)) : nullptr;
  auto weight = [&](const void *w) {
    Rows r{w, Cp * e, (int)(Cp * e / 16)};
    if (plan || (tiles_too && (!whole || !aligned16(w)))) {
      void *dst = ws.take(F * Cp * e);
      if (!plan) lay.add(w, C, dst, F, C, Cp, Cp, false);
      r.p = dst;
    }
    return r;
  };
  const Rows wg = weight(p.w_gate), wu = weight(p.w_up);
  // W_down^T (F, Cp), and [W_gate; W_up]^T (C, 2 Fp): hidden units past F are zero columns
  void *wd_t = ws.take(F * Cp * e), *w_t = ws.take(C * 2 * Fp * e);
  // bf16: dg and du are rounded for their products, their column sums are not
  const int64_t tiles = (M + 31) / 32, parts = tiles < 2048 ? (tiles + 31) / 32 : 64;
  float *sums = e == 2 ? static_cast<float *>(ws.take(tiles * 2 * Fp * 4)) : nullptr;
  float *sum_parts = e == 2 ? static_cast<float *>(ws.take(parts * 2 * Fp * 4)) : nullptr;
  if (plan) return *bytes = ws.used, PA_OK;
  if (tiles_too) lay.add(p.w_down, F, wd_t, F, C, Cp, Cp, true);
  if (dx) {
    lay.add(p.w_gate, C, w_t, C, F, Fp, 2 * Fp, true);
    lay.add(p.w_up, C, static_cast<char *>(w_t) + Fp * e, C, F, Fp, 2 * Fp, true);
  }
  const bool in_biases = out.b_gate || out.b_up, in_weights = out.w_gate || out.w_up || (e == 4 && in_biases);
  int rc = PA_OK;
  bool packed = false;
  for (int64_t r0 = 0; r0 < M; r0 += per) {
    const int64_t rows = M - r0 < per ? M - r0 : per, done = rows_done(rows), rest = rows - done;
    auto from = [](const void *q, int64_t row, int64_t ld) { return const_cast<char *>(static_cast<const char *>(q)) + row * ld; };
    const void *xr = from(x, r0, C * e), *dyr = from(dy, r0, C * e);
    if (copy_x) lay.add(xr, C, room.x, rows, C, Cp, Cp, false), xr = room.x;
    if (copy_dy) lay.add(dyr, C, room.dy, rows, C, Cp, Cp, false), dyr = room.dy;
    if ((rc = tile::lay_out(lay, e, st))) return rc;
    lay = Layout{};  // the weights with the first piece
    float *piece_sums = e == 2 ? sums + r0 / 32 * 2 * Fp : nullptr;
    if (done > 0) {
      if (!packed) rc = hidden_pack(C, F, p, blob, st);
      packed = true;
      if (!rc) rc = rows_hidden_backward(done, Cp, F, Fp, blob, act, xr, dyr, room.dgu, room.h, piece_sums, num_cu, st);
      if (rc) return rc;
    }
    if (rest > 0) {
      Args a{};
      a.X = from(xr, done, Cp * e), a.ldx = Cp * e, a.units = (int)(Cp * e / 16);
      a.X2 = from(dyr, done, Cp * e), a.ldx2 = Cp * e, a.units2 = a.units;
      a.W[0] = wg.p, a.W[1] = wu.p, a.W[2] = wd_t, a.ldw = wg.ld, a.ldw2 = Cp * e;
      a.M = rest, a.N = (int)F, a.limit = (int)Fp;
      a.bias[0] = p.b_gate, a.bias[1] = p.b_up;
      a.sums = e == 2 && in_biases ? piece_sums + done / 32 * 2 * Fp : nullptr;
      a.out = from(room.dgu, done, 2 * Fp * e), a.ldo = 2 * Fp, a.out2 = from(room.h, done, Fp * e), a.ldh = Fp, a.act = act;
      if ((rc = product<E, TO, tile::kBack>(a, num_cu, st))) return rc;
    }
    if (dx) {
      Args d{};
      d.X = room.dgu, d.ldx = 2 * Fp * e, d.units = (int)(2 * Fp * e / 16), d.x_groups = tile::kGrouped<TO>;
      d.W[0] = w_t, d.ldw = 2 * Fp * e;
      d.M = rows, d.N = d.limit = (int)C;
      d.out = from(dx, r0, C * e), d.ldo = C;
      d.vec = whole_rows(d.out, C, e);
      if ((rc = product<E, TO, tile::kPlain>(d, num_cu, st))) return rc;
    }
    if (in_weights && (rc = rows_product<E>(room.in, room.dgu, xr, rows, 1, num_cu, st))) return rc;
    if ((out.w_down || out.b_down) && (rc = rows_product<E>(room.down, dyr, room.h, rows, 2, num_cu, st))) return rc;
  }
  Totals totals;
  const Partials &in = room.in, &down = room.down;
  if (in_weights) {
    totals.add(in.product, in.G, 2 * Fp * Cp, Cp, out.w_gate, F, C, e);
    totals.add(in.product + Fp * Cp, in.G, 2 * Fp * Cp, Cp, out.w_up, F, C, e);
  }
  if (in_biases) {
    if (e == 2) {
      hipLaunchKernelGGL(tile_sums_kernel, dim3((unsigned)((2 * Fp + 255) / 256), (unsigned)parts), dim3(256), 0, st, sums, sum_parts, tiles,
                         (int)(2 * Fp));
      if ((rc = launch_status())) return rc;
    }
    const float *db = e == 2 ? sum_parts : in.sums;
    totals.add(db, e == 2 ? parts : in.G, 2 * Fp, F, out.b_gate, 1, F, 4);
    totals.add(db + Fp, e == 2 ? parts : in.G, 2 * Fp, F, out.b_up, 1, F, 4);
  }
  if (out.w_down || out.b_down) {
    totals.add(down.product, down.G, Cp * Fp, Fp, out.w_down, C, F, e);
    totals.add(down.sums, down.G, Cp, C, out.b_down, 1, C, 4);
  }
  if (totals.count == 0) return PA_OK;
  hipLaunchKernelGGL(totals_kernel, dim3((unsigned)totals.blocks), dim3(256), 0, st, totals);
  return launch_status();
}

int64_t backward_workspace_bytes(int dtype, int64_t M, int64_t C, int64_t F, int num_cu) {
  int64_t bytes = 0;
  const pa_gated_params p{};
  const pa_gated_grads g{};
  if (dtype == PA_F32) backward<tile::F32, float>(M, C, F, p, 0, nullptr, nullptr, nullptr, g, nullptr, &bytes, num_cu, nullptr);
  else backward<tile::Bf16, bf16>(M, C, F, p, 0, nullptr, nullptr, nullptr, g, nullptr, &bytes, num_cu, nullptr);
  return bytes;
}

int backward(int dtype, int64_t M, int64_t C, int64_t F, const pa_gated_params &p, int act, const void *x, const void *dy, void *dx,
             const pa_gated_grads &out, void *workspace, int num_cu, hipStream_t st) {
  char *ws = static_cast<char *>(workspace);
  if (dtype == PA_F32) return backward<tile::F32, float>(M, C, F, p, act, x, dy, dx, out, ws, nullptr, num_cu, st);
  return backward<tile::Bf16, bf16>(M, C, F, p, act, x, dy, dx, out, ws, nullptr, num_cu, st);
}

}  // namespace gated
}  // namespace pa
