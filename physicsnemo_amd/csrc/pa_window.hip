// Attention of points over a window of their neighbours and a few first points, served: y_i = sum_j p_ij v_j, p_i the softmax over the
// visible j of scale q_i . k_j (+ a bias by buckets of j - i).
//
// One pass over the visible keys, a weight one multiply-add and one exp2: a query's reference is the largest score of the first tile that it sees
// something of, and stays.  Where scores outgrow it until the weights pass 2^30, the workgroup looks for those queries' largest scores and goes over
// the keys once more (a running maximum would scale the values' sum in a branch, which costs copies of it around every tile: 193 -> 172 us below).
// A wave owns 32 queries of a head, a lane one of them (with its partner 32 lanes on): the scores of a tile of keys are the rows of a
// C tile, so that reference and sum are per lane, and the weights go back into the product with the values as they lie.  Four waves share the
// tiles of keys and values, two buffers in LDS, the next tile's loads under the present one's products.  Tiles that a wave's
// queries do not see are skipped, and only tiles on an edge are masked.
//
// What it takes: 131 072 x 8 x 32 bf16, 513 keys a query: 174 us (0.27 GB: 49 us; 69 GFLOP: 50 us; 52 vector and 16 exp2 instructions a tile of 32 x 32:
// about 110 us at full issue, which bounds it; 66 % of the issue slots, matrix pipes 20 %); 3 x 9 001 x 8 over 2 x 64, 1 024 keys: 98; 4 x 7 225 x 8 x 16 float32,
// 171 keys: 67; with biases 65 536 x 8 x 32, 257 keys: 77.  Five waves a SIMD instead of four spill (2 to 3 times as long), 64 queries a wave lose a third.
#include "pa_window.h"

#include <math.h>

namespace pa {
namespace window {

constexpr float kMost = 1073741824.f, kSlack = 16.f;  // how far weights may sum up, log2 of one may lie above the reference before it is taken again
// how far from 0 log2 of the reference's own weight may lie: -m c is rounded, at scores of 1e9 to tens and at 1e11 past what a float32 weight holds
constexpr float kSlip = 64.f;
// what the backward pass takes: past 2^22 the denominator's float32 logarithm, with the reference in it, is off by a quarter and more, and with it
// all weights of the row
constexpr float kMostStat = 4194304.f;

__device__ __forceinline__ float most_of(const f32x16 &z) {
  float m = z[0];
#pragma unroll
  for (int r = 1; r < 16; ++r) m = fmaxf(m, z[r]);
  return m;
}

// The softmax of a wave's queries so far, and the values' sum under it.  A query's numbers depend on its own scores alone.
template <class O, int DP>
struct Running {
  f32x16 o[DP / 32];
  float m, l, off;  // reference in units of z, this lane's share of the sum, -m c (0 while nothing was seen)
  bool fresh;       // for the whole wave: some query has seen nothing yet
  __device__ __forceinline__ void start(bool live) {
    zero(o);
    m = live ? -INFINITY : 0.f, l = 0.f, off = 0.f;
    fresh = true;
  }
  // the largest score of the first tile that a query sees something of is its reference
  __device__ __forceinline__ void refer(const f32x16 &z, float c) {
    const float most = half_max(most_of(z));
    m = m == -INFINITY ? most : m;
    off = m == -INFINITY ? 0.f : -m * c;
    fresh = some_lane(m == -INFINITY);
  }
  // z -> weights
  __device__ __forceinline__ typename O::Weights weigh(f32x16 &z, float c) {
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = __builtin_amdgcn_exp2f(fmaf(z[r], c, off));
    const typename O::Weights w = O::pack(z);
    l += O::sum(w, z);
    return w;
  }
};

// The same with the largest score so far for the reference, for the steps, which memory bounds: a weight costs a subtraction more, and is right for scores of
// any size.
template <class O, int DP>
struct Raising {
  f32x16 o[DP / 32];
  float m, l, ref;  // reference in units of z, this lane's share of the sum, m or 0 while nothing was seen
  __device__ __forceinline__ void start(bool live) {
    zero(o);
    m = live ? -INFINITY : 0.f, l = 0.f, ref = 0.f;
  }
  // a larger reference where this tile's largest score asks for it, and all that is summed so far under it
  __device__ __forceinline__ void raise(const f32x16 &z, float c) {
    const float most = half_max(most_of(z));
    const bool need = m == -INFINITY || !((most - ref) * c <= kSlack);
    if (!some_lane(need)) return;
    const float now = need ? fmaxf(m, most) : m;
    ref = now == -INFINITY ? 0.f : now;
    const float alpha = __builtin_amdgcn_exp2f((m - ref) * c);
    m = now;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
  }
  __device__ __forceinline__ float weight(float z, float c) const { return __builtin_amdgcn_exp2f((z - ref) * c); }
  // z -> weights
  __device__ __forceinline__ typename O::Weights weigh(f32x16 &z, float c) {
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = weight(z[r], c);
    const typename O::Weights w = O::pack(z);
    l += O::sum(w, z);
    return w;
  }
};

// z as the products start from it: the bias of a tile of keys from k0 for the query at position i of a wave from q0, or zero
template <bool BIAS>
__device__ __forceinline__ f32x16 start_of(const Args &a, int q0, int i, int k0, int g, const float *table) {
  f32x16 z;
  if constexpr (BIAS) {
    const Reach reach = reach_of(a.bias, k0 - q0 - 31, k0 + 31 - q0);
    if (reach == kNear) {
      const float *t = table + (k0 + 4 * g - i + table_low(a.bias));
#pragma unroll
      for (int r = 0; r < 16; ++r) z[r] = t[8 * (r >> 2) + (r & 3)];
    } else {
      const float far = reach == kFarBehind ? table[0] : table[table_size(a.bias) - 1];
#pragma unroll
      for (int r = 0; r < 16; ++r) z[r] = far;
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
  }
  return z;
}

// Waves a SIMD: bf16 rows to 32 run four, which the bound keeps; float32 rows of 64 take up to 14 registers more than two waves leave where they are
// not held to two.
template <class T, int DP, bool PLAIN, bool BIAS>
__global__ __launch_bounds__(256, DP == 32 && sizeof(T) == 2 ? 4 : DP == 64 && sizeof(T) == 4 ? 2 : 1) void forward_kernel(Args a) {
  constexpr int KT = tile_rows<T, DP>(), SUB = KT / 32, TILE = KT * WindowOps<T, DP>::kStride;
  extern __shared__ u32x4 lds_raw[];
  T *const tiles = reinterpret_cast<T *>(lds_raw);  // [buffer][keys, values][KT][stride]
  float *const table = reinterpret_cast<float *>(tiles + 4 * TILE);
  const uint32_t work = own_work(), at_head = work / (uint32_t)a.blocks;
  const int block = (int)(work - at_head * (uint32_t)a.blocks), b = (int)(at_head / (uint32_t)a.Hq), h = (int)(at_head - (uint32_t)b * (uint32_t)a.Hq);
  const int lane = threadIdx.x & 63, i = lane & 31, g = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int len = length_of(a, b), q0 = block * 128, qw = q0 + 32 * wave, me = qw + i;
  using O = WindowOps<T, DP>;
  Running<O, DP> run;
  run.start(me < len);
  if (q0 < len) {
    const typename O::Raw raw = O::template rows<PLAIN>(head_of<T>(a.q, b, h), a.q.row, me, len, me < len, a.D, g);
    typename O::Rows own;
    const int hk = h / (a.Hq / a.Hk);
    const T *const keys = head_of<T>(a.k, b, hk), *const values = head_of<T>(a.v, b, hk);
    const Tiles list(a, len, q0, q0 + 127 < len ? q0 + 127 : len - 1, KT);
    if constexpr (BIAS) fill_bias_table(a, h, table);
    const Sights sights = sights_of_queries(a, len, qw);
    Stage<O, T, DP, PLAIN, KT, 256> ks, vs;
    auto scores = [&](const T *rows, int r0) {
      f32x16 z = O::scores(rows, own, i, g, start_of<BIAS>(a, qw, me, r0, g, table), a.D);
      if (!sights.all(r0)) hide(z, keys_of(a, len, me), r0, g, -INFINITY);
      return z;
    };
    // all tiles of keys, and of values if they are wanted: f(keys, values, first key) for each sub-tile in sight.  Nothing in it changes the
    // values' sum but the products: a scaling in a branch would cost copies of the sum around every tile.
    auto pass = [&](bool both, auto &&f) {
      if (list.count > 0) {
        ks.load(a.k, keys, list[0] * KT, len, a.D, threadIdx.x);
        if (both) vs.load(a.v, values, list[0] * KT, len, a.D, threadIdx.x);
        if (both) own = O::settle(raw);
        ks.store(tiles, threadIdx.x);
        if (both) vs.store(tiles + TILE, threadIdx.x);
      }
      __syncthreads();
      for (int n = 0; n < list.count; ++n) {
        const T *const kt = tiles + (n & 1) * 2 * TILE, *const vt = kt + TILE;
        T *const next = tiles + ((n + 1) & 1) * 2 * TILE;
        if (n + 1 < list.count) {
          ks.load(a.k, keys, list[n + 1] * KT, len, a.D, threadIdx.x);
          if (both) vs.load(a.v, values, list[n + 1] * KT, len, a.D, threadIdx.x);
        }
        const int k0 = list[n] * KT;
#pragma unroll 1
        for (int s = 0; s < SUB; ++s) {
          if (sights.none(k0 + 32 * s)) continue;
          f(kt + 32 * s * O::kStride, vt + 32 * s * O::kStride, k0 + 32 * s);
        }
        if (n + 1 < list.count) {
          ks.store(next, threadIdx.x);
          if (both) vs.store(next + TILE, threadIdx.x);
        }
        __syncthreads();
      }
    };
    for (bool again = false;; again = true) {
      pass(true, [&](const T *krows, const T *vrows, int r0) {
        f32x16 z = scores(krows, r0);
        if (__builtin_expect(run.fresh, 0)) run.refer(z, a.c);
        O::outcome(vrows, run.weigh(z, a.c), lane, run.o);
      });
      // Scores far above the first ones: those queries take their largest score for the reference, and the workgroup goes over the keys again
      const bool high = half_max(run.l <= kMost ? 0.f : 1.f) > 0.f;
      if (again || !__syncthreads_or(high)) break;
      float most = -INFINITY;
      pass(false, [&](const T *krows, const T *, int r0) { most = fmaxf(most, most_of(scores(krows, r0))); });
      most = half_max(most);
      zero(run.o);
      run.l = 0.f;
      run.m = high ? most : run.m;
      run.off = run.m == -INFINITY ? 0.f : -run.m * a.c;
    }
    // A score of a visible infinite key is infinite, which thirds do not give: a sum of weights that is not finite is formed again, too, and so is one
    // whose reference weighs far from one
    const bool slips = run.m != -INFINITY && !(fabsf(fmaf(run.m, a.c, run.off)) <= kSlip);
    bool again = run.l * 0.f != 0.f || slips, bad = again || not_finite(run.o);
    if (__builtin_expect(some_lane(bad), 0)) {
      again = half_max(again ? 1.f : 0.f) > 0.f;
      bad = half_max(bad ? 1.f : 0.f) > 0.f;
      const Span span = keys_of(a, len, me);
      for (int d = 0; d < DP / 32; ++d)
        for (int r = 0; r < 16; ++r) run.o[d][r] = bad ? 0.f : run.o[d][r];
      auto score = [&](int j) {
        float z = half_sum(O::dot(own, O::template rows<PLAIN>(keys, a.k.row, j, len, true, a.D, g)));
        if constexpr (BIAS) z += bias_at(a.bias, table, j - me);
        return z;
      };
      const int low = qw - a.left > 0 ? qw - a.left : 0, high = qw + 31 + a.right < len - 1 ? qw + 31 + a.right : len - 1;
      float most = -INFINITY;
      bool open = true;  // no score is NaN so far
      for (int j = a.sinks > 0 ? 0 : low; j <= high && some_lane(again && open); j = j + 1 == a.sinks && low > j ? low : j + 1)
        if (const float z = score(j); span.sees(j)) most = fmaxf(most, z), open = open && z == z;
      if (again) run.l = 0.f, run.m = most, run.off = most == -INFINITY ? 0.f : -most * a.c;
      const float ref = run.m == -INFINITY ? 0.f : run.m;
      auto weight = [&](int j, bool &seen) {
        seen = span.sees(j);
        const float z = score(j), w = __builtin_amdgcn_exp2f(again ? (z - ref) * a.c : fmaf(z, a.c, run.off));
        if (again && seen && g == 0) run.l += w;
        return w;
      };
      auto on = [&] { return again && g == 0 && run.l == run.l; };
      add_rows<T, DP>(values, a.v.row, 0, (a.sinks < low ? a.sinks : low) - 1, a.D, g, bad, run.o, weight, on);
      add_rows<T, DP>(values, a.v.row, low, high, a.D, g, bad, run.o, weight, on);
    }
  }
  const float l = half_sum(run.l);
  const bool some = me < len && l != 0.f;
  T *const row = static_cast<T *>(a.y) + (((int64_t)b * a.N + me) * a.Hq + h) * a.D;
  store_rows<T, DP>(run.o, 1.f / l, some, row, me < a.N, a.D, g);
  if (a.stats && g == 0 && me < a.N) {
    const float stat = log2f(l) - run.off;
    a.stats[((int64_t)b * a.Hq + h) * a.N + me] = !some ? INFINITY : fabsf(stat) <= kMostStat ? stat : __builtin_nanf("");
  }
}

// ---------------------------------------------------------------------------------------------------------------
// step: the newest T points over the cache.  The columns of a wave's tile are (new point, query head of the group) pairs that share a
// key head; every wave of every part of the keys has tiles of its own (part + parts x n), keys straight to registers, values through a patch
// of LDS of its own for the transposing read; waves are joined in LDS, parts by a second kernel.
// ---------------------------------------------------------------------------------------------------------------
// LDS accesses of a wave happen in order; this keeps the compiler from exchanging them
__device__ __forceinline__ void wave_meets() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

struct StepArgs {
  Args a;
  int T, G, columns, column_tiles, parts;
  float *part_o, *part_ml;  // [b][hk][column tile][part][32][DP], [..][32][2]
};

template <class T, int DP, bool PLAIN, bool BIAS>
__global__ __launch_bounds__(256) void step_kernel(StepArgs s) {
  using O = Ops<T, DP>;
  constexpr int TILE = 32 * O::kStride, DB = DP / 32;
  const Args &a = s.a;
  extern __shared__ u32x4 lds_raw[];
  const int lane = threadIdx.x & 63, i = lane & 31, g = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  T *const patch = reinterpret_cast<T *>(lds_raw) + wave * TILE;
  float *const join = reinterpret_cast<float *>(lds_raw);              // after the last tile: [wave][column][DP]
  float *const biases = join + (4 * TILE * sizeof(T) > 4 * 32 * DP * 4 ? TILE * sizeof(T) : 32 * DP * 4);  // [bucket][G]
  uint8_t *const buckets = reinterpret_cast<uint8_t *>(biases + a.bias.buckets * s.G);                   // of distance 0 .. M
  __shared__ float most_of_wave[4][32], sum_of_wave[4][32], sum_of_all[32];
  int64_t work = blockIdx.x;
  const int part = (int)(work % s.parts);
  work /= s.parts;
  const int ct = (int)(work % s.column_tiles);
  work /= s.column_tiles;
  const int hk = (int)(work % a.Hk), b = (int)(work / a.Hk);
  const int len = length_of(a, b);
  const int col = ct * 32 + i, t = col / s.G, gq = col - t * s.G, me = len - s.T + t;
  const bool mine = col < s.columns && me >= 0;
  const int t0 = ct * 32 / s.G, t1 = (ct * 32 + 31 < s.columns ? ct * 32 + 31 : s.columns - 1) / s.G;
  const int first_q = len - s.T + t0 > 0 ? len - s.T + t0 : 0, last_q = len - s.T + t1;
  const typename O::Rows own = O::settle(O::template rows<PLAIN>(head_of<T>(a.q, b, hk * s.G + gq), a.q.row, t, s.T, mine, a.D, g));
  const T *const keys = head_of<T>(a.k, b, hk), *const values = head_of<T>(a.v, b, hk);
  const Span span = keys_of(a, mine ? len : 0, me);
  Raising<O, DP> run;
  run.start(mine);
  if constexpr (BIAS) {
    for (int u = threadIdx.x; u < a.bias.buckets * s.G; u += 256)
      biases[u] = bias_start(a.bias.table[(int64_t)(u / s.G) * a.Hq + hk * s.G + u % s.G], a.c);
    for (int u = threadIdx.x; u <= a.bias.distance; u += 256) buckets[u] = (uint8_t)bucket_of(a.bias, u);
    __syncthreads();
  }
  if (last_q >= 0) {
    const Tiles list(a, len, first_q, last_q, 32);
    const int by = 4 * s.parts;
    int n = part * 4 + wave;
    typename O::Rows next;
    Stage<O, T, DP, PLAIN, 32, 64> vs;
    auto fetch = [&](int at) {
      const int k0 = list[at] * 32;
      next = O::template rows<PLAIN>(keys, a.k.row, k0 + i, len, k0 + i < len, a.D, g);
      vs.load(a.v, values, k0, len, a.D, lane);
    };
    if (n < list.count) fetch(n);
    for (; n < list.count; n += by) {
      const int k0 = list[n] * 32;
      vs.store(patch, lane);
      wave_meets();  // lanes read what others wrote
      const typename O::Rows rows = next;
      if (n + by < list.count) fetch(n + by);
      f32x16 z;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        z[r] = 0.f;
        if constexpr (BIAS) {
          int d = me - (k0 + rowmap(r, g));
          d = d < 0 ? 0 : d < a.bias.distance ? d : a.bias.distance;
          z[r] = biases[buckets[d] * s.G + gq];
        }
      }
      z = O::scores(rows, own, z);
      hide(z, span, k0, g, -INFINITY);
      run.raise(z, a.c);
      const typename O::Weights w = run.weigh(z, a.c);
      O::outcome(patch, w, lane, run.o);
      wave_meets();
    }
    bool bad = not_finite(run.o);
    if (__builtin_expect(some_lane(bad), 0)) {
      bad = half_max(bad ? 1.f : 0.f) > 0.f;
      for (int d = 0; d < DB; ++d)
        for (int r = 0; r < 16; ++r) run.o[d][r] = bad ? 0.f : run.o[d][r];
      for (n = part * 4 + wave; n < list.count; n += by) {
        const int k0 = list[n] * 32, k1 = k0 + 31 < len ? k0 + 31 : len - 1;
        add_rows<T, DP>(values, a.v.row, k0, k1, a.D, g, bad, run.o, [&](int j, bool &seen) {
          seen = span.sees(j);
          float z = half_sum(O::dot(own, O::template rows<PLAIN>(keys, a.k.row, j, len, true, a.D, g)));
          if constexpr (BIAS) {
            const int d = me - j;
            z += biases[buckets[d < 0 ? 0 : d < a.bias.distance ? d : a.bias.distance] * s.G + gq];
          }
          return run.weight(z, a.c);
        });
      }
    }
  }
  // the four waves' results under one maximum
  const float l = half_sum(run.l);
  if (g == 0) most_of_wave[wave][i] = l != 0.f ? run.ref : -INFINITY, sum_of_wave[wave][i] = l;
  __syncthreads();  // and all patches have been read
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) top = fmaxf(top, most_of_wave[w][i]);
  const float ref = top == -INFINITY ? 0.f : top;
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w)
    if (sum_of_wave[w][i] != 0.f) total += sum_of_wave[w][i] * __builtin_amdgcn_exp2f((most_of_wave[w][i] - ref) * a.c);
  const float scale = l != 0.f ? __builtin_amdgcn_exp2f((run.ref - ref) * a.c) : 0.f;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) join[(wave * 32 + i) * DP + 32 * db + rowmap(r, g)] = l != 0.f ? run.o[db][r] * scale : 0.f;
  const int64_t slot = (((int64_t)b * a.Hk + hk) * s.column_tiles + ct) * s.parts + part;
  if (s.parts > 1 && wave == 0 && g == 0) {
    s.part_ml[(slot * 32 + i) * 2] = top;
    s.part_ml[(slot * 32 + i) * 2 + 1] = total;
  }
  if (wave == 0 && g == 0) sum_of_all[i] = total;
  __syncthreads();
  const int live = s.columns - ct * 32 < 32 ? s.columns - ct * 32 : 32;
  for (int u = threadIdx.x; u < live * DP; u += 256) {
    const int c = u / DP, d = u - c * DP;
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) o += join[(w * 32 + c) * DP + d];
    if (s.parts > 1) {
      s.part_o[(slot * 32 + c) * DP + d] = o;
    } else if (d < a.D) {
      const int column = ct * 32 + c, tt = column / s.G, hq = hk * s.G + column - tt * s.G;
      const float sum = sum_of_all[c];
      store_from_f32(static_cast<T *>(a.y) + (((int64_t)b * s.T + tt) * a.Hq + hq) * a.D + d, sum != 0.f ? o / sum : 0.f);
    }
  }
}

// joins the parts of the keys: a workgroup per (sequence, key head, column tile, four columns)
template <class T, int DP>
__global__ __launch_bounds__(256) void join_kernel(StepArgs s) {
  const Args &a = s.a;
  int64_t work = blockIdx.x;
  const int quad = (int)(work % 8);
  work /= 8;
  const int c = quad * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int ct = (int)(work % s.column_tiles), hk = (int)(work / s.column_tiles % a.Hk), b = (int)(work / s.column_tiles / a.Hk);
  const int column = ct * 32 + c;
  if (column >= s.columns) return;
  const int64_t slot = work * s.parts;
  // a part's maximum and sum a lane, so that nothing waits for the part before
  const auto most_and_sum = [&](int p) { return reinterpret_cast<const float2 *>(s.part_ml)[(slot + p) * 32 + c]; };
  float top = -INFINITY;
  for (int p = lane; p < s.parts; p += 64) top = fmaxf(top, most_and_sum(p).x);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float ref = top == -INFINITY ? 0.f : top;
  float total = 0.f, o[(DP + 63) / 64] = {};
  for (int first = 0; first < s.parts; first += 64) {
    float w = 0.f;
    if (first + lane < s.parts) {
      const float2 ml = most_and_sum(first + lane);
      if (ml.y != 0.f) w = __builtin_amdgcn_exp2f((ml.x - ref) * a.c), total += ml.y * w;
    }
    const int count = s.parts - first < 64 ? s.parts - first : 64;
#pragma unroll 8
    for (int p = 0; p < count; ++p) {  // parts without a sum hold zeros
      const float by = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), p));
#pragma unroll
      for (int k = 0; k < (DP + 63) / 64; ++k)
        if (lane + 64 * k < DP) o[k] += s.part_o[((slot + first + p) * 32 + c) * DP + lane + 64 * k] * by;
    }
  }
  total = wave_sum(total);
  const int t = column / s.G, hq = hk * s.G + column - t * s.G;
#pragma unroll
  for (int k = 0; k < (DP + 63) / 64; ++k)
    if (lane + 64 * k < a.D)
      store_from_f32(static_cast<T *>(a.y) + (((int64_t)b * s.T + t) * a.Hq + hq) * a.D + lane + 64 * k, total != 0.f ? o[k] / total : 0.f);
}

// ---------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------
// Whether d >= E (M / E)^(b / L), that is d^L E^b >= M^b E^L: by logarithms where they tell, else by the whole numbers themselves
// (up to 2 048^128 128^128: 2 304 bits)
static bool reached(int64_t d, int64_t E, int64_t M, int L, int b) {
  const double lhs = L * log((double)d) + b * log((double)E), rhs = b * log((double)M) + L * log((double)E);
  if (fabs(lhs - rhs) > 1e-9 * (fabs(lhs) + 1)) return lhs > rhs;
  constexpr int WORDS = 80;
  uint32_t x[WORDS] = {1}, y[WORDS] = {1};
  auto times = [](uint32_t *v, int64_t factor, int count) {
    for (; count > 0; --count) {
      uint64_t carry = 0;
      for (int w = 0; w < WORDS; ++w) {
        const uint64_t t = (uint64_t)v[w] * (uint64_t)factor + carry;
        v[w] = (uint32_t)t;
        carry = t >> 32;
      }
    }
  };
  times(x, d, L), times(x, E, b), times(y, M, b), times(y, E, L);
  for (int w = WORDS - 1; w >= 0; --w)
    if (x[w] != y[w]) return x[w] > y[w];
  return true;
}

static BiasArgs make_bias(const pa_window_params &p) {
  static thread_local BiasArgs last = {};  // the borders depend on the three numbers alone
  static thread_local int64_t last_buckets = 0;
  const bool both = p.right != 0;
  if (p.buckets == 0) return BiasArgs{};
  if (last_buckets != p.buckets || last.distance != (int)p.distance || last.both != both) {
    BiasArgs b = {};
    b.buckets = (int)p.buckets, b.distance = (int)p.distance, b.both = both;
    b.side = both ? b.buckets / 2 : b.buckets;
    b.exact = b.side / 2;
    const int L = b.side - b.exact;
    for (int k = 1; k < L; ++k) {
      int d = (int)(b.exact * pow((double)b.distance / b.exact, (double)k / L)) - 1;
      if (d < b.exact) d = b.exact;
      while (!reached(d, b.exact, b.distance, L, k)) ++d;
      b.borders[k - 1] = d;
    }
    last = b, last_buckets = p.buckets;
  }
  BiasArgs b = last;
  b.table = p.bias;
  return b;
}

Args make_args(const pa_window_params &p) {
  Args a = {};
  a.N = (int)p.N, a.Hq = (int)p.Hq, a.Hk = (int)p.Hk, a.D = (int)p.D, a.B = (int)p.B;
  a.left = p.left < 0 || p.left >= p.N ? kNoBound : (int)p.left;
  a.right = p.right < 0 || p.right >= p.N ? kNoBound : (int)p.right;
  a.sinks = a.left == kNoBound ? 0 : (int)p.sinks;  // all that lies behind is seen without them
  a.sink_rows = (a.sinks + 31) / 32 * 32;
  a.scale = (float)p.scale, a.c = (float)(p.scale * 1.4426950408889634);
  a.lengths = p.lengths;
  a.bias = make_bias(p);
  a.blocks = (int)((p.N + 127) / 128);
  return a;
}

template <class T, int DP, bool PLAIN, bool BIAS>
static int launch_forward(const Args &a, hipStream_t st) {
  const size_t lds = 4 * (size_t)tile_rows<T, DP>() * WindowOps<T, DP>::kStride * sizeof(T) + (BIAS ? table_size(a.bias) * sizeof(float) : 0);
  auto kernel = forward_kernel<T, DP, PLAIN, BIAS>;
  if (int rc = allow_dynamic_lds(kernel, lds)) return rc;
  kernel<<<(unsigned)((int64_t)a.blocks * a.Hq * a.B), 256, lds, st>>>(a);
  return launch_status();
}
template <class T>
static int forward_of(const Args &a, hipStream_t st) {
  return by_width(a.D, a.q.plain && a.k.plain && a.v.plain, [&](auto dp, auto plain) {
    constexpr int DP = decltype(dp)::value;
    constexpr bool PLAIN = decltype(plain)::value;
    return a.bias.buckets ? launch_forward<T, DP, PLAIN, true>(a, st) : launch_forward<T, DP, PLAIN, false>(a, st);
  });
}

int forward(int dtype, const pa_window_params &p, const pa_heads &q, const pa_heads &k, const pa_heads &v, void *y, float *stats, hipStream_t st) {
  const int64_t elem = dtype == PA_F32 ? 4 : 2;
  Args a = make_args(p);
  a.q = make_view(q, p.D, elem), a.k = make_view(k, p.D, elem), a.v = make_view(v, p.D, elem);
  a.y = y, a.stats = stats;
  return dtype == PA_F32 ? forward_of<float>(a, st) : forward_of<bf16>(a, st);
}

struct StepPlan {
  int64_t column_tiles, parts, slots;
  int DP;
};
// Parts of the keys: as many as fill the chip twice, but a tile of keys at least for each of a workgroup's waves
static StepPlan step_plan(const pa_window_params &p, int64_t T, int num_cu) {
  StepPlan s;
  const int64_t G = p.Hq / p.Hk;
  s.column_tiles = (T * G + 31) / 32;
  int64_t seen = p.N;
  if (p.left >= 0 && p.left + T + p.sinks < seen) seen = p.left + T + p.sinks;
  const int64_t tiles = (seen + 31) / 32, base = p.B * p.Hk * s.column_tiles;
  int64_t parts = (2 * (int64_t)num_cu + base - 1) / base;
  if (parts > (tiles + 3) / 4) parts = (tiles + 3) / 4;
  s.parts = parts < 1 ? 1 : parts;
  s.slots = base * s.parts;
  s.DP = p.D <= 32 ? 32 : p.D <= 64 ? 64 : 128;
  return s;
}
int64_t step_workspace_bytes(int, const pa_window_params &p, int64_t T, int num_cu) {
  const StepPlan s = step_plan(p, T, num_cu);
  return s.parts > 1 ? s.slots * 32 * (s.DP + 2) * (int64_t)sizeof(float) : 0;
}

template <class T, int DP, bool PLAIN>
static int launch_step(const StepArgs &s, hipStream_t st) {
  const size_t patches = 4 * 32 * Ops<T, DP>::kStride * sizeof(T), joins = 4 * 32 * DP * sizeof(float);
  size_t lds = patches > joins ? patches : joins;
  if (s.a.bias.buckets) lds += (size_t)s.a.bias.buckets * s.G * sizeof(float) + (s.a.bias.distance + 4) / 4 * 4;
  const int64_t base = (int64_t)s.a.B * s.a.Hk * s.column_tiles;
  int rc = 0;
  if (s.a.bias.buckets) {
    auto kernel = step_kernel<T, DP, PLAIN, true>;
    if ((rc = allow_dynamic_lds(kernel, lds))) return rc;
    kernel<<<(unsigned)(base * s.parts), 256, lds, st>>>(s);
  } else {
    auto kernel = step_kernel<T, DP, PLAIN, false>;
    if ((rc = allow_dynamic_lds(kernel, lds))) return rc;
    kernel<<<(unsigned)(base * s.parts), 256, lds, st>>>(s);
  }
  if ((rc = launch_status()) || s.parts == 1) return rc;
  join_kernel<T, DP><<<(unsigned)(base * 8), 256, 0, st>>>(s);
  return launch_status();
}

int step(int dtype, const pa_window_params &p, int64_t T, const pa_heads &q, const pa_heads &k, const pa_heads &v, void *y, void *workspace,
         int num_cu, hipStream_t st) {
  const StepPlan plan = step_plan(p, T, num_cu);
  StepArgs s = {};
  s.a = make_args(p);
  const int64_t elem = dtype == PA_F32 ? 4 : 2;
  s.a.q = make_view(q, p.D, elem), s.a.k = make_view(k, p.D, elem), s.a.v = make_view(v, p.D, elem);
  const bool plain = s.a.q.plain && s.a.k.plain && s.a.v.plain;
  s.a.y = y;
  s.T = (int)T, s.G = (int)(p.Hq / p.Hk), s.columns = (int)(T * (p.Hq / p.Hk));
  s.column_tiles = (int)plan.column_tiles, s.parts = (int)plan.parts;
  s.part_o = static_cast<float *>(workspace);
  s.part_ml = s.part_o + plan.slots * 32 * plan.DP;
  if (dtype == PA_F32) return by_width(s.a.D, plain, [&](auto dp, auto is_plain) { return launch_step<float, decltype(dp)::value, decltype(is_plain)::value>(s, st); });
  return by_width(s.a.D, plain, [&](auto dp, auto is_plain) { return launch_step<bf16, decltype(dp)::value, decltype(is_plain)::value>(s, st); });
}

}  // namespace window
}  // namespace pa
