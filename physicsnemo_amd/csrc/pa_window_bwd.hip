// Gradients of attention over a window: with p_ij formed again from the kept log2 of the softmax's denominators,
//   delta_i = sum_j p_ij dp_ij = dy_i . y_i,  dp_ij = dy_i . v_j,  ds_ij = p_ij (dp_ij - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij dy_i,  d bias[b] = sum over bucket b of ds_ij
// in two passes, so that every sum has an owner and a fixed order: queries_kernel owns 32 queries a wave and goes over the keys they see
// (delta, dq, d bias), keys_kernel owns 32 keys a wave and goes over the queries that see them and over the query heads that share
// them (dk, dv).
//
// What it takes: 65 536 x 8 x 32 bf16, 257 keys a query and 8 sinks: queries 97 us, keys 100 (0.27 GB in all: 49; the eight products' 71 GFLOP: 52;
// vector instructions and registers, three and four waves a SIMD, bound them: 60 and 50 % of the issue slots, matrix pipes 21); 4 x 7 225 x 8 x 16 float32,
// 171 keys: 91 and 108; with the bias gradient, 3 x 5 001 x 8 over 4 x 64, 512 keys: 121 to 127 (six products a tile, not four) and 93.
//
// delta from y carries y's rounding (2^-9 of |dy| |v| for bf16), and with a delta that is off by e a query's score gradients sum up to e, not to zero: dq is
// off by e times the mean of its keys, which may be many times what is left of dq where the keys and values have means of their own.  So the sum of
// ds, as it is multiplied, and the mean key sum_j p_ij k_j are summed along; what the one leaves of the other is taken off dq, and the sum before its rounding is
// added to delta for the second kernel.  Keys and values of mean 8 (6 000 points, 4 001 keys of 32 channels): dq in bf16 3.7 off, now 0.0024, dk 0.0145, now 0.0023; in float32 1.2e-3, now
// 4.5e-6, a plain form 1.4e-4.  It costs an eighth product beside seven (65 536 x 8 x 32: queries 82 -> 97 us; float32
// 4 x 7 225 x 8 x 16: 78 -> 91; 20 000 x 4 x 64, 401 keys: 131 -> 161).
// The bias gradient is float32, and sums single ds: where it is wanted, the first kernel sums p dp before it goes over the keys again.
#include "pa_window.h"

namespace pa {
namespace window {

// Sums of a tile's score gradients by offset key - query, added to a wave's table of them (t: the offset of the tile's first key from the
// wave's first query).  Eight keys at a time go to LDS as [diagonal][key], where 39 lanes add up a diagonal each: what a diagonal lacks at its ends is
// never written and stays zero.  (LDS atomics, one a score, took 96 cycles an instruction: 3 000 a tile, and 150 us of the whole at 11 253 x 8 x 64.)
constexpr int kDiagonals = 39, kDiagonal = 12;
__device__ __forceinline__ void add_diagonals(const f32x16 &ds, float *buffer, float *t, int lane) {
  const int i = lane & 31, g = lane >> 5;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float *const put = buffer + (4 * g - i + 31) * kDiagonal + 4 * g;
#pragma unroll
    for (int j = 0; j < 4; ++j) put[j * kDiagonal + j] = ds[4 * q + j];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // LDS accesses of a wave happen in order; this keeps the compiler from exchanging them
    __builtin_amdgcn_wave_barrier();
    if (lane < kDiagonals) {
      const f32x4 *const d = reinterpret_cast<const f32x4 *>(buffer + lane * kDiagonal);
      const f32x4 a = d[0], b = d[1];
      t[8 * q + lane - 31] += ((a[0] + a[1]) + (a[2] + a[3])) + ((b[0] + b[1]) + (b[2] + b[3]));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// Waves a SIMD.  queries_kernel: bf16 rows to 32 run three by themselves (of odd pieces for ten spilled registers), to 64 two; the thirds of float32 rows take
// 200 registers at widths to 32 (a third wave for 35 spilled ones) and 320 at 64 (a second wave).  keys_kernel: bf16 rows to 32 run four by themselves
// without biases and three with them; float32 rows need 184 at widths to 32 and 271 at 64 (a third wave took 4 x 7 225 x 8 x 16 from 109 to 101 us, a second one
// 20 000 x 4 x 64, 401 keys, from 200 to 175; with the differences behind the products 108 and 184).  Rows of 128 run one: 350 to 450 registers.
template <int DP>
constexpr int kWavesOfQueries = DP == 128 ? 1 : DP == 64 ? 2 : 3;
template <class T, int DP>
constexpr int kWavesOfKeys = sizeof(T) == 2 || DP == 128 ? 1 : DP == 64 ? 2 : 3;

// Products that start from -delta, or from a denominator, are rounded differently, always to the same side, and sums over long windows keep that: with queries
// of mean 8 (6 000 points, 4 001 keys, 128 channels) dk and dv of float32 rows were 6.5e-6 off, 2.2e-6 to 2.7e-6 with the differences taken behind the products,
// where a plain float32 form has 1.7e-6 and 3.3e-6; the far buckets' gradients 1.4e-5, now 1.4e-6 (3 x 5 001 x 8 x 64).  It costs 4 us of the 101 of
// the key pass at 4 x 7 225 x 8 x 16.  bf16 rows start from them: their p and ds are rounded to 2^-9.
template <class T>
constexpr bool kDifferencesAfter = sizeof(T) == 4;

template <class T, int DP, bool PLAIN, bool BIAS, bool DBIAS>
__global__ __launch_bounds__(256, kWavesOfQueries<DP>) void queries_kernel(Args a) {
  constexpr int KT = tile_rows<T, DP>(), SUB = KT / 32, TILE = KT * WindowOps<T, DP>::kStride;
  extern __shared__ u32x4 lds_raw[];
  T *const tiles = reinterpret_cast<T *>(lds_raw);  // [buffer][keys, values][KT][stride]
  float *const table = reinterpret_cast<float *>(tiles + 4 * TILE);
  const int entries = BIAS ? table_size(a.bias) : 0;
  float *const sums = table + entries;  // DBIAS: [wave][offset]
  const uint32_t work = own_work(), at_head = work / (uint32_t)a.blocks;
  const int block = (int)(work - at_head * (uint32_t)a.blocks), b = (int)(at_head / (uint32_t)a.Hq), h = (int)(at_head - (uint32_t)b * (uint32_t)a.Hq);
  const int lane = threadIdx.x & 63, i = lane & 31, g = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int len = length_of(a, b), q0 = block * 128, qw = q0 + 32 * wave, me = qw + i;
  using O = WindowOps<T, DP>;
  constexpr bool kAfter = DBIAS || kDifferencesAfter<T>;
  f32x16 dq[DP / 32];
  zero(dq);
  if constexpr (BIAS) fill_bias_table(a, h, table);
  float *const mine = sums + wave * entries;
  // 16-byte boundaries: the tables' sizes are no multiples of four
  float *const buffer = reinterpret_cast<float *>((reinterpret_cast<uintptr_t>(sums + 4 * entries) + 15) / 16 * 16) + wave * kDiagonals * kDiagonal;
  if constexpr (DBIAS) {
    for (int u = lane; u < entries; u += 64) mine[u] = 0.f;
    for (int u = lane; u < kDiagonals * kDiagonal; u += 64) buffer[u] = 0.f;
  }
  float behind = 0.f, ahead = 0.f;
  if (q0 < len) {
    const typename O::Raw raw = O::template rows<PLAIN>(head_of<T>(a.q, b, h), a.q.row, me, len, me < len, a.D, g);
    const typename O::Raw raw_dy = O::template rows<PLAIN>(head_of<T>(a.dy, b, h), a.dy.row, me, len, me < len, a.D, g);
    const typename O::Rows own = O::settle(raw), dy = O::settle(raw_dy);
    const int64_t at = ((int64_t)b * a.Hq + h) * a.N + me;
    float stat = me < len ? a.saved_stats[at] : INFINITY;
    float delta = 0.f;
    if constexpr (!DBIAS) {
      const typename O::Raw y =
          O::template rows<PLAIN>(static_cast<const T *>(a.saved_y) + ((int64_t)b * a.N * a.Hq + h) * a.D, (int64_t)a.Hq * a.D, me, len, me < len, a.D, g);
      delta = half_sum(O::dot(dy, y));
    }
    const Sights sights = sights_of_queries(a, len, qw);
    const int hk = h / (a.Hq / a.Hk);
    const T *const keys = head_of<T>(a.k, b, hk), *const values = head_of<T>(a.v, b, hk);
    const Tiles list(a, len, q0, q0 + 127 < len ? q0 + 127 : len - 1, KT);
    Stage<O, T, DP, PLAIN, KT, 256> ks, vs;
    // one pass over the keys: f(sub-tile's keys, values, p, dp, first key)
    auto pass = [&](float from, auto &&f) {  // from: what dp starts from, in the last pass less delta
      __syncthreads();
      if (list.count > 0) {
        ks.load(a.k, keys, list[0] * KT, len, a.D, threadIdx.x);
        vs.load(a.v, values, list[0] * KT, len, a.D, threadIdx.x);
        ks.store(tiles, threadIdx.x);
        vs.store(tiles + TILE, threadIdx.x);
      }
      __syncthreads();
      for (int n = 0; n < list.count; ++n) {
        const T *const kt = tiles + (n & 1) * 2 * TILE, *const vt = kt + TILE;
        T *const next = tiles + ((n + 1) & 1) * 2 * TILE;
        if (n + 1 < list.count) {
          ks.load(a.k, keys, list[n + 1] * KT, len, a.D, threadIdx.x);
          vs.load(a.v, values, list[n + 1] * KT, len, a.D, threadIdx.x);
        }
#pragma unroll 1
        for (int s = 0; s < SUB; ++s) {
          const int k0 = list[n] * KT + 32 * s;
          if (sights.none(k0)) continue;
          const T *const krows = kt + 32 * s * O::kStride;
          f32x16 z, dp;
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[r] = from;
          Reach reach = kNear;
          if constexpr (BIAS) {
            reach = reach_of(a.bias, k0 - qw - 31, k0 + 31 - qw);
            if (reach == kNear) {
              const float *t = table + (k0 + 4 * g - me + table_low(a.bias));
#pragma unroll
              for (int r = 0; r < 16; ++r) z[r] = t[8 * (r >> 2) + (r & 3)];
            } else {
              const float far = reach == kFarBehind ? table[0] : table[entries - 1];
#pragma unroll
              for (int r = 0; r < 16; ++r) z[r] = far;
            }
          } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) z[r] = 0.f;
          }
          z = O::scores(krows, own, i, g, z, a.D);
          dp = O::scores(vt + 32 * s * O::kStride, dy, i, g, dp, a.D);
          if (!sights.all(k0)) {
            const Span span = keys_of(a, len, me);
            hide(z, span, k0, g, -INFINITY);
            if constexpr (DBIAS) hide(dp, span, k0, g, 0.f);  // the bias sums take every element
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) z[r] = __builtin_amdgcn_exp2f(fmaf(z[r], a.c, -stat));
          f(krows, z, dp, k0, reach);
        }
        if (n + 1 < list.count) {
          ks.store(next, threadIdx.x);
          vs.store(next + TILE, threadIdx.x);
        }
        __syncthreads();
      }
    };
    if constexpr (DBIAS) {
      // the denominator, too: for bf16 the forward pass summed the weights as it multiplied them, rounded
      float part = 0.f, total = 0.f;
      pass(0.f, [&](const T *, f32x16 &p, f32x16 &dp, int, Reach) {
        float sum = 0.f, weights = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) sum = fmaf(p[r], dp[r], sum), weights += p[r];
        part += sum, total += weights;
      });
      total = half_sum(total);
      if (total > 0.f) {
        delta = half_sum(part) / total;
        stat += log2f(total);
      }
    }
    float exact = 0.f, rest = 0.f;  // the sum of ds, for delta; the sum of ds as it is multiplied; `mean`: sum p k, good to 2^-8, which is enough beside a rest that is small itself
    f32x16 mean[DP / 32];
    zero(mean);
    pass(kAfter ? 0.f : -delta, [&](const T *krows, f32x16 &p, f32x16 &dp, int k0, Reach reach) {
      O::outcome_coarse(krows, p, lane, mean);
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] *= kAfter ? dp[r] - delta : dp[r];
      if constexpr (DBIAS)
        if (!sights.all(k0)) hide(p, keys_of(a, len, me), k0, g, 0.f);  // where delta is NaN
      if constexpr (DBIAS) {
        if (reach == kNear) {
          add_diagonals(p, buffer, mine + (k0 - qw + table_low(a.bias)), lane);
        } else {
          float sum = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) sum += p[r];
          if (reach == kFarBehind) behind += sum;
          else ahead += sum;
        }
      }
      const typename O::Weights ds = O::pack(p);
      rest += O::sum(ds, p);
      if constexpr (sizeof(T) == 2) exact += sum_of(p);
      O::outcome(krows, ds, lane, dq);
    });
    rest = half_sum(rest);
    exact = sizeof(T) == 2 ? half_sum(exact) : rest;
    bool bad = not_finite(dq) || not_finite(mean) || rest * 0.f != 0.f;
    if (__builtin_expect(some_lane(bad), 0)) {
      bad = half_max(bad ? 1.f : 0.f) > 0.f;
      const Span span = keys_of(a, len, me);
      for (int d = 0; d < DP / 32; ++d)
        for (int r = 0; r < 16; ++r) dq[d][r] = bad ? 0.f : dq[d][r];
      auto weight = [&](int j, bool &seen) {
        seen = span.sees(j);
        float z = half_sum(O::dot(own, O::template rows<PLAIN>(keys, a.k.row, j, len, true, a.D, g)));
        const float by = half_sum(O::dot(dy, O::template rows<PLAIN>(values, a.v.row, j, len, true, a.D, g)));
        if constexpr (BIAS) z += bias_at(a.bias, table, j - me);
        return __builtin_amdgcn_exp2f(fmaf(z, a.c, -stat)) * (by - delta);
      };
      const int low = qw - a.left > 0 ? qw - a.left : 0, high = qw + 31 + a.right < len - 1 ? qw + 31 + a.right : len - 1;
      float own_rest = 0.f;  // delta from what is seen alone
      for (int j = a.sinks > 0 ? 0 : low; j <= high && some_lane(bad && own_rest == own_rest); j = j + 1 == a.sinks && low > j ? low : j + 1) {
        bool seen;
        const float w = weight(j, seen);
        own_rest += seen ? w : 0.f;
      }
      if (bad) delta += own_rest, exact = 0.f;
      add_rows<T, DP>(keys, a.k.row, 0, (a.sinks < low ? a.sinks : low) - 1, a.D, g, bad, dq, weight);
      add_rows<T, DP>(keys, a.k.row, low, high, a.D, g, bad, dq, weight);
    }
    if (g == 0 && me < len) a.delta[at] = stat == stat ? delta + exact : 0.f;  // 0: the weights are NaN, and where there are none no NaN of delta's meets them
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[d][r] = bad ? dq[d][r] : fmaf(-rest, mean[d][r], dq[d][r]);
  }
  T *const row = static_cast<T *>(a.dq) + (((int64_t)b * a.N + me) * a.Hq + h) * a.D;
  store_rows<T, DP>(dq, a.scale, me < len, row, me < a.N, a.D, g);
  if constexpr (DBIAS) {
    // this workgroup's share of every bucket: waves added up by offset, then offsets by bucket, one bucket a wave at a time
    __shared__ float far[2][4];
    behind = wave_sum(behind), ahead = wave_sum(ahead);
    if (lane == 0) far[0][wave] = behind, far[1][wave] = ahead;
    __syncthreads();
    for (int u = threadIdx.x; u < entries; u += 256) sums[u] = (sums[u] + sums[entries + u]) + (sums[2 * entries + u] + sums[3 * entries + u]);
    __syncthreads();
    float *const out = a.bias_parts + (((int64_t)b * a.blocks + block) * a.Hq + h) * a.bias.buckets;
    const int low = table_low(a.bias), n = a.bias.side, E = a.bias.exact;
    for (int bucket = wave; bucket < a.bias.buckets; bucket += 4) {
      const bool forward = bucket >= n;
      const int k = forward ? bucket - n : bucket;
      const int from = k <= E ? k : a.bias.borders[k - E - 1];
      const int past = k + 1 <= E ? k + 1 : k + 1 < n ? a.bias.borders[k - E] : a.bias.distance + kPad + 1;
      float sum = 0.f;
      for (int d = from + lane; d < past; d += 64) {
        if (forward) sum += d > 0 ? sums[low + d] : 0.f;
        else sum += sums[low - d];
      }
      sum = wave_sum(sum);
      if (k == n - 1) sum += forward ? (far[1][0] + far[1][1]) + (far[1][2] + far[1][3]) : (far[0][0] + far[0][1]) + (far[0][2] + far[0][3]);
      if (lane == 0) out[bucket] = sum;
    }
  }
}

// d bias: a workgroup per head and bucket, the query blocks' shares in 256 parts that are joined in order
__global__ __launch_bounds__(256) void bias_sums_kernel(const float *parts, int64_t rows, int Hq, int buckets, float *d_bias) {
  __shared__ float part[256];
  const int h = blockIdx.x / buckets, bucket = blockIdx.x % buckets;
  float sum = 0.f;
  for (int64_t r = threadIdx.x; r < rows; r += 256) sum += parts[(r * Hq + h) * buckets + bucket];
  part[threadIdx.x] = sum;
  for (int n = 128; n > 0; n >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < n) part[threadIdx.x] += part[threadIdx.x + n];
  }
  if (threadIdx.x == 0) d_bias[(int64_t)bucket * Hq + h] = part[0];
}

// ---------------------------------------------------------------------------------------------------------------
// keys_kernel: tiles of keys with sinks are seen by all queries behind them, which are cut into sink_chunks parts, each a workgroup of its own
// for those tiles alone, whose sums are joined by sink_sums_kernel.
// ---------------------------------------------------------------------------------------------------------------
template <class T, int DP, bool PLAIN, bool BIAS>
__global__ __launch_bounds__(256, (kWavesOfKeys<T, DP>)) void keys_kernel(Args a) {
  constexpr int QT = tile_rows<T, DP>(), SUB = QT / 32, TILE = QT * WindowOps<T, DP>::kStride;
  extern __shared__ u32x4 lds_raw[];
  T *const tiles = reinterpret_cast<T *>(lds_raw);  // [buffer][queries, gradients][QT][stride]
  float *const stats = reinterpret_cast<float *>(tiles + 4 * TILE);  // [buffer][log2 denominators, deltas][QT]
  float *const table = stats + 4 * QT;
  const int lane = threadIdx.x & 63, i = lane & 31, g = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.Hq / a.Hk, chunks = a.sink_chunks, per_head = a.blocks + chunks;
  const uint32_t work = own_work(), at_head = work / (uint32_t)per_head;
  int block = (int)(work - at_head * (uint32_t)per_head), chunk = -1;
  const int b = (int)(at_head / (uint32_t)a.Hk), hk = (int)(at_head - (uint32_t)b * (uint32_t)a.Hk);
  if (chunks > 0) {
    if (block < chunks) chunk = block, block = 0;
    else block -= chunks;
  }
  const int len = length_of(a, b), k0 = block * 128, kw = k0 + 32 * wave, me = kw + i;
  using O = WindowOps<T, DP>;
  constexpr bool kAfter = kDifferencesAfter<T>;
  f32x16 dk[DP / 32], dv[DP / 32];
  zero(dk);
  zero(dv);
  if (k0 < len) {
    const typename O::Raw raw_key = O::template rows<PLAIN>(head_of<T>(a.k, b, hk), a.k.row, me, len, me < len, a.D, g);
    const typename O::Raw raw_value = O::template rows<PLAIN>(head_of<T>(a.v, b, hk), a.v.row, me, len, me < len, a.D, g);
    const typename O::Rows key = O::settle(raw_key), value = O::settle(raw_value);
    Sights sights = sights_of_keys(a, len, kw);
    if (chunks > 0 && (kw < a.sink_rows) != (chunk >= 0)) sights.high = -1;  // the other workgroups' rows
    // queries that see a key of the block: i >= j - right, and i <= j + left or j a sink
    int first = k0 - a.right > 0 ? k0 - a.right : 0, last = k0 + 127 + a.left;
    if (chunk >= 0 || last > len - 1) last = len - 1;
    int t0 = first / QT, t1 = last / QT;  // tiles of queries
    if (chunk >= 0) {
      const int tiles_of_all = (a.N + QT - 1) / QT, each = (tiles_of_all + chunks - 1) / chunks;
      t0 = t0 > chunk * each ? t0 : chunk * each;
      t1 = t1 < chunk * each + each - 1 ? t1 : chunk * each + each - 1;
    }
    const int tiles_of_head = t1 - t0 + 1, count = tiles_of_head > 0 ? tiles_of_head * G : 0;
    Stage<O, T, DP, PLAIN, QT, 256> qs, gs;
    float stat = 0.f;
    // the tile in work and the one to fetch, counted on: a division an iteration by each of two was half of all scalar work
    int h = hk * G, tile = t0, next_h = hk * G, next_tile = t0;
    auto on = [&](int &head, int &at) {
      if (++at > t1) at = t0, ++head;
    };
    int from = 0;
    auto fetch = [&]() {
      const int h = next_h;
      from = next_tile * QT;
      on(next_h, next_tile);
      qs.load(a.q, head_of<T>(a.q, b, h), from, len, a.D, threadIdx.x);
      gs.load(a.dy, head_of<T>(a.dy, b, h), from, len, a.D, threadIdx.x);
      if (threadIdx.x < 2 * QT) {
        const int row = from + threadIdx.x % QT;
        const float *src = (int)threadIdx.x < QT ? a.saved_stats : a.delta;
        stat = src[((int64_t)b * a.Hq + h) * a.N + (row < len ? row : len - 1)];
      }
    };
    auto put = [&](int n) {
      T *const to = tiles + (n & 1) * 2 * TILE;
      qs.store(to, threadIdx.x);
      gs.store(to + TILE, threadIdx.x);
      // as the products start from them: less the denominator in units of z, less delta; rows that are not there weigh nothing.  Here and not in
      // fetch, where it would wait for the loads: 110 -> 99 us at 65 536 x 8 x 32, 257 keys a query.
      if (threadIdx.x < 2 * QT)
        stats[(n & 1) * 2 * QT + threadIdx.x] = (int)threadIdx.x >= QT ? -stat : from + (int)threadIdx.x < len ? (kAfter ? -stat : -stat / a.c) : -INFINITY;
    };
    if (count > 0) fetch(), put(0);
    int filled = -1;
    for (int n = 0; n < count; ++n, on(h, tile)) {
      if (BIAS && h != filled) {
        __syncthreads();  // the head before is done with
        fill_bias_table(a, h, table);
        filled = h;
      }
      __syncthreads();
      const T *const qt = tiles + (n & 1) * 2 * TILE, *const gt = qt + TILE;
      const float *const lse = stats + (n & 1) * 2 * QT, *const delta = lse + QT;
      if (n + 1 < count) fetch();
#pragma unroll 1
      for (int s = 0; s < SUB; ++s) {
        const int q0 = tile * QT + 32 * s;
        if (sights.none(q0)) continue;
        const T *const qrows = qt + 32 * s * O::kStride, *const grows = gt + 32 * s * O::kStride;
        f32x16 z, dp;
        const auto rows_of = [&](const float *p, int q) { return *reinterpret_cast<const f32x4 *>(p + 32 * s + 8 * q + 4 * g); };
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (kAfter) {
#pragma unroll
            for (int j = 0; j < 4; ++j) z[4 * q + j] = dp[4 * q + j] = 0.f;
          } else {
            const f32x4 l4 = rows_of(lse, q), d4 = rows_of(delta, q);
#pragma unroll
            for (int j = 0; j < 4; ++j) z[4 * q + j] = l4[j], dp[4 * q + j] = d4[j];
          }
        }
        if constexpr (BIAS) {
          const Reach reach = reach_of(a.bias, kw - q0 - 31, kw + 31 - q0);
          if (reach == kNear) {
            const float *t = table + (me - q0 - 4 * g + table_low(a.bias));
#pragma unroll
            for (int r = 0; r < 16; ++r) z[r] += t[-(8 * (r >> 2) + (r & 3))];
          } else {
            const float far = reach == kFarBehind ? table[0] : table[table_size(a.bias) - 1];
#pragma unroll
            for (int r = 0; r < 16; ++r) z[r] += far;
          }
        }
        z = O::scores(qrows, key, i, g, z, a.D);
        dp = O::scores(grows, value, i, g, dp, a.D);
        if constexpr (kAfter) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 l4 = rows_of(lse, q), d4 = rows_of(delta, q);
#pragma unroll
            for (int j = 0; j < 4; ++j) z[4 * q + j] = fmaf(z[4 * q + j], a.c, l4[j]), dp[4 * q + j] += d4[j];
          }
        }
        if (!sights.all(q0)) hide(z, queries_of(a, len, me), q0, g, -INFINITY);  // behind what may be NaN
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] = __builtin_amdgcn_exp2f(kAfter ? z[r] : z[r] * a.c);
        O::outcome(grows, O::pack(z), lane, dv);
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] *= dp[r];
        O::outcome(qrows, O::pack(z), lane, dk);
      }
      if (n + 1 < count) put(n + 1);
    }
    bool bad = not_finite(dk) || not_finite(dv);
    if (__builtin_expect(some_lane(bad), 0)) {
      bad = half_max(bad ? 1.f : 0.f) > 0.f;
      const Span span = queries_of(a, len, me);
      for (int d = 0; d < DP / 32; ++d)
        for (int r = 0; r < 16; ++r) dk[d][r] = bad ? 0.f : dk[d][r], dv[d][r] = bad ? 0.f : dv[d][r];
      const int q_low = t0 * QT > kw - a.right ? t0 * QT : kw - a.right;
      int q_high = t1 * QT + QT - 1 < len - 1 ? t1 * QT + QT - 1 : len - 1;
      if (kw >= a.sinks && kw + 31 + a.left < q_high) q_high = kw + 31 + a.left;
      for (h = hk * G; h < hk * G + G; ++h) {
        const T *const queries = head_of<T>(a.q, b, h), *const grads = head_of<T>(a.dy, b, h);
        const int64_t first_stat = ((int64_t)b * a.Hq + h) * a.N;
        auto p_of = [&](int n, bool &seen) {
          seen = span.sees(n);
          float z = half_sum(O::dot(key, O::template rows<PLAIN>(queries, a.q.row, n, len, true, a.D, g)));
          if constexpr (BIAS) z += bias_start(a.bias.table[(int64_t)bucket_of_offset(a.bias, me - n) * a.Hq + h], a.c);
          return __builtin_amdgcn_exp2f(fmaf(z, a.c, -a.saved_stats[first_stat + n]));
        };
        add_rows<T, DP>(grads, a.dy.row, q_low, q_high, a.D, g, bad, dv, p_of);
        add_rows<T, DP>(queries, a.q.row, q_low, q_high, a.D, g, bad, dk, [&](int n, bool &seen) {
          const float p = p_of(n, seen);
          return p * (half_sum(O::dot(value, O::template rows<PLAIN>(grads, a.dy.row, n, len, true, a.D, g))) - a.delta[first_stat + n]);
        });
      }
    }
  }
  if (chunk < 0) {
    if (kw < a.sink_rows) return;
    const int64_t at = (((int64_t)b * a.N + me) * a.Hk + hk) * a.D;
    store_rows<T, DP>(dk, a.scale, me < len, static_cast<T *>(a.dk) + at, me < a.N, a.D, g);
    store_rows<T, DP>(dv, 1.f, me < len, static_cast<T *>(a.dv) + at, me < a.N, a.D, g);
    return;
  }
  // [b][hk][chunk][dk, dv][sink_rows][D]
  if (kw >= a.sink_rows) return;
  float *const part = a.sink_parts + (((int64_t)b * a.Hk + hk) * chunks + chunk) * 2 * a.sink_rows * a.D + (32 * wave + i) * a.D;
  store_rows<float, DP>(dk, a.scale, me < len, part, true, a.D, g);
  store_rows<float, DP>(dv, 1.f, me < len, part + a.sink_rows * a.D, true, a.D, g);
}

// 32 neighbouring elements a workgroup, the chunks in 8 parts that are joined in order
template <class T>
__global__ __launch_bounds__(256) void sink_sums_kernel(Args a) {
  __shared__ float parts[8][32];
  const int64_t per = 2 * a.sink_rows * (int64_t)a.D, all = (int64_t)a.B * a.Hk * per;
  const int part = threadIdx.x >> 5, each = (a.sink_chunks + 7) / 8, last = part * each + each < a.sink_chunks ? part * each + each : a.sink_chunks;
  for (int64_t first = (int64_t)blockIdx.x * 32; first < all; first += (int64_t)gridDim.x * 32) {
    const int64_t e = first + (threadIdx.x & 31);  // `per` is whole thirty-twos
    const int64_t head = e / per, at = e - head * per;
    const float *p = a.sink_parts + head * a.sink_chunks * per + at;
    float sum = 0.f;
#pragma unroll 4
    for (int c = part * each; c < last; ++c) sum += p[c * per];
    parts[part][threadIdx.x & 31] = sum;
    __syncthreads();
    if (part == 0) {
#pragma unroll
      for (int k = 1; k < 8; ++k) sum += parts[k][threadIdx.x];
      const int b = (int)(head / a.Hk), hk = (int)(head % a.Hk), side = (int)(at / (a.sink_rows * a.D));
      const int row = (int)(at / a.D % a.sink_rows), d = (int)(at % a.D);
      T *const out = static_cast<T *>(side ? a.dv : a.dk);
      if (row < a.N) store_from_f32(out + (((int64_t)b * a.N + row) * a.Hk + hk) * a.D + d, sum);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------
template <class T, int DP, bool PLAIN, bool BIAS, bool DBIAS>
static int launch_queries(const Args &a, hipStream_t st) {
  const size_t lds = 4 * (size_t)tile_rows<T, DP>() * WindowOps<T, DP>::kStride * sizeof(T) +
                     (BIAS ? (DBIAS ? 5 : 1) * table_size(a.bias) * sizeof(float) : 0) + (DBIAS ? 16 + 4 * kDiagonals * kDiagonal * sizeof(float) : 0);
  auto kernel = queries_kernel<T, DP, PLAIN, BIAS, DBIAS>;
  if (int rc = allow_dynamic_lds(kernel, lds)) return rc;
  kernel<<<(unsigned)((int64_t)a.blocks * a.Hq * a.B), 256, lds, st>>>(a);
  return launch_status();
}
template <class T, int DP, bool PLAIN, bool BIAS>
static int launch_keys(const Args &a, hipStream_t st) {
  constexpr int QT = tile_rows<T, DP>();
  const size_t lds = 4 * (size_t)QT * WindowOps<T, DP>::kStride * sizeof(T) + 4 * QT * sizeof(float) + (BIAS ? table_size(a.bias) * sizeof(float) : 0);
  auto kernel = keys_kernel<T, DP, PLAIN, BIAS>;
  if (int rc = allow_dynamic_lds(kernel, lds)) return rc;
  const int64_t per_head = a.blocks + a.sink_chunks;
  kernel<<<(unsigned)(per_head * a.Hk * a.B), 256, lds, st>>>(a);
  if (int rc = launch_status()) return rc;
  if (a.sink_chunks == 0) return PA_OK;
  const int64_t n = (int64_t)a.B * a.Hk * 2 * a.sink_rows * a.D;
  sink_sums_kernel<T><<<(unsigned)(n / 32 < 16384 ? n / 32 : 16384), 256, 0, st>>>(a);
  return launch_status();
}
template <class T>
static int backward_of(const Args &a, float *d_bias, hipStream_t st) {
  return by_width(a.D, a.q.plain && a.k.plain && a.v.plain && a.dy.plain, [&](auto dp, auto plain) {
    constexpr int DP = decltype(dp)::value;
    constexpr bool PLAIN = decltype(plain)::value;
    const bool bias = a.bias.buckets != 0;
    int rc = d_bias ? launch_queries<T, DP, PLAIN, true, true>(a, st)
             : bias ? launch_queries<T, DP, PLAIN, true, false>(a, st) : launch_queries<T, DP, PLAIN, false, false>(a, st);
    if (!rc && d_bias) {
      bias_sums_kernel<<<(unsigned)(a.Hq * a.bias.buckets), 256, 0, st>>>(a.bias_parts, (int64_t)a.B * a.blocks, a.Hq, a.bias.buckets, d_bias);
      rc = launch_status();
    }
    if (rc) return rc;
    return bias ? launch_keys<T, DP, PLAIN, true>(a, st) : launch_keys<T, DP, PLAIN, false>(a, st);
  });
}

// what the workspace holds, in floats
struct Room {
  int64_t delta, bias_parts, sink_parts;
  int chunks;
};
static Room room_of(const Args &a, bool want_bias) {
  Room r;
  r.delta = ((int64_t)a.B * a.Hq * a.N + 3) / 4 * 4;
  r.bias_parts = want_bias ? ((int64_t)a.B * a.blocks * a.Hq * a.bias.buckets + 3) / 4 * 4 : 0;
  // Parts of 1 024 queries.  Where the workgroups fill the card few times over, the longest counts: there parts of about as many queries as see
  // a block of keys without sinks (5 001 x 3 x 4 x 64, 512 keys: 98 us with parts of 640, 119 of 1 024; 65 536 x 8 x 32, 257 keys: 121 of 384, 115 of 1 024).
  int64_t queries = 1024;
  if ((int64_t)a.blocks * a.Hk * a.B <= 2048) {
    queries = 128 + (int64_t)a.left + (a.right == kNoBound ? 0 : a.right);
    queries = queries < 512 ? 512 : queries > 1024 ? 1024 : (queries + 63) / 64 * 64;
  }
  r.chunks = a.sinks > 0 ? (int)((a.N + queries - 1) / queries) : 0;
  r.sink_parts = (int64_t)a.B * a.Hk * r.chunks * 2 * a.sink_rows * a.D;
  return r;
}
int64_t backward_workspace_bytes(int dtype, const pa_window_params &p, bool want_bias) {
  const Room r = room_of(make_args(p), want_bias);
  return (r.delta + r.bias_parts + r.sink_parts) * (int64_t)sizeof(float);
}
int backward(int dtype, const pa_window_params &p, const pa_heads &q, const pa_heads &k, const pa_heads &v, const void *y, const float *stats,
             const pa_heads &dy, void *dq, void *dk, void *dv, float *d_bias, void *workspace, hipStream_t st) {
  const int64_t elem = dtype == PA_F32 ? 4 : 2;
  Args a = make_args(p);
  const Room r = room_of(a, d_bias != nullptr);
  a.q = make_view(q, p.D, elem), a.k = make_view(k, p.D, elem), a.v = make_view(v, p.D, elem), a.dy = make_view(dy, p.D, elem);
  a.saved_y = y, a.saved_stats = stats;
  a.dq = dq, a.dk = dk, a.dv = dv;
  a.delta = static_cast<float *>(workspace);
  a.bias_parts = a.delta + r.delta;
  a.sink_parts = a.bias_parts + r.bias_parts;
  a.sink_chunks = r.chunks;
  return dtype == PA_F32 ? backward_of<float>(a, d_bias, st) : backward_of<bf16>(a, d_bias, st);
}

}  // namespace window
}  // namespace pa
