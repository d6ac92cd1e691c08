// Choice of the next token from a row of logits with temperature, top-k, top-p, min-p and a given random number (sm_100a).
//
// With w_i = e^((x_i - max) / T) a token is kept when its rank is below k, when the weights ahead of it (larger ones, and
// equal ones of lower index) sum to less than p times the weight of the first k, and when w_i >= min_p; the result is the
// first kept index whose running sum, in index order, exceeds u times the kept weight.
//
// A row is read once: a cluster of up to eight CTAs shares it and each keeps its slice in shared memory (rows too long for
// that are read again from L2 instead).  No sort of the row: rank and sum are thresholds on the value.  A histogram of 2048
// buckets, linear in the value so that the bulk of a row does not meet in a few of them, gives the bucket a threshold lies
// in, whose values are collected and sorted; one with too many is narrowed by further histograms over its range of keys
// until equal values are left, which are taken in index order.  For a small k the histogram is of the threads' own maxima:
// the buckets that hold k of those hold the k largest values, which are collected, and the rest of the work is comparing
// all pairs of them.
// Weights are whole numbers, round(w 2^b), b = 46 below 2^18 tokens and one less from each doubling on (their sum stays below
// 2^64): sums are then exact, the same in any order, so atomics cannot change the result.  A weight is off by at most 2^-(b+1)
// of the largest (one below that is nothing) and a running sum by V of those: 2^-30 for 128000 tokens, 2^-24 for 2^20, which is
// the step of u; longer rows are refused.  The
// exponential is 64-bit: 2^y = 2^(i / 256) (from a table) e^t, |t| <= ln 2 / 512, the last factor by its series to t^4
// (4 * 10^-17 dropped): ten 64-bit operations.
// Bound: barriers between the phases and the latency behind them; the 64-bit pipe is 12 %, the issue slots 37 %, DRAM 2 %
// busy.  Measured: 200 rows of 128001, bf16, p 0.95, 250 us, k 50 102 us (8 us to read the rows); 8 rows of 32000, fp32,
// k 50, p 0.9, 14.4 us.  A first histogram of an eighth of the values to estimate the threshold cost more than it saved
// (322 us).
#include "serving.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>
#include <math_constants.h>

namespace cg = cooperative_groups;

namespace bg {
namespace {

typedef unsigned long long u64;
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBuckets = 2048, kCoarse = 64;
constexpr int kMaxCluster = 8;
constexpr int kMaxListed = kThreads; // values of one bucket that are sorted, one a thread
constexpr int kMaxPairs = 256;       // values that are ranked by comparing all pairs

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

// What can never be drawn is -inf (NaN too); -0 and +0 are one value.
__device__ __forceinline__ float canonical(float x) { return x > -CUDART_INF_F ? x + 0.0f : -CUDART_INF_F; }
// Order-preserving 32-bit key of a canonical value.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr uint32_t kLowestKey = 0x00800000u;           // of the lowest finite value

// A bucket's sum in two words: 64-bit atomics on shared memory run at 1.1 a clock and SM (measured), 32-bit ones at 4.8, and
// a weight below 2^-14 touches the upper word only with its carry.
struct Shared {
  uint32_t low[kBuckets], high[kBuckets];
  u64 coarse[kCoarse];
  u64 listed[kMaxListed];              // this CTA's values of a bucket: key << 32 | ~index, so that larger means ranked earlier
  u64 pair_weight[kMaxPairs];
  double table[256];                   // 2^(i / 256) times the weight of the largest
  u64 seg_sum[kWarps], warp_sum[kWarps];
  uint32_t seg_ties[kWarps];
  uint32_t top, bottom, first;         // this CTA's part of a cluster-wide maximum, minimum, first index
  uint32_t warp_a[kWarps], warp_b[kWarps];
  uint32_t n_listed;
  // what one warp or thread found for all
  uint32_t all_top, all_bottom;
  uint32_t bucket;
  u64 above, in_bucket, total, rest;
  int seg;
  uint32_t seg_tie_base;
  uint32_t cut_key, cut_ties;
  // the cluster's list, in the place of the sums: they have been read by then (collect())
  __device__ u64* all_listed() { return reinterpret_cast<u64*>(low); }
  __device__ void add(uint32_t b, u64 f) {
    const uint32_t v = (uint32_t)f, old = atomicAdd(&low[b], v);
    const uint32_t h = (uint32_t)(f >> 32) + (old + v < old ? 1u : 0u);
    if (h) atomicAdd(&high[b], h);
  }
  __device__ u64 sum(int b) const { return (u64)high[b] << 32 | low[b]; }
};
static_assert(kMaxListed * 8 <= 2 * kBuckets * 4, "the list fits where the sums were");

// Kept: values above `x`, and the first `ties` of those equal to it.
struct Cut {
  float x;
  uint32_t ties;
};

struct Row {
  float top, floor_x;      // the largest value; lower ones than floor_x weigh as little as it: nothing
  double top_wide, step;   // 256 / (T ln 2)
  double least;            // smallest weight min_p keeps
  const double* table;
  // the weight times 2^bits, before its rounding
  __device__ __forceinline__ double scaled(float x) const {
    const double magic = 6755399441055744.0;                // 1.5 * 2^52: its sum with a small number rounds it to a whole one
    const double a = (double)fmaxf(x, floor_x) - top_wide;
    const double s = fma(a, step, magic);
    const int n = __double2loint(s);
    const double r = fma(a, step, magic - s);               // step a = n + r, |r| <= 1/2
    const double u = 0.0027076061740622863;                 // ln 2 / 256
    double q = fma(r, u * u * u * u / 24.0, u * u * u / 6.0);
    q = fma(r, q, u * u / 2.0);
    q = fma(r, q, u);
    const double t = table[n & 255];
    const double w = fma(t, r * q, t);
    return __hiloint2double(__double2hiint(w) + (int)((uint32_t)(n & ~255) << 12), __double2loint(w));       // * 2^(n >> 8)
  }
  __device__ __forceinline__ u64 fixed(double w) const { return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull; }     // to nearest, w < 2^51
  __device__ __forceinline__ u64 fixed_of(float x) const { return fixed(scaled(x)); }
  __device__ __forceinline__ u64 drawn(float x) const {     // weight in the final draw: min_p applied
    const double w = scaled(x);
    return x == top || w >= least ? fixed(w) : 0ull;
  }
};

__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const u64 o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  return v;
}
__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

template <typename T, bool RES>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleProblem p, int slice) {
  extern __shared__ __align__(16) unsigned char dyn[];
  Shared& sh = *reinterpret_cast<Shared*>(dyn);
  float* kept_values = reinterpret_cast<float*>(dyn + ((sizeof(Shared) + 15) & ~(size_t)15));
  cg::cluster_group cluster = cg::this_cluster();
  const int nc = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x / nc;
  constexpr int VEC = 16 / sizeof(T);
  struct alignas(4 * sizeof(T)) Four {
    T v[4];
  };
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.vocab;
  // slices begin on 16-byte boundaries of the row's address, so that a row of odd length is still read in vectors
  const int mis = (int)((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % VEC);
  const int64_t begin = (int64_t)rank * slice - mis;
  bool infinite = false;                 // the largest is +inf: all such are taken as equal, nothing else can be drawn
  auto finite_form = [&](float v) { return infinite ? (v == CUDART_INF_F ? 0.0f : -CUDART_INF_F) : v; };
  auto value_at = [&](int j) -> float {
    if (RES) return kept_values[j];
    const int64_t e = begin + j;
    return e >= 0 && e < p.vocab ? finite_form(canonical(widen(x[e]))) : -CUDART_INF_F;
  };
  // f(four values, place of the first in the slice) for [j0, j1) by `lanes` threads of which this is number `me`; j0 a multiple of four
  auto each_four = [&](int j0, int j1, int me, int lanes, auto&& f) {
    for (int j = j0 + 4 * me; j < j1; j += 4 * lanes) {
      float v[4];
      if (RES) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(kept_values + j);
      else if (begin + j >= 0 && begin + j + 4 <= p.vocab) {
        const Four q = *reinterpret_cast<const Four*>(x + begin + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = finite_form(canonical(widen(q.v[i])));
      } else
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = value_at(j + i);
      f(v, j);
    }
  };

  // ---- read the slice; every thread's largest value ----
  float mine = -CUDART_INF_F;
  for (int i = tid; i < kBuckets; i += kThreads) { sh.low[i] = 0u; sh.high[i] = 0u; }
  const int bits = min(46, __clzll((long long)p.vocab));      // vocab 2^bits < 2^64
  if (tid < 256) sh.table[tid] = exp2((double)tid / 256.0) * (double)(1ull << bits);
  if (tid == 0) sh.n_listed = 0u;
#pragma unroll 4
  for (int j = tid * VEC; j < slice; j += kThreads * VEC) {
    const int64_t e = begin + j;
    float v[VEC];
    if (e >= 0 && e + VEC <= p.vocab) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(x + e));
      const T* q = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = canonical(widen(q[i]));
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = e + i >= 0 && e + i < p.vocab ? canonical(widen(x[e + i])) : -CUDART_INF_F;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) mine = fmaxf(mine, v[i]);
    if (RES)
#pragma unroll
      for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4*>(kept_values + j + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  }
  // the cluster's largest value, and the smallest of the threads' own largest
  {
    uint32_t top = mine > -CUDART_INF_F ? key_of(mine) : 0u, low = top ? top : 0xffffffffu;
    top = __reduce_max_sync(0xffffffffu, top);
    low = __reduce_min_sync(0xffffffffu, low);
    if (lane == 0) { sh.warp_a[warp] = top; sh.warp_b[warp] = low; }
    __syncthreads();
    if (warp == 0) {
      top = __reduce_max_sync(0xffffffffu, lane < kWarps ? sh.warp_a[lane] : 0u);
      low = __reduce_min_sync(0xffffffffu, lane < kWarps ? sh.warp_b[lane] : 0xffffffffu);
      if (lane == 0) { sh.top = top; sh.bottom = low; }
    }
    cluster.sync();
    if (warp == 0) {
      const Shared* r = cluster.map_shared_rank(&sh, lane < nc ? lane : 0);
      top = __reduce_max_sync(0xffffffffu, r->top);
      low = __reduce_min_sync(0xffffffffu, r->bottom);
      if (lane == 0) { sh.all_top = top; sh.all_bottom = low; }
    }
    __syncthreads();
  }
  const bool nothing = sh.all_top == 0u;
  Row w;
  w.top = nothing ? 0.0f : value_of(sh.all_top);
  float least_maximum = nothing ? 0.0f : value_of(sh.all_bottom);
  if (w.top == CUDART_INF_F) {
    infinite = true;
    if (RES) {
      for (int j = tid; j < slice; j += kThreads) kept_values[j] = finite_form(kept_values[j]);
      __syncthreads();
    }
    mine = finite_form(mine);
    w.top = least_maximum = 0.0f;
  }

  const float t = p.temperatures ? p.temperatures[row] : p.temperature;
  if (nothing || !(t > 0.0f)) {
    // nothing to draw from, or greedy: the first of the largest
    uint32_t first = 0xffffffffu;
    if (!nothing)
      for (int j = tid; j < slice; j += kThreads)
        if (value_at(j) == w.top) { first = (uint32_t)(begin + j); break; }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) sh.warp_a[warp] = first;
    __syncthreads();
    if (warp == 0) {
      first = __reduce_min_sync(0xffffffffu, lane < kWarps ? sh.warp_a[lane] : 0xffffffffu);
      if (lane == 0) sh.first = first;
    }
    cluster.sync();
    if (rank == 0 && warp == 0) {
      first = __reduce_min_sync(0xffffffffu, cluster.map_shared_rank(&sh, lane < nc ? lane : 0)->first);
      if (lane == 0) {
        p.tokens[row] = nothing ? -1 : (int64_t)first;
        if (p.probabilities) p.probabilities[row] = nothing ? 0.0f : 1.0f;
      }
    }
    cluster.sync();
    return;
  }

  // Values next to the largest are at least 2^-24 of it away: at a temperature below 2^-30 of it their weights are below
  // e^-64 and vanish, as they do at 2^-30.  The floor then still lies below the largest value, and y within 2^16.
  const float warm = fmaxf(t, fabsf(w.top) * 9.313225746154785e-10f);
  w.floor_x = fmaxf(w.top - 100.0f * warm, -FLT_MAX);
  w.top_wide = (double)w.top;
  w.step = 369.3299304675746 / (double)warm;               // 256 / ln 2
  w.table = sh.table;
  const float min_p = p.min_ps ? p.min_ps[row] : p.min_p;
  w.least = min_p > 0.0f ? (double)(1ull << bits) * (double)fminf(min_p, 1.0f) : 0.0;
  float u = p.uniforms[row];
  u = u > 0.0f ? u : 0.0f;
  // what the running sum has to exceed
  auto draw_target = [&](u64 total) -> u64 {
    const u64 at = u < 1.0f ? (u64)((double)u * (double)total) : total;
    return at < total ? at : total - 1;
  };

  // Buckets of values, 0 at the largest: never increasing with the value (the sum with 2^23 leaves whole numbers).
  auto scale_of = [&](float x_low) -> float {
    const float span = w.top - x_low;
    return span > 0.0f && span < CUDART_INF_F ? (float)(kBuckets - 1) / span : 0.0f;
  };
  auto bucket_of_value = [&](float v, float sc) -> uint32_t {
    return __float_as_uint(fminf(fmaf(w.top - v, sc, 8388608.0f), 8388608.0f + (float)(kBuckets - 1))) - 0x4b000000u;
  };

  int round = 0;
  // One round: `fill()` adds this CTA's part and `once()` the cluster's, then the bucket in which the running sum (bucket 0
  // first) reaches the target is found.  target_of(total) gives the target from the round's total.
  auto search = [&](auto&& fill, auto&& once, auto&& target_of) {
    if (round > 0) {
      cluster.sync();                        // the other CTAs have read the last round's
      for (int i = tid; i < kBuckets; i += kThreads) { sh.low[i] = 0u; sh.high[i] = 0u; }
      __syncthreads();
    }
    ++round;
    if (rank == 0 && tid == 0) once();
    fill();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kCoarse / kWarps; ++i) {
      const int c = warp + i * kWarps;
      const u64 s = warp_sum(sh.sum(c * 32 + lane));
      if (lane == 0) sh.coarse[c] = s;
    }
    cluster.sync();
    if (warp == 0) {
      u64 a = 0, b = 0;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        if (r < nc) {
          const ulonglong2 q = reinterpret_cast<const ulonglong2*>(cluster.map_shared_rank(&sh, r)->coarse)[lane];
          a += q.x;
          b += q.y;
        }
      const u64 incl = warp_scan(a + b, lane);
      const u64 total = __shfl_sync(0xffffffffu, incl, 31);
      u64 target = target_of(total);
      if (target > total) target = total;
      if (target < 1) target = 1;
      const int at = __ffs(__ballot_sync(0xffffffffu, incl >= target)) - 1;      // total >= 1: some lane reaches it
      u64 above = __shfl_sync(0xffffffffu, incl - a - b, at);
      const u64 a_at = __shfl_sync(0xffffffffu, a, at);
      int c = 2 * at;
      if (above + a_at < target) { above += a_at; ++c; }
      u64 f = 0;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        if (r < nc) f += cluster.map_shared_rank(&sh, r)->sum(c * 32 + lane);
      const u64 fi = warp_scan(f, lane);
      const int fl = __ffs(__ballot_sync(0xffffffffu, above + fi >= target)) - 1;
      if (lane == fl) {
        sh.bucket = (uint32_t)(c * 32 + fl);
        sh.above = above + fi - f;
        sh.total = total;
        sh.rest = target - (above + fi - f);       // how much of the bucket is wanted
        sh.in_bucket = f;
      }
    }
    __syncthreads();
  };
  // Collects the cluster's values that `wanted` names into all_listed and returns their number; the list holds them when
  // there are at most kMaxListed.  `n_listed` is zero before; the lists may be read until the next cluster barrier.
  auto collect = [&](auto&& wanted) -> uint32_t {
    each_four(0, slice, tid, kThreads, [&](const float* v, int j) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v[i] > -CUDART_INF_F && wanted(v[i])) {
          const uint32_t at = atomicAdd(&sh.n_listed, 1u);
          if (at < kMaxListed) sh.listed[at] = (u64)key_of(v[i]) << 32 | (uint32_t)~(uint32_t)(begin + j + i);
        }
    });
    cluster.sync();
    u64* all = sh.all_listed();
    uint32_t m[kMaxCluster], n = 0;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) m[r] = r < nc ? cluster.map_shared_rank(&sh, r)->n_listed : 0u;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      if (tid < m[r] && n + tid < kMaxListed) all[n + tid] = cluster.map_shared_rank(&sh, r)->listed[tid];
      n += m[r];
    }
    __syncthreads();
    return n;
  };
  auto forget_list = [&] {
    cluster.sync();                          // every list has been read
    if (tid == 0) sh.n_listed = 0u;
  };

  // From the bucket a first round found: the cut among its values, which count for one or for their weights.
  auto resolve = [&](float sc, bool counting, Cut cut) -> Cut {
    const uint32_t b0 = sh.bucket;
    u64 wanted = sh.rest;
    const bool splits_ties = !counting && cut.ties && bucket_of_value(cut.x, sc) == b0;     // then the earlier cut's own ties are in it
    if (!splits_ties && (!counting || sh.in_bucket <= kMaxListed)) {
      const uint32_t held = collect([&](float v) { return v > cut.x && bucket_of_value(v, sc) == b0 && (counting || w.fixed_of(v)); });
      if (held <= kMaxListed) {
        // Bitonic, largest first, an element a thread: by shuffles inside a warp, through shared memory across warps.
        const int n = (int)held, log = n <= 1 ? 0 : 32 - __clz(n - 1);
        u64* all = sh.all_listed();
        u64 e = tid < n ? all[tid] : 0ull;
        __syncthreads();
        for (int ls = 1; ls <= log; ++ls)
          for (int ld = ls - 1; ld >= 0; --ld) {
            u64 o;
            if (ld >= 5) {
              all[tid] = e;
              __syncthreads();
              o = all[tid ^ (1 << ld)];
              __syncthreads();
            } else if (warp * 32 < 1 << log) o = __shfl_xor_sync(0xffffffffu, e, 1 << ld);
            else continue;
            const bool first = !(tid >> ld & 1), down = !(tid >> ls & 1);
            e = (e > o) == (first == down) ? e : o;
          }
        all[tid] = e;
        // running sums; the element that reaches what is wanted is the cut
        const u64 f = !e ? 0ull : counting ? 1ull : w.fixed_of(value_of((uint32_t)(e >> 32)));
        const u64 in_warp = warp_scan(f, lane);
        if (lane == 31) sh.warp_sum[warp] = in_warp;
        __syncthreads();
        u64 before = in_warp - f;
        for (int i = 0; i < warp; ++i) before += sh.warp_sum[i];
        if (before < wanted && before + f >= wanted) {       // exactly one thread
          const uint32_t key = (uint32_t)(e >> 32);
          uint32_t same = 1;
          while ((int)same <= tid && (uint32_t)(all[tid - (int)same] >> 32) == key) ++same;
          sh.cut_key = key;
          sh.cut_ties = same;
        }
        forget_list();                       // (its barrier also shows the cut to all)
        return Cut{value_of(sh.cut_key), sh.cut_ties};
      }
      forget_list();
    }
    // the keys of that bucket: [smallest key in a bucket <= b0, smallest key in a bucket < b0), 32 probes at a time
    auto smallest = [&](uint32_t bucket) {              // smallest key of a number whose bucket is at most `bucket`
      uint32_t a = kLowestKey, z = key_of(w.top);       // the answer lies in [a, z]
      while (a < z) {
        const uint32_t step = (z - a) / 33u + 1u;
        const uint32_t at = z - a > step * (uint32_t)lane ? a + step * (uint32_t)lane : z;
        const uint32_t yes = __ballot_sync(0xffffffffu, bucket_of_value(value_of(at), sc) <= bucket);
        const int l = __ffs(yes) - 1;                   // probes grow with the lane; the first that qualifies
        if (l < 0) { a = min(z, a + 31u * step) + 1u; if (a > z) a = z; }
        else {
          const uint32_t nz = __shfl_sync(0xffffffffu, at, l);
          const uint32_t na = l == 0 ? nz : __shfl_sync(0xffffffffu, at, l - 1) + 1u;
          a = na; z = nz;
        }
      }
      return a;
    };
    uint32_t lo = smallest(b0), hi = b0 == 0u ? key_of(w.top) : smallest(b0 - 1u) - 1u;
    const uint32_t cut_key = cut.ties ? key_of(cut.x) : 0u;
    while (lo < hi) {
      const int shift = max(0, 21 - __clz(hi - lo));     // 2048 buckets over the range
      auto bucket_of = [&](uint32_t k) { return (hi - k) >> shift; };
      const u64 want = wanted;
      search(
          [&] {
            each_four(0, slice, tid, kThreads, [&](const float* v, int) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t k = key_of(v[i]);
                if (k < lo || k > hi || !(v[i] > cut.x)) continue;
                if (counting) atomicAdd(&sh.low[bucket_of(k)], 1u);
                else if (const u64 f = w.fixed_of(v[i])) sh.add(bucket_of(k), f);
              }
            });
          },
          [&] {
            if (!counting && cut.ties && cut_key >= lo && cut_key <= hi) sh.add(bucket_of(cut_key), w.fixed_of(cut.x) * cut.ties);
          },
          [&](u64) { return want; });
      wanted = sh.rest;
      const uint32_t b = sh.bucket, old = hi;
      hi = old - (b << shift);
      const uint32_t width = (1u << shift) - 1u;
      lo = max(lo, hi > width ? hi - width : 0u);
      __syncthreads();                                   // (the found bucket has been read)
    }
    const float at = value_of(lo);
    if (counting) return Cut{at, (uint32_t)wanted};
    const u64 each = w.fixed_of(at);
    u64 ties = each ? (wanted + each - 1) / each : 1ull;
    if (cut.ties && at == cut.x && ties > cut.ties) ties = cut.ties;
    return Cut{at, (uint32_t)min(max(ties, 1ull), 0xffffffffull)};
  };

  Cut cut{-CUDART_INF_F, 0u};
  const float top_p = p.top_ps ? p.top_ps[row] : p.top_p;
  auto nucleus = [&](u64 total) -> u64 { return (u64)ceil((double)fmaxf(top_p, 0.0f) * (double)total); };
  const int top_k = p.top_ks ? p.top_ks[row] : p.top_k;
  if (top_k > 0 && top_k < p.vocab) {
    const float sc = scale_of(least_maximum);
    uint32_t n = kMaxPairs + 1;
    if (top_k <= kMaxPairs / 2) {
      search([&] { if (mine > -CUDART_INF_F) atomicAdd(&sh.low[bucket_of_value(mine, sc)], 1u); }, [] {}, [&](u64) { return (u64)top_k; });
      if (sh.total >= (u64)top_k) {          // else there are not k maxima to go by
        const uint32_t b0 = sh.bucket;
        n = collect([&](float v) { return bucket_of_value(v, sc) <= b0; });
        if (n > kMaxPairs) forget_list();
      }
    }
    if (n > kMaxPairs) {
      search(
          [&] {
            each_four(0, slice, tid, kThreads, [&](const float* v, int) {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (v[i] > -CUDART_INF_F) atomicAdd(&sh.low[bucket_of_value(v[i], sc)], 1u);
            });
          },
          [] {}, [&](u64) { return (u64)top_k; });
      if (sh.above + sh.in_bucket <= kMaxPairs) {
        const uint32_t b0 = sh.bucket;
        n = collect([&](float v) { return bucket_of_value(v, sc) <= b0; });
      }
    }
    if (n <= kMaxPairs) {
      // few enough to finish on a list that holds the k largest: ranks, the nucleus, and the draw in index order
      if (rank == 0) {
        const u64* all = sh.all_listed();
        const u64 me = tid < n ? all[tid] : 0ull;
        const float v = value_of((uint32_t)(me >> 32));
        const u64 weight = tid < n ? w.fixed_of(v) : 0ull;
        if (tid < n) sh.pair_weight[tid] = weight;
        __syncthreads();
        u64 before = 0;
        int ahead = 0;
        if (tid < n)
          for (uint32_t j = 0; j < n; ++j)
            if (all[j] > me) { before += sh.pair_weight[j]; ++ahead; }
        const bool ranked = tid < n && ahead < top_k;
        auto block_sum = [&](u64 s) -> u64 {
          s = warp_sum(s);
          __syncthreads();
          if (lane == 0) sh.warp_sum[warp] = s;
          __syncthreads();
          s = 0;
#pragma unroll
          for (int i = 0; i < kMaxPairs / 32; ++i) s += sh.warp_sum[i];
          return s;
        };
        const u64 reach = top_p < 1.0f ? nucleus(block_sum(ranked ? weight : 0ull)) : ~0ull;
        const bool kept = ranked && (ahead == 0 || before < reach);
        const u64 drawn = kept ? w.drawn(v) : 0ull;
        const u64 total = block_sum(drawn);
        if (tid < n) sh.pair_weight[tid] = drawn;
        __syncthreads();
        const u64 target = draw_target(total);
        if (drawn) {
          u64 run = 0;
          for (uint32_t j = 0; j < n; ++j)
            if ((uint32_t)all[j] > (uint32_t)me) run += sh.pair_weight[j];       // of lower index
          if (run <= target && target < run + drawn) {
            p.tokens[row] = (int64_t)(uint32_t)~(uint32_t)me;
            if (p.probabilities) p.probabilities[row] = (float)(w.scaled(v) / (double)total);
          }
        }
      }
      cluster.sync();
      return;
    }
    cut = resolve(sc, true, cut);
  }
  if (top_p < 1.0f) {
    const float sc = scale_of(fmaxf(w.top - 34.0f * warm, -FLT_MAX));
    const Cut by_rank = cut;
    search(
        [&] {
          each_four(0, slice, tid, kThreads, [&](const float* v, int) {
            u64 f[4];                        // all four ahead of the first atomic, which the table's loads cannot pass
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = w.fixed_of(v[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (v[i] > by_rank.x && f[i]) sh.add(bucket_of_value(v[i], sc), f[i]);
          });
        },
        [&] { if (by_rank.ties) sh.add(bucket_of_value(by_rank.x, sc), w.fixed_of(by_rank.x) * by_rank.ties); },
        nucleus);
    cut = resolve(sc, false, by_rank);
  }

  // ---- the draw: sums per warp segment in index order, then the segment, then the token ----
  const u64 tie_weight = cut.ties ? w.drawn(cut.x) : 0ull;
  const int seg_len = ((slice + kWarps * 128 - 1) / (kWarps * 128)) * 128;
  const int s0 = min(slice, warp * seg_len), s1 = min(slice, s0 + seg_len);
  {
    u64 sum = 0;
    uint32_t ties = 0;
    each_four(s0, s1, lane, 32, [&](const float* v, int) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u64 f = w.drawn(v[i]);
        sum += v[i] > cut.x ? f : 0ull;
        ties += v[i] == cut.x;
      }
    });
    sum = warp_sum(sum);
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) { sh.seg_sum[warp] = sum; sh.seg_ties[warp] = ties; }
  }
  cluster.sync();
  if (warp == 0) {
    // lane l holds segments 4 l to 4 l + 3 of the cluster's, in index order
    constexpr int PER = kMaxCluster * kWarps / 32;
    u64 sums[PER], mine = 0;
    uint32_t tied[PER], ties = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int sg = lane * PER + i;
      const bool there = sg < nc * kWarps;
      const Shared* r = cluster.map_shared_rank(&sh, there ? sg / kWarps : 0);
      sums[i] = there ? r->seg_sum[sg % kWarps] : 0ull;
      tied[i] = there ? r->seg_ties[sg % kWarps] : 0u;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) ties += tied[i];
    const uint32_t ties_before = (uint32_t)(warp_scan(ties, lane) - ties);
    uint32_t tb = ties_before;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      sums[i] += tie_weight * (u64)min(tied[i], cut.ties > tb ? cut.ties - tb : 0u);
      mine += sums[i];
      tb += tied[i];
    }
    const u64 incl = warp_scan(mine, lane);
    const u64 total = __shfl_sync(0xffffffffu, incl, 31);
    const u64 target = draw_target(total);
    const int at = __ffs(__ballot_sync(0xffffffffu, incl > target)) - 1;
    if (lane == at) {
      u64 before = incl - mine;
      tb = ties_before;
      int found = -1;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (found < 0) {
          if (before + sums[i] > target) found = lane * PER + i;
          else { before += sums[i]; tb += tied[i]; }
        }
      sh.seg = found;
      sh.rest = target - before;
      sh.seg_tie_base = tb;
      sh.total = total;
    }
  }
  __syncthreads();
  if (sh.seg / kWarps == rank && sh.seg % kWarps == warp) {
    u64 rest = sh.rest;
    uint32_t tb = sh.seg_tie_base;
    const int n = s1 - s0, per = ((n + 31) / 32) | 1;       // an odd stride between lanes: no bank conflicts
    const int a0 = min(n, lane * per), a1 = min(n, a0 + per);
    u64 sum = 0;
    uint32_t ties = 0;
#pragma unroll 4
    for (int j = a0; j < a1; ++j) {
      const float v = value_at(s0 + j);
      const u64 f = w.drawn(v);
      sum += v > cut.x ? f : 0ull;
      ties += v == cut.x;
    }
    const uint32_t before = tb + (uint32_t)(warp_scan(ties, lane) - ties);
    const uint32_t left = cut.ties > before ? cut.ties - before : 0u;
    sum += tie_weight * (u64)min(ties, left);
    const u64 incl = warp_scan(sum, lane);
    const int at = __ffs(__ballot_sync(0xffffffffu, incl > rest)) - 1;
    rest -= __shfl_sync(0xffffffffu, incl - sum, at);
    tb = __shfl_sync(0xffffffffu, before, at);
    const int c0 = __shfl_sync(0xffffffffu, a0, at), c1 = __shfl_sync(0xffffffffu, a1, at);
    for (int j = c0; j < c1; j += 32) {
      const float v = j + lane < c1 ? value_at(s0 + j + lane) : -CUDART_INF_F;
      const bool tie = cut.ties && v == cut.x;
      const uint32_t tied = __ballot_sync(0xffffffffu, tie);
      u64 f = 0;
      if (v > cut.x) f = w.drawn(v);
      else if (tie && tb + __popc(tied & ((1u << lane) - 1u)) < cut.ties) f = tie_weight;
      const u64 run = warp_scan(f, lane);
      const uint32_t hit = __ballot_sync(0xffffffffu, run > rest);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          p.tokens[row] = begin + s0 + j + lane;
          if (p.probabilities) p.probabilities[row] = (float)(w.scaled(v) / (double)sh.total);
        }
        break;
      }
      rest -= __shfl_sync(0xffffffffu, run, 31);
      tb += __popc(tied);
    }
  }
  cluster.sync();         // no CTA leaves while another still reads its sums
}

template <typename T>
cudaError_t launch_typed(const SampleProblem& p, cudaStream_t s, int sm_count) {
  constexpr int VEC = 16 / sizeof(T);
  const size_t fixed = (sizeof(Shared) + 15) & ~(size_t)15;
  const int64_t room = (int64_t)(110 * 1024 - fixed) / 4;      // values of a slice, with two CTAs on an SM
  // Enough CTAs to hold the row; more while SMs are idle and slices stay above 4096 (below, a round's barriers cost more
  // than the shorter slices save).
  int nc = 1;
  while (nc < kMaxCluster && (p.vocab + VEC + nc - 1) / nc > room) nc *= 2;
  while (nc < kMaxCluster && p.n * nc * 2 <= sm_count && p.vocab / (nc * 2) >= 2048) nc *= 2;
  int64_t slice = (p.vocab + VEC - 1 + nc - 1) / nc;           // an unaligned row begins up to VEC - 1 values into its first slice
  slice = (slice + 31) / 32 * 32;
  const bool res = slice <= room;
  void (*kern)(const SampleProblem, int) = res ? sample_kernel<T, true> : sample_kernel<T, false>;
  const size_t smem = fixed + (res ? (size_t)slice * 4 : 0);
  cudaError_t e = allow_shared(kern, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  if (p.n * nc > 0x7fffffffll) return cudaErrorInvalidValue;
  cfg.gridDim = dim3((unsigned)(p.n * nc));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)nc;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p, (int)slice);
}

}  // namespace

cudaError_t launch_sample(const SampleProblem& p, int dtype, cudaStream_t s, int sm_count) {
  if (dtype == BG_F32) return launch_typed<float>(p, s, sm_count);
  if (dtype == BG_F16) return launch_typed<__half>(p, s, sm_count);
  return launch_typed<__nv_bfloat16>(p, s, sm_count);
}

}  // namespace bg
