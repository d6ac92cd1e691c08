// Choice of the next token from a row of logits with temperature, top-k, top-p, min-p and a given random number (sm_100a).
//
// With w_i = e^((x_i - max) / T) a token is kept when its rank is below k, when the weights ahead of it (larger ones, and
// equal ones of lower index) sum to less than p times the weight of the first k, and when w_i >= min_p; the result is the
// first kept index whose running sum, in index order, exceeds u times the kept weight.
//
// A row is read once: a cluster of up to eight CTAs shares it and each keeps its slice in shared memory as ordered 32-bit
// keys (rows too long for that are read again from L2 instead).  No sort: the rank and the sum are thresholds on the
// value.  A histogram of 2048 buckets, linear in the value so that the bulk of a row does not meet in a few of them, gives
// the bucket a threshold lies in, whose keys are collected and sorted (where top-k leaves few keys, all the kept ones are
// collected, and the rest of the work is comparing all pairs).  A bucket with too many keys for that is narrowed by further
// histograms over its range of keys until equal values are left, which are taken in index order.
// Weights are whole numbers, round(w 2^46) (fewer bits for a vocabulary whose sum would pass 2^62): sums are then exact,
// the same in any order, so atomics cannot change the result.  A weight is off by at most 2^-46 of the largest and a
// running sum by some 2^-46 sqrt(V), while u has 24 bits; 32-bit weights would move one choice in a thousand.  The
// exponential is 64-bit: 2^y = 2^(i / 256) (from a table) e^t, |t| <= ln 2 / 512, the last factor by its series to t^4
// (4 * 10^-17 dropped), a dozen operations against some forty of the general function.
#include "serving.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

namespace cg = cooperative_groups;

namespace bg {
namespace {

typedef unsigned long long u64;
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBuckets = 2048, kCoarse = 64;
constexpr int kMaxCluster = 8;
constexpr int kMaxListed = kThreads; // keys of one bucket that are sorted, one a thread
constexpr int kMaxPairs = 256;       // keys that are ranked by comparing all pairs

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

// Order-preserving key; 0 for what can never be drawn (-inf, NaN), which keeps every other key above it.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -CUDART_INF_F)) return 0u;
  const uint32_t b = __float_as_uint(x + 0.0f);        // -0 and +0 are equal values: one key
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

constexpr uint32_t kLowestKey = 0x00800000u;           // of the lowest finite value

// A bucket's sum in two words: 64-bit atomics on shared memory are a loop (1.1 a clock and SM measured, 32-bit ones 4.8), and
// a weight below 2^-14 touches the upper word only with its carry.
struct Shared {
  uint32_t low[kBuckets], high[kBuckets];
  u64 coarse[kCoarse];
  u64 listed[kMaxListed];              // this CTA's keys of a bucket: key << 32 | ~index, so that larger means ranked earlier
  u64 pair_weight[kMaxPairs];
  double table[256];                   // 2^(i / 256)
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

// Kept: keys above `key`, and the first `ties` of those equal to it.
struct Cut {
  uint32_t key, ties;
};

struct Row {
  uint32_t top;            // largest key
  float top_value;
  double top_wide, step;   // 256 / (T ln 2)
  double one, floor;       // weight of the largest, 2^bits; and the smallest weight min_p keeps
  int bits;                // fraction bits of a weight
  bool finite;             // the largest is not +inf
  const double* table;
  // the weight times 2^bits, before its rounding (k > 0)
  __device__ __forceinline__ double scaled(uint32_t k) const {
    const double magic = 6755399441055744.0;                // 1.5 * 2^52: its sum with a small number rounds it to a whole one
    double y = ((double)value_of(k) - top_wide) * step;
    y = y > -12800.0 ? y : -12800.0;                        // 2^-50 and less, which 2^46 times rounds to zero; NaN too
    const double s = y + magic;
    const int n = __double2loint(s);
    const double r = y - (s - magic);                       // y = n + r, |r| <= 1/2
    const double u = 0.0027076061740622863;                 // ln 2 / 256
    double q = fma(r, u * u * u * u / 24.0, u * u * u / 6.0);
    q = fma(r, q, u * u / 2.0);
    q = fma(r, q, u);
    const double t = table[n & 255];
    const double w = fma(t, r * q, t);
    const double e = __hiloint2double(__double2hiint(w) + (((n >> 8) + bits) << 20), __double2loint(w));
    return finite ? e : (k == top ? one : 0.0);
  }
  __device__ u64 fixed(double w) const { return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull; }     // to nearest, w < 2^51
  __device__ u64 fixed_of(uint32_t k) const { return fixed(scaled(k)); }
  __device__ u64 drawn(uint32_t k) const {                  // weight in the final draw: min_p applied
    const double w = scaled(k);
    return k == top || w >= floor ? fixed(w) : 0ull;
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
  uint32_t* keys = reinterpret_cast<uint32_t*>(dyn + ((sizeof(Shared) + 15) & ~(size_t)15));
  cg::cluster_group cluster = cg::this_cluster();
  const int nc = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x / nc;
  constexpr int VEC = 16 / sizeof(T);
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.vocab;
  // slices begin on 16-byte boundaries of the row's address, so that a row of odd length is still read in vectors
  const int mis = (int)((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % VEC);
  const int64_t begin = (int64_t)rank * slice - mis;
  auto key_at = [&](int j) -> uint32_t {
    if (RES) return keys[j];
    const int64_t e = begin + j;
    return e >= 0 && e < p.vocab ? key_of(widen(x[e])) : 0u;
  };

  // f(four keys, place of the first in the slice) for [j0, j1) by `lanes` threads of which this is number `me`; j0 a multiple of four
  auto each_four = [&](int j0, int j1, int me, int lanes, auto&& f) {
    for (int j = j0 + 4 * me; j < j1; j += 4 * lanes) {
      uint32_t k[4];
      if (RES) *reinterpret_cast<uint4*>(k) = *reinterpret_cast<const uint4*>(keys + j);
      else
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = key_at(j + i);
      f(k, j);
    }
  };

  // ---- read the slice; largest and smallest key ----
  uint32_t top = 0u, low = 0xffffffffu;
  for (int i = tid; i < kBuckets; i += kThreads) { sh.low[i] = 0u; sh.high[i] = 0u; }
  if (tid < 256) sh.table[tid] = exp2((double)tid / 256.0);
  if (tid == 0) sh.n_listed = 0u;
#pragma unroll 4
  for (int j = tid * VEC; j < slice; j += kThreads * VEC) {
    const int64_t e = begin + j;
    uint32_t k[VEC];
    if (e >= 0 && e + VEC <= p.vocab) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(x + e));
      const T* v = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < VEC; ++i) k[i] = key_of(widen(v[i]));
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) k[i] = e + i >= 0 && e + i < p.vocab ? key_of(widen(x[e + i])) : 0u;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      top = max(top, k[i]);
      if (k[i]) low = min(low, k[i]);
    }
    if (RES)
#pragma unroll
      for (int i = 0; i < VEC; i += 4) *reinterpret_cast<uint4*>(keys + j + i) = make_uint4(k[i], k[i + 1], k[i + 2], k[i + 3]);
  }
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
  top = sh.all_top;
  low = sh.all_bottom;

  const float t = p.temperatures ? p.temperatures[row] : p.temperature;
  if (top == 0u || !(t > 0.0f)) {
    // nothing to draw from, or greedy: the first of the largest
    uint32_t first = 0xffffffffu;
    if (top != 0u)
      for (int j = tid; j < slice; j += kThreads)
        if (key_at(j) == top) { first = (uint32_t)(begin + j); break; }
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
        p.tokens[row] = top == 0u ? -1 : (int64_t)first;
        if (p.probabilities) p.probabilities[row] = top == 0u ? 0.0f : 1.0f;
      }
    }
    cluster.sync();
    return;
  }

  Row w;
  w.top = top;
  w.top_value = value_of(top);
  w.top_wide = (double)w.top_value;
  w.finite = w.top_value < CUDART_INF_F;
  w.step = 369.3299304675746 / (double)t;                 // 256 / ln 2
  w.bits = min(46, 62 - (64 - __clzll((long long)p.vocab)));
  w.one = (double)(1ull << w.bits);
  w.table = sh.table;
  const float min_p = p.min_ps ? p.min_ps[row] : p.min_p;
  w.floor = min_p > 0.0f ? w.one * (double)fminf(min_p, 1.0f) : 0.0;
  float u = p.uniforms[row];
  u = u > 0.0f ? u : 0.0f;
  // what the running sum has to exceed
  auto draw_target = [&](u64 total) -> u64 {
    const u64 at = u < 1.0f ? (u64)((double)u * (double)total) : total;
    return at < total ? at : total - 1;
  };

  int round = 0;
  // One round: `add(four keys)` for this CTA's keys and `once()` for the cluster, then the bucket
  // in which the running sum (bucket 0 first) reaches the target.  target_of(total) gives the target from the round's
  // total.
  auto search = [&](auto&& add, auto&& once, auto&& target_of) {
    if (round > 0) {
      cluster.sync();                        // the other CTAs have read the last round's
      for (int i = tid; i < kBuckets; i += kThreads) { sh.low[i] = 0u; sh.high[i] = 0u; }
      __syncthreads();
    }
    ++round;
    if (rank == 0 && tid == 0) once();
    each_four(0, slice, tid, kThreads, [&](const uint32_t* k, int) { add(k); });
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
  // Collects the cluster's keys that `wanted` names into all_listed and returns their number; the list holds them when
  // there are at most kMaxListed.  `n_listed` is zero before; the lists may be read until the next cluster barrier.
  auto collect = [&](auto&& wanted) -> uint32_t {
    each_four(0, slice, tid, kThreads, [&](const uint32_t* k, int j) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (k[i] && wanted(k[i])) {
          const uint32_t at = atomicAdd(&sh.n_listed, 1u);
          if (at < kMaxListed) sh.listed[at] = (u64)k[i] << 32 | (uint32_t)~(uint32_t)(begin + j + i);
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
  // The value at which the sum of what the kept keys count for (one, or their weights), largest first, reaches a target.
  auto linear_of = [&](float x_low) -> float {
    const float span = w.top_value - x_low;
    return span > 0.0f && span < CUDART_INF_F ? (float)kBuckets / span : 0.0f;
  };
  auto linear = [&](uint32_t k, float sc) -> uint32_t {   // never increases with the key
    const float v = (w.top_value - value_of(k)) * sc;
    return v >= (float)(kBuckets - 1) ? kBuckets - 1 : (uint32_t)(int)v;      // NaN (infinite top) becomes bucket 0
  };
  // From the bucket a first round found: the cut among its keys.  `before` is what lies above the bucket, sh.rest what
  // is wanted of it.
  auto resolve = [&](float sc, bool counting, Cut cut) -> Cut {
    const uint32_t b0 = sh.bucket;
    u64 wanted = sh.rest;
    const bool splits_ties = !counting && cut.ties && linear(cut.key, sc) == b0;     // then the earlier cut's own ties are in it
    // the bucket as a range of (top - value) sc, as linear() rounds it
    const float v0 = b0 == 0u ? -CUDART_INF_F : (float)b0, v1 = b0 == kBuckets - 1u || sc == 0.0f ? CUDART_INF_F : (float)(b0 + 1u);
    uint32_t held = kMaxListed + 1;
    if (!splits_ties && (!counting || sh.in_bucket <= kMaxListed)) {
      held = collect([&](uint32_t k) {
        const float v = (w.top_value - value_of(k)) * sc;
        return k > cut.key && !(v < v0) && !(v >= v1) && (counting || w.fixed_of(k));
      });
      if (held > kMaxListed) {
        cluster.sync();                    // every count has been read
        if (tid == 0) sh.n_listed = 0u;
      }
    }
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
      const u64 f = !e ? 0ull : counting ? 1ull : w.fixed_of((uint32_t)(e >> 32));
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
      cluster.sync();                      // every list has been read, the cut is there
      if (tid == 0) sh.n_listed = 0u;
      return Cut{sh.cut_key, sh.cut_ties};
    }
    // the keys of that bucket: [smallest key in a bucket <= b0, smallest key in a bucket < b0), 32 probes at a time
    auto smallest = [&](uint32_t bucket) {              // smallest key of a number whose bucket is at most `bucket`
      uint32_t a = kLowestKey, z = w.top;               // the answer lies in [a, z]
      while (a < z) {
        const uint32_t step = (z - a) / 33u + 1u;
        const uint32_t at = z - a > step * (uint32_t)lane ? a + step * (uint32_t)lane : z;
        const uint32_t yes = __ballot_sync(0xffffffffu, linear(at, sc) <= bucket);
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
    uint32_t lo = smallest(b0), hi = b0 == 0u ? w.top : smallest(b0 - 1u) - 1u;
    while (lo < hi) {
      const int shift = max(0, 21 - __clz(hi - lo));     // 2048 buckets over the range
      auto bucket_of = [&](uint32_t k) { return (hi - k) >> shift; };
      const u64 want = wanted;
      search([&](const uint32_t* four) {
#pragma unroll
               for (int i = 0; i < 4; ++i) {
                 const uint32_t k = four[i];
                 if (k < lo || k > hi || k <= cut.key) continue;
                 if (counting) atomicAdd(&sh.low[bucket_of(k)], 1u);
                 else if (const u64 f = w.fixed_of(k)) sh.add(bucket_of(k), f);
               }
             },
             [&] {
               if (!counting && cut.ties && cut.key >= lo && cut.key <= hi) sh.add(bucket_of(cut.key), w.fixed_of(cut.key) * cut.ties);
             },
             [&](u64) { return want; });
      wanted = sh.rest;
      const uint32_t b = sh.bucket, old = hi;
      hi = old - (b << shift);
      const uint32_t width = (1u << shift) - 1u;
      lo = max(lo, hi > width ? hi - width : 0u);
      __syncthreads();                                   // (the found bucket has been read)
    }
    if (counting) return Cut{lo, (uint32_t)wanted};
    const u64 each = w.fixed_of(lo);
    u64 ties = each ? (wanted + each - 1) / each : 1ull;
    if (lo == cut.key && ties > cut.ties) ties = cut.ties;
    return Cut{lo, (uint32_t)min(max(ties, 1ull), 0xffffffffull)};
  };

  Cut cut{0u, 0u};
  const float top_p = p.top_ps ? p.top_ps[row] : p.top_p;
  auto nucleus = [&](u64 total) -> u64 { return (u64)ceil((double)fmaxf(top_p, 0.0f) * (double)total); };
  const int top_k = p.top_ks ? p.top_ks[row] : p.top_k;
  if (top_k > 0 && top_k < p.vocab) {
    const float sc = linear_of(value_of(low));
    search([&](const uint32_t* k) {
#pragma unroll
             for (int i = 0; i < 4; ++i)
               if (k[i]) atomicAdd(&sh.low[linear(k[i], sc)], 1u);
           },
           [] {}, [&](u64) { return (u64)top_k; });
    if (sh.above + sh.in_bucket <= kMaxPairs) {
      // few enough to finish on a list: ranks, the nucleus, and the draw in index order, by comparing all pairs
      const uint32_t b0 = sh.bucket;
      const int n = (int)collect([&](uint32_t k) { return linear(k, sc) <= b0; });
      if (rank == 0) {
        const u64* all = sh.all_listed();
        const u64 me = tid < n ? all[tid] : 0ull;
        const uint32_t key = (uint32_t)(me >> 32);
        const u64 mine = tid < n ? w.fixed_of(key) : 0ull;
        if (tid < n) sh.pair_weight[tid] = mine;
        __syncthreads();
        u64 before = 0;
        int ahead = 0;
        if (tid < n)
          for (int j = 0; j < n; ++j)
            if (all[j] > me) { before += sh.pair_weight[j]; ++ahead; }
        const bool ranked = tid < n && ahead < top_k;
        auto block_sum = [&](u64 v) -> u64 {
          v = warp_sum(v);
          __syncthreads();
          if (lane == 0) sh.warp_sum[warp] = v;
          __syncthreads();
          u64 s = 0;
#pragma unroll
          for (int i = 0; i < kMaxPairs / 32; ++i) s += sh.warp_sum[i];
          return s;
        };
        const u64 reach = top_p < 1.0f ? nucleus(block_sum(ranked ? mine : 0ull)) : ~0ull;
        const bool kept = ranked && (ahead == 0 || before < reach);
        const u64 drawn = kept ? w.drawn(key) : 0ull;
        const u64 total = block_sum(drawn);
        if (tid < n) sh.pair_weight[tid] = drawn;
        __syncthreads();
        const u64 target = draw_target(total);
        if (drawn) {
          u64 run = 0;
          for (int j = 0; j < n; ++j)
            if ((uint32_t)all[j] > (uint32_t)me) run += sh.pair_weight[j];       // of lower index
          if (run <= target && target < run + drawn) {
            p.tokens[row] = (int64_t)(uint32_t)~(uint32_t)me;
            if (p.probabilities) p.probabilities[row] = (float)(w.scaled(key) / (double)total);
          }
        }
      }
      cluster.sync();
      return;
    }
    cut = resolve(sc, true, Cut{0u, 0u});
  }
  if (top_p < 1.0f) {
    const float sc = linear_of(fmaxf(value_of(low), w.top_value - 34.0f * t));
    const Cut by_rank = cut;
    search([&](const uint32_t* k) {
             u64 f[4];                     // all four ahead of the first atomic, which the table's loads cannot pass
#pragma unroll
             for (int i = 0; i < 4; ++i) f[i] = w.fixed_of(k[i]);
#pragma unroll
             for (int i = 0; i < 4; ++i)
               if (k[i] > by_rank.key && f[i]) sh.add(linear(k[i], sc), f[i]);
           },
           [&] { if (by_rank.ties) sh.add(linear(by_rank.key, sc), w.fixed_of(by_rank.key) * by_rank.ties); },
           nucleus);
    cut = resolve(sc, false, by_rank);
  }

  // ---- the draw: sums per warp segment in index order, then the segment, then the token ----
  const u64 tie_weight = cut.key ? w.drawn(cut.key) : 0ull;
  const int seg_len = ((slice + kWarps * 128 - 1) / (kWarps * 128)) * 128;
  const int s0 = min(slice, warp * seg_len), s1 = min(slice, s0 + seg_len);
  {
    u64 sum = 0;
    uint32_t ties = 0;
    each_four(s0, s1, lane, 32, [&](const uint32_t* k, int) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u64 f = w.drawn(k[i]);
        sum += k[i] > cut.key ? f : 0ull;
        ties += k[i] == cut.key;
      }
    });
    if (cut.key == 0u) ties = 0u;
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
      const uint32_t k = key_at(s0 + j);
      const u64 f = w.drawn(k);
      sum += k > cut.key ? f : 0ull;
      ties += k == cut.key;
    }
    if (cut.key == 0u) ties = 0u;
    const uint32_t before = tb + (uint32_t)(warp_scan(ties, lane) - ties);
    const uint32_t left = cut.ties > before ? cut.ties - before : 0u;
    sum += tie_weight * (u64)min(ties, left);
    const u64 incl = warp_scan(sum, lane);
    const int at = __ffs(__ballot_sync(0xffffffffu, incl > rest)) - 1;
    rest -= __shfl_sync(0xffffffffu, incl - sum, at);
    tb = __shfl_sync(0xffffffffu, before, at);
    const int c0 = __shfl_sync(0xffffffffu, a0, at), c1 = __shfl_sync(0xffffffffu, a1, at);
    for (int j = c0; j < c1; j += 32) {
      const uint32_t k = j + lane < c1 ? key_at(s0 + j + lane) : 0u;
      const bool tie = k && k == cut.key;
      const uint32_t tied = __ballot_sync(0xffffffffu, tie);
      u64 f = 0;
      if (k > cut.key) f = w.drawn(k);
      else if (tie && tb + __popc(tied & ((1u << lane) - 1u)) < cut.ties) f = tie_weight;
      const u64 run = warp_scan(f, lane);
      const uint32_t hit = __ballot_sync(0xffffffffu, run > rest);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          p.tokens[row] = begin + s0 + j + lane;
          if (p.probabilities) p.probabilities[row] = (float)(w.scaled(k) / (double)sh.total);
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
  const int64_t room = (int64_t)(110 * 1024 - fixed) / 4;      // keys of a slice, with two CTAs on an SM
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
