// Choice of the next token from a row of logits with temperature, top-k, top-p, min-p and a given random number (sm_100a).
//
// With w_i = e^((x_i - max) / T) a token is kept when its rank is below k, when the weights ahead of it (larger ones, and
// equal ones of lower index) sum to less than p times the weight of the first k, and when w_i >= min_p; the result is the
// first kept index whose running sum, in index order, exceeds u times the kept weight.
//
// A row is read once: a cluster of up to eight CTAs shares it and each keeps its slice in shared memory as ordered 32-bit
// keys (rows too long for that are read again from L2 instead).  No sort: the rank and the sum are thresholds on the
// value, found by histograms over ever narrower ranges of keys -- 2048 buckets, the first round linear in the value so
// that the bulk of a row does not meet in a few buckets -- and what is left at the threshold itself are equal values,
// taken in index order.  Each round ends in one cluster barrier.
// Weights are whole numbers, round(w 2^46) (fewer bits for a vocabulary whose sum would pass 2^62): sums are then exact,
// the same in any order, so atomics cannot change the result.  A weight is off by at most 2^-47 of the largest and a
// running sum by some 2^-47 sqrt(V), while u has 24 bits; 32-bit weights would move one choice in a thousand.  Exponentials
// are 64-bit, and the part of a row that is below 2^-47 is skipped ahead of them.
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

struct Shared {
  u64 hist[2][kBuckets];
  u64 coarse[2][kCoarse];
  u64 seg_sum[kWarps];
  uint32_t seg_ties[kWarps];
  uint32_t top, low, first;            // this CTA's part of a cluster-wide maximum, minimum, first index
  uint32_t warp_a[kWarps], warp_b[kWarps];
  // what one warp found for all
  uint32_t bucket, all_top, all_low, all_first;
  u64 above, total, rest;
  int seg;
  uint32_t seg_tie_base;
};

// Kept: keys above `key`, and the first `ties` of those equal to it.
struct Cut {
  uint32_t key, ties;
};

struct Row {
  uint32_t top;            // largest key
  float top_value;
  double top_wide, inv_t;
  float inv_t32;
  int bits;                // fraction bits of a weight
  float min_p;
  __device__ double weight(uint32_t k) const {
    if (k == top) return 1.0;
    if (k == 0u || isinf(top_value)) return 0.0;
    const float x = value_of(k);
    if ((x - top_value) * inv_t32 < -34.0f) return 0.0;     // rounds to zero
    return exp(((double)x - top_wide) * inv_t);
  }
  __device__ u64 fixed(double w) const { return (u64)(w * (double)(1ull << bits) + 0.5); }
  __device__ u64 fixed_of(uint32_t k) const { return fixed(weight(k)); }
  __device__ u64 drawn(uint32_t k) const {                  // weight in the final draw: min_p applied
    const double w = weight(k);
    return k == top || w >= (double)min_p ? fixed(w) : 0ull;
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

  // ---- read the slice; largest and smallest key ----
  uint32_t top = 0u, low = 0xffffffffu;
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
    if (lane == 0) { sh.top = top; sh.low = low; }
  }
  cluster.sync();
  if (warp == 0) {
    const Shared* r = cluster.map_shared_rank(&sh, lane < nc ? lane : 0);
    top = __reduce_max_sync(0xffffffffu, r->top);
    low = __reduce_min_sync(0xffffffffu, r->low);
    if (lane == 0) { sh.all_top = top; sh.all_low = low; }
  }
  __syncthreads();
  top = sh.all_top;
  low = sh.all_low;

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
  w.inv_t = 1.0 / (double)t;
  w.inv_t32 = (float)w.inv_t;
  w.bits = min(46, 62 - (64 - __clzll((long long)p.vocab)));
  w.min_p = p.min_ps ? p.min_ps[row] : p.min_p;
  w.min_p = w.min_p > 0.0f ? fminf(w.min_p, 1.0f) : 0.0f;

  int round = 0;
  // One round: `add(key, hist)` for this CTA's keys and `once(hist)` for the cluster, then the bucket in which the running
  // sum (bucket 0 first) reaches the target.  target_of(total) gives the target from the round's total.
  auto search = [&](auto&& add, auto&& once, auto&& target_of) {
    const int par = round & 1;
    ++round;
    u64* hist = sh.hist[par];
    for (int i = tid; i < kBuckets; i += kThreads) hist[i] = 0ull;
    __syncthreads();
    if (rank == 0 && tid == 0) once(hist);
    for (int j = tid; j < slice; j += kThreads) add(key_at(j), hist);
    __syncthreads();
    for (int c = warp; c < kCoarse; c += kWarps) {
      const u64 s = warp_sum(hist[c * 32 + lane]);
      if (lane == 0) sh.coarse[par][c] = s;
    }
    cluster.sync();
    if (warp == 0) {
      u64 a = 0, b = 0;
      for (int r = 0; r < nc; ++r) {
        const u64* q = cluster.map_shared_rank(&sh, r)->coarse[par];
        a += q[2 * lane];
        b += q[2 * lane + 1];
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
      for (int r = 0; r < nc; ++r) f += cluster.map_shared_rank(&sh, r)->hist[par][c * 32 + lane];
      const u64 fi = warp_scan(f, lane);
      const int fl = __ffs(__ballot_sync(0xffffffffu, above + fi >= target)) - 1;
      if (lane == fl) {
        sh.bucket = (uint32_t)(c * 32 + fl);
        sh.above = above + fi - f;
        sh.total = total;
        sh.rest = target - (above + fi - f);       // how much of the bucket is wanted
      }
    }
    __syncthreads();
  };
  // Narrows [lo, hi] until one key is left: the key at which the sum of `amount(key)` over the kept keys, largest first,
  // reaches the target; returns what is wanted of that key's own group.
  auto threshold = [&](float x_low, bool counting, Cut cut, auto&& target_of, uint32_t* key) -> u64 {
    const float span = w.top_value - x_low;
    const float sc = span > 0.0f && span < CUDART_INF_F ? (float)kBuckets / span : 0.0f;
    auto linear = [&](uint32_t k) -> uint32_t {         // never increases with the key
      const float v = (w.top_value - value_of(k)) * sc;
      return v >= (float)(kBuckets - 1) ? kBuckets - 1 : (uint32_t)(int)v;      // NaN (infinite top) becomes bucket 0
    };
    auto amount = [&](uint32_t k, u64* slot) {
      if (counting) atomicAdd(reinterpret_cast<unsigned int*>(slot), 1u);       // the low word: counts stay below 2^31
      else if (const u64 f = w.fixed_of(k)) atomicAdd(slot, f);
    };
    auto cut_ties = [&](uint32_t lo, uint32_t hi, auto&& bucket_of, u64* hist) {  // the kept ones of the earlier cut, together
      if (!counting && cut.ties && cut.key >= lo && cut.key <= hi) {
        const u64 f = w.fixed_of(cut.key) * cut.ties;
        if (f) atomicAdd(&hist[bucket_of(cut.key)], f);
      }
    };
    search([&](uint32_t k, u64* hist) { if (k > cut.key) amount(k, &hist[linear(k)]); },
           [&](u64* hist) { cut_ties(kLowestKey, w.top, linear, hist); }, target_of);
    const uint32_t b0 = sh.bucket;
    u64 wanted = sh.rest;
    // the keys of that bucket: [smallest key in a bucket <= b0, smallest key in a bucket < b0), 32 probes at a time
    auto smallest = [&](uint32_t bucket) {              // smallest key of a number whose bucket is at most `bucket`
      uint32_t a = kLowestKey, z = w.top;                       // the answer lies in [a, z]
      while (a < z) {
        const uint32_t step = (z - a) / 33u + 1u;
        const uint32_t at = z - a > step * (uint32_t)lane ? a + step * (uint32_t)lane : z;
        const uint32_t yes = __ballot_sync(0xffffffffu, linear(at) <= bucket);
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
      search([&](uint32_t k, u64* hist) { if (k >= lo && k <= hi && k > cut.key) amount(k, &hist[bucket_of(k)]); },
             [&](u64* hist) { cut_ties(lo, hi, bucket_of, hist); }, [&](u64) { return want; });
      wanted = sh.rest;
      const uint32_t b = sh.bucket, old = hi;
      hi = old - (b << shift);
      const uint32_t width = (1u << shift) - 1u;
      lo = max(lo, hi > width ? hi - width : 0u);
    }
    *key = lo;
    return wanted;
  };

  Cut cut{0u, 0u};
  const int top_k = p.top_ks ? p.top_ks[row] : p.top_k;
  if (top_k > 0 && top_k < p.vocab) {
    uint32_t key;
    const u64 ties = threshold(value_of(low), true, Cut{0u, 0u}, [&](u64) { return (u64)top_k; }, &key);
    cut = Cut{key, (uint32_t)ties};
  }
  const float top_p = p.top_ps ? p.top_ps[row] : p.top_p;
  if (top_p < 1.0f) {
    uint32_t key;
    const float reach = 34.0f * t;
    const float x_low = fmaxf(value_of(low), w.top_value - reach);
    const u64 weight = threshold(x_low, false, cut, [&](u64 total) { return (u64)ceil((double)fmaxf(top_p, 0.0f) * (double)total); }, &key);
    const u64 each = w.fixed_of(key);
    u64 ties = each ? (weight + each - 1) / each : 1ull;
    if (ties < 1) ties = 1;
    if (key == cut.key && ties > cut.ties) ties = cut.ties;
    cut = Cut{key, (uint32_t)min(ties, 0xffffffffull)};
  }

  // ---- the draw: sums per warp segment in index order, then the segment, then the token ----
  const u64 tie_weight = cut.key ? w.drawn(cut.key) : 0ull;
  const int seg_len = ((slice + kWarps * 32 - 1) / (kWarps * 32)) * 32;
  const int s0 = min(slice, warp * seg_len), s1 = min(slice, s0 + seg_len);
  {
    u64 sum = 0;
    uint32_t ties = 0;
    for (int j = s0 + lane; j < s1; j += 32) {
      const uint32_t k = key_at(j);
      if (k > cut.key) sum += w.drawn(k);
      else if (k && k == cut.key) ++ties;
    }
    sum = warp_sum(sum);
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) { sh.seg_sum[warp] = sum; sh.seg_ties[warp] = ties; }
  }
  cluster.sync();
  if (warp == 0) {
    // lane l holds the segments l * per ... of the cluster's nc * kWarps, in index order
    const int n_seg = nc * kWarps, per = (n_seg + 31) / 32;
    u64 mine = 0;
    uint32_t ties = 0;
    for (int i = 0; i < per; ++i) {
      const int sg = lane * per + i;
      if (sg < n_seg) ties += cluster.map_shared_rank(&sh, sg / kWarps)->seg_ties[sg % kWarps];
    }
    const uint32_t ties_before = (uint32_t)(warp_scan(ties, lane) - ties);
    uint32_t tb = ties_before;
    for (int i = 0; i < per; ++i) {
      const int sg = lane * per + i;
      if (sg >= n_seg) break;
      const Shared* r = cluster.map_shared_rank(&sh, sg / kWarps);
      const uint32_t n = r->seg_ties[sg % kWarps], left = cut.ties > tb ? cut.ties - tb : 0u;
      mine += r->seg_sum[sg % kWarps] + tie_weight * (u64)min(n, left);
      tb += n;
    }
    const u64 incl = warp_scan(mine, lane);
    const u64 total = __shfl_sync(0xffffffffu, incl, 31);
    float u = p.uniforms[row];
    u = u > 0.0f ? u : 0.0f;
    u64 target = u < 1.0f ? (u64)((double)u * (double)total) : total;      // the running sum has to exceed this
    if (target >= total) target = total - 1;
    const int at = __ffs(__ballot_sync(0xffffffffu, incl > target)) - 1;
    if (lane == at) {
      u64 before = incl - mine;
      tb = ties_before;
      int found = -1;
      for (int i = 0; i < per && found < 0; ++i) {
        const int sg = lane * per + i;
        if (sg >= n_seg) break;
        const Shared* r = cluster.map_shared_rank(&sh, sg / kWarps);
        const uint32_t n = r->seg_ties[sg % kWarps], left = cut.ties > tb ? cut.ties - tb : 0u;
        const u64 here = r->seg_sum[sg % kWarps] + tie_weight * (u64)min(n, left);
        if (before + here > target) found = sg;
        else { before += here; tb += n; }
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
    for (int j = a0; j < a1; ++j) {
      const uint32_t k = key_at(s0 + j);
      if (k > cut.key) sum += w.drawn(k);
      else if (k && k == cut.key) ++ties;
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
          if (p.probabilities) p.probabilities[row] = (float)(w.weight(k) * (double)(1ull << w.bits) / (double)sh.total);
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
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
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
