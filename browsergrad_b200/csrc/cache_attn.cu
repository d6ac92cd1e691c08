// Launch planning of the attention over a cache, and the per-block document ranges it skips keys by.
#include <math.h>

#include "cache_attn.cuh"

namespace bg {
namespace {

// Smallest and largest id of each 128 keys (ids below zero belong to no document, see DecoderAttention::doc_ranges).
// One warp per block.
__global__ void doc_ranges_kernel(const int* documents, int b, int sk, int blocks, int2* ranges) {
  grid_launch_dependents();
  const long long w = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  if (w >= (long long)b * blocks) return;
  const int batch = (int)(w / blocks), blk = (int)(w % blocks), lane = threadIdx.x & 31;
  int lo = INT_MAX, hi = -1;
  bool none = false;
  for (int i = lane; i < kDocBlock; i += 32) {
    const int key = blk * kDocBlock + i;
    const int id = key < sk ? documents[(long long)batch * sk + key] : -1;
    if (id >= 0) { lo = min(lo, id); hi = max(hi, id); }
    else none = true;
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  none = __any_sync(0xffffffffu, none);
  if (lane == 0) ranges[w] = make_int2(none ? lo | (int)0x80000000 : lo, hi);
}

}  // namespace

cudaError_t launch_doc_ranges(const int* documents, int b, int sk, int2* ranges, cudaStream_t s) {
  const int blocks = (sk + kDocBlock - 1) / kDocBlock;
  const long long warps = (long long)b * blocks;
  doc_ranges_kernel<<<(unsigned)((warps + 7) / 8), 256, 0, s>>>(documents, b, sk, blocks, ranges);
  return cudaGetLastError();
}

CacheAttnPlan cache_attention_plan(const DecoderAttention& p, int dtype, int sm_count) {
  CacheAttnPlan plan;
  const int rows = p.group * p.sq;
  plan.row_tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const int per_cta = 16 * plan.row_tiles;
  const long long units = (long long)p.b * p.hkv * ((rows + per_cta - 1) / per_cta);
  // How many CTAs share the keys: the number estimated to take the least time, in keys that an SM slot works through.  A
  // CTA costs its keys and about 384 more (start, join of its groups, partial result), the kernel that joins the splits
  // about 700.  Sequences of equal length run in whole rounds of CTAs; with one row tile the memory is the bound, and three
  // quarters of the slots draw nearly all of it (64 sets of 2048 keys of 128, bf16: 34 us in one part each, 20 in the four it
  // takes; 256 sets of 2048: 50 in the one it takes, 57 in three; 256 of 8192: 177 in the three it takes, where one would be
  // 166).  Where lengths are given they are taken to differ: few CTAs then wait for the longest (a third more), three rounds of
  // not too short ones even out (32 sequences of about 5000 of 8192 keys, 8 key heads: 155 us in two parts each, 128 in six; one
  // of 131077, 4 key heads of two row tiles: 89 us in 112 parts, 79 in 37, 65 in the 74 of one round).  Heads above 128 run one
  // CTA an SM, and so do few rows of fp32 heads above 64; counting two there costs up to 8 % on the longest caches (131072 keys,
  // 8 heads of 256, bf16: 219 us, with one 202) and gains as much on 8192 keys (24.0, with one 26.6).
  const int head = cache_attn::padded_head(p.d);
  // Keys that a group of warps adds one after another.  The tensor core adds with truncation, which makes results of 16-bit
  // operands smaller by some 10^-7 for every 16 keys: 10^-4 after 16384, a fifth of the half step of float16 (500000 keys in two
  // groups lost 1.6 * 10^-3); bfloat16 stands eight times as many.  fp32 tiles are added in 32 bits.
  const long long group_keys = dtype == BG_F16 ? 16384 : dtype == BG_BF16 ? 131072 : (long long)1 << 40;
  const int groups = (plan.row_tiles == 4 && head <= 128) || head <= 64 ? 8 / plan.row_tiles : 4 / plan.row_tiles;
  const long long least = p.sk <= groups * group_keys ? 1 : (p.sk + groups * group_keys - 1) / (groups * group_keys);
  const double slots = (plan.row_tiles == 1 && dtype != BG_F32 && head > 64 && head <= 128 ? 3.0 : 2.0) * sm_count;      // CTAs that run at once
  long long splits = 1, most = (p.sk + 511) / 512;
  if (most > 128) most = 128;
  if (most < least) most = least;
  double best = 1e300;
  for (long long s = least; s <= most; ++s) {
    const double keys = (double)p.sk / (double)s, cta = keys + 384.0, ctas = (double)(units * s);
    const double rounds = ceil(ctas / slots);
    double t = plan.row_tiles == 1 ? fmax(ctas * cta / slots, 0.75 * cta * rounds) : rounds * cta;
    if (p.lengths) t = ctas >= 3.0 * slots && keys >= 1024.0 ? ctas * cta / slots + 0.25 * cta : 1.3 * rounds * cta;
    if (s > 1) t += 700.0;
    if (t < best) { best = t; splits = s; }
  }
  plan.splits = (int)splits;
  plan.partial_bytes = splits > 1 ? units * splits * per_cta * (cache_attn::padded_head(p.d) + 2) * 4 : 0;
  return plan;
}

cudaError_t launch_cache_attention(const DecoderAttention& p, int dtype, const CacheAttnPlan& plan, float* partials, cudaStream_t s) {
  if (dtype == BG_BF16) return cache_attn::launch_bf16(p, plan, partials, s);
  if (dtype == BG_F16) return cache_attn::launch_f16(p, plan, partials, s);
  return cache_attn::launch_f32(p, plan, partials, s);
}

}  // namespace bg
