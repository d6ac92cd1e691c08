// Attention of fp32 prompts over a cache, head dimensions up to 64 (sm_100a): the rules of cache_attn.cuh with every
// contraction as three tf32 products on the tensor cores.
//
// The structure is that of the fp32 attention of a plan (attn_tf32_row.cu): one CTA owns 128 query rows of a head and
// walks tiles of 64 keys; Q, K and V arrive as the caller's rows (TMA), converter warps round them to hi = tf32(x) in place
// and write lo = x - hi; S = lo.hi + hi.lo + hi.hi in a double-buffered accumulator; one thread per query row takes the
// maximum, the exponentials and the sum without exchange and leaves P as hi / lo planes in tensor memory; P V of a key tile
// starts from zero in one of two accumulators and is added to O in registers while the next tile's runs, because the tensor core
// adds with truncation: eight tiles added there, three products each, left a bias of 5 * 10^-6 of the result, this way 3 * 10^-7.
//   warp 0 producer, warp 1 issues the products, warps 2 and 3 convert V, warps 4-7 softmax, warps 8-11 convert Q and K
// What differs is that addition (there O is folded every eight tiles) and what the rules ask: shared key heads, a visible range
// and a document per row instead of a mask tensor, cap and bias, and value rows behind the sequence's length become zeros as
// they are converted.  The cap is the library's tanhf: its error is scaled by the cap into the exponent, and fp32 results are
// held to some 10^-6.
// Rounded to fewer bits than 32: nothing is left out but the products lo.lo and the bits of lo that tf32 drops, 2^-21 of a term.
// Measured: 8 x 12 heads of 1024 tokens of 64, biased, 137 us, causal without bias 132 (the eight-tile sums 141 and 133; 29 us as
// three tf32 products at half the bf16 rate); products and softmax of the one query tile an SM holds take turns.
// No cluster multicast; every wait is clock-bounded.
#include "serving.h"

#include <cuda.h>
#include <math_constants.h>

#include "attn_common.cuh"
#include "prompt_common.cuh"
#include "tc_common.cuh"

namespace bg {
namespace {

using namespace tc;
using namespace prompt;
using attn::ex2_approx;
using attn::fmax3;
using attn::tma_load_4d;

constexpr int kRows = 128, kKeys = 64, kDim = 64, kThreads = 384;
constexpr int kStagesK = 3, kStagesV = 2;        // the converters stand between a K tile and its product: a third stage covers that hop
// planes of a tile: hi values 0-31, hi values 32-63, then lo likewise; a row of 32 values is 128 bytes
constexpr int kQBytes = 4 * kRows * 128, kKBytes = 4 * kKeys * 128, kVBytes = 4 * kKeys * 128;
constexpr int kSmem = kQBytes + kStagesK * kKBytes + kStagesV * kVBytes;
constexpr int kLaunchRegs = 168, kLightRegs = 72, kSoftmaxRegs = 248;
static_assert(256 * kLightRegs + 128 * kSoftmaxRegs <= kLaunchRegs * kThreads, "setmaxnreg requests exceed the CTA's registers");
constexpr int kColS = 0, kColP = 128, kColO = 384;      // 2 x 64, 2 x (hi 64 | lo 64), 2 x 64
constexpr float kLazyLog2 = 8.0f, kLog2e = 1.4426950408889634f;
constexpr uint32_t kVHalf = kKeys * 128;

__device__ __forceinline__ void umma_ts_tf32(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t}"
      :
      : "r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Splits what the TMA unit left in a tile's hi planes: hi = tf32(x) in place, lo = x - hi behind.  Rows of 128 bytes from
// `rows` on (of each plane's kKeys) become zeros.
template <int THREADS, bool CUT>
__device__ __forceinline__ void split_planes(unsigned char* planes, int bytes, int tid, int rows) {
  float4* h = reinterpret_cast<float4*>(planes);
  float4* l = reinterpret_cast<float4*>(planes + bytes);
#pragma unroll 4
  for (int c = tid; c < bytes / 16; c += THREADS) {
    float4 x = h[c];
    if (CUT && ((c >> 3) & (kKeys - 1)) >= rows) x = make_float4(0.f, 0.f, 0.f, 0.f);
    uint32_t w[4];
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(w[0]) : "f"(x.x));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(w[1]) : "f"(x.y));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(w[2]) : "f"(x.z));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(w[3]) : "f"(x.w));
    const float4 hi = make_float4(__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]), __uint_as_float(w[3]));
    h[c] = hi;
    l[c] = make_float4(x.x - hi.x, x.y - hi.y, x.z - hi.z, x.w - hi.w);
  }
}

// Rows of V as an MN-major operand of 32-bit values: 128-byte swizzle of 32-byte pieces, whose pattern repeats every four
// keys (512 bytes, the stride); the second 32 values of a row are a tile of their own (the leading offset).
__device__ __forceinline__ uint64_t make_v_rows_desc(uint32_t smem_addr) {
  return (uint64_t)((smem_addr & 0x3FFFF) >> 4) | (uint64_t)(kVHalf >> 4) << 16 | (uint64_t)(512 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)1 << 61;
}

struct Prompt32Params {
  DecoderAttention a;
  uint32_t idesc_qk, idesc_pv;
};

template <bool CAP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 1)
prompt_attention32_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                          const __grid_constant__ Prompt32Params pp) {
  const DecoderAttention& a = pp.a;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* sQ = smem;
  unsigned char* sK = sQ + kQBytes;
  unsigned char* sV = sK + kStagesK * kKBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + kStagesV * kVBytes);
  uint64_t* q_full = bars;
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + kStagesK;
  uint64_t* v_full = k_empty + kStagesK;
  uint64_t* v_empty = v_full + kStagesV;
  uint64_t* s_full = v_empty + kStagesV;   // [2]
  uint64_t* s_empty = s_full + 2;          // [2]
  uint64_t* p_full = s_empty + 2;          // [2]
  uint64_t* pv_full = p_full + 2;          // [2]
  uint64_t* q_raw = pv_full + 2;           // rows as the caller has them have landed
  uint64_t* k_raw = q_raw + 1;
  uint64_t* v_raw = k_raw + kStagesK;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(v_raw + kStagesV);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  unsigned char* s_need = reinterpret_cast<unsigned char*>(tmem_holder + 4);     // [n_kv]

  if (a.documents) grid_dependency_wait();       // the ranges of their ids come from the launch before
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int n_bh = a.b * a.hq;
  const int q_tile = (a.sq + kRows - 1) / kRows - 1 - (int)(blockIdx.x / (unsigned)n_bh);     // the last rows see the most keys: they go first
  const int bh = (int)(blockIdx.x % (unsigned)n_bh);
  const int b = bh / a.hq, h = bh % a.hq, hk = h / a.group;
  const int q0 = q_tile * kRows;
  const Sequence seq = sequence_of(a, b);
  const int len = seq.len;
  const int n_kv = (len + kKeys - 1) / kKeys;
  const int2* ranges = a.documents ? a.doc_ranges + (long long)b * ((a.sk + kDocBlock - 1) / kDocBlock) : nullptr;
  const int* docs = a.documents ? a.documents + (long long)b * a.sk : nullptr;
  needed_tiles<kKeys>(a, b, seq, q0, min(q0 + kRows, a.sq) - 1, s_need, threadIdx.x, kThreads);
  if (threadIdx.x == 0) {
    mbar_init(q_full, 4);
    mbar_init(q_raw, 1);
    for (int s = 0; s < kStagesK; ++s) { mbar_init(&k_full[s], 4); mbar_init(&k_empty[s], 1); mbar_init(&k_raw[s], 1); }
    for (int s = 0; s < kStagesV; ++s) { mbar_init(&v_full[s], 2); mbar_init(&v_empty[s], 1); mbar_init(&v_raw[s], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], 4);
      mbar_init(&p_full[i], 4); mbar_init(&pv_full[i], 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_holder)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  auto next = [&](int j) { while (j < n_kv && !s_need[j]) ++j; return j; };

  if (warp < 4 || warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLightRegs));
    if (warp == 0) {
      if (lane == 0) {
        mbar_expect_tx(q_raw, kQBytes / 2);
        for (int x = 0; x < 2; ++x) tma_load_4d(&tmQ, sQ + x * (kRows * 128), q_raw, x * 32, q0, h, b);
        int t = 0;
        for (int j = next(0); j < n_kv; j = next(j + 1), ++t) {
          const int s = t % kStagesK;
          if (!mbar_wait(&k_empty[s], ((uint32_t)(t / kStagesK) & 1u) ^ 1u, abort_flag)) break;
          mbar_expect_tx(&k_raw[s], kKBytes / 2);
          for (int x = 0; x < 2; ++x) tma_load_4d(&tmK, sK + s * kKBytes + x * (kKeys * 128), &k_raw[s], x * 32, j * kKeys, hk, b);
        }
      } else if (lane == 1) {
        int t = 0;
        for (int j = next(0); j < n_kv; j = next(j + 1), ++t) {
          const int s = t % kStagesV;
          if (!mbar_wait(&v_empty[s], ((uint32_t)(t / kStagesV) & 1u) ^ 1u, abort_flag)) break;
          mbar_expect_tx(&v_raw[s], kVBytes / 2);
          for (int x = 0; x < 2; ++x) tma_load_4d(&tmV, sV + s * kVBytes + x * kVHalf, &v_raw[s], x * 32, j * kKeys, hk, b);
        }
      }
    } else if (warp == 1) {
      int n_tiles = 0;
      for (int j = 0; j < n_kv; ++j) n_tiles += s_need[j] != 0;
      auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0; };
      const uint32_t q_addr = smem_u32(sQ), idesc_qk = pp.idesc_qk, idesc_pv = pp.idesc_pv;
      auto issue_qk = [&](int t) -> bool {
        const int s = t % kStagesK, buf = t & 1;
        if (t >= 2 && !wait_all(&s_empty[buf], (uint32_t)((t >> 1) - 1) & 1u)) return false;
        if (!wait_all(&k_full[s], (uint32_t)(t / kStagesK) & 1u)) return false;
        tc_fence_after();
        const uint32_t k_addr = smem_u32(sK + s * kKBytes), d_s = tmem_base + (uint32_t)(kColS + buf * kKeys);
        if (elect_one()) {
#pragma unroll
          for (int pass = 0; pass < 3; ++pass) {          // lo.hi, hi.lo, hi.hi: small terms first
            const uint32_t qa = q_addr + (pass == 0 ? 2 * (kRows * 128) : 0), ka = k_addr + (pass == 1 ? 2 * (kKeys * 128) : 0);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const uint64_t da = make_kmajor_sw128_desc(qa + x * (kRows * 128)), db = make_kmajor_sw128_desc(ka + x * (kKeys * 128));
#pragma unroll
              for (int k = 0; k < 4; ++k) umma<true>(d_s, da + (uint64_t)(k * 2), db + (uint64_t)(k * 2), idesc_qk, (pass | x | k) ? 1u : 0u);
            }
          }
          umma_commit(&s_full[buf]);
          umma_commit(&k_empty[s]);
        }
        __syncwarp();
        return true;
      };
      auto issue_pv = [&](int t) -> bool {
        const int s = t % kStagesV, buf = t & 1;
        if (!wait_all(&p_full[buf], (uint32_t)(t >> 1) & 1u)) return false;
        if (!wait_all(&v_full[s], (uint32_t)(t / kStagesV) & 1u)) return false;
        tc_fence_after();
        const uint32_t v_addr = smem_u32(sV + s * kVBytes), t_p = tmem_base + (uint32_t)(kColP + buf * 2 * kKeys), d_o = tmem_base + (uint32_t)(kColO + buf * kDim);
        if (elect_one()) {
#pragma unroll
          for (int pass = 0; pass < 3; ++pass) {
            const uint32_t pa = t_p + (pass == 0 ? (uint32_t)kKeys : 0u), va = v_addr + (pass == 1 ? 2 * kVHalf : 0);
#pragma unroll
            for (int g = 0; g < 8; ++g)      // groups of 8 keys
              umma_ts_tf32(d_o, pa + (uint32_t)(g * 8), make_v_rows_desc(va + (uint32_t)(g * 1024)), idesc_pv, (pass | g) ? 1u : 0u);
          }
          umma_commit(&pv_full[buf]);
          umma_commit(&v_empty[s]);
        }
        __syncwarp();
        return true;
      };
      bool ok = n_tiles == 0 || wait_all(q_full, 0);
      if (ok && n_tiles > 0) ok = issue_qk(0);
      if (ok && n_tiles > 1) ok = issue_qk(1);
      for (int t = 0; t < n_tiles && ok; ++t) {
        if (t + 2 < n_tiles) ok = issue_qk(t + 2);
        if (ok) ok = issue_pv(t);
      }
    } else if (warp >= 8) {
      const int tid = (int)threadIdx.x - 256;
      auto publish = [&](uint64_t* bar) {
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
      };
      bool ok = __all_sync(0xffffffffu, mbar_wait(q_raw, 0, abort_flag)) != 0;
      if (ok) {
        split_planes<128, false>(sQ, kQBytes / 2, tid, 0);
        publish(q_full);
      }
      int t = 0;
      for (int j = next(0); j < n_kv && ok; j = next(j + 1), ++t) {
        const int s = t % kStagesK;
        ok = __all_sync(0xffffffffu, mbar_wait(&k_raw[s], (uint32_t)(t / kStagesK) & 1u, abort_flag)) != 0;
        if (!ok) break;
        split_planes<128, false>(sK + s * kKBytes, kKBytes / 2, tid, 0);
        publish(&k_full[s]);
      }
    } else {
      const int tid = (int)threadIdx.x - 64;
      bool ok = true;
      int t = 0;
      for (int j = next(0); j < n_kv && ok; j = next(j + 1), ++t) {
        const int s = t % kStagesV;
        ok = __all_sync(0xffffffffu, mbar_wait(&v_raw[s], (uint32_t)(t / kStagesV) & 1u, abort_flag)) != 0;
        if (!ok) break;
        // rows behind the sequence: a probability of zero times what an unwritten cache holds would not be zero
        if (j * kKeys + kKeys > len) split_planes<64, true>(sV + s * kVBytes, kVBytes / 2, tid, len - j * kKeys);
        else split_planes<64, false>(sV + s * kVBytes, kVBytes / 2, tid, 0);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[s]);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int quarter = warp & 3, row = q0 + quarter * 32 + lane;
    const bool row_ok = row < a.sq;
    const uint32_t lane_sel = (uint32_t)(quarter * 32) << 16;
    float o[kDim];                                   // the key tiles added so far, relative to m_ref
#pragma unroll
    for (int d = 0; d < kDim; ++d) o[d] = 0.f;
    float m_ref = -CUDART_INF_F, l = 0.f;            // in powers of two
    const Reach me = reach_of(a, seq, row, row_ok ? row : row - 1);
    int hi = me.keys, doc = -1;
    if (docs) {
      doc = me.keys > 0 && me.first >= 0 && me.first < a.sk ? __ldg(docs + me.first) : -1;
      if (doc < 0) hi = 0;
    }
    const int pos = distance_origin(seq, me.first);
    const float slope = BIAS && a.slopes ? a.slopes[h] * kLog2e : 0.f;
    const float to_log2 = CAP ? a.cap * kLog2e : a.scale * kLog2e, to_cap = CAP ? a.scale / a.cap : 0.f;
    constexpr bool FOLD = !CAP && !BIAS;             // the scale is applied in the exponent (it is positive then)
    bool ok = true;
    int t = 0;
    auto wait_warp = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0; };
    // Adds P V of tile u, once it has completed, and takes the sum to the reference that tile u + 1 set.
    auto add_tile = [&](int u, float alpha) -> bool {
      if (!wait_warp(&pv_full[u & 1], (uint32_t)(u >> 1) & 1u)) return false;
      tc_fence_after();
      const uint32_t t_o = tmem_base + (uint32_t)(kColO + (u & 1) * kDim) + lane_sel;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t r[32];
        tmem_ld32(t_o + (uint32_t)(half * 32), r);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[half * 32 + i] = __fadd_rn(o[half * 32 + i], __uint_as_float(r[i]));
      }
      if (__any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll
        for (int d = 0; d < kDim; ++d) o[d] *= alpha;
      }
      tc_fence_before();
      return true;
    };
    for (int j = 0; j < n_kv && ok; ++j) {
      if (!s_need[j]) continue;
      const int buf = t & 1, k0 = j * kKeys;
      bool whole = hi >= k0 + kKeys;
      if (docs) {
        const int2 x = __ldg(ranges + k0 / kDocBlock);
        whole = whole && x.x == doc && x.y == doc;
      }
      const bool hide = !__all_sync(0xffffffffu, whole);
      uint32_t w[2] = {0xffffffffu, 0xffffffffu};         // the keys seen, made while the scores are
      if (hide) {
        const int n = min(max(hi - k0, 0), kKeys);
        w[0] = n >= 32 ? 0xffffffffu : (1u << n) - 1u;
        w[1] = n >= 64 ? 0xffffffffu : n <= 32 ? 0u : (1u << (n - 32)) - 1u;
        if (docs) {
          const uint4 mine = document_bits(docs + k0, min(a.sk - k0, kKeys), doc);
          w[0] &= mine.x;
          w[1] &= mine.y;
        }
      }
      ok = wait_warp(&s_full[buf], (uint32_t)(t >> 1) & 1u);
      if (!ok) break;
      tc_fence_after();
      float x[kKeys];
      {
        uint32_t* xu = reinterpret_cast<uint32_t*>(x);
        const uint32_t t_s = tmem_base + (uint32_t)(kColS + buf * kKeys) + lane_sel;
        tmem_ld32_issue(t_s, xu);
        tmem_ld32_issue(t_s + 32, xu + 32);
        tmem_ld_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_empty[buf]);
      if (CAP) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i) x[i] = to_log2 * tanhf(x[i] * to_cap);
      } else if (BIAS) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i) x[i] *= to_log2;
      }
      if (BIAS) {
        const float gap = (float)(pos - k0);
#pragma unroll
        for (int i = 0; i < kKeys; ++i) x[i] = fmaf(-slope, fabsf(gap - (float)i), x[i]);
      }
      if (hide) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
          if (!((w[i >> 5] >> (i & 31)) & 1u)) x[i] = -CUDART_INF_F;
      }
      float mt;
      {
        float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int i = 4; i < kKeys; i += 2) mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], x[i], x[i + 1]);
        mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (FOLD) mt *= to_log2;
      }
      const bool coarse = FOLD && fabsf(mt) >= kCoarse && mt != -CUDART_INF_F;
      const bool raise = m_ref != -CUDART_INF_F && mt - m_ref > kLazyLog2;
      float unit = to_log2;                           // FOLD: what the scores are still to be multiplied by
      if (FOLD && __any_sync(0xffffffffu, coarse)) {
#pragma unroll
        for (int i = 0; i < kKeys; ++i) x[i] *= to_log2;
        unit = 1.0f;
      }
      const float alpha = raise ? ex2_approx(m_ref - mt) : 1.0f;
      if (raise) { l *= alpha; m_ref = mt; }
      if (m_ref == -CUDART_INF_F) m_ref = mt;
      const float off = m_ref == -CUDART_INF_F ? 0.f : -m_ref;
      {
        float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kKeys; ++i) {
          x[i] = ex2_approx(FOLD ? fmaf(x[i], unit, off) : x[i] + off);
          ps[i & 3] += x[i];
        }
        l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
      }
      {
        // (P V of tile t - 2, which read this buffer, has been added)
        const uint32_t t_p = tmem_base + (uint32_t)(kColP + buf * 2 * kKeys) + lane_sel;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t ph[32], pl[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float v = x[half * 32 + i];
            asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(ph[i]) : "f"(v));
            pl[i] = __float_as_uint(v - __uint_as_float(ph[i]));
          }
          tmem_st32_issue(t_p + (uint32_t)(half * 32), ph);
          tmem_st32_issue(t_p + (uint32_t)(kKeys + half * 32), pl);
        }
        tmem_st_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[buf]);
      if (t > 0) ok = add_tile(t - 1, alpha);         // while P V of this tile runs
      ++t;
    }
    if (ok && t > 0) ok = add_tile(t - 1, 1.0f);
    if (ok) {
      if (row_ok) {
        const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);      // a row without keys is zero; NaN stays NaN
        float* out = reinterpret_cast<float*>(const_cast<void*>(a.out.ptr)) + b * a.out.sb + (long long)h * a.out.sh + (long long)row * a.out.sr;
#pragma unroll
        for (int d = 0; d < kDim; d += 4)
          if (d < a.d) *reinterpret_cast<float4*>(out + d) = l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o[d] * inv, o[d + 1] * inv, o[d + 2] * inv, o[d + 3] * inv);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) { *a.status.host = kStatusPromptWait; *a.status.device = kStatusPromptWait; }
    const long long t0 = clock64();
    while (clock64() - t0 < 200000) {}
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
  }
}

size_t smem_bytes(int sk) { return (size_t)kSmem + 1024 + 256 + (size_t)((sk + kKeys - 1) / kKeys); }

template <bool CAP, bool BIAS>
cudaError_t launch_kernel(const Prompt32Params& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
  auto kern = prompt_attention32_kernel<CAP, BIAS>;
  static const int regs = [&] {
    cudaFuncAttributes fa;
    return cudaFuncGetAttributes(&fa, kern) == cudaSuccess ? fa.numRegs : 0;
  }();
  if (regs < kLaunchRegs) return cudaErrorLaunchOutOfResources;      // the pool that setmaxnreg draws on
  const size_t smem = smem_bytes(p.a.sk);
  cudaError_t e = allow_shared(kern, smem);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)((long long)((p.a.sq + kRows - 1) / kRows) * p.a.b * p.a.hq));
  if (p.a.documents) return launch_dependent(kern, grid, dim3(kThreads), smem, s, q, k, v, p);
  kern<<<grid, kThreads, smem, s>>>(q, k, v, p);
  return cudaGetLastError();
}

}  // namespace

bool prompt_attention32_usable(const DecoderAttention& p) {
  if (p.d > kDim || p.d % 4 || p.sk == 0 || p.sq < 64 || !encode_fn()) return false;
  if (smem_bytes(p.sk) > 227 * 1024) return false;
  if ((long long)((p.sq + kRows - 1) / kRows) * p.b * p.hq > 0x7fffffffll) return false;
  return view_fits(p.q, BG_F32, p.b, p.sq, p.hq) && view_fits(p.k, BG_F32, p.b, p.sk, p.hkv) && view_fits(p.v, BG_F32, p.b, p.sk, p.hkv) &&
         view_fits(p.out, BG_F32, p.b, p.sq, p.hq);
}

cudaError_t launch_prompt_attention32(const DecoderAttention& p, cudaStream_t s) {
  CUtensorMap q, k, v;
  if (!make_map(&q, p.q, BG_F32, p.b, p.sq, p.hq, p.d, kRows) || !make_map(&k, p.k, BG_F32, p.b, p.sk, p.hkv, p.d, kKeys) ||
      !make_map(&v, p.v, BG_F32, p.b, p.sk, p.hkv, p.d, kKeys, CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B))
    return cudaErrorInvalidValue;
  Prompt32Params pp;
  pp.a = p;
  pp.idesc_qk = (1u << 4) | (2u << 7) | (2u << 10) | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
  pp.idesc_pv = (1u << 4) | (2u << 7) | (2u << 10) | (1u << 16) | ((uint32_t)(kDim >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);      // V is MN-major
  const bool bias = p.slopes || !(p.scale > 0.f), cap = p.cap > 0.f;
  if (cap) return bias ? launch_kernel<true, true>(pp, q, k, v, s) : launch_kernel<true, false>(pp, q, k, v, s);
  return bias ? launch_kernel<false, true>(pp, q, k, v, s) : launch_kernel<false, false>(pp, q, k, v, s);
}

}  // namespace bg
