// Attention of prompts over a cache, 16-bit operands, head dimensions up to 128 (sm_100a): the rules of cache_attn.cuh on
// the tensor cores of this generation.
//
// A CTA owns 256 consecutive query rows of one head as two tiles of 128 (A, B) that share the key and value tiles in
// shared memory; while the softmax of one tile runs, the products of the other do.  (Or one tile of 128, with two CTAs on
// an SM: launch_prompt_attention says when.)
//   warp 0       producer (lane 0: Q, then K tiles; lane 1: V tiles; TMA)
//   warps 1, 2   issue the products of tile A and of tile B: S = Q K^T into tensor memory, O += P V with P read from there
//   warp 3       clears the value rows of the tile the sequence ends in that lie behind its length, between the tile's landing
//                and its products: a probability of zero times what an unwritten cache holds would not be zero
//   warps 4-7    softmax of tile A, one thread per query row; warps 8-11: of tile B
// With 64 values a head P has columns of its own in tensor memory, and the scores of the next key tile are computed
// while a tile's softmax still runs; with 128 values the 512 columns are S and O of both tiles, P takes the place of the
// scores it was made from, and the next scores wait for P V.  The reference of the exponentials follows the row maximum
// lazily: O is rescaled when the maximum has grown by more than 2^8.  P is rounded to the operand type, which is what the
// tensor core multiplies: each probability is off by at most 2^-8 (bf16) or 2^-11 (f16) of itself, f16 ones below 2^-21 of the
// reference (kRoomF16) by up to 2^-32 of it.
// Which keys a row sees is one number, the end of its visible range, and for packed documents the row's id: tiles nobody
// sees are not loaded, tiles everybody sees are not masked, for the rest the bits of the keys seen are made while the
// tile's scores are (packed documents of 4 x 2048: 53 us with a pass over the scores, 49 this way).
// Bound: 4 D flops a visible pair on the tensor pipe (1024 clocks a tile of 128 x 128 x 128) against one exponential a
// pair on the MUFU (16 a clock: 1024 clocks).  A cap would add two more MUFU operations; within |s| <= cap, where scores
// nearly always lie, tanh is an odd polynomial on the FMA pipe instead, two values an instruction.
// Measured: 4 x 16 heads of 4096 keys of 128, bf16, 549 us = 1001 TFLOP/s, causal 865; 2 x 16 heads of 4099 keys of 128, f16,
// prefix and cap, 274 us = 517 TFLOP/s of visible pairs (tensor pipe 27 %, FMA pipe 39 %, MUFU 25 %: the chain of a tile,
// scores - maximum - cap - exponentials - P V, is what it waits for).  P handed over in two halves gained nothing.
// No cluster multicast; every wait is clock-bounded.
#include "serving.h"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
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

constexpr int kRows = 128, kKeys = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazyLog2 = 8.0f;
// Key tiles that are added in tensor memory before O goes to a sum in memory (LONG: caches that have more).  The tensor core adds
// with truncation, which makes a result smaller by some 10^-7 for each addition, eight a tile: 5 * 10^-5 after 64 tiles, but
// 8 * 10^-4 after 131072 keys, more than the half step of float16.  64 rows of 8 heads of 128 over 131072 keys: 2144 us without
// the sums in memory, 2212 with them; their code alone would cost plain prompts of heads of 64 a tenth (394 -> 430 us), hence
// kernels of their own.
constexpr int kFoldTiles = 64;
// float16 probabilities lie up to 2^7 above the reference, 2^15 with the lazy maximum, where the type still has room: against
// the maximum itself they would vanish below 2^-25 of it while their sum still counted them.  It cancels in the division.
constexpr float kRoomF16 = 7.0f;
// D: values of a head, padded; NT: query tiles of a CTA.
template <int D, int NT>
struct Cfg {
  static constexpr bool Alias = D == 128;                    // P in the columns of S
  static constexpr int Threads = 128 + 128 * NT, PerSm = NT == 1 ? 2 : 1;
  static constexpr int Boxes = D / 64;                       // 128-byte wide boxes of a row
  static constexpr int BoxBytes = 128 * 128;                 // 128 rows of 64 values
  static constexpr int TileBytes = Boxes * BoxBytes;
  static constexpr int Stages = 2;
  static constexpr int TmemCols = 256 * NT;
  static constexpr int ColS = 0, ColO = 128 * NT, ColP = Alias ? 0 : 192 * NT, StepP = Alias ? 128 : 64;
  static constexpr int Smem = NT * TileBytes + 2 * Stages * TileBytes;
  // Registers move from warps 0-3 to the softmax warps, within what the CTA is launched with (checked at launch; a request
  // beyond the pool would wait for ever).
  static constexpr int LaunchRegs = NT == 1 ? 128 : 168, LightRegs = NT == 1 ? 56 : 72, SoftmaxRegs = NT == 1 ? 200 : 216;
  static_assert(128 * LightRegs + 128 * NT * SoftmaxRegs <= LaunchRegs * Threads, "setmaxnreg requests exceed the CTA's registers");
  static_assert(Alias ? NT == 2 : true, "tensor memory");
};

struct PromptParams {
  DecoderAttention a;
  uint32_t idesc_qk, idesc_pv;
};

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a0, float a1) {
  if (BF16) { __nv_bfloat162 v = __floats2bfloat162_rn(a0, a1); return *reinterpret_cast<uint32_t*>(&v); }
  __half2 v = __floats2half2_rn(a0, a1);
  return *reinterpret_cast<uint32_t*>(&v);
}
// two values an instruction
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float c, float d, float e, float f) {      // (x, y) = (a c + e, b d + f)
  asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmov.b64 r, {%6, %7};\n\t"
      "fma.rn.f32x2 p, p, q, r;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "=f"(x), "=f"(y) : "f"(a), "f"(b), "f"(c), "f"(d), "f"(e), "f"(f));
}
__device__ __forceinline__ void mul2(float& x, float& y, float a, float b, float c, float d) {
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmul.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "=f"(x), "=f"(y) : "f"(a), "f"(b), "f"(c), "f"(d));
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b, float c, float d) {
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tadd.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "=f"(x), "=f"(y) : "f"(a), "f"(b), "f"(c), "f"(d));
}

__device__ __forceinline__ void tanh_ratio2(float& p, float& q, float z, float w) {      // tanh_ratio of z and of w
  fma2(p, q, z, w, -0.003067060373723507f, -0.003067060373723507f, 0.016743116080760956f, 0.016743116080760956f);
  fma2(p, q, z, w, p, q, -0.051605675369501114f, -0.051605675369501114f);
  fma2(p, q, z, w, p, q, 0.13281433284282684f, 0.13281433284282684f);
  fma2(p, q, z, w, p, q, -0.3332904279232025f, -0.3332904279232025f);
  fma2(p, q, z, w, p, q, 0.9999994039535522f, 0.9999994039535522f);
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
      "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15]) : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// ---- rare work, out of the main path ----

template <int D>
__device__ __noinline__ void rescale_row(uint32_t t_o, float alpha) {
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t r[32];
    tmem_ld32(t_o + (uint32_t)(c * 32), r);
#pragma unroll
    for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
    tmem_st32(t_o + (uint32_t)(c * 32), r);
  }
}

// Adds a row's O to its sum in memory, [D] values and their reference, 128 rows side by side: O goes on from zero.
template <int D>
__device__ __noinline__ void fold_row(uint32_t t_o, float* sum, float m_ref, bool first) {
  const float from = first ? -CUDART_INF_F : sum[D * kRows];
  const float f = from == -CUDART_INF_F ? 0.f : ex2_approx(from - m_ref);
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t r[32];
    tmem_ld32(t_o + (uint32_t)(c * 32), r);
    float* p = sum + c * 32 * kRows;
    float before[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) before[i] = first ? 0.f : p[i * kRows];
#pragma unroll
    for (int i = 0; i < 32; ++i) p[i * kRows] = fmaf(before[i], f, __uint_as_float(r[i]));
  }
  sum[D * kRows] = m_ref;
}

// Caps the scores of a row's key tile in tensor memory, some of them beyond the cap.  Each value takes the form that is accurate
// relative to it; within the cap that is the polynomial with the very operations of the main path, so that a score's bits do
// not depend on its neighbours.  Beyond it 1 - 2 / (1 + e^2x) is off by at most 2^-21, of a value above 0.76.  Out of line and
// sixteen at a time because it is the instruction cache that the two paths compete for: 4 x 16 heads of 4096 keys of 64, some
// scores of a tile beyond the cap, 1314 us; 32 at a time 1622, in line 2970 (and 727 instead of 687 where none is beyond).
__device__ __noinline__ void cap_mixed_row(uint32_t t_s, float to_cap, float to_log2) {
#pragma unroll 1
  for (int c = 0; c < kKeys / 16; ++c) {
    uint32_t r[16];
    tmem_ld16(t_s + (uint32_t)(c * 16), r);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      float x = __uint_as_float(r[i]), y = __uint_as_float(r[i + 1]), z, w, p, q;
      mul2(x, y, x, y, to_cap, to_cap);
      mul2(z, w, x, y, x, y);
      tanh_ratio2(p, q, z, w);
      float u, v, e, f;
      mul2(e, f, x, y, 2.0f * kLog2e, 2.0f * kLog2e);
      e = rcp_approx(1.0f + ex2_approx(e));
      f = rcp_approx(1.0f + ex2_approx(f));
      fma2(e, f, e, f, -2.0f, -2.0f, 1.0f, 1.0f);
      mul2(e, f, e, f, to_log2, to_log2);
      mul2(u, v, x, y, to_log2, to_log2);
      mul2(u, v, u, v, p, q);
      r[i] = __float_as_uint(within_one(z, u, e));
      r[i + 1] = __float_as_uint(within_one(w, v, f));
    }
    tmem_st16(t_s + (uint32_t)(c * 16), r);
  }
}

template <bool BF16, int D, int NT, bool CAP, bool BIAS, bool LONG>
__global__ void __launch_bounds__(Cfg<D, NT>::Threads, Cfg<D, NT>::PerSm)
prompt_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const __grid_constant__ PromptParams pp) {
  using C = Cfg<D, NT>;
  constexpr int kThreads = C::Threads;
  const DecoderAttention& a = pp.a;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* sQ = smem;
  unsigned char* sK = sQ + NT * C::TileBytes;
  unsigned char* sV = sK + C::Stages * C::TileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + C::Stages * C::TileBytes);
  uint64_t* q_full = bars;                       // [2]
  uint64_t* k_full = q_full + 2;                 // [Stages]
  uint64_t* k_empty = k_full + C::Stages;
  uint64_t* v_full = k_empty + C::Stages;
  uint64_t* v_empty = v_full + C::Stages;
  uint64_t* s_full = v_empty + C::Stages;        // [2] the scores of a tile are there
  uint64_t* s_empty = s_full + 2;                // [2] its softmax warps hold them in registers (unused when P takes their place)
  uint64_t* p_full = s_empty + 2;                // [2] P is there
  uint64_t* pv_full = p_full + 2;                // [2] P V has completed
  uint64_t* turn = pv_full + 2;                  // [2][4] a warp of tile A (0) / B (1) has its exponentials of a shared key tile behind it
  uint64_t* v_raw = turn + 8;                    // the value tile the sequence ends in has landed, still to be cleared behind it
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(v_raw + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  unsigned char* s_need = reinterpret_cast<unsigned char*>(tmem_holder + 4);     // [2][n_kv]

  if (a.documents) grid_dependency_wait();       // the ranges of their ids come from the launch before
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int n_bh = a.b * a.hq;
  const int n_qt = (a.sq + kRows - 1) / kRows, n_pairs = (n_qt + NT - 1) / NT;
  const int pair = n_pairs - 1 - (int)(blockIdx.x / (unsigned)n_bh);       // the last rows see the most keys: they go first
  const int bh = (int)(blockIdx.x % (unsigned)n_bh);
  const int b = bh / a.hq, h = bh % a.hq, hk = h / a.group;
  const bool has_b = NT == 2 && 2 * pair + 1 < n_qt;

  const Sequence seq = sequence_of(a, b);
  const int len = seq.len;
  const int n_kv = (len + kKeys - 1) / kKeys;
  const int2* ranges = a.documents ? a.doc_ranges + (long long)b * ((a.sk + kDocBlock - 1) / kDocBlock) : nullptr;
  const int* docs = a.documents ? a.documents + (long long)b * a.sk : nullptr;
#pragma unroll
  for (int g = 0; g < NT; ++g)
    needed_tiles<kKeys>(a, b, seq, (NT * pair + g) * kRows, min((NT * pair + g + 1) * kRows, a.sq) - 1, s_need + g * n_kv, threadIdx.x, kThreads);
  if (threadIdx.x == 0) {
    for (int g = 0; g < 2; ++g) {
      mbar_init(&q_full[g], 1);
      mbar_init(&s_full[g], 1); mbar_init(&s_empty[g], 4);
      mbar_init(&p_full[g], 4); mbar_init(&pv_full[g], 1);
    }
    for (int s = 0; s < C::Stages; ++s) {
      mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], NT);      // a slot is free once the issuers are done with it
      mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], NT);
    }
    for (int i = 0; i < 8; ++i) mbar_init(&turn[i], 1);
    mbar_init(v_raw, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)), "n"(C::TmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  auto next = [&](int j) { while (j < n_kv && !s_need[j] && (NT == 1 || !s_need[n_kv + j])) ++j; return j; };
  // the tile that holds both keys of the sequence and rows behind it (rows behind the buffer arrive as zeros anyway)
  const int ragged = len < a.sk && (len % kKeys) != 0 ? len / kKeys : -1;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::LightRegs));
    if (warp == 0) {
      if (lane == 0) {
        for (int g = 0; g < (has_b ? 2 : 1); ++g) {
          mbar_expect_tx(&q_full[g], C::TileBytes);
          for (int x = 0; x < C::Boxes; ++x)
            tma_load_4d(&tmQ, sQ + g * C::TileBytes + x * C::BoxBytes, &q_full[g], x * 64, (NT * pair + g) * kRows, h, b);
        }
        int u = 0;
        for (int j = next(0); j < n_kv; j = next(j + 1), ++u) {
          const int s = u % C::Stages;
          if (!mbar_wait(&k_empty[s], ((uint32_t)(u / C::Stages) & 1u) ^ 1u, abort_flag)) break;
          mbar_expect_tx(&k_full[s], C::TileBytes);
          for (int x = 0; x < C::Boxes; ++x) tma_load_4d(&tmK, sK + s * C::TileBytes + x * C::BoxBytes, &k_full[s], x * 64, j * kKeys, hk, b);
        }
        // the query tiles have landed before this warp may leave
        for (int g = 0; g < (has_b ? 2 : 1); ++g) mbar_wait(&q_full[g], 0, abort_flag);
      } else if (lane == 1) {
        int u = 0;
        for (int j = next(0); j < n_kv; j = next(j + 1), ++u) {
          const int s = u % C::Stages;
          if (!mbar_wait(&v_empty[s], ((uint32_t)(u / C::Stages) & 1u) ^ 1u, abort_flag)) break;
          uint64_t* landed = j == ragged ? v_raw : &v_full[s];       // warp 3 passes the cleared tile on
          mbar_expect_tx(landed, C::TileBytes);
          for (int x = 0; x < C::Boxes; ++x) tma_load_4d(&tmV, sV + s * C::TileBytes + x * C::BoxBytes, landed, x * 64, j * kKeys, hk, b);
        }
      }
    } else if (warp <= NT) {
      const int g = warp - 1;
      const unsigned char* need = s_need + g * n_kv;
      const uint32_t q_addr = smem_u32(sQ + g * C::TileBytes);
      const uint32_t d_s = tmem_base + (uint32_t)(C::ColS + g * kKeys);
      const uint32_t d_o = tmem_base + (uint32_t)(C::ColO + g * D);
      const uint32_t d_p = tmem_base + (uint32_t)(C::ColP + g * C::StepP);
      const uint32_t idesc_qk = pp.idesc_qk, idesc_pv = pp.idesc_pv;
      int n_qk = 0, n_pv = 0;
      auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0; };
      auto issue_qk = [&](int slot) -> bool {
        const int n = n_qk++;
        if (n == 0 && !wait_all(&q_full[g], 0)) return false;
        if (n > 0 && !wait_all(C::Alias ? &pv_full[g] : &s_empty[g], (uint32_t)(n - 1) & 1u)) return false;
        tc_fence_after();
        const uint32_t k_addr = smem_u32(sK + slot * C::TileBytes);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint64_t da = make_kmajor_sw128_desc(q_addr + (uint32_t)((k >> 2) * C::BoxBytes)) + (uint64_t)((k & 3) * 2);
            const uint64_t db = make_kmajor_sw128_desc(k_addr + (uint32_t)((k >> 2) * C::BoxBytes)) + (uint64_t)((k & 3) * 2);
            umma<false>(d_s, da, db, idesc_qk, k ? 1u : 0u);
          }
          umma_commit(&s_full[g]);
        }
        __syncwarp();
        return true;
      };
      auto issue_pv = [&](int slot) -> bool {
        const int n = n_pv++;
        if (!wait_all(&p_full[g], (uint32_t)n & 1u)) return false;
        tc_fence_after();
        const uint32_t v_addr = smem_u32(sV + slot * C::TileBytes);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            // rows of V are the K index: 16 of them are 2048 bytes; the second 64 values of a row lie a box further on
            uint64_t db = make_mnmajor_sw128_desc(v_addr + (uint32_t)(k * 2048));
            if (C::Boxes == 2) db = (db & ~((uint64_t)0x3fff << 16)) | ((uint64_t)(C::BoxBytes >> 4) << 16);
            umma_ts_f16(d_o, d_p + (uint32_t)(k * 8), db, idesc_pv, (LONG ? n % kFoldTiles != 0 : n > 0) || k > 0 ? 1u : 0u);
          }
          umma_commit(&pv_full[g]);
        }
        __syncwarp();
        return true;
      };
      auto release = [&](uint64_t* bar, bool used) {
        if (elect_one()) { if (used) umma_commit(bar); else mbar_arrive(bar); }
        __syncwarp();
      };
      // A tile this query tile skips is released once it has landed, so that the arrival counts for that tile.
      // P of its own: the next scores are issued ahead of P V.  P in the place of the scores: behind it.
      bool ok = true;
      int jc = next(0), u = 0;
      auto scores = [&](int j, int n) {
        const int slot = n % C::Stages;
        ok = wait_all(&k_full[slot], (uint32_t)(n / C::Stages) & 1u);
        const bool used = need[j] != 0;
        if (ok && used) ok = issue_qk(slot);
        if (ok) release(&k_empty[slot], used);
      };
      if (jc < n_kv) scores(jc, 0);
      while (jc < n_kv && ok) {
        const int jn = next(jc + 1);
        if (!C::Alias && jn < n_kv) scores(jn, u + 1);
        const int slot = u % C::Stages;
        if (ok) ok = wait_all(&v_full[slot], (uint32_t)(u / C::Stages) & 1u);
        const bool used = need[jc] != 0;
        if (ok && used) ok = issue_pv(slot);
        if (ok) release(&v_empty[slot], used);
        if (C::Alias && ok && jn < n_kv) scores(jn, u + 1);
        jc = jn;
        ++u;
      }
    } else if (warp == 3 && ragged >= 0) {
      // warp 3: the value rows behind the sequence in its last tile
      int u = 0, j = next(0);
      for (; j < n_kv && j != ragged; j = next(j + 1)) ++u;
      if (j == ragged) {
        const int slot = u % C::Stages;
        if (mbar_wait(v_raw, 0, abort_flag)) {
          const int r0 = len - ragged * kKeys;
          for (int i = lane; i < (kKeys - r0) * 8 * C::Boxes; i += 32) {      // a row is 128 bytes of each box, wherever its pieces lie
            const int x = i / ((kKeys - r0) * 8), c = i - x * ((kKeys - r0) * 8);
            *reinterpret_cast<uint4*>(sV + slot * C::TileBytes + x * C::BoxBytes + r0 * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_full[slot]);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SoftmaxRegs));
    const int g = (warp - 4) >> 2, quarter = warp & 3;
    const int r_in_tile = quarter * 32 + lane;
    const int row = (NT * pair + g) * kRows + r_in_tile;
    const bool active = g == 0 || has_b, row_ok = active && row < a.sq;
    if (active) {
      const uint32_t lane_sel = (uint32_t)(quarter * 32) << 16;
      const uint32_t t_s = tmem_base + (uint32_t)(C::ColS + g * kKeys) + lane_sel;
      const uint32_t t_o = tmem_base + (uint32_t)(C::ColO + g * D) + lane_sel;
      const uint32_t t_p = tmem_base + (uint32_t)(C::ColP + g * C::StepP) + lane_sel;
      const unsigned char* need = s_need + g * n_kv;
      const Reach me = reach_of(a, seq, row, row_ok ? row : row - 1);
      int hi = me.keys, doc = -1;
      if (docs) {
        doc = me.keys > 0 && me.first >= 0 && me.first < a.sk ? __ldg(docs + me.first) : -1;
        if (doc < 0) hi = 0;
      }
      const int pos = distance_origin(seq, me.first);
      const float slope = BIAS && a.slopes ? a.slopes[h] * kLog2e : 0.f;
      const float to_log2 = CAP ? a.cap * kLog2e : a.scale * kLog2e, to_cap = CAP ? a.scale / a.cap : 0.f;
      constexpr bool TURNS = NT == 2 && (C::Alias || CAP || BIAS);      // (4 x 16 heads, 4096 rows: plain scores of heads of 64 are 8 % slower with turns, the others 2 to 9 % faster)
      constexpr bool FOLD = !CAP && !BIAS;        // the scale is applied in the exponent (it is positive then)
      float m_ref = -CUDART_INF_F, l = 0.f;
      bool ok = true;
      int t = 0, n_shared = 0;
      for (int j = 0; j < n_kv && ok; ++j) {
        if (!need[j]) continue;
        const bool shared = NT == 2 && s_need[j] && s_need[n_kv + j];
        const int k0 = j * kKeys;
        bool whole = hi >= k0 + kKeys;
        if (docs) {
          const int2 x = __ldg(ranges + j);
          whole = whole && x.x == doc && x.y == doc;      // a block with keys of no document has its sign bit set
        }
        const bool hide = !__all_sync(0xffffffffu, whole);
        // the bits of the keys seen, made while the scores are (warp-uniform; all set where nothing is hidden)
        uint32_t seen[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
        if (hide) {
          const int n = min(max(hi - k0, 0), kKeys);
#pragma unroll
          for (int c = 0; c < 4; ++c) seen[c] = n >= 32 * c + 32 ? 0xffffffffu : n <= 32 * c ? 0u : (1u << (n - 32 * c)) - 1u;
          if (docs) {
            const uint4 mine = document_bits(docs + k0, min(a.sk - k0, kKeys), doc);
            seen[0] &= mine.x; seen[1] &= mine.y; seen[2] &= mine.z; seen[3] &= mine.w;
          }
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[g], (uint32_t)t & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after();
        float x[kKeys];
        uint32_t* xu = reinterpret_cast<uint32_t*>(x);
        tmem_ld32_issue(t_s, xu);
        tmem_ld32_issue(t_s + 32, xu + 32);
        tmem_ld32_issue(t_s + 64, xu + 64);
        tmem_ld32_issue(t_s + 96, xu + 96);
        tmem_ld_wait();
        float base = 0.f;                                  // added to every score of the row
        if (CAP) {
          float z0 = 0.f, z1 = 0.f;
#pragma unroll
          for (int i = 0; i < kKeys; i += 2) {
            mul2(x[i], x[i + 1], x[i], x[i + 1], to_cap, to_cap);
            if (i & 2) z1 = fmax3(z1, fabsf(x[i]), fabsf(x[i + 1]));
            else z0 = fmax3(z0, fabsf(x[i]), fabsf(x[i + 1]));
          }
          if (__all_sync(0xffffffffu, fmaxf(z0, z1) <= 1.0f)) {
#pragma unroll
            for (int i = 0; i < kKeys; i += 2) {
              float z, y, q, r;
              mul2(z, y, x[i], x[i + 1], x[i], x[i + 1]);
              tanh_ratio2(q, r, z, y);
              mul2(x[i], x[i + 1], x[i], x[i + 1], to_log2, to_log2);
              mul2(x[i], x[i + 1], x[i], x[i + 1], q, r);
            }
          } else {                                         // a score beyond the cap among them, or what lies behind the keys
            cap_mixed_row(t_s, to_cap, to_log2);
            tmem_ld32_issue(t_s, xu);
            tmem_ld32_issue(t_s + 32, xu + 32);
            tmem_ld32_issue(t_s + 64, xu + 64);
            tmem_ld32_issue(t_s + 96, xu + 96);
            tmem_ld_wait();
          }
        } else if (BIAS) {
#pragma unroll
          for (int i = 0; i < kKeys; i += 2) mul2(x[i], x[i + 1], x[i], x[i + 1], to_log2, to_log2);
        }
        if (BIAS) {
          if (__all_sync(0xffffffffu, k0 + kKeys - 1 <= pos)) {        // every key behind the row: the distance is linear
            base = slope * (float)(k0 - pos);
#pragma unroll
            for (int i = 0; i < kKeys; ++i) x[i] = fmaf(slope, (float)i, x[i]);
          } else {
            const float gap = (float)(pos - k0);
#pragma unroll
            for (int i = 0; i < kKeys; ++i) x[i] = fmaf(-slope, fabsf(gap - (float)i), x[i]);
          }
        }
        uint32_t dead = 0u;                                 // 32-key pieces that no row of this warp sees
        if (hide) {
#pragma unroll
          for (int i = 0; i < kKeys; ++i)
            if (!((seen[i >> 5] >> (i & 31)) & 1u)) x[i] = -CUDART_INF_F;
          dead = __reduce_and_sync(0xffffffffu, (seen[0] == 0u ? 1u : 0u) | (seen[1] == 0u ? 2u : 0u) | (seen[2] == 0u ? 4u : 0u) | (seen[3] == 0u ? 8u : 0u));
        }
        if (!C::Alias) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[g]);
        }
        float mt;
        {
          float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
          for (int i = 4; i < kKeys; i += 2) mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], x[i], x[i + 1]);
          mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          if (FOLD) mt *= to_log2;
          else mt += base;
        }
        const bool coarse = fabsf(mt) >= kCoarse && mt != -CUDART_INF_F;
        if (!BF16 && !coarse) mt -= kRoomF16;
        // O is rescaled by whole warps once the P V before it has completed (with P in the place of the scores these
        // scores are younger than that product)
        bool pv_done = t == 0 || C::Alias;
        const bool raise = m_ref != -CUDART_INF_F && mt - m_ref > kLazyLog2;
        float unit = to_log2;                               // FOLD: what the scores are still to be multiplied by
        const bool fold = LONG && t % kFoldTiles == 0 && t > 0;
        if (FOLD ? __any_sync(0xffffffffu, raise || coarse || fold) : __any_sync(0xffffffffu, raise || fold)) {
          if (FOLD && __any_sync(0xffffffffu, coarse)) {
#pragma unroll
            for (int i = 0; i < kKeys; ++i) x[i] *= to_log2;
            unit = 1.0f;
          }
          if (!pv_done) {
            ok = __all_sync(0xffffffffu, mbar_wait(&pv_full[g], (uint32_t)(t - 1) & 1u, abort_flag));
            if (!ok) break;
            pv_done = true;
            tc_fence_after();
          }
          const float alpha = raise ? ex2_approx(m_ref - mt) : 1.0f;
          if (fold) fold_row<D>(t_o, a.sums + ((size_t)blockIdx.x * NT + g) * ((D + 1) * kRows) + r_in_tile, m_ref, t == kFoldTiles);
          else rescale_row<D>(t_o, alpha);
          if (raise) { l *= alpha; m_ref = mt; }
        }
        if (m_ref == -CUDART_INF_F) m_ref = mt;
        const float off = (m_ref == -CUDART_INF_F ? 0.f : -m_ref) + base;
        // The two warps of this SM quarter take turns at the exponentials of key tiles both need: left alone they fall into
        // step, both at the MUFU and then both away from it.
        if (TURNS && shared && (g == 1 || n_shared > 0)) {
          ok = __all_sync(0xffffffffu, mbar_wait(&turn[(1 - g) * 4 + quarter], (uint32_t)(n_shared - (g == 0)) & 1u, abort_flag));
          if (!ok) break;
        }
        {
          float ps[4] = {0.f, 0.f, 0.f, 0.f};
          auto exponentials = [&](int i) {                 // of x[i], x[i + 1]
            if (FOLD) fma2(x[i], x[i + 1], x[i], x[i + 1], unit, unit, off, off);
            else add2(x[i], x[i + 1], x[i], x[i + 1], off, off);
            x[i] = ex2_approx(x[i]);
            x[i + 1] = ex2_approx(x[i + 1]);
            add2(ps[i & 2], ps[(i & 2) + 1], ps[i & 2], ps[(i & 2) + 1], x[i], x[i + 1]);
          };
          if (!dead) {                                     // one straight block: a branch per piece would drain the MUFU at each
#pragma unroll
            for (int i = 0; i < kKeys; i += 2) exponentials(i);
          } else {
#pragma unroll
            for (int c = 0; c < kKeys / 32; ++c) {
              if ((dead >> c) & 1u) {
#pragma unroll
                for (int i = c * 32; i < c * 32 + 32; ++i) x[i] = 0.f;
              } else {
#pragma unroll
                for (int i = c * 32; i < c * 32 + 32; i += 2) exponentials(i);
              }
            }
          }
          l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        }
        if (TURNS && shared) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&turn[g * 4 + quarter]);
          ++n_shared;
        }
        if (!pv_done) {             // P of the previous key tile has been consumed
          ok = __all_sync(0xffffffffu, mbar_wait(&pv_full[g], (uint32_t)(t - 1) & 1u, abort_flag));
          if (!ok) break;
          tc_fence_after();
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) w[i] = pack16<BF16>(x[half * 64 + 2 * i], x[half * 64 + 2 * i + 1]);
          tmem_st32_issue(t_p + (uint32_t)(half * 32), w);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g]);
        ++t;
      }
      if (ok && t > 0) ok = __all_sync(0xffffffffu, mbar_wait(&pv_full[g], (uint32_t)(t - 1) & 1u, abort_flag));
      if (ok) {
        tc_fence_after();
        const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);      // a row without keys is zero; NaN stays NaN
        const float* sum = LONG && t > kFoldTiles ? a.sums + ((size_t)blockIdx.x * NT + g) * ((D + 1) * kRows) + r_in_tile : nullptr;
        const float from = sum ? sum[D * kRows] : -CUDART_INF_F, f = from == -CUDART_INF_F ? 0.f : ex2_approx(from - m_ref);
        uint16_t* out = reinterpret_cast<uint16_t*>(const_cast<void*>(a.out.ptr)) + b * a.out.sb + (long long)h * a.out.sh + (long long)(row_ok ? row : 0) * a.out.sr;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          if (t > 0) tmem_ld32(t_o + (uint32_t)(c * 32), r);
          if (LONG && sum)
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(fmaf(sum[(c * 32 + i) * kRows], f, __uint_as_float(r[i])));
          if (row_ok) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              if (c * 32 + i >= a.d) continue;
              float o[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) o[e] = t > 0 && l != 0.f ? __uint_as_float(r[i + e]) * inv : 0.f;
              *reinterpret_cast<uint4*>(out + c * 32 + i) =
                  make_uint4(pack16<BF16>(o[0], o[1]), pack16<BF16>(o[2], o[3]), pack16<BF16>(o[4], o[5]), pack16<BF16>(o[6], o[7]));
            }
          }
        }
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
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "n"(C::TmemCols) : "memory");
  }
}

template <int D, int NT>
size_t smem_bytes(int sk) { return (size_t)Cfg<D, NT>::Smem + 1024 + 256 + NT * (size_t)((sk + kKeys - 1) / kKeys); }

template <bool BF16, int D, int NT, bool CAP, bool BIAS, bool LONG>
cudaError_t launch_kernel(const PromptParams& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
  auto kern = prompt_attention_kernel<BF16, D, NT, CAP, BIAS, LONG>;
  static const int regs = [&] {
    cudaFuncAttributes fa;
    return cudaFuncGetAttributes(&fa, kern) == cudaSuccess ? fa.numRegs : 0;
  }();
  if (regs < Cfg<D, NT>::LaunchRegs) return cudaErrorLaunchOutOfResources;
  const size_t smem = smem_bytes<D, NT>(p.a.sk);
  cudaError_t e = allow_shared(kern, smem);
  if (e != cudaSuccess) return e;
  const int pairs = ((p.a.sq + kRows - 1) / kRows + NT - 1) / NT;
  const dim3 grid((unsigned)((long long)pairs * p.a.b * p.a.hq)), block(Cfg<D, NT>::Threads);
  if (p.a.documents) return launch_dependent(kern, grid, block, smem, s, q, k, v, p);
  kern<<<grid, block, smem, s>>>(q, k, v, p);
  return cudaGetLastError();
}

template <bool BF16, int D, int NT, bool CAP, bool BIAS>
cudaError_t launch_length(const PromptParams& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
  return p.a.sums ? launch_kernel<BF16, D, NT, CAP, BIAS, true>(p, q, k, v, s) : launch_kernel<BF16, D, NT, CAP, BIAS, false>(p, q, k, v, s);
}

template <bool BF16, int D, int NT>
cudaError_t launch_rules(const PromptParams& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
  // a scale that is not positive cannot be taken out of the row maximum: such scores are scaled like biased ones
  const bool bias = p.a.slopes || !(p.a.scale > 0.f), cap = p.a.cap > 0.f;
  if (cap) return bias ? launch_length<BF16, D, NT, true, true>(p, q, k, v, s) : launch_length<BF16, D, NT, true, false>(p, q, k, v, s);
  return bias ? launch_length<BF16, D, NT, false, true>(p, q, k, v, s) : launch_length<BF16, D, NT, false, false>(p, q, k, v, s);
}

// Query tiles of a CTA.
int query_tiles(const DecoderAttention& p) {
  if (p.d > 64) return 2;
  // One query tile a CTA and two CTAs an SM where there is little work behind a CTA's start, which the other then covers:
  // 32 x 128 tokens 18 us against 24, 16 x 512 33 against 35 (capped 45 against 49), packed documents of 400 in 4 x 2048
  // 46 against 49; from 2048 keys on two tiles that share their keys and take turns win (capped 99.5 us against 101.5,
  // 16 heads of 4096 keys 683 against 773).  Packed documents in 4 x 12 heads of 4096 tokens, one tile against two: of 100 tokens
  // 71 us against 77, of 1024 91 against 98, of 2048 126 against 127, one of 4096 199 against 188.
  return p.documents || p.sk <= 1024 ? 1 : 2;
}

}  // namespace

bool prompt_attention_usable(const DecoderAttention& p, int dtype) {
  if (dtype == BG_F32) return prompt_attention32_usable(p);
  if ((dtype != BG_BF16 && dtype != BG_F16) || p.d > 128 || p.d % 8 || p.sk == 0 || !encode_fn()) return false;
  // Below 64 rows a head most of a 128-row tile would stand empty, and the key-split kernel reads each key once for the
  // whole group: 63 rows there against 64 here, 8 x 12 heads of 64 over 1024 keys 28 us against 20, over 64 keys 10.9 against
  // 11.7, 8 x 8 heads of 128 in groups of four over 1024 keys 44 against 25.  These kernels do not split the keys, so few query
  // tiles over a long cache leave most SMs idle, and there the key-split kernel would be the faster one: 64 rows of 8 heads of
  // 128 over 16384 keys 261 us against its 42 for 63 rows, over 131072 keys 2.2 ms against 185 us.
  if (p.sq < 64) return false;
  if (smem_bytes<128, 2>(p.sk) > 227 * 1024) return false;
  if ((long long)((p.sq + 127) / 128) * p.b * p.hq > 0x7fffffffll) return false;
  return view_fits(p.q, dtype, p.b, p.sq, p.hq) && view_fits(p.k, dtype, p.b, p.sk, p.hkv) && view_fits(p.v, dtype, p.b, p.sk, p.hkv) && view_fits(p.out, dtype, p.b, p.sq, p.hq);
}

int64_t prompt_attention_scratch(const DecoderAttention& p, int dtype) {
  if (dtype == BG_F32 || p.sk <= kFoldTiles * kKeys) return 0;
  const int64_t nt = query_tiles(p), ctas = (((p.sq + kRows - 1) / kRows + nt - 1) / nt) * (int64_t)p.b * p.hq;
  return ctas * nt * ((p.d > 64 ? 128 : 64) + 1) * kRows * (int64_t)sizeof(float);
}

cudaError_t launch_prompt_attention(const DecoderAttention& p, int dtype, cudaStream_t s) {
  if (dtype == BG_F32) return launch_prompt_attention32(p, s);
  CUtensorMap q, k, v;
  if (!make_map(&q, p.q, dtype, p.b, p.sq, p.hq, p.d, kRows) || !make_map(&k, p.k, dtype, p.b, p.sk, p.hkv, p.d, kKeys) || !make_map(&v, p.v, dtype, p.b, p.sk, p.hkv, p.d, kKeys))
    return cudaErrorInvalidValue;
  const bool bf = dtype == BG_BF16, wide = p.d > 64;
  const uint32_t fmt = bf ? 1u : 0u;
  PromptParams pp;
  pp.a = p;
  pp.idesc_qk = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
  pp.idesc_pv = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((uint32_t)((wide ? 128 : 64) >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);   // V is MN-major
  if (wide) return bf ? launch_rules<true, 128, 2>(pp, q, k, v, s) : launch_rules<false, 128, 2>(pp, q, k, v, s);
  if (query_tiles(p) == 1) return bf ? launch_rules<true, 64, 1>(pp, q, k, v, s) : launch_rules<false, 64, 1>(pp, q, k, v, s);
  return bf ? launch_rules<true, 64, 2>(pp, q, k, v, s) : launch_rules<false, 64, 2>(pp, q, k, v, s);
}

}  // namespace bg
