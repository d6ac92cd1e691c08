// Attention over a key / value cache with the keys split over warps and CTAs (sm_100a): single tokens and short rows of
// queries of every type, and prompts the tensor-memory kernel (prompt_attn.cu) does not take.
//
// For a query row at position t and a key j of the same sequence
//     s = scale q.k_j,   s <- cap tanh(s / cap),   s <- s - slope |t - j|,
//     o = sum_j e^(s - m) v_j / sum_j e^(s - m)    over the keys the row sees (rules in bgcuda.h); no key: o = 0.
// One generated token reads every key and value once and computes 4 D flops with each pair: the bound is memory, so the
// layout serves the loads.  The query rows that share a key head (group x tokens) are the M rows of mma.sync tiles:
// sixteen rows cost what one costs, and each key is read once for all of them.  tcgen05 has nothing to add here (its 128
// rows would stand empty) and would need its operands in a swizzled layout.  A CTA's warps form groups of RT; a group owns
// RT 16-row tiles and walks its own key tiles through a ring of cp.async stages, synchronised by a barrier of the group
// alone.  Groups keep a running maximum and sum in 32 bits and are joined in shared memory at the end; with few rows the
// keys are also split over CTAs, whose partial results a second kernel joins in split order, a CTA per row.
// fp32 operands are multiplied as three tf32 products (hi hi + hi lo + lo hi); each tile's P V starts from zero and is
// added to O in registers, because the tensor core's own accumulation truncates.  16-bit P is rounded to the operand
// type, because the tensor core multiplies two operands of one type: each probability is off by at most 2^-8 (bf16) or 2^-11
// (f16) of itself, the half step the result is rounded by too; f16 ones below 2^-28 of the largest by up to 2^-39 of it.
// Measured: 32 x 8 key heads of 8192 keys of 128, bf16, 177 us = 6.1 TB/s in the three parts the plan takes (166 in one);
// 131077 keys, 4 key heads of two row tiles, f16, 65 to 69 us on different machines (41 us at the copy rate; 8 warps an SM wait
// for their own tile's products and exponentials, DRAM 59 % busy); 64 x 12 heads of 2048 keys of 64, fp32, 128 us = 6.3 TB/s;
// fp32 prompts of heads of 128 (2 x 16 x 2048, causal) 42 TFLOP/s.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "serving.h"

namespace bg {
namespace cache_attn {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t* r, const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_addr(p)) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t* r, const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_addr(p)) : "memory");
}
template <typename T> __device__ __forceinline__ void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float* c, const uint32_t* a, const uint32_t* b) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// x = hi + lo, hi on the tf32 grid; lo keeps its own upper bits in the product.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  lo = __float_as_uint(x - __uint_as_float(hi));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<float>(float, float) { return 0u; }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh(x) for 16-bit results, |x| > 1: 1 - 2 / (1 + e^2x) is off by at most 2^-21, of a value above 0.76.
__device__ __forceinline__ float tanh_beyond_one(float x) { return 1.0f - __fdividef(2.0f, 1.0f + ex2(x * (2.0f * kLog2e))); }
// The cap of n scores: scale s / cap in, cap log2(e) tanh of it out.  fp32 results take the library function.  For 16-bit ones
// the scores nearly always lie within the cap, and then the polynomial serves; else each value takes the form that is
// accurate relative to it (the other one's error is absolute, and the cap multiplies it into the exponent: 6 % at a cap of 10^6).
template <typename T, int N> __device__ __forceinline__ void cap_scores(float* x, float to_log2) {
  if (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_log2 * tanhf(x[i]);
    return;
  }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(x[i]));
  if (__all_sync(0xffffffffu, top <= 1.0f)) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= to_log2 * tanh_ratio(x[i] * x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_log2 * within_one(x[i] * x[i], x[i] * tanh_ratio(x[i] * x[i]), tanh_beyond_one(x[i]));
  }
}

// The reference of the exponentials of scores of at most mx.  float16 probabilities lie up to 2^14 above it, where the type has
// its room: against a reference of mx itself they would lose bits from 2^-14 on and vanish at 2^-25, while their sum below the
// line still counted them (131077 keys 2^-26 below the largest add up to 2^-9 of it).  Scores from 2^21 on, which 32 bits
// hold to a quarter, keep mx: the difference would be rounded into the exponent.  The running reference is the largest of the tiles', so no
// exponent passes 14; sums, rescaling and joins are relative to it, and it cancels in the division.
template <typename T> __device__ __forceinline__ float below(float mx) { return mx; }
template <> __device__ __forceinline__ float below<__half>(float mx) { return fabsf(mx) < 2097152.0f ? mx - 14.0f : mx; }

template <typename T, int DP_, int RT_>
struct Cfg {
  static constexpr int DP = DP_, RT = RT_, ES = sizeof(T);
  static constexpr int Warps = (RT == 4 && DP <= 128) || DP <= 64 ? 8 : 4;
  // CTAs that share an SM (their start and end overlap).  With one row tile of 16-bit heads above 64 a third one fits when
  // the ring has two stages: 32 x 8 heads of 8192 keys of 128 at 6.4 TB/s against 6.0; with two row tiles it does not pay.
  static constexpr int PerSm = DP > 128 ? 1 : ES == 2 && RT == 1 && DP > 64 ? 3 : 2;
  static constexpr int KG = Warps / RT;                 // key groups
  static constexpr int Threads = Warps * 32;
  static constexpr int KT = ES == 2 ? (RT == 1 ? 16 : 32) : (RT == 1 ? 8 : 16);   // keys of a tile
  static constexpr int LD = DP + 16 / ES;               // row stride in shared memory: 16 bytes of padding, no bank conflicts
  static constexpr int TileBytes = KT * LD * ES;        // one K or V tile
  static constexpr int SetBytes = KG * 2 * TileBytes;   // a stage of every group
  static constexpr int QBytes = 16 * RT * LD * ES;
  static constexpr int Stages = RT == 4 || PerSm == 3 ? 2 : (4 * SetBytes + QBytes <= 108 * 1024 ? 4 : 3 * SetBytes + QBytes <= 109 * 1024 ? 3 : 2);
  static constexpr int MergeLd = DP + 4;
  static constexpr int MergeBytes = Warps * 16 * MergeLd * 4;
  static constexpr int RingBytes = Stages * SetBytes;
  static constexpr int Smem = QBytes + (RingBytes > MergeBytes ? RingBytes : MergeBytes);
};

template <typename T, int DP, int RT>
__global__ void __launch_bounds__(Cfg<T, DP, RT>::Threads, Cfg<T, DP, RT>::PerSm)
cache_attention_kernel(const __grid_constant__ DecoderAttention p, int splits, int row_tiles, int vec, float* partials) {
  using C = Cfg<T, DP, RT>;
  constexpr int KT = C::KT, LD = C::LD, KG = C::KG, ST = C::Stages, ROWS = 16 * RT, GT = RT * 32;
  extern __shared__ __align__(128) unsigned char smem[];
  T* sQ = reinterpret_cast<T*>(smem);
  unsigned char* ring = smem + C::QBytes;
  __shared__ int s_hi[ROWS], s_pos[ROWS], s_doc[ROWS];
  __shared__ int s_top, s_doc_min, s_doc_max;
  __shared__ float s_m[C::Warps * 16], s_l[C::Warps * 16];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kg = warp / RT, rt = warp % RT, gt = tid % GT;
  const int unit = blockIdx.x / splits, split = blockIdx.x % splits;
  const int n_bh = p.b * p.hkv;
  const int row_tile = row_tiles - 1 - unit / n_bh;      // the last rows see the most keys: they go first
  const int bh = unit % n_bh, b = bh / p.hkv, hk = bh % p.hkv;
  const int n_rows = p.group * p.sq, row0 = row_tile * ROWS;

  // (all three requested before the first is used)
  const int len_in = p.lengths ? __ldg(p.lengths + b) : p.sk, start_in = p.starts ? __ldg(p.starts + b) : 0, prefix = p.prefixes ? __ldg(p.prefixes + b) : 0;
  int len = len_in;
  if (p.lengths) {
    if (len < 0 || len > p.sk) {
      if (tid == 0) { *p.status.host = kStatusLength; *p.status.device = kStatusLength; }
      len = min(max(len, 0), p.sk);
    }
  }
  if (tid == 0) { s_top = 0; s_doc_min = INT_MAX; s_doc_max = -1; }
  __syncthreads();
  // what each row sees: keys [0, hi) of its own document
  if (tid < ROWS) {
    const int r = row0 + tid;
    int hi = 0, doc = -1;
    long long pos = 0;
    if (r < n_rows) {
      pos = (p.starts ? (long long)start_in : (long long)len - p.sq) + r / p.group;
      if (!p.causal) hi = len;
      else if (pos >= 0 && pos < len) hi = min((long long)len, max(pos + 1, (long long)prefix));
      if (p.documents) {
        doc = pos >= 0 && pos < p.sk ? p.documents[(long long)b * p.sk + pos] : -1;
        if (doc < 0) hi = 0;
      }
    }
    s_hi[tid] = hi;
    // (for distances alone: moving a row that lies outside the keys up to them adds one number to all its scores, which the
    // softmax does not see and 32 bits hold better)
    s_pos[tid] = (int)min(max(pos, 0ll), (long long)len);
    s_doc[tid] = doc;
    if (hi > 0) {
      atomicMax(&s_top, hi);
      if (p.documents) { atomicMin(&s_doc_min, doc); atomicMax(&s_doc_max, doc); }
    }
  }
  __syncthreads();

  const int n_tiles = (s_top + KT - 1) / KT;
  const int per = ((n_tiles + splits * KG - 1) / (splits * KG)) * KG;    // tiles of this CTA, a whole number per group
  const int t_begin = split * per, t_end = min(n_tiles, t_begin + per);
  const int2* ranges = p.documents ? p.doc_ranges + (long long)b * ((p.sk + kDocBlock - 1) / kDocBlock) : nullptr;
  const int doc_min = s_doc_min, doc_max = s_doc_max;
  auto next = [&](int t) {       // the first tile from t on, in steps of this group, that holds a key some row may see
    if (ranges)
      while (t < t_end) {
        const int2 rg = __ldg(ranges + t * KT / kDocBlock);
        if ((rg.x & 0x7fffffff) <= doc_max && rg.y >= doc_min) break;
        t += KG;
      }
    return t;
  };
  const T* kp = reinterpret_cast<const T*>(p.k.ptr) + b * p.k.sb + hk * p.k.sh;
  const T* vp = reinterpret_cast<const T*>(p.v.ptr) + b * p.v.sb + hk * p.v.sh;
  auto tile_ptr = [&](int stage, int which) { return reinterpret_cast<T*>(ring + ((stage * KG + kg) * 2 + which) * C::TileBytes); };
  // K and V rows of a tile; rows at or behind the sequence's length become zeros whatever the cache holds there
  auto load = [&](int tile, int stage) {
    const int key0 = tile * KT;
    T* dk = tile_ptr(stage, 0);
    T* dv = tile_ptr(stage, 1);
    constexpr int PER = 16 / C::ES, CPR = DP / PER;
    if ((vec & 1) && GT % CPR == 0) {
      // a thread keeps its column and steps down the rows
      const int r0 = gt / CPR, c = (gt - r0 * CPR) * PER;
      constexpr int STEP = GT / CPR;
      const T* ks = kp + (long long)(key0 + r0) * p.k.sr + c;
      const T* vs = vp + (long long)(key0 + r0) * p.v.sr + c;
      const int rows = c < p.d ? len - key0 - r0 : 0;          // of this column, counted from r0
#pragma unroll
      for (int r = 0; r < KT; r += STEP) {
        const bool there = r < rows;
        cp_async16(dk + (r0 + r) * LD + c, there ? ks : kp, there);
        cp_async16(dv + (r0 + r) * LD + c, there ? vs : vp, there);
        ks += STEP * p.k.sr;
        vs += STEP * p.v.sr;
      }
    } else if (vec & 1) {
#pragma unroll
      for (int i0 = 0; i0 < KT * CPR; i0 += GT) {
        const int i = i0 + gt;
        if (KT * CPR % GT == 0 || i < KT * CPR) {
          const int r = i / CPR, c = (i - r * CPR) * PER;
          const bool there = key0 + r < len && c < p.d;
          const long long key = there ? key0 + r : 0;
          const int col = there ? c : 0;
          cp_async16(dk + r * LD + c, kp + key * p.k.sr + col, there);
          cp_async16(dv + r * LD + c, vp + key * p.v.sr + col, there);
        }
      }
    } else {
      for (int i = gt; i < KT * DP; i += GT) {
        const int r = i / DP, c = i - r * DP;
        const bool there = key0 + r < len && c < p.d;
        dk[r * LD + c] = there ? kp[(long long)(key0 + r) * p.k.sr + c] : narrow<T>(0.0f);
        dv[r * LD + c] = there ? vp[(long long)(key0 + r) * p.v.sr + c] : narrow<T>(0.0f);
      }
    }
  };
  auto group_sync = [&]() {
    if (RT == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(kg + 1), "n"(GT) : "memory");
  };

  const int g = lane >> 2, t4 = lane & 3;
  const int ra = rt * 16 + g;                             // this lane's rows of the CTA's: ra and ra + 8
  const int hi_r[2] = {s_hi[ra], s_hi[ra + 8]}, pos_r[2] = {s_pos[ra], s_pos[ra + 8]}, doc_r[2] = {s_doc[ra], s_doc[ra + 8]};
  float slope_r[2] = {0.f, 0.f};
  if (p.slopes)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (row0 + ra + 8 * i < n_rows) slope_r[i] = p.slopes[hk * p.group + (row0 + ra + 8 * i) % p.group] * kLog2e;
  const float to_log2 = p.cap > 0.f ? p.cap * kLog2e : p.scale * kLog2e, to_cap = p.cap > 0.f ? p.scale / p.cap : 0.f;

  float o[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m_r[2] = {-CUDART_INF_F, -CUDART_INF_F}, l_r[2] = {0.f, 0.f};

  int lt = next(t_begin + kg), ct = lt, issued = 0, done = 0;
  // query rows -> shared memory, zeros where there is none; they arrive with the first key tile
  if (vec & 2) {
    constexpr int PER = 16 / C::ES, CPR = DP / PER;
    for (int i = tid; i < ROWS * CPR; i += C::Threads) {
      const int r = i / CPR, c = (i - r * CPR) * PER;
      const bool there = row0 + r < n_rows && c < p.d;
      const int row = there ? row0 + r : 0, tok = row / p.group, gh = row - tok * p.group;
      cp_async16(sQ + r * LD + c, reinterpret_cast<const T*>(p.q.ptr) + b * p.q.sb + tok * p.q.sr + (long long)(hk * p.group + gh) * p.q.sh + (there ? c : 0), there);
    }
  } else {
    for (int i = tid; i < ROWS * DP; i += C::Threads) {
      const int r = i / DP, d = i - r * DP;
      T v = narrow<T>(0.0f);
      if (row0 + r < n_rows && d < p.d) {
        const int tok = (row0 + r) / p.group, gh = (row0 + r) - tok * p.group;
        v = reinterpret_cast<const T*>(p.q.ptr)[b * p.q.sb + tok * p.q.sr + (long long)(hk * p.group + gh) * p.q.sh + d];
      }
      sQ[r * LD + d] = v;
    }
  }
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) {
    if (lt < t_end) { load(lt, issued % ST); lt = next(lt + KG); }
    ++issued;
    cp_async_commit();
  }
  cp_async_wait<ST - 2>();
  __syncthreads();
  constexpr bool QREG = C::ES == 2 && DP <= 128;
  uint32_t q_frag[QREG ? DP / 16 : 1][4];
  if (QREG)
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) ldsm4(q_frag[QREG ? kk : 0], sQ + (rt * 16 + (lane & 15)) * LD + kk * 16 + (lane >> 4) * 8);

  while (ct < t_end) {
    cp_async_wait<ST - 2>();
    group_sync();
    if (lt < t_end) { load(lt, issued % ST); lt = next(lt + KG); }
    ++issued;
    cp_async_commit();
    const T* tk = tile_ptr(done % ST, 0);
    const T* tv = tile_ptr(done % ST, 1);
    const int key0 = ct * KT;
    ++done;
    ct = next(ct + KG);
    float s[KT / 8][4];
#pragma unroll
    for (int n = 0; n < KT / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
    if constexpr (C::ES == 2) {
      // a chain of dependent products is as long as the head: odd steps go to one of their own
      float s2[KT / 8][4];
#pragma unroll
      for (int n = 0; n < KT / 8; ++n) s2[n][0] = s2[n][1] = s2[n][2] = s2[n][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        uint32_t a[4];
        if (QREG) {
#pragma unroll
          for (int i = 0; i < 4; ++i) a[i] = q_frag[QREG ? kk : 0][i];
        } else ldsm4(a, sQ + (rt * 16 + (lane & 15)) * LD + kk * 16 + (lane >> 4) * 8);
#pragma unroll
        for (int n = 0; n < KT / 16; ++n) {
          uint32_t kf[4];
          ldsm4(kf, tk + (n * 16 + (lane >> 4) * 8 + (lane & 7)) * LD + kk * 16 + ((lane >> 3) & 1) * 8);
          mma16<T>(kk & 1 ? s2[2 * n] : s[2 * n], a, kf[0], kf[1]);
          mma16<T>(kk & 1 ? s2[2 * n + 1] : s[2 * n + 1], a, kf[2], kf[3]);
        }
      }
#pragma unroll
      for (int n = 0; n < KT / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] += s2[n][e];
    } else {
      const float* qf = reinterpret_cast<const float*>(sQ) + ra * LD + t4;
      const float* kf = reinterpret_cast<const float*>(tk) + g * LD + t4;
      // Four chains for hi.hi and one for the small products: the tensor core truncates as it adds, a bias of half a step
      // each time, which a single chain of the whole head would raise to 10^-6 of the score; and they run side by side.
      float c[KT / 8][5][4];
#pragma unroll
      for (int n = 0; n < KT / 8; ++n)
#pragma unroll
        for (int j = 0; j < 5; ++j) c[n][j][0] = c[n][j][1] = c[n][j][2] = c[n][j][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < DP / 8; ++kk) {
        uint32_t ah[4], al[4];
        split_tf32(qf[kk * 8], ah[0], al[0]);
        split_tf32(qf[kk * 8 + 8 * LD], ah[1], al[1]);
        split_tf32(qf[kk * 8 + 4], ah[2], al[2]);
        split_tf32(qf[kk * 8 + 8 * LD + 4], ah[3], al[3]);
#pragma unroll
        for (int n = 0; n < KT / 8; ++n) {
          uint32_t bh2[2], bl2[2];
          split_tf32(kf[n * 8 * LD + kk * 8], bh2[0], bl2[0]);
          split_tf32(kf[n * 8 * LD + kk * 8 + 4], bh2[1], bl2[1]);
          mma_tf32(c[n][4], al, bh2);
          mma_tf32(c[n][kk & 3], ah, bh2);
          mma_tf32(c[n][4], ah, bl2);
        }
      }
#pragma unroll
      for (int n = 0; n < KT / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = ((c[n][0][e] + c[n][1][e]) + (c[n][2][e] + c[n][3][e])) + c[n][4][e];
    }
    // scores -> the exponent's unit (powers of two), rules, maximum
    const float to_exponent = p.cap > 0.f ? to_cap : to_log2;
#pragma unroll
    for (int n = 0; n < KT / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] *= to_exponent;
    if (p.cap > 0.f) cap_scores<T, KT / 2>(&s[0][0], to_log2);
    float mx[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
    for (int n = 0; n < KT / 8; ++n) {
      const int key = key0 + n * 8 + 2 * t4;
      int kd[2] = {0, 0};
      if (p.documents) {
        const int* dp = p.documents + (long long)b * p.sk;
        kd[0] = key < p.sk ? __ldg(dp + key) : -1;
        kd[1] = key + 1 < p.sk ? __ldg(dp + key + 1) : -1;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = e >> 1, kx = key + (e & 1);
        float y = s[n][e];
        if (p.slopes) y = fmaf(-slope_r[r], fabsf((float)(pos_r[r] - kx)), y);
        const bool seen = kx < hi_r[r] && (!p.documents || kd[e & 1] == doc_r[r]);
        s[n][e] = seen ? y : -CUDART_INF_F;
        mx[r] = fmaxf(mx[r], s[n][e]);
      }
    }
    float alpha[2], m_use[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      mx[r] = below<T>(mx[r]);
      const float m_new = fmaxf(m_r[r], mx[r]);
      m_use[r] = m_new == -CUDART_INF_F ? 0.f : m_new;
      alpha[r] = ex2(m_r[r] - m_use[r]);
      m_r[r] = m_new;
    }
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < KT / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = ex2(s[n][e] - m_use[e >> 1]);
        sum[e >> 1] += s[n][e];
      }
    l_r[0] = l_r[0] * alpha[0] + sum[0];
    l_r[1] = l_r[1] * alpha[1] + sum[1];
    if constexpr (C::ES == 2) {
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) { o[n][0] *= alpha[0]; o[n][1] *= alpha[0]; o[n][2] *= alpha[1]; o[n][3] *= alpha[1]; }
      }
#pragma unroll
      for (int kk = 0; kk < KT / 16; ++kk) {
        const uint32_t a[4] = {pack2<T>(s[2 * kk][0], s[2 * kk][1]), pack2<T>(s[2 * kk][2], s[2 * kk][3]),
                               pack2<T>(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack2<T>(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
          uint32_t vf[4];
          ldsm4_t(vf, tv + (kk * 16 + (lane & 15)) * LD + n * 16 + (lane >> 4) * 8);
          mma16<T>(o[2 * n], a, vf[0], vf[1]);
          mma16<T>(o[2 * n + 1], a, vf[2], vf[3]);
        }
      }
    } else {
      // the k index of this product is a key: its column t4 is taken as key 2 t4 and column t4 + 4 as key 2 t4 + 1, which
      // is where the score product left them
      uint32_t ph[KT / 8][4], pl[KT / 8][4];
#pragma unroll
      for (int n = 0; n < KT / 8; ++n) {
        split_tf32(s[n][0], ph[n][0], pl[n][0]);
        split_tf32(s[n][2], ph[n][1], pl[n][1]);
        split_tf32(s[n][1], ph[n][2], pl[n][2]);
        split_tf32(s[n][3], ph[n][3], pl[n][3]);
      }
      const float* vf = reinterpret_cast<const float*>(tv) + 2 * t4 * LD + g;
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KT / 8; ++kk) {
          uint32_t bh2[2], bl2[2];
          split_tf32(vf[kk * 8 * LD + n * 8], bh2[0], bl2[0]);
          split_tf32(vf[(kk * 8 + 1) * LD + n * 8], bh2[1], bl2[1]);
          mma_tf32(acc, pl[kk], bh2);
          mma_tf32(acc, ph[kk], bl2);
          mma_tf32(acc, ph[kk], bh2);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = fmaf(o[n][e], alpha[e >> 1], acc[e]);
      }
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l_r[r] += __shfl_xor_sync(0xffffffffu, l_r[r], 1);
    l_r[r] += __shfl_xor_sync(0xffffffffu, l_r[r], 2);
  }
  // ---- join the key groups: every warp leaves its 16 rows in shared memory ----
  grid_launch_dependents();
  __syncthreads();
  float* mo = reinterpret_cast<float*>(ring) + warp * 16 * C::MergeLd;
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) {
    *reinterpret_cast<float2*>(mo + g * C::MergeLd + n * 8 + 2 * t4) = make_float2(o[n][0], o[n][1]);
    *reinterpret_cast<float2*>(mo + (g + 8) * C::MergeLd + n * 8 + 2 * t4) = make_float2(o[n][2], o[n][3]);
  }
  if (t4 == 0) {
    s_m[warp * 16 + g] = m_r[0]; s_m[warp * 16 + g + 8] = m_r[1];
    s_l[warp * 16 + g] = l_r[0]; s_l[warp * 16 + g + 8] = l_r[1];
  }
  __syncthreads();
  T* op = reinterpret_cast<T*>(const_cast<void*>(p.out.ptr)) + b * p.out.sb;
  auto store = [&](int r, int d, const float4& v) {      // four values of row r, from d on
    const int tok = (row0 + r) / p.group, gh = (row0 + r) - tok * p.group;
    T* dst = op + tok * p.out.sr + (long long)(hk * p.group + gh) * p.out.sh + d;
    const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < p.d) dst[i] = narrow<T>(x[i]);
  };
  constexpr int Q4 = DP / 4;
  const int live = min(ROWS, n_rows - row0);
  float* part = partials ? partials + ((long long)unit * splits + split) * (ROWS * (DP + 2)) : nullptr;
  for (int i = tid; i < live * Q4; i += C::Threads) {
    const int r = i / Q4, d = (i - r * Q4) * 4;
    float m = -CUDART_INF_F, l = 0.f;
#pragma unroll
    for (int k = 0; k < KG; ++k) m = fmaxf(m, s_m[(k * RT + (r >> 4)) * 16 + (r & 15)]);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (m != -CUDART_INF_F)
#pragma unroll
      for (int k = 0; k < KG; ++k) {
        const int w = (k * RT + (r >> 4)) * 16 + (r & 15);
        const float f = ex2(s_m[w] - m);
        const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<float*>(ring) + w * C::MergeLd + d);
        l = fmaf(f, s_l[w], l);
        a.x = fmaf(f, v.x, a.x); a.y = fmaf(f, v.y, a.y); a.z = fmaf(f, v.z, a.z); a.w = fmaf(f, v.w, a.w);
      }
    if (!part) {
      const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);     // a row without keys is zero; NaN stays NaN
      store(r, d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
    } else {
      *reinterpret_cast<float4*>(part + r * DP + d) = a;
      if (d == 0) { part[ROWS * DP + r] = m; part[ROWS * DP + ROWS + r] = l; }
    }
  }
}

// fp32 with at most four query rows a key head: no tensor core.  Sixteen MMA rows would stand empty, and splitting every
// key and value into tf32 parts costs more instructions than the products (8 heads of 53307 keys of 128: 121 us that way).
// A warp owns tiles of eight keys.  Scores: four lanes a key, each a quarter of the head, for every row; then each of the
// four has one row's score.  P V: a lane holds four values of the result of every row and takes the probabilities by
// shuffle.  All in plain 32-bit arithmetic; groups and splits are joined as above.
template <int DP_, int R_>
struct FewCfg {
  static constexpr int DP = DP_, R = R_, KT = 8, Warps = DP > 128 ? 4 : 8, Threads = Warps * 32;
  static constexpr int LD = DP % 32 == 0 ? DP + 16 : DP;         // rows of two keys lie 16 banks apart
  static constexpr int TileFloats = KT * LD;
  static constexpr int Stages = 2;
  static constexpr int RingBytes = Stages * Warps * 2 * TileFloats * 4;
  static constexpr int QBytes = R * DP * 4;
  static constexpr int MergeBytes = Warps * R * DP * 4;
  static constexpr int Smem = QBytes + (RingBytes > MergeBytes ? RingBytes : MergeBytes);
};

template <int DP, int R>
__global__ void __launch_bounds__(FewCfg<DP, R>::Threads, DP <= 64 ? 2 : 1)
few_rows_kernel(const __grid_constant__ DecoderAttention p, int splits, int vec, float* partials) {
  using C = FewCfg<DP, R>;
  constexpr int KT = C::KT, LD = C::LD, KG = C::Warps, ST = C::Stages, ROWS = 16;      // (partial results keep the layout of 16 rows)
  extern __shared__ __align__(128) unsigned char smem[];
  float* sQ = reinterpret_cast<float*>(smem);
  float* ring = reinterpret_cast<float*>(smem + C::QBytes);
  __shared__ int s_hi[4], s_pos[4], s_doc[4];
  __shared__ float s_m[C::Warps * 4], s_l[C::Warps * 4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int unit = blockIdx.x / splits, split = blockIdx.x % splits;
  const int b = unit / p.hkv, hk = unit % p.hkv, n_rows = p.group * p.sq;
  const int len_in = p.lengths ? __ldg(p.lengths + b) : p.sk, start_in = p.starts ? __ldg(p.starts + b) : 0, prefix = p.prefixes ? __ldg(p.prefixes + b) : 0;
  const int len = min(max(len_in, 0), p.sk);
  if (len != len_in && tid == 0) { *p.status.host = kStatusLength; *p.status.device = kStatusLength; }
  if (tid < 4) {
    int hi = 0, doc = -1;
    long long pos = 0;
    if (tid < n_rows) {
      pos = (p.starts ? (long long)start_in : (long long)len - p.sq) + tid / p.group;
      if (!p.causal) hi = len;
      else if (pos >= 0 && pos < len) hi = min((long long)len, max(pos + 1, (long long)prefix));
      if (p.documents) {
        doc = pos >= 0 && pos < p.sk ? p.documents[(long long)b * p.sk + pos] : -1;
        if (doc < 0) hi = 0;
      }
    }
    s_hi[tid] = hi;
    // (for distances alone: moving a row that lies outside the keys up to them adds one number to all its scores, which the
    // softmax does not see and 32 bits hold better)
    s_pos[tid] = (int)min(max(pos, 0ll), (long long)len);
    s_doc[tid] = doc;
  }
  for (int i = tid; i < R * DP; i += C::Threads) {
    const int r = i / DP, d = i - r * DP, tok = r / p.group, gh = r - tok * p.group;
    sQ[i] = r < n_rows && d < p.d ? reinterpret_cast<const float*>(p.q.ptr)[b * p.q.sb + tok * p.q.sr + (long long)(hk * p.group + gh) * p.q.sh + d] : 0.f;
  }
  __syncthreads();
  int top = 0, doc_min = INT_MAX, doc_max = -1;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (s_hi[r] > 0) { top = max(top, s_hi[r]); doc_min = min(doc_min, s_doc[r]); doc_max = max(doc_max, s_doc[r]); }
  const int n_tiles = (top + KT - 1) / KT;
  const int per = ((n_tiles + splits * KG - 1) / (splits * KG)) * KG;
  const int t_begin = split * per, t_end = min(n_tiles, t_begin + per);
  const int2* ranges = p.documents ? p.doc_ranges + (long long)b * ((p.sk + kDocBlock - 1) / kDocBlock) : nullptr;
  auto next = [&](int t) {
    if (ranges)
      while (t < t_end) {
        const int2 rg = __ldg(ranges + t * KT / kDocBlock);
        if ((rg.x & 0x7fffffff) <= doc_max && rg.y >= doc_min) break;
        t += KG;
      }
    return t;
  };
  const float* kp = reinterpret_cast<const float*>(p.k.ptr) + b * p.k.sb + hk * p.k.sh;
  const float* vp = reinterpret_cast<const float*>(p.v.ptr) + b * p.v.sb + hk * p.v.sh;
  auto tile_ptr = [&](int stage, int which) { return ring + ((stage * KG + warp) * 2 + which) * C::TileFloats; };
  auto load = [&](int tile, int stage) {
    const int key0 = tile * KT;
    float* dk = tile_ptr(stage, 0);
    float* dv = tile_ptr(stage, 1);
    if (vec) {
      constexpr int CPR = DP / 4;
#pragma unroll
      for (int i = lane; i < KT * CPR; i += 32) {
        const int r = i / CPR, c = (i - r * CPR) * 4;
        const bool there = key0 + r < len && c < p.d;
        const long long key = there ? key0 + r : 0;
        const int col = there ? c : 0;
        cp_async16(dk + r * LD + c, kp + key * p.k.sr + col, there);
        cp_async16(dv + r * LD + c, vp + key * p.v.sr + col, there);
      }
    } else {
      for (int i = lane; i < KT * DP; i += 32) {
        const int r = i / DP, c = i - r * DP;
        const bool there = key0 + r < len && c < p.d;
        dk[r * LD + c] = there ? kp[(long long)(key0 + r) * p.k.sr + c] : 0.f;
        dv[r * LD + c] = there ? vp[(long long)(key0 + r) * p.v.sr + c] : 0.f;
      }
    }
  };
  const int part = lane & 3, my_row = part < R ? part : part % R;
  const int hi = s_hi[my_row], pos = s_pos[my_row], doc = s_doc[my_row];
  const float slope = p.slopes && my_row < n_rows ? p.slopes[hk * p.group + my_row % p.group] * kLog2e : 0.f;
  const float to_log2 = p.cap > 0.f ? p.cap * kLog2e : p.scale * kLog2e, to_cap = p.cap > 0.f ? p.scale / p.cap : 0.f;
  constexpr int PER = (DP + 127) / 128;
  float4 o[R][PER];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < PER; ++i) o[r][i] = make_float4(0.f, 0.f, 0.f, 0.f);
  float m = -CUDART_INF_F, l = 0.f;                     // of my_row, the same in the eight lanes that share it
  int lt = next(t_begin + warp), ct = lt, issued = 0, done = 0;
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) {
    if (lt < t_end) { load(lt, issued % ST); lt = next(lt + KG); }
    ++issued;
    cp_async_commit();
  }
  while (ct < t_end) {
    cp_async_wait<ST - 2>();
    __syncwarp();
    if (lt < t_end) { load(lt, issued % ST); lt = next(lt + KG); }
    ++issued;
    cp_async_commit();
    const float* tk = tile_ptr(done % ST, 0) + (lane >> 2) * LD + part * 4;
    const float* tv = tile_ptr(done % ST, 1) + lane * 4;
    const int key = ct * KT + (lane >> 2);
    ++done;
    ct = next(ct + KG);
    float acc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = 0.f;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const float4 kv = *reinterpret_cast<const float4*>(tk + i * 16);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float4 qv = *reinterpret_cast<const float4*>(sQ + r * DP + i * 16 + part * 4);
        acc[r] = fmaf(kv.x, qv.x, fmaf(kv.y, qv.y, fmaf(kv.z, qv.z, fmaf(kv.w, qv.w, acc[r]))));
      }
    }
    float y = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], 1);
      acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], 2);
      if (r == my_row) y = acc[r];
    }
    y = p.cap > 0.f ? to_log2 * tanhf(y * to_cap) : y * to_log2;
    if (p.slopes) y = fmaf(-slope, fabsf((float)(pos - key)), y);
    bool seen = key < hi;
    if (p.documents) seen = seen && __ldg(p.documents + (long long)b * p.sk + min(key, p.sk - 1)) == doc;
    y = seen ? y : -CUDART_INF_F;
    float mx = y;
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    const float m_new = fmaxf(m, mx), m_use = m_new == -CUDART_INF_F ? 0.f : m_new;
    const float alpha = ex2(m - m_use), pr = ex2(y - m_use);
    m = m_new;
    float sum = pr;
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    l = fmaf(l, alpha, sum);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float al = __shfl_sync(0xffffffffu, alpha, r);
#pragma unroll
      for (int i = 0; i < PER; ++i) { o[r][i].x *= al; o[r][i].y *= al; o[r][i].z *= al; o[r][i].w *= al; }
    }
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      float pk[R];
#pragma unroll
      for (int r = 0; r < R; ++r) pk[r] = __shfl_sync(0xffffffffu, pr, k * 4 + r);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (DP % 128 != 0 && i * 128 + lane * 4 >= DP) continue;
        const float4 v = *reinterpret_cast<const float4*>(tv + k * LD + i * 128);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          o[r][i].x = fmaf(pk[r], v.x, o[r][i].x); o[r][i].y = fmaf(pk[r], v.y, o[r][i].y);
          o[r][i].z = fmaf(pk[r], v.z, o[r][i].z); o[r][i].w = fmaf(pk[r], v.w, o[r][i].w);
        }
      }
    }
  }
  cp_async_wait<0>();
  grid_launch_dependents();
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i * 128 + lane * 4 < DP) *reinterpret_cast<float4*>(ring + (warp * R + r) * DP + i * 128 + lane * 4) = o[r][i];
  if (lane < R) { s_m[warp * 4 + lane] = m; s_l[warp * 4 + lane] = l; }
  __syncthreads();
  float* part_out = partials ? partials + ((long long)unit * splits + split) * (ROWS * (DP + 2)) : nullptr;
  const int live = min(R, n_rows);
  for (int i = tid; i < live * DP; i += C::Threads) {
    const int r = i / DP, d = i - r * DP;
    float top_m = -CUDART_INF_F, sum = 0.f, v = 0.f;
#pragma unroll
    for (int k = 0; k < KG; ++k) top_m = fmaxf(top_m, s_m[k * 4 + r]);
    if (top_m != -CUDART_INF_F)
#pragma unroll
      for (int k = 0; k < KG; ++k) {
        const float f = ex2(s_m[k * 4 + r] - top_m);
        sum = fmaf(f, s_l[k * 4 + r], sum);
        v = fmaf(f, ring[(k * R + r) * DP + d], v);
      }
    if (!part_out) {
      const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);
      const int tok = r / p.group, gh = r - tok * p.group;
      if (d < p.d) reinterpret_cast<float*>(const_cast<void*>(p.out.ptr))[b * p.out.sb + tok * p.out.sr + (long long)(hk * p.group + gh) * p.out.sh + d] = v * inv;
    } else {
      part_out[r * DP + d] = v;
      if (d == 0) { part_out[ROWS * DP + r] = top_m; part_out[ROWS * DP + ROWS + r] = sum; }
    }
  }
}

// Joins the parts of one row: four warps take the splits in turn, 16 bytes a lane.
template <typename T, int DP, int RT>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ DecoderAttention p, int splits, int row_tiles, const float* partials) {
  constexpr int ROWS = 16 * RT, STEP = ROWS * (DP + 2);
  __shared__ float s_part[4][DP], s_sum[4];
  grid_dependency_wait();
  const int unit = blockIdx.x / ROWS, r = blockIdx.x % ROWS, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_bh = p.b * p.hkv, row_tile = row_tiles - 1 - unit / n_bh, bh = unit % n_bh, b = bh / p.hkv, hk = bh % p.hkv;
  const int row = row_tile * ROWS + r;
  if (row >= p.group * p.sq) return;
  const float* all = partials + (long long)unit * splits * STEP;
  float top = -CUDART_INF_F;
  for (int k = lane; k < splits; k += 32) top = fmaxf(top, __ldg(all + (long long)k * STEP + ROWS * DP + r));
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  constexpr int PER = (DP + 127) / 128;
  float4 acc[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  if (top != -CUDART_INF_F)
#pragma unroll 4
    for (int k = warp; k < splits; k += 4) {
      const float* q = all + (long long)k * STEP;
      const float f = ex2(__ldg(q + ROWS * DP + r) - top);
      sum = fmaf(f, __ldg(q + ROWS * DP + ROWS + r), sum);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int d = i * 128 + lane * 4;
        if (d >= DP) continue;
        const float4 v = __ldg(reinterpret_cast<const float4*>(q + r * DP + d));
        acc[i].x = fmaf(f, v.x, acc[i].x); acc[i].y = fmaf(f, v.y, acc[i].y); acc[i].z = fmaf(f, v.z, acc[i].z); acc[i].w = fmaf(f, v.w, acc[i].w);
      }
    }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (i * 128 + lane * 4 < DP) *reinterpret_cast<float4*>(&s_part[warp][i * 128 + lane * 4]) = acc[i];
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  const float l = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
  const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
  const int tok = row / p.group, gh = row - tok * p.group;
  T* dst = reinterpret_cast<T*>(const_cast<void*>(p.out.ptr)) + b * p.out.sb + tok * p.out.sr + (long long)(hk * p.group + gh) * p.out.sh;
  for (int d = threadIdx.x; d < p.d; d += 128) dst[d] = narrow<T>(((s_part[0][d] + s_part[1][d]) + (s_part[2][d] + s_part[3][d])) * inv);
}

template <typename T, int DP, int RT>
cudaError_t launch_one(const DecoderAttention& p, const CacheAttnPlan& plan, float* partials, cudaStream_t s) {
  using C = Cfg<T, DP, RT>;
  static_assert(C::Smem + 4096 <= 227 * 1024, "shared memory of a CTA");
  const int row_tiles = (p.group * p.sq + 16 * RT - 1) / (16 * RT);
  const long long grid = (long long)p.b * p.hkv * row_tiles * plan.splits;
  if (grid <= 0 || grid > 0x7fffffffll) return cudaErrorInvalidValue;
  constexpr int per = 16 / C::ES;
  const int vec = p.d % per == 0 && (reinterpret_cast<uintptr_t>(p.k.ptr) & 15) == 0 && (reinterpret_cast<uintptr_t>(p.v.ptr) & 15) == 0 &&
                  p.k.sr % per == 0 && p.v.sr % per == 0 && p.k.sb % per == 0 && p.v.sb % per == 0 && p.k.sh % per == 0 && p.v.sh % per == 0 ? 1 : 0;
  const int qvec = p.d % per == 0 && (reinterpret_cast<uintptr_t>(p.q.ptr) & 15) == 0 && p.q.sr % per == 0 && p.q.sb % per == 0 && p.q.sh % per == 0 ? 2 : 0;
  cudaError_t e = allow_shared(cache_attention_kernel<T, DP, RT>, C::Smem);
  if (e != cudaSuccess) return e;
  cache_attention_kernel<T, DP, RT><<<(unsigned)grid, C::Threads, C::Smem, s>>>(p, plan.splits, row_tiles, vec | qvec, plan.splits > 1 ? partials : nullptr);
  e = cudaGetLastError();
  if (e != cudaSuccess || plan.splits == 1) return e;
  return launch_dependent(join_kernel<T, DP, RT>, dim3((unsigned)(grid / plan.splits * 16 * RT)), dim3(128), 0, s, p, plan.splits, row_tiles, (const float*)partials);
}

template <int DP, int R>
cudaError_t launch_few(const DecoderAttention& p, const CacheAttnPlan& plan, float* partials, cudaStream_t s) {
  using C = FewCfg<DP, R>;
  static_assert(C::Smem + 1024 <= 227 * 1024, "shared memory of a CTA");
  const long long grid = (long long)p.b * p.hkv * plan.splits;
  if (grid <= 0 || grid > 0x7fffffffll) return cudaErrorInvalidValue;
  const int vec = p.d % 4 == 0 && (reinterpret_cast<uintptr_t>(p.k.ptr) & 15) == 0 && (reinterpret_cast<uintptr_t>(p.v.ptr) & 15) == 0 &&
                  p.k.sr % 4 == 0 && p.v.sr % 4 == 0 && p.k.sb % 4 == 0 && p.v.sb % 4 == 0 && p.k.sh % 4 == 0 && p.v.sh % 4 == 0;
  cudaError_t e = allow_shared(few_rows_kernel<DP, R>, C::Smem);
  if (e != cudaSuccess) return e;
  few_rows_kernel<DP, R><<<(unsigned)grid, C::Threads, C::Smem, s>>>(p, plan.splits, vec, plan.splits > 1 ? partials : nullptr);
  e = cudaGetLastError();
  if (e != cudaSuccess || plan.splits == 1) return e;
  return launch_dependent(join_kernel<float, DP, 1>, dim3((unsigned)(grid / plan.splits * 16)), dim3(128), 0, s, p, plan.splits, 1, (const float*)partials);
}

template <typename T, int DP>
cudaError_t launch_rows(const DecoderAttention& p, const CacheAttnPlan& plan, float* partials, cudaStream_t s) {
  if constexpr (sizeof(T) == 4) {
    const int rows = p.group * p.sq;
    if (rows == 1) return launch_few<DP, 1>(p, plan, partials, s);
    if (rows == 2) return launch_few<DP, 2>(p, plan, partials, s);
    if (rows <= 4) return launch_few<DP, 4>(p, plan, partials, s);
  }
  return plan.row_tiles == 1 ? launch_one<T, DP, 1>(p, plan, partials, s)
         : plan.row_tiles == 2 ? launch_one<T, DP, 2>(p, plan, partials, s) : launch_one<T, DP, 4>(p, plan, partials, s);
}

inline int padded_head(int d) { return d <= 64 ? 64 : d <= 80 ? 80 : d <= 96 ? 96 : d <= 128 ? 128 : 256; }

template <typename T>
cudaError_t launch_typed(const DecoderAttention& p, const CacheAttnPlan& plan, float* partials, cudaStream_t s) {
  switch (padded_head(p.d)) {
    case 64: return launch_rows<T, 64>(p, plan, partials, s);
    case 80: return launch_rows<T, 80>(p, plan, partials, s);
    case 96: return launch_rows<T, 96>(p, plan, partials, s);
    case 128: return launch_rows<T, 128>(p, plan, partials, s);
    default: return launch_rows<T, 256>(p, plan, partials, s);
  }
}

// one translation unit per type
cudaError_t launch_bf16(const DecoderAttention& p, const CacheAttnPlan& plan, float* partials, cudaStream_t s);
cudaError_t launch_f16(const DecoderAttention& p, const CacheAttnPlan& plan, float* partials, cudaStream_t s);
cudaError_t launch_f32(const DecoderAttention& p, const CacheAttnPlan& plan, float* partials, cudaStream_t s);

}  // namespace cache_attn
}  // namespace bg
