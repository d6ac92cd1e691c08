// Rotary positions, alone or together with the append of new keys and values to a cache (sm_100a).
//
// A pair (a, b) of a head at position t becomes (a cos w - b sin w, a sin w + b cos w), w = t f_j.  The work is bound by
// memory: every value is read and written once.  A CTA takes a few consecutive tokens of one sequence with all their
// heads, so the angles -- which all heads share -- are computed once per token into shared memory and the loop over heads
// only loads, multiplies and stores, 16 bytes per access, both halves of a pair's vectors in flight together.
// Angles: t f_j reaches 10^6 radians and more, where 32 bits leave no fraction; the product is formed in 64 bits as turns
// (f_j / 2 pi comes from the host), its whole part is taken off, and sine and cosine of the fraction are 32-bit.  The
// rotation is done in 32 bits and rounded once to the stored type.
// Eight CTAs an SM (32 registers a thread) hide the load latency: 32771 tokens of 32 heads of 128, bf16, 96 to 108 us on different
// machines = 5.0 to 5.6 TB/s; on the fastest of them 104 us at 40 registers and 121 with the next item fetched ahead.  Ragged
// prompts into a cache (6 x 1537 tokens, 32 + 8 + 8 heads of 128, f16, interleaved pairs) 39 to 41 us = 5.1 to 5.3 TB/s,
// instruction issue 68 % busy.
#include "serving.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace bg {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Vec {
  T v[VEC];
};

// One item: the vectors at elements c * VEC of the first half and of the second half of the rotated part.  The sines and
// cosines of a token lie so that threads of neighbouring c read neighbouring words: the i-th value of every item together.
template <typename T, int VEC, bool INTER>
__device__ __forceinline__ void turn_item(Vec<T, VEC>& lo, Vec<T, VEC>& hi, const float2* cs, int c, int items) {
  if (!INTER) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float2 w = cs[i * items + c];
      const float a = to_f(lo.v[i]), b = to_f(hi.v[i]);
      lo.v[i] = from_f<T>(a * w.x - b * w.y);
      hi.v[i] = from_f<T>(a * w.y + b * w.x);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const float2 w = cs[(i >> 1) * items + c], z = cs[((VEC + i) >> 1) * items + c];
      const float a = to_f(lo.v[i]), b = to_f(lo.v[i + 1]), e = to_f(hi.v[i]), f = to_f(hi.v[i + 1]);
      lo.v[i] = from_f<T>(a * w.x - b * w.y);
      lo.v[i + 1] = from_f<T>(a * w.y + b * w.x);
      hi.v[i] = from_f<T>(e * z.x - f * z.y);
      hi.v[i + 1] = from_f<T>(e * z.y + f * z.x);
    }
  }
}
// Where turn_item looks for pair j's sine and cosine.
template <int VEC, bool INTER>
__device__ __forceinline__ int place_of(int j, int half) {
  const int items = half / VEC;
  if (VEC == 1) return j;
  if (!INTER) return (j % VEC) * items + j / VEC;
  constexpr int PER = VEC / 2 > 0 ? VEC / 2 : 1;          // pairs of one vector
  const int second = j >= half / 2 ? 1 : 0, q = j - second * (half / 2);
  return (second * PER + q % PER) * items + q / PER;
}

// VEC = 1 handles what vectors cannot: odd sizes, strides or addresses that are not multiples of a vector.  An item is
// then one pair of values, wherever the layout puts its two members.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kThreads, 8) rotary_kernel(const __grid_constant__ RotaryProblem p, int tokens_per_cta, int tiles) {
  __shared__ float2 s_cs[kMaxTokens * kRotaryMaxPairs];
  const int batch = blockIdx.x / tiles;
  const int s0 = (blockIdx.x % tiles) * tokens_per_cta;
  const int n_tok = min(tokens_per_cta, p.s - s0);
  const int half = p.rot >> 1;
  const int64_t first = p.starts ? (int64_t)p.starts[batch] : p.start;
  int64_t count = p.s;
  if (p.counts) {
    count = p.counts[batch];
    if (count < 0 || count > p.s) {
      if (threadIdx.x == 0) { *p.status.host = kStatusAppend; *p.status.device = kStatusAppend; }
      count = count < 0 ? 0 : p.s;
    }
  }
  for (int i = threadIdx.x; i < n_tok * half; i += kThreads) {
    const int tok = i / half, j = i - tok * half;
    const int64_t at = p.positions ? (int64_t)p.positions[(int64_t)batch * p.s + s0 + tok] : first + s0 + tok;
    const double turns = (double)at * p.turns[j];
    const float frac = (float)(turns - rint(turns));
    float sn, cs;
    sincospif(2.0f * frac, &sn, &cs);
    s_cs[tok * half + place_of<VEC, INTER>(j, half)] = make_float2(cs * p.magnitude, sn * p.magnitude);
  }
  __syncthreads();
  // items of a head: those of the rotated part, then the values behind it, two vectors an item
  const int pairs = half / VEC, rest = (p.d - p.rot) / VEC, rest_items = (rest + 1) / 2;
  const int per_head = pairs + rest_items;
  int h_total = 0;
  for (int g = 0; g < p.n_seg; ++g) h_total += p.seg[g].heads;
  using V = Vec<T, VEC>;
  // (c, head, tok) of this thread's items, advanced without divisions
  const int dc = kThreads % per_head, dh = (kThreads / per_head) % h_total, dt = kThreads / per_head / h_total;
  int c = threadIdx.x % per_head, head = (int)threadIdx.x / per_head % h_total, tok = (int)threadIdx.x / per_head / h_total;
  while (tok < n_tok) {
    int h = head, g = 0;
    while (h >= p.seg[g].heads) h -= p.seg[g++].heads;
    const RotarySegment& sg = p.seg[g];
    int64_t row_out = s0 + tok;
    bool keep = true;
    if (sg.cached) {
      keep = s0 + tok < count;
      row_out += first;
      if (keep && (row_out < 0 || row_out >= p.capacity)) {
        *p.status.host = kStatusAppend;
        *p.status.device = kStatusAppend;
        keep = false;
      }
    }
    if (keep) {
      const T* x = reinterpret_cast<const T*>(sg.in.ptr) + batch * sg.in.sb + (int64_t)(s0 + tok) * sg.in.sr + h * sg.in.sh;
      T* y = reinterpret_cast<T*>(const_cast<void*>(sg.out.ptr)) + batch * sg.out.sb + row_out * sg.out.sr + h * sg.out.sh;
      const bool turned = c < pairs;
      const int k = c - pairs;
      const int e0 = turned ? (VEC == 1 && INTER ? 2 * c : c * VEC) : p.rot + k * VEC;
      const int e1 = turned ? (VEC == 1 && INTER ? 2 * c + 1 : half + c * VEC) : p.rot + (k + rest_items) * VEC;
      const bool both = turned || k + rest_items < rest;
      V lo = *reinterpret_cast<const V*>(x + e0), hi = lo;
      if (both) hi = *reinterpret_cast<const V*>(x + e1);
      if (turned && sg.turn) turn_item<T, VEC, INTER && VEC != 1>(lo, hi, s_cs + tok * half, c, pairs);
      *reinterpret_cast<V*>(y + e0) = lo;
      if (both) *reinterpret_cast<V*>(y + e1) = hi;
    }
    c += dc;
    head += dh;
    tok += dt;
    if (c >= per_head) { c -= per_head; ++head; }
    if (head >= h_total) { head -= h_total; ++tok; }
  }
}

template <typename T, int VEC>
cudaError_t launch_vec(const RotaryProblem& p, cudaStream_t s) {
  int heads = 0;
  for (int g = 0; g < p.n_seg; ++g) heads += p.seg[g].heads;
  const int per_token = heads * (p.rot / 2 / VEC + ((p.d - p.rot) / VEC + 1) / 2);
  // four items a thread: enough loads in flight without emptying the grid
  int tok = (4 * kThreads + per_token - 1) / per_token;
  if (tok > kMaxTokens) tok = kMaxTokens;
  if (tok > p.s) tok = p.s;
  const int64_t tiles = (p.s + tok - 1) / tok;
  if (tiles * p.b > 0x7fffffffll) return cudaErrorInvalidValue;
  const unsigned grid = (unsigned)(tiles * p.b);
  if (p.interleaved) rotary_kernel<T, VEC, true><<<grid, kThreads, 0, s>>>(p, tok, (int)tiles);
  else rotary_kernel<T, VEC, false><<<grid, kThreads, 0, s>>>(p, tok, (int)tiles);
  return cudaGetLastError();
}

// Whether every access of `vec` elements is aligned to its own size.
bool vectors_fit(const RotaryProblem& p, int vec, int es) {
  if ((p.rot / 2) % vec || (p.d - p.rot) % vec) return false;
  for (int g = 0; g < p.n_seg; ++g)
    for (const HeadPtr* h : {&p.seg[g].in, &p.seg[g].out})
      if (reinterpret_cast<uintptr_t>(h->ptr) % (uintptr_t)(vec * es) || h->sb % vec || h->sr % vec || h->sh % vec) return false;
  return true;
}

}  // namespace

cudaError_t launch_rotary(const RotaryProblem& p, int dtype, cudaStream_t s, int) {
  const int es = dtype_size(dtype);
  if (dtype == BG_F32) return vectors_fit(p, 4, es) ? launch_vec<float, 4>(p, s) : launch_vec<float, 1>(p, s);
  const bool bf = dtype == BG_BF16;
  if (vectors_fit(p, 8, es)) return bf ? launch_vec<__nv_bfloat16, 8>(p, s) : launch_vec<__half, 8>(p, s);
  if (vectors_fit(p, 4, es)) return bf ? launch_vec<__nv_bfloat16, 4>(p, s) : launch_vec<__half, 4>(p, s);
  return bf ? launch_vec<__nv_bfloat16, 1>(p, s) : launch_vec<__half, 1>(p, s);
}

}  // namespace bg
