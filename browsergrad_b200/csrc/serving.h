// Internal declarations of the serving operators: rotary positions, attention over a key / value cache, token sampling.
#pragma once

#include "common.h"

namespace bg {

// A resolved bg_head_view: element strides over batch, row and head; the values of one head are contiguous.
struct HeadPtr {
  const void* ptr;
  int64_t sb, sr, sh;
};
// Where a kernel reports refused data: the context's device word, and its pinned host copy (device-visible), so that no
// copy has to follow the launch.
struct StatusWords {
  int* device;
  int* host;
};
// What they report there: a bg_status in the low byte, the operator above it.
constexpr int kStatusAppend = BG_ERR_INDEX_RANGE | 1 << 8;
constexpr int kStatusLength = BG_ERR_INDEX_RANGE | 2 << 8;
constexpr int kStatusPromptWait = BG_ERR_DEVICE_TIMEOUT | 3 << 8;

// Raises a kernel's limit of dynamic shared memory where it is below `bytes`, which is remembered (the call costs about a
// microsecond).  The limit belongs to the kernel on its device and is shared by all threads and contexts: it is never
// lowered, and the lock is held across the change, so that a larger one of another thread is not overwritten.
cudaError_t allow_shared(const void* kern, size_t bytes);
template <typename... Args>
cudaError_t allow_shared(void (*kern)(Args...), size_t bytes) { return allow_shared(reinterpret_cast<const void*>(kern), bytes); }

// ---- rotary.cu ---------------------------------------------------------------------------------------------------
constexpr int kRotaryMaxPairs = 128;
struct RotarySegment {
  HeadPtr in, out;
  int heads;
  int turn;        // rotate (else copy)
  int cached;      // rows go to start + s of the cache, those at or behind counts[b] nowhere
};
struct RotaryProblem {
  RotarySegment seg[3];
  int n_seg;
  int b, s, d, rot, interleaved;
  int64_t capacity;           // rows of the caches
  int64_t start;
  const int* starts;          // [b] or null (then `start`)
  const int* positions;       // [b, s] or null (then start + s)
  const int* counts;          // [b] or null (then s)
  float magnitude;
  double turns[kRotaryMaxPairs];   // full turns per position of each pair, signed by the direction
  StatusWords status;
};
cudaError_t launch_rotary(const RotaryProblem& p, int dtype, cudaStream_t s, int sm_count);

// ---- attention over a cache --------------------------------------------------------------------------------------
struct DecoderAttention {
  int b, hq, hkv, group, sq, sk, d;
  HeadPtr q, k, v, out;       // k, v: heads are the hkv shared ones
  float scale;
  float cap;                  // 0: none
  const float* slopes;        // [hq] or null
  const int* documents;       // [b, sk] or null
  const int* prefixes;        // [b] or null
  const int* lengths;         // [b] or null (then sk)
  const int* starts;          // [b] or null (then lengths[b] - sq)
  int causal;
  const int2* doc_ranges;     // [b, ceil(sk / 128)] smallest and largest id of each 128 keys, the smallest with its sign bit
                              // set when some of them belong to no document; set with documents
  float* sums;                // prompt_attention_scratch() bytes, or null where that is none
  StatusWords status;
};
constexpr int kDocBlock = 128;
cudaError_t launch_doc_ranges(const int* documents, int b, int sk, int2* ranges, cudaStream_t s);

#ifdef __CUDACC__
// tanh(x) / x from z = x^2 <= 1, fitted to a largest relative error of 6.2e-7: what 16-bit attention caps its scores with.
// Relative, so that a cap far above the scores costs them no digits.
__device__ __forceinline__ float tanh_ratio(float z) {
  float p = fmaf(z, -0.003067060373723507f, 0.016743116080760956f);
  p = fmaf(z, p, -0.051605675369501114f);
  p = fmaf(z, p, 0.13281433284282684f);
  p = fmaf(z, p, -0.3332904279232025f);
  return fmaf(z, p, 0.9999994039535522f);
}
// `within` where z <= 1, else `beyond`: a selection between two values at hand (a branch for each score would diverge).
__device__ __forceinline__ float within_one(float z, float within, float beyond) {
  float y;
  asm("{\n\t.reg .pred p;\n\tsetp.le.f32 p, %1, 0f3F800000;\n\tselp.f32 %0, %2, %3, p;\n\t}" : "=f"(y) : "f"(z), "f"(within), "f"(beyond));
  return y;
}
#endif

// Key-split kernel (cache_attn.cu): every type and head size up to 256, few rows per key head or many.
struct CacheAttnPlan {
  int row_tiles;        // 16-row tiles one CTA works on
  int splits;           // CTAs that share the keys of one set of rows
  int64_t partial_bytes;
};
CacheAttnPlan cache_attention_plan(const DecoderAttention& p, int dtype, int sm_count);
cudaError_t launch_cache_attention(const DecoderAttention& p, int dtype, const CacheAttnPlan& plan, float* partials, cudaStream_t s);

// Prompts of 16-bit operands (prompt_attn.cu).
bool prompt_attention_usable(const DecoderAttention& p, int dtype);
int64_t prompt_attention_scratch(const DecoderAttention& p, int dtype);
cudaError_t launch_prompt_attention(const DecoderAttention& p, int dtype, cudaStream_t s);

// ---- sample.cu ---------------------------------------------------------------------------------------------------
constexpr int64_t kSampleMaxVocab = 1 << 20;     // up to here a running sum is good to the step of the numbers drawn with
struct SampleProblem {
  const void* logits;
  int64_t n, vocab;
  const float* uniforms;
  const float* temperatures; float temperature;
  const int* top_ks; int top_k;
  const float* top_ps; float top_p;
  const float* min_ps; float min_p;
  int64_t* tokens;
  float* probabilities;       // or null
};
cudaError_t launch_sample(const SampleProblem& p, int dtype, cudaStream_t s, int sm_count);

}  // namespace bg
