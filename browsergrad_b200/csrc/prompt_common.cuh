// What the prompt attention kernels (prompt_attn.cu, prompt_attn32.cu) share: which keys a row and a tile of rows see, and
// the tensor maps of strided heads.
#pragma once

#include <cuda.h>
#include <stdint.h>

#include "serving.h"

namespace bg {

// fp32 operands (prompt_attn32.cu)
bool prompt_attention32_usable(const DecoderAttention& p);
cudaError_t launch_prompt_attention32(const DecoderAttention& p, cudaStream_t s);

namespace prompt {

constexpr int kMaxPos = 1 << 30;
// Scores (in powers of two) from here on are a quarter or more apart in 32 bits.  The reference of their exponentials is then the
// largest of the rounded scores: an unrounded product, what the exponent takes otherwise, may lie half a step above it, and
// the exponential of that would pass the type (float16 from scores of 2^27 on).
constexpr float kCoarse = 2097152.0f;

// Bits of the keys (of `keys` that exist from docs on) whose document is this lane's.  Each key's id is read once per warp;
// the rows of a warp belong to few documents, so the words are made per document, by ballots, not per row.
__device__ __forceinline__ uint4 document_bits(const int* docs, int keys, int doc) {
  const int lane = threadIdx.x & 31;
  int id[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) id[c] = c * 32 + lane < keys ? __ldg(docs + c * 32 + lane) : -1;
  uint4 w = make_uint4(0u, 0u, 0u, 0u);
  uint32_t left = __ballot_sync(0xffffffffu, doc >= 0);
  while (left) {
    const int d = __shfl_sync(0xffffffffu, doc, __ffs(left) - 1);
    const uint4 v = make_uint4(__ballot_sync(0xffffffffu, id[0] == d), __ballot_sync(0xffffffffu, id[1] == d),
                               __ballot_sync(0xffffffffu, id[2] == d), __ballot_sync(0xffffffffu, id[3] == d));
    if (doc == d) w = v;
    left &= ~__ballot_sync(0xffffffffu, doc == d);
  }
  return w;
}
// What a CTA's sequence is about; the three are requested together.  A length outside the cache is reported and cut.
struct Sequence {
  int len, prefix;
  long long start;
};
__device__ __forceinline__ Sequence sequence_of(const DecoderAttention& a, int b) {
  const int n = a.lengths ? __ldg(a.lengths + b) : a.sk, st = a.starts ? __ldg(a.starts + b) : 0, pre = a.prefixes ? __ldg(a.prefixes + b) : 0;
  if ((n < 0 || n > a.sk) && threadIdx.x == 0) { *a.status.host = kStatusLength; *a.status.device = kStatusLength; }
  const int len = min(max(n, 0), a.sk);
  return Sequence{len, pre, a.starts ? (long long)st : (long long)len - a.sq};
}

// The position distances are taken from.  Moving a row that lies outside the keys up to them adds one number to all its
// scores, which the softmax does not see and 32 bits hold better.
__device__ __forceinline__ int distance_origin(const Sequence& q, int pos) { return min(max(pos, 0), q.len); }

// Rows [i0, i1] of sequence b: the positions among them that see any key, and how many keys the last of them sees.
struct Reach {
  int first, last, keys;       // first > last: none
};
__device__ __forceinline__ Reach reach_of(const DecoderAttention& a, const Sequence& q, int i0, int i1) {
  const int len = q.len;
  long long p0 = q.start + i0, p1 = q.start + i1;
  if (!a.causal) {
    p0 = min(max(p0, (long long)-kMaxPos), (long long)kMaxPos);
    p1 = min(max(p1, (long long)-kMaxPos), (long long)kMaxPos);
    return Reach{(int)p0, (int)p1, i0 <= i1 ? len : 0};
  }
  p0 = max(p0, 0ll);
  p1 = min(p1, (long long)len - 1);
  if (i0 > i1 || p0 > p1) return Reach{1, 0, 0};
  return Reach{(int)p0, (int)p1, (int)min((long long)len, max(p1 + 1, (long long)q.prefix))};
}

// Which tiles of KEYS keys rows [i0, i1] need: those in front of the last row's reach that, with documents, hold an id
// between the rows' smallest and largest.
template <int KEYS>
__device__ __forceinline__ void needed_tiles(const DecoderAttention& a, int b, const Sequence& q, int i0, int i1, unsigned char* need, int tid, int threads) {
  const int n_kv = (q.len + KEYS - 1) / KEYS, blocks = (a.sk + kDocBlock - 1) / kDocBlock;
  const int2* ranges = a.documents ? a.doc_ranges + (long long)b * blocks : nullptr;
  const Reach r = reach_of(a, q, i0, i1);
  int lo = INT_MAX, hi = -1;
  if (ranges && r.first <= r.last && r.last >= 0) {
    // at most 128 rows lie in two blocks
    const int t0 = min(max(r.first, 0) / kDocBlock, blocks - 1), t1 = min(r.last / kDocBlock, blocks - 1);
    const int2 x = __ldg(ranges + t0), y = __ldg(ranges + t1);
    lo = min(x.x & 0x7fffffff, y.x & 0x7fffffff);
    hi = max(x.y, y.y);
  }
  const int end = (r.keys + KEYS - 1) / KEYS;
  for (int j = tid; j < n_kv; j += threads) {
    bool n = j < end;
    if (ranges) {
      const int2 x = __ldg(ranges + j * KEYS / kDocBlock);
      n = n && (x.x & 0x7fffffff) <= hi && x.y >= lo;
    }
    need[j] = n;
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult qr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr) == cudaSuccess && qr == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(p);
    cudaGetLastError();
    return (EncodeTiledFn) nullptr;
  }();
  return fn;
}

// Boxes of `box_rows` rows x 128 bytes; values behind d and rows behind the last arrive as zeros.
inline bool make_map(CUtensorMap* map, const HeadPtr& v, int dtype, int b, int rows, int heads, int d, int box_rows,
                     CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
  const int es = dtype_size(dtype);
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)b};
  // an axis of extent one has no stride: any legal value will do
  const cuuint64_t any = ((cuuint64_t)d * es + 15) / 16 * 16;
  cuuint64_t strides[3] = {rows > 1 ? (cuuint64_t)(v.sr * es) : any, heads > 1 ? (cuuint64_t)(v.sh * es) : any, b > 1 ? (cuuint64_t)(v.sb * es) : any};
  cuuint32_t box[4] = {(cuuint32_t)(128 / es), (cuuint32_t)box_rows, 1, 1}, step[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = dtype == BG_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : dtype == BG_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  return fn(map, type, 4, const_cast<void*>(v.ptr), dims, strides,
            box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What TMA asks of a view: 16-byte steps below 2^40 bytes, no axis that stands still.
inline bool view_fits(const HeadPtr& v, int dtype, int b, int rows, int heads) {
  const int per = 16 / dtype_size(dtype);
  if (reinterpret_cast<uintptr_t>(v.ptr) & 15) return false;
  const int64_t st[3] = {v.sr, v.sh, v.sb};
  const int ext[3] = {rows, heads, b};
  for (int i = 0; i < 3; ++i)
    if (ext[i] > 1 && (st[i] <= 0 || st[i] % per || st[i] >= ((int64_t)1 << 37))) return false;
  return true;
}

}  // namespace prompt
}  // namespace bg
