// C ABI entry points of the serving operators (bgcuda.h): arguments are checked here, against the buffers they name, so
// that no kernel can leave them; the kernels check what only the device knows (lengths, cache rows) and report it through
// the status word.
#include "serving.h"

#include <math.h>
#include <string.h>

#include <algorithm>
#include <map>
#include <mutex>

#include "runtime.h"

namespace bg {
namespace {

// The largest extent the kernels' 32-bit indexes take.
constexpr int64_t kMaxExtent = (int64_t)1 << 30;

struct Call {
  bg_context* ctx;
  const char* op;
  int error(int code, const std::string& msg) const { return fail(ctx, code, std::string(op) + ": " + msg); }
};

// What every call checks first: a refusal of earlier work is reported before anything else runs, and nothing is issued
// into a stream that is being captured (buffers and scratch are taken from the context's allocator per call).
int begin(const Call& c) {
  cudaSetDevice(c.ctx->device);
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  cudaError_t e = cudaStreamIsCapturing(c.ctx->stream, &cap);
  if (e != cudaSuccess) return cuda_fail(c.ctx, e, c.op);
  if (cap != cudaStreamCaptureStatusNone) return c.error(BG_ERR_UNSUPPORTED, "the bridge's stream is being captured into a graph");
  if (const int st = take_early_status(c.ctx)) return fail_device_status(c.ctx, st, kInEarlierWork);
  return BG_OK;
}

int find(const Call& c, bg_handle h, const char* what, HandleRec** out) {
  auto it = c.ctx->handles.find(h);
  if (it == c.ctx->handles.end()) return c.error(BG_ERR_UNKNOWN_HANDLE, std::string(what) + ": unknown handle " + std::to_string(h));
  *out = &it->second;
  return BG_OK;
}

// A buffer of exactly n values of `dtype`; handle 0 gives null where `optional`.
template <typename T>
int vector_of(const Call& c, bg_handle h, int64_t n, int dtype, const char* what, bool optional, T** out) {
  *out = nullptr;
  if (h == 0 && optional) return BG_OK;
  HandleRec* r;
  if (int rc = find(c, h, what, &r)) return rc;
  if (r->dtype != dtype) return c.error(BG_ERR_INVALID, std::string(what) + " must be " + dtype_name(dtype) + ", the buffer holds " + dtype_name(r->dtype));
  if (r->bytes != n * dtype_size(dtype))
    return c.error(BG_ERR_INVALID, std::string(what) + ": buffer holds " + std::to_string(r->bytes) + " bytes, the call implies " + std::to_string(n * dtype_size(dtype)));
  *out = reinterpret_cast<T*>(r->ptr);
  return BG_OK;
}

// Resolves a view of b x rows x heads runs of d values and checks that all of them lie inside the buffer; for a view
// that is written also that no two of them share a value.
int view_of(const Call& c, const bg_head_view* v, int64_t b, int64_t rows, int64_t heads, int64_t d, int dtype, const char* what,
            bool written, HeadPtr* out) {
  if (!v) return c.error(BG_ERR_INVALID, std::string(what) + ": null view");
  HandleRec* r;
  if (int rc = find(c, v->handle, what, &r)) return rc;
  if (r->dtype != dtype) return c.error(BG_ERR_INVALID, std::string(what) + " must be " + dtype_name(dtype) + ", the buffer holds " + dtype_name(r->dtype));
  const int64_t numel = r->bytes / dtype_size(dtype), ext[3] = {b, rows, heads};
  if (v->offset < 0) return c.error(BG_ERR_INVALID, std::string(what) + ": negative offset");
  const bool empty = b == 0 || rows == 0 || heads == 0;
  __int128 last = (__int128)v->offset + d;
  for (int i = 0; i < 3; ++i) {
    if (v->stride[i] < 0) return c.error(BG_ERR_INVALID, std::string(what) + ": negative stride");
    if (ext[i] > 1) last += (__int128)(ext[i] - 1) * v->stride[i];
  }
  if (!empty && last > numel)
    return c.error(BG_ERR_INVALID, std::string(what) + ": the view reaches beyond the buffer's " + std::to_string(numel) + " values");
  if (written && !empty) {
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int x, int y) { return v->stride[x] < v->stride[y]; });
    __int128 span = d;
    for (int i : order) {
      if (ext[i] <= 1) continue;
      if (v->stride[i] < span) return c.error(BG_ERR_INVALID, std::string(what) + ": rows of the view overlap");
      span += (__int128)(ext[i] - 1) * v->stride[i];
    }
  }
  out->ptr = empty ? r->ptr : reinterpret_cast<char*>(r->ptr) + v->offset * dtype_size(dtype);
  // an extent of one never moves: its stride is not looked at again
  out->sb = b > 1 ? v->stride[0] : 0;
  out->sr = rows > 1 ? v->stride[1] : 0;
  out->sh = heads > 1 ? v->stride[2] : 0;
  return BG_OK;
}

// What the context remembers about a buffer's contents ends when the buffer is written in place.
void forget_contents(bg_context* ctx, bg_handle h) {
  auto it = ctx->handles.find(h);
  if (it == ctx->handles.end()) return;
  uniform_flag_drop(ctx, it->second.ptr);
  mask_classes_drop(ctx, it->second.ptr);
  split_planes_drop(ctx, it->second.ptr);
  cast_copy_drop(ctx, it->second.ptr);
}

// The result: the caller's view, or a fresh dense [b, heads, rows, d] buffer that is given up again unless kept.
struct Result {
  bg_context* ctx;
  bg_handle handle = 0;
  void* fresh = nullptr;
  int64_t bytes = 0;
  HeadPtr view{};
  explicit Result(bg_context* c) : ctx(c) {}
  ~Result() { if (fresh) dev_free(ctx, fresh, bytes); }
};

int result_of(const Call& c, const bg_head_view* out, int64_t b, int64_t rows, int64_t heads, int64_t d, int dtype, Result* r) {
  if (out) {
    if (int rc = view_of(c, out, b, rows, heads, d, dtype, "out", true, &r->view)) return rc;
    r->handle = out->handle;
    return BG_OK;
  }
  r->bytes = b * heads * rows * d * dtype_size(dtype);
  if (int rc = dev_alloc(c.ctx, r->bytes, &r->fresh)) { r->fresh = nullptr; return rc; }
  r->view = HeadPtr{r->fresh, b > 1 ? heads * rows * d : 0, rows > 1 ? d : 0, heads > 1 ? rows * d : 0};
  return BG_OK;
}

bg_handle keep(Result* r, int dtype, int64_t b, int64_t rows, int64_t heads, int64_t d) {
  if (r->fresh) {
    const int64_t shape[4] = {b, heads, rows, d};
    r->handle = mint_handle(r->ctx, r->fresh, r->bytes, dtype, shape, 4);
    r->fresh = nullptr;
  }
  return r->handle;
}

// Runs the launches of one operator the way a plan's unit is run: counted, named in the trace, timed when profiling.
template <typename F>
int launch(const Call& c, const std::string& name, int launches, F&& fn) {
  bg_context* ctx = c.ctx;
  cudaEvent_t e0 = nullptr, e1 = nullptr;
  if (ctx->profiling) {
    cudaEventCreate(&e0);
    cudaEventCreate(&e1);
    cudaEventRecord(e0, ctx->stream);
  }
  cudaError_t e = fn();
  if (ctx->profiling) {
    cudaEventRecord(e1, ctx->stream);
    ctx->pending_events.push_back({name, {e0, e1}});
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return cuda_fail(ctx, e, c.op);
  }
  ctx->launches += launches;
  ctx->last_trace += name + "\n";
  return BG_OK;
}

int check_type(const Call& c, int dtype) {
  if (dtype != BG_F32 && dtype != BG_F16 && dtype != BG_BF16) return c.error(BG_ERR_UNSUPPORTED, "float32, float16 or bfloat16 required");
  return BG_OK;
}
int check_extent(const Call& c, int64_t v, int64_t low, const char* what) {
  if (v < low || v > kMaxExtent) return c.error(BG_ERR_INVALID, std::string(what) + " = " + std::to_string(v) + " is out of range");
  return BG_OK;
}
int check_sizes(const Call& c, int64_t b, int64_t h, int64_t s, int64_t d) {
  if (int rc = check_extent(c, b, 0, "batch")) return rc;
  if (int rc = check_extent(c, h, 1, "heads")) return rc;
  if (int rc = check_extent(c, s, 0, "rows")) return rc;
  if (int rc = check_extent(c, d, 1, "head dimension")) return rc;
  // keeps every product of extents (and its bytes) inside 64 bits, and the grids inside 31
  if ((__int128)b * h * s * d > ((__int128)1 << 50) || b * h > kMaxExtent) return c.error(BG_ERR_INVALID, "the operands are too large");
  return BG_OK;
}

// Full turns per position of every rotated pair.
int turns_of(const Call& c, const bg_rotary_spec* sp, int64_t d, int inverse, RotaryProblem* p) {
  if (!sp) return c.error(BG_ERR_INVALID, "null rotary specification");
  if (sp->dim < 2 || sp->dim % 2 || sp->dim > d || sp->dim > 2 * kRotaryMaxPairs)
    return c.error(BG_ERR_INVALID, "the rotated dimension must be even, at most the head dimension and at most 256");
  if (!(sp->base > 0.0) || !std::isfinite(sp->base)) return c.error(BG_ERR_INVALID, "base must be positive");
  if (!std::isfinite(sp->magnitude)) return c.error(BG_ERR_INVALID, "magnitude must be finite");
  if (sp->scaling < BG_ROTARY_PLAIN || sp->scaling > BG_ROTARY_RAMP) return c.error(BG_ERR_INVALID, "unknown frequency scaling");
  if (sp->scaling != BG_ROTARY_PLAIN && (!(sp->factor > 0.0) || !std::isfinite(sp->factor))) return c.error(BG_ERR_INVALID, "factor must be positive");
  if (sp->scaling == BG_ROTARY_RAMP && (!(sp->low < sp->high) || !std::isfinite(sp->low) || !std::isfinite(sp->high) || !(sp->original_length > 0.0) || !std::isfinite(sp->original_length)))
    return c.error(BG_ERR_INVALID, "ramp scaling needs low < high and a positive original length");
  const double two_pi = 6.283185307179586476925286766559, step = -2.0 * log(sp->base) / sp->dim;
  for (int j = 0; j < sp->dim / 2; ++j) {
    double f = exp(step * j) / two_pi;
    if (sp->scaling == BG_ROTARY_LINEAR) f /= sp->factor;
    if (sp->scaling == BG_ROTARY_RAMP) {
      double keep = (sp->original_length * f - sp->low) / (sp->high - sp->low);
      keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
      f *= keep + (1.0 - keep) / sp->factor;
    }
    p->turns[j] = inverse ? -f : f;
  }
  p->rot = sp->dim;
  p->interleaved = sp->interleaved != 0;
  p->magnitude = (float)sp->magnitude;
  return BG_OK;
}

int rotary(const Call& c, const bg_head_view* x, const bg_rotary_spec* spec, int64_t b, int64_t h, int64_t s, int64_t d, int dtype,
           bg_handle positions, int64_t start, int inverse, const bg_head_view* out_view, bg_handle* out) {
  if (int rc = begin(c)) return rc;
  if (int rc = check_type(c, dtype)) return rc;
  if (int rc = check_sizes(c, b, h, s, d)) return rc;
  if ((__int128)h * d > kMaxExtent) return c.error(BG_ERR_INVALID, "a row of heads is too long");
  if (start < -((int64_t)1 << 40) || start > ((int64_t)1 << 40)) return c.error(BG_ERR_INVALID, "start is out of range");
  RotaryProblem p{};
  if (int rc = turns_of(c, spec, d, inverse, &p)) return rc;
  if (int rc = view_of(c, x, b, s, h, d, dtype, "x", false, &p.seg[0].in)) return rc;
  int* pos = nullptr;
  if (int rc = vector_of(c, positions, b * s, BG_I32, "positions", true, &pos)) return rc;
  // in place means the very same view: any other sharing would read values already turned
  if (out_view && out_view->handle == x->handle && (out_view->offset != x->offset || memcmp(out_view->stride, x->stride, sizeof(x->stride)) != 0))
    return c.error(BG_ERR_INVALID, "out shares x's buffer without being the same view");
  Result r(c.ctx);
  if (int rc = result_of(c, out_view, b, s, h, d, dtype, &r)) return rc;
  p.seg[0].out = r.view;
  p.seg[0].heads = (int)h;
  p.seg[0].turn = 1;
  p.n_seg = 1;
  p.b = (int)b; p.s = (int)s; p.d = (int)d;
  p.start = start;
  p.positions = pos;
  p.status = {c.ctx->d_status, c.ctx->h_status};
  c.ctx->last_trace.clear();
  if (b > 0 && s > 0) {
    if (out_view) forget_contents(c.ctx, r.handle);
    if (int rc = launch(c, std::string("rotary[") + dtype_name(dtype) + "]", 1, [&] { return launch_rotary(p, dtype, c.ctx->stream, c.ctx->sm_count); })) return rc;
  }
  *out = keep(&r, dtype, b, s, h, d);
  return BG_OK;
}

int rotary_append(const Call& c, const bg_head_view* q, const bg_head_view* k, const bg_head_view* v, const bg_head_view* kc,
                  const bg_head_view* vc, const bg_rotary_spec* spec, int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t capacity,
                  int64_t d, int dtype, bg_handle starts, int64_t start, bg_handle counts, const bg_head_view* out_view, bg_handle* out) {
  if (int rc = begin(c)) return rc;
  if (int rc = check_type(c, dtype)) return rc;
  if (int rc = check_sizes(c, b, hq, s, d)) return rc;
  if (int rc = check_sizes(c, b, hkv, capacity, d)) return rc;
  if (int rc = check_sizes(c, b, hkv, s, d)) return rc;
  if ((__int128)(hq + 2 * hkv) * d > kMaxExtent) return c.error(BG_ERR_INVALID, "a row of heads is too long");
  RotaryProblem p{};
  if (int rc = turns_of(c, spec, d, 0, &p)) return rc;
  if (int rc = view_of(c, q, b, s, hq, d, dtype, "q", false, &p.seg[0].in)) return rc;
  if (int rc = view_of(c, k, b, s, hkv, d, dtype, "k", false, &p.seg[1].in)) return rc;
  if (int rc = view_of(c, v, b, s, hkv, d, dtype, "v", false, &p.seg[2].in)) return rc;
  if (int rc = view_of(c, kc, b, capacity, hkv, d, dtype, "k_cache", true, &p.seg[1].out)) return rc;
  if (int rc = view_of(c, vc, b, capacity, hkv, d, dtype, "v_cache", true, &p.seg[2].out)) return rc;
  int *st = nullptr, *ct = nullptr;
  if (int rc = vector_of(c, starts, b, BG_I32, "starts", true, &st)) return rc;
  if (int rc = vector_of(c, counts, b, BG_I32, "counts", true, &ct)) return rc;
  if (!st && (start < 0 || start > capacity || (!ct && start > capacity - s))) return c.error(BG_ERR_INVALID, "the new rows do not fit the cache");
  const bg_handle written[3] = {kc->handle, vc->handle, out_view ? out_view->handle : 0};
  const bg_handle read[5] = {q->handle, k->handle, v->handle, starts, counts};
  for (int i = 0; i < 3; ++i) {
    if (!written[i]) continue;
    for (bg_handle r : read)
      if (r == written[i]) return c.error(BG_ERR_INVALID, "a buffer that is written is also an operand");
    for (int j = 0; j < i; ++j)
      if (written[j] == written[i]) return c.error(BG_ERR_INVALID, "k_cache, v_cache and out must be different buffers");
  }
  Result r(c.ctx);
  if (int rc = result_of(c, out_view, b, s, hq, d, dtype, &r)) return rc;
  p.seg[0].out = r.view;
  p.seg[0].heads = (int)hq;
  p.seg[0].turn = p.seg[1].turn = 1;
  p.seg[1].heads = p.seg[2].heads = (int)hkv;
  p.seg[1].cached = p.seg[2].cached = 1;
  p.n_seg = 3;
  p.b = (int)b; p.s = (int)s; p.d = (int)d;
  p.capacity = capacity;
  p.start = start;
  p.starts = st;
  p.counts = ct;
  p.status = {c.ctx->d_status, c.ctx->h_status};
  c.ctx->last_trace.clear();
  if (b > 0 && s > 0) {
    for (bg_handle h : written) forget_contents(c.ctx, h);
    if (int rc = launch(c, std::string("rotary_append[") + dtype_name(dtype) + "]", 1, [&] { return launch_rotary(p, dtype, c.ctx->stream, c.ctx->sm_count); })) return rc;
    c.ctx->status_pending = true;
  }
  *out = keep(&r, dtype, b, s, hq, d);
  return BG_OK;
}

int decoder_attention(const Call& c, const bg_head_view* q, const bg_head_view* k, const bg_head_view* v, int64_t b, int64_t hq,
                      int64_t hkv, int64_t sq, int64_t sk, int64_t d, int dtype, const bg_attention_rules* rules,
                      const bg_head_view* out_view, bg_handle* out) {
  if (int rc = begin(c)) return rc;
  if (!rules) return c.error(BG_ERR_INVALID, "null rules");
  if (int rc = check_type(c, dtype)) return rc;
  if (int rc = check_sizes(c, b, hq, sq, d)) return rc;
  if (int rc = check_sizes(c, b, hkv, sk, d)) return rc;
  if (hq % hkv) return c.error(BG_ERR_INVALID, "query heads must be a multiple of the key heads");
  if (hq * sq > kMaxExtent) return c.error(BG_ERR_INVALID, "too many query rows");
  if (d > 256) return c.error(BG_ERR_UNSUPPORTED, "head dimensions above 256");
  // (within these the kernels' factors, scale log2 e, cap log2 e and scale / cap, are all numbers of 32 bits)
  if (!(fabs(rules->scale) <= 1e18)) return c.error(BG_ERR_INVALID, "scale must be a number of at most 1e18");
  if (rules->softcap != 0.0 && !(rules->softcap >= 1e-6 && rules->softcap <= 1e6)) return c.error(BG_ERR_INVALID, "softcap must be zero (none) or lie between 1e-6 and 1e6");
  if (rules->prefixes && !rules->causal) return c.error(BG_ERR_INVALID, "prefixes need causal attention");
  DecoderAttention p{};
  if (int rc = view_of(c, q, b, sq, hq, d, dtype, "q", false, &p.q)) return rc;
  if (int rc = view_of(c, k, b, sk, hkv, d, dtype, "k", false, &p.k)) return rc;
  if (int rc = view_of(c, v, b, sk, hkv, d, dtype, "v", false, &p.v)) return rc;
  float* slopes = nullptr;
  int *documents = nullptr, *prefixes = nullptr, *lengths = nullptr, *starts = nullptr;
  if (int rc = vector_of(c, rules->slopes, hq, BG_F32, "slopes", true, &slopes)) return rc;
  if (int rc = vector_of(c, rules->documents, b * sk, BG_I32, "documents", true, &documents)) return rc;
  if (int rc = vector_of(c, rules->prefixes, b, BG_I32, "prefixes", true, &prefixes)) return rc;
  if (int rc = vector_of(c, rules->lengths, b, BG_I32, "lengths", true, &lengths)) return rc;
  if (int rc = vector_of(c, rules->starts, b, BG_I32, "starts", true, &starts)) return rc;
  if (out_view)
    for (bg_handle h : {q->handle, k->handle, v->handle, rules->slopes, rules->documents, rules->prefixes, rules->lengths, rules->starts})
      if (h == out_view->handle) return c.error(BG_ERR_INVALID, "out is also an operand");
  Result r(c.ctx);
  if (int rc = result_of(c, out_view, b, sq, hq, d, dtype, &r)) return rc;
  p.out = r.view;
  p.b = (int)b; p.hq = (int)hq; p.hkv = (int)hkv; p.group = (int)(hq / hkv); p.sq = (int)sq; p.sk = (int)sk; p.d = (int)d;
  p.scale = (float)rules->scale;
  p.cap = (float)rules->softcap;
  p.slopes = slopes;
  p.documents = documents;
  p.prefixes = prefixes;
  p.lengths = lengths;
  p.starts = starts;
  p.causal = rules->causal != 0;
  p.status = {c.ctx->d_status, c.ctx->h_status};
  c.ctx->last_trace.clear();
  if (b > 0 && sq > 0) {
    if (out_view) forget_contents(c.ctx, r.handle);
    // scratch: freed behind the launches, in stream order
    struct Scratch {
      bg_context* ctx;
      void* p = nullptr;
      int64_t n = 0;
      ~Scratch() { if (p) dev_free(ctx, p, n); }
      int get(int64_t bytes) {
        n = bytes;
        return dev_alloc(ctx, bytes, &p);
      }
    } ranges{c.ctx}, partials{c.ctx};
    if (documents && sk > 0) {
      if (int rc = ranges.get(b * ((sk + kDocBlock - 1) / kDocBlock) * (int64_t)sizeof(int2))) return rc;
      p.doc_ranges = reinterpret_cast<const int2*>(ranges.p);
      if (int rc = launch(c, "doc_ranges", 1, [&] { return launch_doc_ranges(documents, p.b, p.sk, reinterpret_cast<int2*>(ranges.p), c.ctx->stream); })) return rc;
    }
    if (prompt_attention_usable(p, dtype)) {
      if (const int64_t bytes = prompt_attention_scratch(p, dtype)) {
        if (int rc = partials.get(bytes)) return rc;
        p.sums = reinterpret_cast<float*>(partials.p);
      }
      if (int rc = launch(c, std::string("prompt_attention[") + dtype_name(dtype) + "]", 1, [&] { return launch_prompt_attention(p, dtype, c.ctx->stream); })) return rc;
      c.ctx->status_pending = true;
      *out = keep(&r, dtype, b, sq, hq, d);
      return BG_OK;
    }
    const CacheAttnPlan plan = cache_attention_plan(p, dtype, c.ctx->sm_count);
    if (plan.partial_bytes)
      if (int rc = partials.get(plan.partial_bytes)) return rc;
    const std::string name = std::string("cache_attention[") + dtype_name(dtype) + "] x" + std::to_string(plan.splits);
    if (int rc = launch(c, name, plan.splits > 1 ? 2 : 1, [&] { return launch_cache_attention(p, dtype, plan, reinterpret_cast<float*>(partials.p), c.ctx->stream); })) return rc;
    c.ctx->status_pending = true;
  }
  *out = keep(&r, dtype, b, sq, hq, d);
  return BG_OK;
}

int sample_tokens(const Call& c, bg_handle logits, bg_handle uniforms, int64_t n, int64_t vocab, int dtype, const bg_sampling* sp,
                  bg_handle probabilities, bg_handle out_handle, bg_handle* out) {
  if (int rc = begin(c)) return rc;
  if (!sp) return c.error(BG_ERR_INVALID, "null sampling parameters");
  if (int rc = check_type(c, dtype)) return rc;
  if (int rc = check_extent(c, n, 0, "rows")) return rc;
  if (int rc = check_extent(c, vocab, 1, "vocabulary")) return rc;
  if (vocab > kSampleMaxVocab) return c.error(BG_ERR_UNSUPPORTED, "vocabularies above 1048576");
  if (!(sp->temperature >= 0.0) || !std::isfinite(sp->temperature)) return c.error(BG_ERR_INVALID, "temperature must be zero (greedy) or positive");
  if (sp->top_k < 0) return c.error(BG_ERR_INVALID, "top_k must be zero (all) or positive");
  if (std::isnan(sp->top_p)) return c.error(BG_ERR_INVALID, "top_p is not a number");
  if (!(sp->min_p >= 0.0 && sp->min_p <= 1.0)) return c.error(BG_ERR_INVALID, "min_p must lie in [0, 1]");
  SampleProblem p{};
  char* x = nullptr;
  if (int rc = vector_of(c, logits, n * vocab, dtype, "logits", false, &x)) return rc;
  float *u = nullptr, *ts = nullptr, *ps = nullptr, *ms = nullptr, *prob = nullptr;
  int* ks = nullptr;
  if (int rc = vector_of(c, uniforms, n, BG_F32, "uniforms", false, &u)) return rc;
  if (int rc = vector_of(c, sp->temperatures, n, BG_F32, "temperatures", true, &ts)) return rc;
  if (int rc = vector_of(c, sp->top_ks, n, BG_I32, "top_ks", true, &ks)) return rc;
  if (int rc = vector_of(c, sp->top_ps, n, BG_F32, "top_ps", true, &ps)) return rc;
  if (int rc = vector_of(c, sp->min_ps, n, BG_F32, "min_ps", true, &ms)) return rc;
  if (int rc = vector_of(c, probabilities, n, BG_F32, "probabilities", true, &prob)) return rc;
  int64_t* tokens = nullptr;
  if (int rc = vector_of(c, out_handle, n, BG_I64, "out", true, &tokens)) return rc;
  const bg_handle read[6] = {logits, uniforms, sp->temperatures, sp->top_ks, sp->top_ps, sp->min_ps};
  for (bg_handle w : {probabilities, out_handle})
    for (bg_handle h : read)
      if (w && w == h) return c.error(BG_ERR_INVALID, "a buffer that is written is also an operand");
  struct Fresh {
    bg_context* ctx;
    void* p = nullptr;
    int64_t n = 0;
    ~Fresh() { if (p) dev_free(ctx, p, n); }
  } fresh{c.ctx};
  if (!tokens) {
    fresh.n = n * 8;
    if (int rc = dev_alloc(c.ctx, fresh.n, &fresh.p)) { fresh.p = nullptr; return rc; }
    tokens = reinterpret_cast<int64_t*>(fresh.p);
  }
  p.logits = x;
  p.n = n; p.vocab = vocab;
  p.uniforms = u;
  p.temperatures = ts; p.temperature = (float)sp->temperature;
  p.top_ks = ks; p.top_k = (int)std::min<int64_t>(sp->top_k, INT32_MAX);
  p.top_ps = ps; p.top_p = (float)sp->top_p;
  p.min_ps = ms; p.min_p = (float)sp->min_p;
  p.tokens = tokens;
  p.probabilities = prob;
  c.ctx->last_trace.clear();
  if (n > 0) {
    if (out_handle) forget_contents(c.ctx, out_handle);
    if (prob) forget_contents(c.ctx, probabilities);
    if (int rc = launch(c, std::string("sample[") + dtype_name(dtype) + "]", 1, [&] { return launch_sample(p, dtype, c.ctx->stream, c.ctx->sm_count); })) return rc;
  }
  if (fresh.p) {
    const int64_t shape[1] = {n};
    *out = mint_handle(c.ctx, fresh.p, fresh.n, BG_I64, shape, 1);
    fresh.p = nullptr;
  } else *out = out_handle;
  return BG_OK;
}

// Nothing throws across the boundary: a failed host allocation becomes a status.
template <typename F>
int guarded(bg_context* ctx, const char* op, bg_handle* out, F&& fn) {
  if (!ctx || !out) return BG_ERR_INVALID;
  try {
    return fn(Call{ctx, op});
  } catch (...) {
    return BG_ERR_OOM;
  }
}

}  // namespace

cudaError_t allow_shared(const void* kern, size_t bytes) {
  static std::mutex lock;
  static std::map<std::pair<int, const void*>, size_t> limits;
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  std::lock_guard<std::mutex> hold(lock);
  size_t& limit = limits[{dev, kern}];
  if (limit >= bytes) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) limit = bytes;
  return e;
}

}  // namespace bg

using namespace bg;

extern "C" {

int bg_rotary(bg_context* ctx, const bg_head_view* x, const bg_rotary_spec* spec, int64_t b, int64_t h, int64_t s, int64_t d, int dtype,
              bg_handle positions, int64_t start, int inverse, const bg_head_view* out_view, bg_handle* out) {
  return guarded(ctx, "rotary", out, [&](const Call& c) { return rotary(c, x, spec, b, h, s, d, dtype, positions, start, inverse, out_view, out); });
}

int bg_rotary_append(bg_context* ctx, const bg_head_view* q, const bg_head_view* k, const bg_head_view* v, const bg_head_view* k_cache,
                     const bg_head_view* v_cache, const bg_rotary_spec* spec, int64_t b, int64_t hq, int64_t hkv, int64_t s, int64_t capacity,
                     int64_t d, int dtype, bg_handle starts, int64_t start, bg_handle counts, const bg_head_view* out_view, bg_handle* out) {
  return guarded(ctx, "rotary_append", out, [&](const Call& c) {
    return rotary_append(c, q, k, v, k_cache, v_cache, spec, b, hq, hkv, s, capacity, d, dtype, starts, start, counts, out_view, out);
  });
}

int bg_decoder_attention(bg_context* ctx, const bg_head_view* q, const bg_head_view* k, const bg_head_view* v, int64_t b, int64_t hq,
                         int64_t hkv, int64_t sq, int64_t sk, int64_t d, int dtype, const bg_attention_rules* rules,
                         const bg_head_view* out_view, bg_handle* out) {
  return guarded(ctx, "decoder_attention", out, [&](const Call& c) { return decoder_attention(c, q, k, v, b, hq, hkv, sq, sk, d, dtype, rules, out_view, out); });
}

int bg_sample_tokens(bg_context* ctx, bg_handle logits, bg_handle uniforms, int64_t n, int64_t vocab, int dtype, const bg_sampling* sampling,
                     bg_handle probabilities, bg_handle out_handle, bg_handle* out) {
  return guarded(ctx, "sample_tokens", out, [&](const Call& c) { return sample_tokens(c, logits, uniforms, n, vocab, dtype, sampling, probabilities, out_handle, out); });
}

}  // extern "C"
