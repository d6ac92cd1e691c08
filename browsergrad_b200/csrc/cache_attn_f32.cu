// cache_attn.cuh instantiated for one operand type.
#include "cache_attn.cuh"

namespace bg {
namespace cache_attn {
cudaError_t launch_f32(const DecoderAttention& p, const CacheAttnPlan& plan, float* partials, cudaStream_t s) {
  return launch_typed<float>(p, plan, partials, s);
}
}  // namespace cache_attn
}  // namespace bg
