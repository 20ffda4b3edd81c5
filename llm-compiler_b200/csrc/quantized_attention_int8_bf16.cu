// Decode attention of bf16 queries over a paged cache of int8 codes (quantized_attention.cuh).
#include "quantized_attention.cuh"

namespace b200 {
namespace cache_attention {
int launch_int8_bf16(const Params& p, const void* keys, const void* values, int64_t batch, int64_t dim, cudaStream_t stream) {
  return launch_code<__nv_bfloat16, Int8Code>(p, keys, values, batch, dim, stream);
}
}  // namespace cache_attention
}  // namespace b200
