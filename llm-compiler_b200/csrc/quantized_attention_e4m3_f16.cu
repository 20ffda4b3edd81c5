// Decode attention of fp16 queries over a paged cache of e4m3 codes (quantized_attention.cuh).
#include "quantized_attention.cuh"

namespace b200 {
namespace cache_attention {
int launch_e4m3_f16(const Params& p, const void* keys, const void* values, int64_t batch, int64_t dim, cudaStream_t stream) {
  return launch_code<__half, E4m3Code>(p, keys, values, batch, dim, stream);
}
}  // namespace cache_attention
}  // namespace b200
