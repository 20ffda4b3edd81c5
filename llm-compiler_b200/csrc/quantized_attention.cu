// Decode attention over a paged cache in 8 bits: checks, the split of the work, and the instances for integer codes
// (quantized_attention.cuh).
#include "quantized_attention.cuh"

namespace b200 {
namespace cache_attention {
int launch_int8(const Params& p, const void* keys, const void* values, int64_t batch, int64_t dim, cudaStream_t stream) {
  return launch_code<Int8Code>(p, keys, values, batch, dim, stream);
}

namespace {
struct Plan {
  int64_t head_blocks, block_heads, split_tokens, splits;
  int64_t parts(int64_t batch, int64_t kv_heads) const {
    return splits > 1 ? batch * kv_heads * head_blocks * splits * block_heads : 0;
  }
};
Plan plan_of(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t max_length, int64_t split_tokens) {
  Plan plan;
  const int64_t group = q_heads / kv_heads;
  plan.head_blocks = ceil_div(group, dim == 256 ? 8 : 16);
  plan.block_heads = ceil_div(group, plan.head_blocks);
  const int64_t items = batch * kv_heads * plan.head_blocks;
  if (split_tokens <= 0) {
    const int64_t resident = static_cast<int64_t>(kNumSMs) * (dim == 64 ? 3 : dim == 128 ? 2 : 1);
    const int64_t most = std::max<int64_t>(1, resident / items);
    split_tokens = std::max<int64_t>(ceil_div(max_length, most), 128);
  }
  plan.split_tokens = ceil_div(split_tokens, kTile) * kTile;
  plan.splits = ceil_div(max_length, plan.split_tokens);
  if (items > kMaxCounters) {  // (that many sequences fill the GPU by themselves)
    plan.splits = 1;
    plan.split_tokens = std::max(plan.split_tokens, ceil_div(max_length, kTile) * kTile);
  }
  return plan;
}
}  // namespace
}  // namespace cache_attention
}  // namespace b200

using namespace b200;
using namespace b200::cache_attention;

extern "C" int64_t b200_paged_decode_attention_8bit_workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                                    int64_t head_dim, int64_t max_length,
                                                                    int64_t split_tokens) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || head_dim <= 0 || max_length <= 0) return 0;
  const int64_t parts = plan_of(batch, q_heads, kv_heads, head_dim, max_length, split_tokens).parts(batch, kv_heads);
  return parts > 0 ? kCounterBytes + parts * (head_dim + 2) * 4 : 0;
}

extern "C" int b200_paged_decode_attention_8bit(
    const void* query, const void* key_pool, const void* value_pool, const float* key_scales, const float* value_scales,
    const int32_t* block_table, const int64_t* lengths, const void* mask, void* output, int64_t batch, int64_t q_heads,
    int64_t kv_heads, int64_t head_dim, int64_t num_blocks, int64_t block_size, int64_t max_blocks_per_sequence,
    int64_t mask_len, int64_t q_batch_stride, int64_t q_head_stride, int64_t mask_batch_stride, int mask_dtype, double scale,
    int dtype, int cache_dtype, int64_t split_tokens, int64_t max_length_hint, void* workspace, int64_t workspace_bytes,
    int32_t* status, void* stream) {
  if (!query || !key_pool || !value_pool || !key_scales || !value_scales || !block_table || !lengths || !output || !status ||
      batch < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || num_blocks <= 0 || block_size <= 0 ||
      max_blocks_per_sequence <= 0 || mask_len <= 0 || mask_len > max_blocks_per_sequence * block_size || split_tokens < 0)
    return B200_ERR_BAD_ARGUMENT;
  if (mask && !known_dtype(mask_dtype)) return B200_ERR_BAD_ARGUMENT;
  if ((dtype != B200_BF16 && dtype != B200_F16) || (cache_dtype != B200_I8 && cache_dtype != B200_E4M3) ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256) || block_size % kTile != 0)
    return B200_ERR_UNSUPPORTED;
  if (!aligned16(key_pool) || !aligned16(value_pool) || (reinterpret_cast<uintptr_t>(output) & 7u) != 0)
    return B200_ERR_ALIGNMENT;
  if (batch > 65535 || q_heads > 65535 || num_blocks * kv_heads > INT32_MAX || num_blocks > INT32_MAX ||
      block_size > (1 << 20) || mask_len > (int64_t(1) << 40))
    return B200_ERR_TOO_LARGE;
  if (batch == 0) return B200_OK;
  const int64_t longest = max_length_hint > 0 && max_length_hint < mask_len ? max_length_hint : mask_len;
  const Plan plan = plan_of(batch, q_heads, kv_heads, head_dim, longest, split_tokens);
  if (plan.splits > 65535) return B200_ERR_TOO_LARGE;
  Params p = {};
  const int64_t parts = plan.parts(batch, kv_heads);
  if (parts > 0) {
    if (!workspace || workspace_bytes < kCounterBytes + parts * (head_dim + 2) * 4) return B200_ERR_WORKSPACE;
    p.counters = static_cast<int*>(workspace);
    p.ws_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
    p.ws_ml = p.ws_o + parts * head_dim;
  }
  p.q = query; p.key_scales = key_scales; p.value_scales = value_scales; p.table = block_table; p.lengths = lengths;
  p.mask = mask; p.out = output; p.status = status;
  p.q_batch_stride = q_batch_stride; p.q_head_stride = q_head_stride; p.mask_batch_stride = mask_batch_stride;
  p.num_blocks = num_blocks; p.max_blocks = max_blocks_per_sequence; p.mask_len = mask_len;
  p.split_tokens = plan.split_tokens; p.num_splits = static_cast<int>(plan.splits);
  p.q_heads = static_cast<int>(q_heads); p.kv_heads = static_cast<int>(kv_heads);
  p.group = static_cast<int>(q_heads / kv_heads);
  p.head_blocks = static_cast<int>(plan.head_blocks); p.block_heads = static_cast<int>(plan.block_heads);
  p.block_size = static_cast<int>(block_size); p.mask_dtype = mask_dtype; p.half = dtype == B200_F16;
  p.q_vector = aligned16(query) && q_batch_stride % 8 == 0 && q_head_stride % 8 == 0;
  p.scale = static_cast<float>(scale); p.wait_limit = wait_limit(); p.drop_loads = drop_loads();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return cache_dtype == B200_I8 ? launch_int8(p, key_pool, value_pool, batch, head_dim, s)
                                : launch_e4m3(p, key_pool, value_pool, batch, head_dim, s);
}
