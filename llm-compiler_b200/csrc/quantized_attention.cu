// Decode attention over a paged cache in 8 bits: checks and the split of the work (quantized_attention.cuh has the kernel).
#include "quantized_attention.cuh"

namespace b200 {
namespace cache_attention {
namespace {
struct Plan {
  int64_t head_blocks, block_heads, splits, rounds;  // rounds of the CTAs that the GPU holds at once
  bool cluster;
  int64_t parts(int64_t batch, int64_t kv_heads) const {
    return splits > 1 && !cluster ? batch * kv_heads * head_blocks * splits * block_heads : 0;
  }
};
Plan plan_of(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t longest, int64_t split_tokens) {
  Plan plan;
  const int64_t group = q_heads / kv_heads;
  plan.head_blocks = ceil_div(group, dim == 256 ? 8 : 16);
  plan.block_heads = ceil_div(group, plan.head_blocks);
  const int64_t items = batch * kv_heads * plan.head_blocks;
  const int64_t resident = dim == 256 ? 1 : dim == 64 && plan.block_heads <= 8 ? 4 : 3, slots = kNumSMs * resident;
  if (split_tokens > 0) {
    plan.splits = ceil_div(longest, split_tokens);
  } else {
    // One round of the clusters that the GPU holds at once: a CTA streams nothing for some 5 us at its start and end, and a
    // second round waits for that (32 x 4096 tokens, 4 heads of 128: 28 us in 256 CTAs, 39 in 512; 25 x 4096, 2 of 128: 15.5 in
    // 50 clusters of 7, 16.2 of 4, 22 of 8, two of which wait; 18 x 8192, one of 256: 23 in 6, 28 in 4, 35 in 8). Beyond a
    // cluster's eight only 1024 tokens and more a CTA (16 x 4096, 2 heads of 64: 9.5 in 8 splits, 11 in 16; 1 x 32768, 4 heads of
    // 128: 36 in 8, 20 in 32, 22 in 64). Where one round cannot split at all, several of short CTAs even out lengths that
    // differ (64 ragged to 8192, 4 heads of 128: 79 in one split, 63 in two, 59 in four; 64 x 4096 of one length 47, 64 and 62).
    plan.splits = 8;
    while (plan.splits > 1 && items > clusters_at_once(resident, plan.splits)) --plan.splits;
    if (plan.splits == 8)
      while (items * plan.splits * 2 <= slots && plan.splits * 2 * 1024 <= longest) plan.splits *= 2;
    if (plan.splits == 1 && items <= slots) plan.splits = 2;
  }
  // (a CTA has a tile for each of its warps)
  plan.splits = std::max<int64_t>(1, std::min(plan.splits, ceil_div(longest, 32 * kWarps)));
  if (items > kMaxCounters) plan.splits = std::min<int64_t>(plan.splits, 8);
  plan.cluster = plan.splits > 1 && plan.splits <= 8;
  plan.rounds = plan.cluster ? ceil_div(items, clusters_at_once(resident, plan.splits)) : ceil_div(items * plan.splits, slots);
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

extern "C" int b200_paged_decode_attention_8bit(const b200_cache_attention_call* call, void* stream) {
  if (!call) return B200_ERR_BAD_ARGUMENT;
  const b200_cache_attention_call& c = *call;
  if (!c.query || !c.key_pool || !c.value_pool || !c.key_scales || !c.value_scales || !c.block_table || !c.lengths ||
      !c.output || !c.status || c.batch < 0 || c.q_heads <= 0 || c.kv_heads <= 0 || c.q_heads % c.kv_heads != 0 ||
      c.num_blocks <= 0 || c.block_size <= 0 || c.max_blocks_per_sequence <= 0 || c.mask_len <= 0 ||
      c.mask_len > c.max_blocks_per_sequence * c.block_size || c.split_tokens < 0 ||
      (c.mask && (c.mask_dtype < 0 || c.mask_dtype > B200_F16)))
    return B200_ERR_BAD_ARGUMENT;
  if ((c.dtype != B200_BF16 && c.dtype != B200_F16) || (c.cache_dtype != B200_I8 && c.cache_dtype != B200_E4M3) ||
      (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) || c.block_size % 32 != 0)
    return B200_ERR_UNSUPPORTED;
  if (!aligned16(c.key_pool) || !aligned16(c.value_pool) || (reinterpret_cast<uintptr_t>(c.output) & 7u) != 0)
    return B200_ERR_ALIGNMENT;
  if (c.batch > 65535 || c.q_heads > 65535 || c.num_blocks > INT32_MAX || c.num_blocks * c.kv_heads > INT32_MAX ||
      c.block_size > (1 << 20) || c.max_blocks_per_sequence * c.block_size > INT32_MAX / 2)
    return B200_ERR_TOO_LARGE;
  if (c.batch == 0) return B200_OK;
  const int64_t longest = c.max_length_hint > 0 && c.max_length_hint < c.mask_len ? c.max_length_hint : c.mask_len;
  const Plan plan = plan_of(c.batch, c.q_heads, c.kv_heads, c.head_dim, longest, c.split_tokens);
  if (plan.splits > 65535) return B200_ERR_TOO_LARGE;
  Params p = {};
  const int64_t parts = plan.parts(c.batch, c.kv_heads);
  if (parts > 0) {
    if (!c.workspace || c.workspace_bytes < kCounterBytes + parts * (c.head_dim + 2) * 4) return B200_ERR_WORKSPACE;
    p.counters = static_cast<int*>(c.workspace);
    p.ws_o = reinterpret_cast<float*>(static_cast<char*>(c.workspace) + kCounterBytes);
    p.ws_ml = p.ws_o + parts * c.head_dim;
  }
  p.q = c.query; p.key_scales = c.key_scales; p.value_scales = c.value_scales; p.table = c.block_table;
  p.lengths = c.lengths; p.mask = c.mask; p.out = c.output; p.status = c.status;
  p.q_batch_stride = c.q_batch_stride; p.q_head_stride = c.q_head_stride; p.mask_batch_stride = c.mask_batch_stride;
  p.num_blocks = c.num_blocks; p.max_blocks = c.max_blocks_per_sequence; p.mask_len = c.mask_len;
  p.num_splits = static_cast<int>(plan.splits); p.cluster = plan.cluster;
  p.batch = static_cast<int>(c.batch);
  p.sorted = plan.rounds > 1 && c.batch > 1 && c.batch <= kTableCache;
  p.q_heads = static_cast<int>(c.q_heads); p.kv_heads = static_cast<int>(c.kv_heads);
  p.group = static_cast<int>(c.q_heads / c.kv_heads);
  p.head_blocks = static_cast<int>(plan.head_blocks); p.block_heads = static_cast<int>(plan.block_heads);
  p.block_size = static_cast<int>(c.block_size); p.mask_dtype = static_cast<int>(c.mask_dtype);
  const uint64_t block_tiles = static_cast<uint64_t>(c.block_size / 32);
  p.block_magic = ((uint64_t(1) << 63) + block_tiles - 1) / block_tiles;
  p.q_vector = aligned16(c.query) && c.q_batch_stride % 8 == 0 && c.q_head_stride % 8 == 0;
  p.scale = static_cast<float>(c.scale); p.wait_limit = wait_limit(); p.drop_loads = drop_loads();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto launch = c.cache_dtype == B200_I8 ? (c.dtype == B200_BF16 ? launch_int8_bf16 : launch_int8_f16)
                                               : (c.dtype == B200_BF16 ? launch_e4m3_bf16 : launch_e4m3_f16);
  return launch(p, c.key_pool, c.value_pool, c.batch, c.head_dim, s);
}
