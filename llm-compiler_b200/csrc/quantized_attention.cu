// Decode attention over a paged cache in 8 bits.
//
//     out = sum_t softmax_t(scale * ks * (q . ck_t) + mask_t) vs cv_t,   t < length,
// where ck, cv are the codes of token t and ks, vs the scales of its block. One CTA per (sequence, query head): its warps
// take the tokens in turn, each with a running maximum and sum of its own, and merge them at the end.
#include "quantized.cuh"

namespace b200 {
namespace {

constexpr int kWarps = 4;

struct CacheAttentionParams {
  const void* q;
  const uint8_t* pool[2];
  const float* scales[2];
  const int32_t* table;
  const int64_t* lengths;
  const void* mask;
  void* out;
  int32_t* status;
  int64_t q_batch_stride, q_head_stride, mask_batch_stride, num_blocks, max_blocks, mask_len;
  int q_heads, kv_heads, block_size, mask_dtype;
  float scale;
};

__device__ __forceinline__ float mask_value(const CacheAttentionParams& p, int64_t b, int64_t t) {
  const int64_t i = b * p.mask_batch_stride + t;
  if (p.mask_dtype == B200_F32) return static_cast<const float*>(p.mask)[i];
  if (p.mask_dtype == B200_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p.mask)[i]);
  return __half2float(static_cast<const __half*>(p.mask)[i]);
}

template <typename T, typename Code, int D>
__global__ void __launch_bounds__(kWarps * 32) cache_attention_kernel(const CacheAttentionParams p) {
  constexpr int kEach = D / 32;
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][D];
  grid_launch_dependents();
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.x, kv = head / (p.q_heads / p.kv_heads);
  const int64_t b = blockIdx.y;
  int64_t length = max(p.lengths[b], static_cast<int64_t>(0));
  if (length > p.mask_len) {
    length = p.mask_len;
    if (threadIdx.x == 0) atomicOr(p.status, B200_STATUS_LENGTH_OVER_MASK);
  }
  const T* q = static_cast<const T*>(p.q) + b * p.q_batch_stride + head * p.q_head_stride;
  float qv[kEach], acc[kEach], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    qv[e] = Elem<T>::load(q + lane * kEach + e);
    acc[e] = 0.0f;
  }
  for (int64_t t = warp; t < length; t += kWarps) {
    const int64_t block = p.table[b * p.max_blocks + t / p.block_size];
    if (block < 0 || block >= p.num_blocks) {
      if (lane == 0) atomicOr(p.status, B200_STATUS_BAD_POSITION);
      continue;
    }
    const int64_t slab = block * p.kv_heads + kv, row = (slab * p.block_size + t % p.block_size) * D + lane * kEach;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < kEach; ++e) s = fmaf(qv[e], Code::decode(p.pool[0][row + e]), s);
    s = warp_sum(s) * (p.scale * p.scales[0][slab]);
    if (p.mask != nullptr) s += mask_value(p, b, t);
    const float m_new = fmaxf(m, s), m_safe = m_new == -INFINITY ? 0.0f : m_new;
    const float keep = expf(m - m_safe), w = s == s ? expf(s - m_safe) : s, wv = w * p.scales[1][slab];
    l = l * keep + w;
#pragma unroll
    for (int e = 0; e < kEach; ++e) acc[e] = fmaf(acc[e], keep, wv * Code::decode(p.pool[1][row + e]));
    m = m_new;
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) so[warp][lane * kEach + e] = acc[e];
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kWarps * 32) {
    float top = -INFINITY, sum = 0.0f, o = 0.0f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w]);
    for (int w = 0; w < kWarps; ++w) {
      const float weight = sm[w] == -INFINITY ? (sl[w] == sl[w] ? 0.0f : sl[w]) : expf(sm[w] - top);
      sum += weight * sl[w];
      o += weight * so[w][d];
    }
    // (0 / 0 = NaN for a sequence without tokens)
    Elem<T>::store(static_cast<T*>(p.out) + (b * p.q_heads + head) * D + d, o / sum);
  }
}

template <typename T, typename Code>
cudaError_t launch_attention(const CacheAttentionParams& p, int64_t batch, int64_t dim, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.q_heads), static_cast<unsigned>(batch)), block(kWarps * 32);
  if (dim == 64) return launch_chained(cache_attention_kernel<T, Code, 64>, grid, block, 0, stream, p);
  if (dim == 128) return launch_chained(cache_attention_kernel<T, Code, 128>, grid, block, 0, stream, p);
  return launch_chained(cache_attention_kernel<T, Code, 256>, grid, block, 0, stream, p);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int64_t b200_paged_decode_attention_8bit_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) {
  return 0;
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
      (head_dim != 64 && head_dim != 128 && head_dim != 256) || block_size % 32 != 0)
    return B200_ERR_UNSUPPORTED;
  if (!aligned16(key_pool) || !aligned16(value_pool)) return B200_ERR_ALIGNMENT;
  if (batch > 65535) return B200_ERR_TOO_LARGE;
  if (batch == 0) return B200_OK;
  CacheAttentionParams p = {};
  p.q = query;
  p.pool[0] = static_cast<const uint8_t*>(key_pool); p.pool[1] = static_cast<const uint8_t*>(value_pool);
  p.scales[0] = key_scales; p.scales[1] = value_scales;
  p.table = block_table; p.lengths = lengths; p.mask = mask; p.out = output; p.status = status;
  p.q_batch_stride = q_batch_stride; p.q_head_stride = q_head_stride; p.mask_batch_stride = mask_batch_stride;
  p.num_blocks = num_blocks; p.max_blocks = max_blocks_per_sequence; p.mask_len = mask_len;
  p.q_heads = static_cast<int>(q_heads); p.kv_heads = static_cast<int>(kv_heads);
  p.block_size = static_cast<int>(block_size); p.mask_dtype = mask_dtype; p.scale = static_cast<float>(scale);
  (void)workspace; (void)workspace_bytes; (void)max_length_hint;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t error;
  if (dtype == B200_BF16)
    error = cache_dtype == B200_I8 ? launch_attention<__nv_bfloat16, Int8Code>(p, batch, head_dim, s)
                                   : launch_attention<__nv_bfloat16, E4m3Code>(p, batch, head_dim, s);
  else
    error = cache_dtype == B200_I8 ? launch_attention<__half, Int8Code>(p, batch, head_dim, s)
                                   : launch_attention<__half, E4m3Code>(p, batch, head_dim, s);
  return error == cudaSuccess ? launch_status() : B200_ERR_LAUNCH;
}
