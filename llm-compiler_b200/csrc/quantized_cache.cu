// A paged KV cache in 8 bits: the store that quantises new tokens into it, and copies of its blocks (of any paged cache's).
//
// Pools are [num_blocks, kv_heads, block_size, head_dim] codes with one fp32 scale per (block, KV head) for K and one for V.
// A (block, head) is the unit of everything here: it is contiguous (the attention's tile copies read it as one run, and
// need no stride over the heads of a token), and it is what a scale belongs to.
#include <string.h>

#include <algorithm>

#include "quantized.cuh"

namespace b200 {
namespace {

// ---------------------------------------------------------------------------------------------------------- store ----
// One CTA per (block that receives rows, KV head, sequence, K or V). With x the new rows, T the code's largest value and s
// the block's scale so far (0 where the block is entered at its first row):
//     s' = max(s, amax|x| * fp32(1/T)),  rows held: c' = round(c * (s / s')),  new rows: c = round(x * (1 / s')).
// s' only grows while a block fills, so a row is rounded anew only when a later token is larger than all before it.
// Every step is one IEEE operation in fp32, so the codes do not depend on how the work is split.
// What bounds it: reading x once (4 x 4096 tokens, 4 heads of 128: 12.9 us for 50 MB, part of them from L2), and for a single
// token per sequence the chain position, table row, scale, largest magnitude (64 sequences, 4 heads of 128: 5.3 us).
constexpr int kStoreThreads = 256;
constexpr int kStoreVectors = 8;  // 16-byte loads a thread keeps: a 128 x 128 block is read once

struct StoreParams {
  const void* x[2];        // new keys, new values
  int64_t strides[2][4];   // batch, head, token, element
  uint8_t* pool[2];
  float* scales[2];
  const int32_t* table;
  const int64_t* positions;
  int32_t* status;
  int64_t tokens, max_blocks, num_blocks;
  int heads, dim, block_size;
};

template <typename T, typename Code, bool kVector>
__global__ void __launch_bounds__(kStoreThreads, 3)
quantized_store_kernel(const StoreParams p) {
  constexpr int per = kVector ? 8 : 1;  // elements a load takes
  grid_launch_dependents();
  __shared__ uint32_t parts[kStoreThreads / 32];
  const int h = blockIdx.y % p.heads, which = blockIdx.y / p.heads;
  const int64_t b = blockIdx.z;
  grid_dependency_wait();
  const int64_t position = p.positions[b];
  if (position < 0) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0) atomicOr(p.status, B200_STATUS_BAD_POSITION);
    return;
  }
  if (position >= p.max_blocks * p.block_size) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0) atomicOr(p.status, B200_STATUS_KV_OVERFLOW);
    return;
  }
  const int64_t column = position / p.block_size + blockIdx.x;
  const int64_t first = position > column * p.block_size ? position : column * p.block_size;
  const int64_t end = min(position + p.tokens, (column + 1) * p.block_size);
  if (first >= end) return;
  if (column >= p.max_blocks) {
    if (threadIdx.x == 0) atomicOr(p.status, B200_STATUS_KV_OVERFLOW);
    return;
  }
  const int64_t block = p.table[b * p.max_blocks + column];
  const int held = static_cast<int>(first - column * p.block_size), rows = static_cast<int>(end - first);
  const int64_t* st = p.strides[which];
  const T* x = static_cast<const T*>(p.x[which]) + b * st[0] + h * st[1] + (first - position) * st[2];
  const int per_row = p.dim / per, items = rows * per_row;
  // item i is load i % per_row of row i / per_row; a thread stays in its column where a row divides the CTA's threads
  const int my_row = threadIdx.x / per_row, my_column = threadIdx.x - my_row * per_row;
  const int row_step = kStoreThreads % per_row == 0 ? kStoreThreads / per_row : 0;
  auto address = [&](int j) {  // the thread's j-th
    if (row_step > 0) return x + (my_row + j * row_step) * st[2] + my_column * per * st[3];
    const int i = threadIdx.x + j * kStoreThreads, row = i / per_row;
    return x + row * st[2] + (i - row * per_row) * per * st[3];
  };

  // The largest magnitude of the new rows: without their signs, 16-bit floats compare as integers, two in a word. The rows
  // are asked for beside the block.
  constexpr uint32_t kInfinity = IsHalf<T>::value ? 0x7c00u : 0x7f80u;
  uint4 kept[kStoreVectors];
  uint32_t pair = 0;
  auto look_at = [&](const uint4& raw) {
    pair = __vmaxu2(__vmaxu2(pair, raw.x & 0x7fff7fffu), raw.y & 0x7fff7fffu);
    pair = __vmaxu2(__vmaxu2(pair, raw.z & 0x7fff7fffu), raw.w & 0x7fff7fffu);
  };
  auto bits_of = [&](int j) { return static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(address(j))) & 0x7fffu; };
  auto largest_of_all = [&](uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    __syncthreads();  // (what was there has been read)
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kStoreThreads / 32; ++w) v = max(v, parts[w]);
    return v;
  };
  const int mine = items > static_cast<int>(threadIdx.x) ? (items - threadIdx.x + kStoreThreads - 1) / kStoreThreads : 0;
  if constexpr (kVector) {
#pragma unroll
    for (int j = 0; j < kStoreVectors; ++j) {
      kept[j] = make_uint4(0u, 0u, 0u, 0u);
      if (j < mine) kept[j] = *reinterpret_cast<const uint4*>(address(j));
    }
  }
  if (block < 0 || block >= p.num_blocks) {
    if (threadIdx.x == 0) atomicOr(p.status, B200_STATUS_BAD_POSITION);
    return;
  }
  const int64_t slab = block * p.heads + h;
  uint8_t* codes = p.pool[which] + slab * p.block_size * p.dim;
  const float before = held > 0 ? p.scales[which][slab] : 0.0f;
  if constexpr (kVector) {
#pragma unroll
    for (int j = 0; j < kStoreVectors; ++j) look_at(kept[j]);
    for (int j = kStoreVectors; j < mine; ++j) look_at(*reinterpret_cast<const uint4*>(address(j)));
  } else {
    for (int j = 0; j < mine; ++j) pair = max(pair, bits_of(j));
  }
  uint32_t most = largest_of_all(max(pair & 0xffffu, pair >> 16));
  const bool all_bad = most >= kInfinity;
  if (all_bad) {  // once more, of the finite ones
    pair = 0;
    for (int i = threadIdx.x; i < rows * p.dim; i += kStoreThreads) {
      const int row = i / p.dim;
      const uint32_t bits = *reinterpret_cast<const uint16_t*>(x + row * st[2] + (i - row * p.dim) * st[3]) & 0x7fffu;
      if (bits < kInfinity) pair = max(pair, bits);
    }
    most = largest_of_all(pair);
  }
  const uint16_t most_bits = static_cast<uint16_t>(most);
  const float largest = Elem<T>::load(reinterpret_cast<const T*>(&most_bits));
  float scale = most > 0 ? fmaxf(__fmul_rn(largest, 1.0f / Code::kTop), kSmallestScale) : 0.0f;
  scale = fmaxf(scale, before);
  const float inverse = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
  __syncthreads();  // every thread has read the scale
  if (threadIdx.x == 0) {
    p.scales[which][slab] = scale;
    if (all_bad) atomicOr(p.status, B200_STATUS_NOT_FINITE);
  }
  if (held > 0 && scale != before) {  // the rows in front, on the larger scale (dim is a multiple of 16)
    const float ratio = __fdiv_rn(before, scale);
    uint4* words = reinterpret_cast<uint4*>(codes);
    for (int i = threadIdx.x; i < held * p.dim / 16; i += kStoreThreads) {
      uint4 raw = words[i];
      uint32_t* w = reinterpret_cast<uint32_t*>(&raw);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t packed = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          packed |= Code::encode(__fmul_rn(Code::decode((w[j] >> (8 * e)) & 0xffu), ratio)) << (8 * e);
        w[j] = packed;
      }
      words[i] = raw;
    }
  }
  uint8_t* out = codes + held * p.dim;
  auto put = [&](const uint4& raw, int j) {
    Vec16<T> v;
    v.load(reinterpret_cast<const T*>(&raw));
    uint2 packed = make_uint2(0u, 0u);
#pragma unroll
    for (int e = 0; e < 8; ++e) v.v[e] = __fmul_rn(v.v[e], inverse);
    if (!all_bad) {
      packed = make_uint2(Code::encode_four(v.v[0], v.v[1], v.v[2], v.v[3]), Code::encode_four(v.v[4], v.v[5], v.v[6], v.v[7]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        packed.x |= Code::encode(v.v[e]) << (8 * e);
        packed.y |= Code::encode(v.v[e + 4]) << (8 * e);
      }
    }
    *reinterpret_cast<uint2*>(out + (threadIdx.x + j * kStoreThreads) * 8) = packed;
  };
  if constexpr (kVector) {
#pragma unroll
    for (int j = 0; j < kStoreVectors; ++j)
      if (j < mine) put(kept[j], j);
    for (int j = kStoreVectors; j < mine; ++j) put(*reinterpret_cast<const uint4*>(address(j)), j);
  } else {
    for (int j = 0; j < mine; ++j)
      out[threadIdx.x + j * kStoreThreads] = static_cast<uint8_t>(Code::encode(__fmul_rn(Elem<T>::load(address(j)), inverse)));
  }
}

// ----------------------------------------------------------------------------------------------------------- copy ----
// pool[layer, destinations[i]] = pool[layer, sources[i]] of every pool and layer in one launch. Nothing but bytes move:
// each is read once and written once (150 blocks of 28 layers, 1.1 GB read: 329 us, 6.7 TB/s, a copy's rate).
constexpr int kCopyThreads = 256;
constexpr int kCopyChunk = 16384;  // bytes of a block that one CTA moves
constexpr int kMaxPools = B200_MAX_COPY_POOLS;

struct CopyParams {
  uint8_t* base[kMaxPools];
  int64_t layer_stride[kMaxPools];  // bytes
  int64_t block_bytes[kMaxPools];
  int64_t first_unit[kMaxPools + 1];  // CTAs of the pools before
  const int32_t* sources;
  const int32_t* destinations;
  int32_t* status;
  int64_t num_blocks, layers, count;
  int pools;
};

template <typename V>
__device__ __forceinline__ void copy_run(uint8_t* to, const uint8_t* from, int64_t bytes) {
  const int64_t n = bytes / static_cast<int64_t>(sizeof(V));
  const V* src = reinterpret_cast<const V*>(from);
  V* dst = reinterpret_cast<V*>(to);
  for (int64_t i = threadIdx.x; i < n; i += kCopyThreads * 4) {
    V held[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j * kCopyThreads < n) held[j] = src[i + j * kCopyThreads];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j * kCopyThreads < n) dst[i + j * kCopyThreads] = held[j];
  }
}

__global__ void __launch_bounds__(kCopyThreads) copy_blocks_kernel(const CopyParams p) {
  grid_launch_dependents();
  grid_dependency_wait();
  int pool = 0;
  while (pool + 1 < p.pools && static_cast<int64_t>(blockIdx.x) >= p.first_unit[pool + 1]) ++pool;
  const int64_t unit = blockIdx.x - p.first_unit[pool], bytes = p.block_bytes[pool];
  auto place = [&](int64_t pair, int64_t layer, uint8_t** to, const uint8_t** from) {
    const int64_t source = p.sources[pair], destination = p.destinations[pair];
    if (source < 0 || source >= p.num_blocks || destination < 0 || destination >= p.num_blocks) {
      atomicOr(p.status, B200_STATUS_BAD_POSITION);
      return false;
    }
    uint8_t* base = p.base[pool] + layer * p.layer_stride[pool];
    *to = base + destination * bytes;
    *from = base + source * bytes;
    return source != destination;
  };
  uint8_t* to;
  const uint8_t* from;
  if (bytes >= kCopyChunk / 16) {  // a CTA moves a piece of one block
    const int64_t pieces = (bytes + kCopyChunk - 1) / kCopyChunk, piece = unit % pieces, pair = unit / pieces % p.count;
    if (!place(pair, unit / pieces / p.count, &to, &from)) return;
    const int64_t offset = piece * kCopyChunk, size = min(bytes - offset, static_cast<int64_t>(kCopyChunk));
    if ((bytes & 15) == 0 && ((reinterpret_cast<uintptr_t>(p.base[pool]) | p.layer_stride[pool]) & 15) == 0)
      copy_run<uint4>(to + offset, from + offset, size);
    else
      copy_run<uint8_t>(to + offset, from + offset, size);
    return;
  }
  // small blocks (scales): a thread moves whole blocks
  const int64_t i = unit * kCopyThreads + threadIdx.x;
  if (i >= p.count * p.layers || !place(i % p.count, i / p.count, &to, &from)) return;
  if ((bytes & 3) == 0 && ((reinterpret_cast<uintptr_t>(p.base[pool]) | p.layer_stride[pool]) & 3) == 0) {
    for (int64_t e = 0; e < bytes; e += 4) *reinterpret_cast<uint32_t*>(to + e) = *reinterpret_cast<const uint32_t*>(from + e);
  } else {
    for (int64_t e = 0; e < bytes; ++e) to[e] = from[e];
  }
}

template <typename T, typename Code>
cudaError_t launch_store(const StoreParams& p, bool vector, int64_t batch, cudaStream_t stream) {
  // a portion of T tokens touches at most this many blocks, wherever it starts
  const int64_t columns = std::min<int64_t>((p.tokens + p.block_size - 2) / p.block_size + 1, p.max_blocks + 1);
  const dim3 grid(static_cast<unsigned>(columns), static_cast<unsigned>(2 * p.heads), static_cast<unsigned>(batch));
  return vector ? launch_chained(quantized_store_kernel<T, Code, true>, grid, dim3(kStoreThreads), 0, stream, p)
                : launch_chained(quantized_store_kernel<T, Code, false>, grid, dim3(kStoreThreads), 0, stream, p);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_paged_kv_store_8bit(const b200_cache_store_call* call, void* stream) {
  if (!call) return B200_ERR_BAD_ARGUMENT;
  const b200_cache_store_call& c = *call;
  if (!c.key_pool || !c.value_pool || !c.key_scales || !c.value_scales || !c.block_table || !c.key || !c.value ||
      !c.positions || !c.status || c.batch < 0 || c.heads <= 0 || c.tokens < 0 || c.head_dim <= 0 || c.num_blocks <= 0 ||
      c.block_size <= 0 || c.max_blocks_per_sequence <= 0)
    return B200_ERR_BAD_ARGUMENT;
  const int64_t dtype = c.dtype, cache_dtype = c.cache_dtype;
  if ((dtype != B200_BF16 && dtype != B200_F16) || (cache_dtype != B200_I8 && cache_dtype != B200_E4M3) || c.head_dim % 16 != 0)
    return B200_ERR_UNSUPPORTED;
  if (!aligned16(c.key_pool) || !aligned16(c.value_pool)) return B200_ERR_ALIGNMENT;
  if (c.batch > 65535 || c.heads > 32767 || c.head_dim * c.block_size > (int64_t(1) << 30)) return B200_ERR_TOO_LARGE;
  if (c.batch == 0 || c.tokens == 0) return B200_OK;
  StoreParams p = {};
  p.x[0] = c.key; p.x[1] = c.value;
  for (int i = 0; i < 4; ++i) { p.strides[0][i] = c.key_strides[i]; p.strides[1][i] = c.value_strides[i]; }
  p.pool[0] = static_cast<uint8_t*>(c.key_pool); p.pool[1] = static_cast<uint8_t*>(c.value_pool);
  p.scales[0] = c.key_scales; p.scales[1] = c.value_scales;
  p.table = c.block_table; p.positions = c.positions; p.status = c.status;
  p.tokens = c.tokens; p.max_blocks = c.max_blocks_per_sequence; p.num_blocks = c.num_blocks;
  p.heads = static_cast<int>(c.heads); p.dim = static_cast<int>(c.head_dim); p.block_size = static_cast<int>(c.block_size);
  bool vector = aligned16(c.key) && aligned16(c.value);
  for (int i = 0; i < 2; ++i) {
    vector = vector && p.strides[i][3] == 1;
    for (int j = 0; j < 3; ++j) vector = vector && p.strides[i][j] % 8 == 0;
  }
  const int64_t batch = c.batch;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t error;
  if (dtype == B200_BF16)
    error = cache_dtype == B200_I8 ? launch_store<__nv_bfloat16, Int8Code>(p, vector, batch, s)
                                   : launch_store<__nv_bfloat16, E4m3Code>(p, vector, batch, s);
  else
    error = cache_dtype == B200_I8 ? launch_store<__half, Int8Code>(p, vector, batch, s)
                                   : launch_store<__half, E4m3Code>(p, vector, batch, s);
  return error == cudaSuccess ? launch_status() : B200_ERR_LAUNCH;
}

extern "C" int b200_copy_kv_blocks(const b200_block_pool* pools, int64_t pool_count, const int32_t* sources,
                                   const int32_t* destinations, int64_t count, int64_t layers, int64_t num_blocks,
                                   int32_t* status, void* stream) {
  if (!pools || !sources || !destinations || !status || pool_count <= 0 || count < 0 || layers <= 0 || num_blocks <= 0)
    return B200_ERR_BAD_ARGUMENT;
  if (pool_count > kMaxPools) return B200_ERR_TOO_LARGE;
  CopyParams p = {};
  p.sources = sources; p.destinations = destinations; p.status = status;
  p.num_blocks = num_blocks; p.layers = layers; p.count = count;
  p.pools = static_cast<int>(pool_count);
  for (int i = 0; i < p.pools; ++i) {
    if (!pools[i].base || pools[i].block_bytes <= 0 || (layers > 1 && pools[i].layer_stride < num_blocks * pools[i].block_bytes))
      return B200_ERR_BAD_ARGUMENT;
    p.base[i] = static_cast<uint8_t*>(pools[i].base);
    p.layer_stride[i] = pools[i].layer_stride;
    p.block_bytes[i] = pools[i].block_bytes;
    const int64_t units = p.block_bytes[i] >= kCopyChunk / 16 ? ceil_div(p.block_bytes[i], kCopyChunk) * count * layers
                                                              : ceil_div(count * layers, kCopyThreads);
    p.first_unit[i + 1] = p.first_unit[i] + units;
  }
  if (count == 0) return B200_OK;
  if (p.first_unit[p.pools] > 0x7fffffff) return B200_ERR_TOO_LARGE;
  const cudaError_t error = launch_chained(copy_blocks_kernel, dim3(static_cast<unsigned>(p.first_unit[p.pools])),
                                           dim3(kCopyThreads), 0, static_cast<cudaStream_t>(stream), p);
  return error == cudaSuccess ? launch_status() : B200_ERR_LAUNCH;
}
