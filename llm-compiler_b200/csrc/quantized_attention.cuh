// Decode attention over a paged cache in 8 bits: the kernel and its launch, instantiated per code and query type in a .cu of
// its own.
//
//     out = sum_t softmax_t(scale * ks * (q . ck_t) + mask_t) vs cv_t,   t < length,
// with ck, cv the codes of token t and ks, vs the scales of its block. The G query heads of a KV head share one read of its
// codes. What bounds it is that read: 2 * length * D bytes per KV head; per byte there are 2 G operations, which the tensor
// cores take, and one conversion, which the CUDA cores do.
//
// Products. Codes become fp16, which holds every int8 and e4m3 value exactly, and are multiplied on mma m16n8k16 with the
// TOKENS (or the elements of D) along M and the heads along N = 8: S^T = K Q^T, O^T = V^T P^T. Up to eight heads of a group
// then cost one n-tile, where heads along M would pad them to sixteen. No element is shuffled:
//  - the sum over D may run in any order, so a lane reads 16 consecutive bytes of a token as its part of four k-steps, and q
//    is laid out once to match;
//  - V comes through ldmatrix.trans in units of two bytes: a lane gets d and d + 1 of two tokens, and splits them into the
//    two tokens' even and odd element, which are rows of two halves of an A operand;
//  - P^T is transposed 8 x 8 by movmatrix.
// q is brought to [1, 2) per head by a power of two, which goes back into the scores: exact but for elements below 2^-14 of the
// head's largest, which are off by at most 2^-25 of it (fp16 alone would overflow).
//
// Scales. ks multiplies the scores. vs is folded into the probabilities relative to a running reference `vref`, which the
// accumulators are carried in: a power of two that follows vs (accumulators rescaled, exactly) only when vs is more than twice it
// or less than a quarter of it. It follows any distance up, where what is in the accumulators may underflow, and down as far as
// they stay within fp32's range, where it is the tile that may; a tile that no head gives any weight does not move it.
//
// Probabilities. The running maximum moves only when a score passes it by more than 3 (in units of log 2): the softmax is the
// same, and most tiles need no reduction across lanes. So P, at most 2^3 * 2, is carried 2^11 higher, which fills fp16: P is
// rounded by 2^-11 of it, an eighth of the rounding of a bf16 result, down to 2^-23 of the largest probability, and by 2^-34 of
// the largest below (carried at 1 and with wider limits, the tail behind a token e^14 above it came out 1 % off, and behind one
// e^18 above it as nothing); its sum stays fp32. An fp16 result's own rounding is no larger than P's, so there P is two fp16
// numbers, what the first leaves in the second (2^-22, and 2^-34 of the largest as before): one more product per V fragment.
//
// Work. The tiles (32 tokens) of one (sequence, KV head, up to 8 NT heads) are dealt to `splits` CTAs of four warps, a tile
// to a warp in turn. Each warp has a ring of its own that TMA fills: a tile never spans two blocks (block sizes are multiples
// of 32), is contiguous in the pool, and is one box for K and one for V. Warps merge through shared memory. Up to eight
// splits are a cluster, whose CTAs merge through distributed shared memory; more leave partials in the workspace, which the
// CTA that arrives last adds in split order. Either way results do not depend on timing.
//
// Measured: 64 x 4096 tokens, 2 heads of 64 (67 MB): 16.7 us, 4.0 TB/s; 64 ragged to 8192, 4 heads of 128 (270 MB): 52 us,
// 5.2 TB/s; 3 x 30001, 8 heads of 128 with a mask (185 MB): 37 us, 5.0 TB/s; 1 x 1000: 4.8 us. A CTA streams nothing for some
// 5 us at its start and end (length, table row, first copies; merge, exchange in the cluster, stores), which is what is left
// beside the rate: in between the SMs' rings keep 96 KB and more in flight.
#pragma once

#include <float.h>

#include <algorithm>
#include <type_traits>

#include "quantized.cuh"
#include "tensor_map.cuh"

namespace b200 {
namespace cache_attention {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 3.0f;      // how far a score may pass the running maximum before it moves, in units of log 2
constexpr float kUnseen = 36.0f;    // a probability that far below the running maximum is 0 in fp16
constexpr float kLift = 2048.0f;    // what the probabilities are carried times: 2^kSlack * 2 (block scales) * kLift = 2^15
constexpr int64_t kCounterBytes = 65536;
constexpr int64_t kMaxCounters = kCounterBytes / 4;
constexpr int kTableCache = 512;  // entries of a sequence's row of the block table that wait in shared memory

struct Params {
  const void* q;
  const float* key_scales;
  const float* value_scales;
  const int32_t* table;
  const int64_t* lengths;
  const void* mask;
  void* out;
  float* ws_o;     // more splits than a cluster holds: [items, splits, heads of a block, D]
  float* ws_ml;    // [items, splits, heads of a block, 2]
  int* counters;   // [items], zero between calls
  int32_t* status;
  int64_t q_batch_stride, q_head_stride, mask_batch_stride, num_blocks, max_blocks, mask_len;
  int q_heads, kv_heads, group, head_blocks, block_heads, block_size, mask_dtype, num_splits, batch;
  int cluster;     // the splits are a cluster
  int sorted;      // CTAs take the sequences from the longest to the shortest
  int q_vector;    // rows of q may be read 16 bytes at a time
  uint64_t block_magic;  // 2^63 / tiles of a block, rounded up: tile * it >> 63 is the tile's block (it is off by less than the
                         // divisor, at most 2^15, and a tile is below 2^25: their product stays below 2^63)
  float scale;
  uint32_t wait_limit;
  int drop_loads;
};

// Four codes of a word as fp16: neighbours (bytes 0, 1 and 2, 3) for K, and every other (0, 2 and 1, 3) for V.
template <typename Code>
struct Convert;
template <>
struct Convert<Int8Code> {
  // 0x64xx is 1024 + xx: a code with its sign bit turned, 0 .. 255, lands there by a byte permutation; 1152 comes off.
  __device__ static uint32_t back(uint32_t pair) {
    const uint32_t bias = 0x64806480u;
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&pair), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  __device__ static void neighbours(uint32_t w, uint32_t& lo, uint32_t& hi) {
    w ^= 0x80808080u;
    lo = back(__byte_perm(w, 0x64646464u, 0x4140));
    hi = back(__byte_perm(w, 0x64646464u, 0x4342));
  }
  __device__ static void every_other(uint32_t w, uint32_t& even, uint32_t& odd) {
    w ^= 0x80808080u;
    even = back(__byte_perm(w, 0x64646464u, 0x4240));
    odd = back(__byte_perm(w, 0x64646464u, 0x4341));
  }
};
template <>
struct Convert<E4m3Code> {
  __device__ static uint32_t two(uint16_t codes) {
    uint32_t pair;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(pair) : "h"(codes));
    return pair;
  }
  __device__ static void neighbours(uint32_t w, uint32_t& lo, uint32_t& hi) {
    lo = two(static_cast<uint16_t>(w));
    hi = two(static_cast<uint16_t>(w >> 16));
  }
  __device__ static void every_other(uint32_t w, uint32_t& even, uint32_t& odd) {
    neighbours(__byte_perm(w, 0u, 0x3120), even, odd);
  }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / x of a sum of probabilities, good to 2^-23; 0 where there are none (a sum is 0, or from 1 to 2^44)
__device__ __forceinline__ float inverse_of(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return x != 0.0f ? y : 0.0f;
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float load_mask(const Params& p, int64_t i) {
  if (p.mask_dtype == B200_F32) return static_cast<const float*>(p.mask)[i];
  if (p.mask_dtype == B200_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p.mask)[i]);
  return __half2float(static_cast<const __half*>(p.mask)[i]);
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void store_cluster_f32x4(uint32_t local_smem_addr, int rank, const float4& v) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_smem_addr), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void store_cluster_f32x2(uint32_t local_smem_addr, int rank, const float2& v) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_smem_addr), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote), "f"(v.x), "f"(v.y) : "memory");
}

template <int D>
struct Shape {
  static constexpr int kTile = 32;                             // tokens of a tile (D 128: 16 and a fourth CTA, 37 -> 41 us at 3 x 30001)
  static constexpr int kRowBytes = D < 128 ? D : 128;         // a box is one swizzle span wide
  static constexpr int kBoxes = D / kRowBytes;
  static constexpr int kBoxBytes = kTile * kRowBytes;
  static constexpr int kTileBytes = kTile * D;                 // K or V
  static constexpr int kStages = D == 128 ? 2 : 3;  // (shorter rings, more CTAs: 61 us where 96 KB of rings take 72, ragged to 8192)
  static constexpr int kResident(int n_tiles) { return D == 256 ? 1 : D == 64 && n_tiles == 1 ? 4 : 3; }  // CTAs of an SM
  static constexpr int kRingBytes = kWarps * kStages * 2 * kTileBytes;
  // What the CTAs of a cluster give this one: beside the ring where it fits without costing a CTA, else in it
  __host__ __device__ static constexpr int kGivenBytes(int n_tiles) { return n_tiles * 8 * D * 4 + 128; }
  __host__ __device__ static constexpr bool kBeside(int n_tiles) { return !(D == 128 && n_tiles == 2); }
  __host__ __device__ static constexpr int kPartBytes(int n_tiles) { return kWarps * n_tiles * 8 * D * 4; }
  __host__ __device__ static constexpr int kGivenAt(int n_tiles) { return kBeside(n_tiles) ? kRingBytes : kPartBytes(n_tiles); }
  static constexpr int kBytes(int n_tiles) {
    return kBeside(n_tiles) ? kRingBytes + kGivenBytes(n_tiles) : std::max(kRingBytes, kPartBytes(n_tiles) + kGivenBytes(n_tiles));
  }
  // byte offset of 16-byte chunk `chunk` of row `row` in a tile
  __device__ static uint32_t at(int row, int chunk) {
    if (D == 64) return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
    return (chunk >> 3) * kBoxBytes + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
  }
  // Which of eight tokens is row r of a fragment: rows that one 128-byte phase of a read takes together differ in bit 2,
  // so that their swizzled chunks lie in different halves of the banks (64-byte rows: two rows make 128 bytes anyway).
  __device__ static int token(int r) { return D == 64 ? r : (r >> 1) | ((r & 1) << 2); }
};

template <typename T, typename Code, int D, int NT, bool kMask>
__global__ void __launch_bounds__(kThreads, (Shape<D>::kResident(NT)))
cache_attention_kernel(const Params p, const __grid_constant__ CUtensorMap key_map,
                       const __grid_constant__ CUtensorMap value_map) {
  using S = Shape<D>;
  constexpr int kTile = S::kTile, kParts = kTile / 16, kEach = kTile / 8;  // m-tiles; a lane's tokens
  constexpr int kStages = S::kStages, kSteps = D / 16, kHeads = 8 * NT;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ __align__(8) uint64_t full[kWarps * kStages];
  __shared__ float merge_m[kWarps][kHeads], merge_l[kWarps][kHeads];
  __shared__ __align__(8) float2 joined[8][kHeads];  // of the cluster's CTAs: their maximum and sum
  __shared__ int last_flag;
  __shared__ __align__(16) int row_cache[kTableCache];

  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  const int split = blockIdx.x, item_head = blockIdx.y, kv = item_head / p.head_blocks, hb = item_head % p.head_blocks;
  int64_t b = blockIdx.z;
  const int head0 = kv * p.group + hb * p.block_heads;
  const int heads = min(p.block_heads, p.group - hb * p.block_heads);
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbarrier_init(smem_u32(&full[warp * kStages + s]), 1);
    fence_mbarrier_init();
  }
  const int tiles_per_block = p.block_size / kTile, my_first = split * kWarps + warp;
  grid_dependency_wait_cta();
  if (p.sorted) {
    // Several rounds of CTAs: the longest sequences first, so that the last round is short (64 ragged to 8192, 4 heads of
    // 128: 62 us in the order of the batch). The CTAs at z take the sequence that z others are longer than.
    for (int i = threadIdx.x; i < kTableCache; i += kThreads) {
      const int64_t n = i < p.batch ? min(p.lengths[i], p.mask_len) : -1;
      row_cache[i] = i < p.batch ? static_cast<int>(max(n, static_cast<int64_t>(0))) : -1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.batch; i += kThreads) {
      const int mine = row_cache[i];
      int longer = 0;
      for (int other = 0; other < p.batch; other += 4) {
        const int4 four = *reinterpret_cast<const int4*>(row_cache + other);  // (-1 beyond the batch)
        longer += (four.x > mine || (four.x == mine && other < i)) + (four.y > mine || (four.y == mine && other + 1 < i)) +
                  (four.z > mine || (four.z == mine && other + 2 < i)) + (four.w > mine || (four.w == mine && other + 3 < i));
      }
      if (longer == static_cast<int>(blockIdx.z)) last_flag = i;
    }
    __syncthreads();
    b = last_flag;
  }
  const int32_t* table = p.table + b * p.max_blocks;

  // The row of the block table is asked for beside the length.
  const int cached = static_cast<int>(min(p.max_blocks, static_cast<int64_t>(kTableCache)));
  int entries[kTableCache / kThreads];
#pragma unroll
  for (int i = 0; i < kTableCache / kThreads; ++i) {
    const int column = threadIdx.x + i * kThreads;
    entries[i] = column < cached ? table[column] : -1;
  }
  int64_t length64 = max(p.lengths[b], static_cast<int64_t>(0));
  if (length64 > p.mask_len) {
    length64 = p.mask_len;
    if (threadIdx.x == 0 && split == 0 && item_head == 0) atomicOr(p.status, B200_STATUS_LENGTH_OVER_MASK);
  }
#pragma unroll
  for (int i = 0; i < kTableCache / kThreads; ++i) row_cache[threadIdx.x + i * kThreads] = entries[i];
  __syncthreads();
  const int length = static_cast<int>(length64), tiles = (length + kTile - 1) / kTile;
  const int active = max(min((tiles + kWarps - 1) / kWarps, p.num_splits), 1);  // splits with a tile for each warp
  if (split >= active) return;  // (a cluster's barriers do not wait for CTAs that have left)
  const bool alone = active == 1;
  if (S::kBeside(NT) && p.cluster && !alone) cluster_arrive();  // this CTA's memory is there
  const int stride = kWarps * active;
  const int mine = tiles > my_first ? (tiles - my_first + stride - 1) / stride : 0;

  // Places of this warp's tiles, 32 tiles ahead in the lanes: lane i of a window that starts at `it` holds tile it + i.
  struct Window { int slab, row; float ks, vs; };  // (block, head), row in the block
  bool bad = false;
  auto look_up = [&](int it) {
    Window w = {-1, 0, 0.0f, 0.0f};
    if (it >= mine) return w;
    const int tile = my_first + it * stride, column = static_cast<int>(__umul64hi(2 * static_cast<uint64_t>(tile), p.block_magic));
    const int block = column < kTableCache ? row_cache[column] : table[column];
    if (block < 0 || block >= p.num_blocks) {
      bad = true;
      return w;
    }
    w.slab = block * p.kv_heads + kv;
    w.row = (tile - column * tiles_per_block) * kTile;
    w.ks = p.key_scales[w.slab];
    w.vs = p.value_scales[w.slab];
    return w;
  };
  const uint32_t ring = smem_u32(smem) + warp * kStages * 2 * S::kTileBytes;
  const uint32_t bars = smem_u32(&full[warp * kStages]);
  Window now = look_up(lane), next = {-1, 0, 0.0f, 0.0f};
  if (mine > 32) next = look_up(lane + 32);
  int base = 0, issued = 0;  // of `now`; tiles asked for
  int issue_stage = 0;
  auto issue = [&]() {  // the lane that holds the tile's place asks for it; a tile without a block has no copy
    const Window& w = issued - base < 32 ? now : next;
    if (lane == (issued & 31) && w.slab >= 0 && !p.drop_loads) {
      const uint32_t bar = bars + issue_stage * 8, dst = ring + issue_stage * 2 * S::kTileBytes;
      mbarrier_arrive_expect_tx(bar, 2 * S::kTileBytes);
#pragma unroll
      for (int x = 0; x < S::kBoxes; ++x) {
        tma_load_3d(dst + x * S::kBoxBytes, &key_map, bar, x * S::kRowBytes, w.row, w.slab);
        tma_load_3d(dst + S::kTileBytes + x * S::kBoxBytes, &value_map, bar, x * S::kRowBytes, w.row, w.slab);
      }
    }
    __syncwarp();
    ++issued;
    issue_stage = issue_stage + 1 == kStages ? 0 : issue_stage + 1;
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s)
    if (s < mine) issue();

  // Scores without a mask are in units of log 2; with one they stay natural, since a mask of the type's lowest value would
  // leave its range.
  constexpr float kUnit = kMask ? 1.0f : kLog2e, kToLog2 = kMask ? kLog2e : 1.0f;

  // ---- q as B operands: lane (g, j) holds head g, elements 64 c + 16 j .. + 15 of every 64 ----
  uint32_t qb[NT][kSteps][2];
  float factor[NT][2];  // score of one product, for this lane's columns (heads 2 j, 2 j + 1)
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int head = 8 * t + g;
    float v[D / 4];
    if (head < heads) {
      const int64_t offset = b * p.q_batch_stride + (head0 + head) * p.q_head_stride + 16 * j;
      const uint16_t* q = static_cast<const uint16_t*>(p.q) + offset;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        uint32_t raw[8];
        if (p.q_vector) {
          const uint4 a = *reinterpret_cast<const uint4*>(q + 64 * c), d = *reinterpret_cast<const uint4*>(q + 64 * c + 8);
          raw[0] = a.x; raw[1] = a.y; raw[2] = a.z; raw[3] = a.w;
          raw[4] = d.x; raw[5] = d.y; raw[6] = d.z; raw[7] = d.w;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            raw[e] = q[64 * c + 2 * e] | (static_cast<uint32_t>(q[64 * c + 2 * e + 1]) << 16);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[16 * c + 2 * e] = Elem<T>::lo(raw[e]);
          v[16 * c + 2 * e + 1] = Elem<T>::hi(raw[e]);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < D / 4; ++e) v[e] = 0.0f;
    }
    float most = 0.0f;
#pragma unroll
    for (int e = 0; e < D / 4; ++e) most = fmaxf(most, fabsf(v[e]));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const uint32_t exponent = min(max(__float_as_uint(most) >> 23, 1u), 253u);
    const float down = __uint_as_float((254u - exponent) << 23), up = __uint_as_float(exponent << 23);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {  // k-step i: bytes 4 (i % 4) .. + 3 of the lane's 16 in 64-element group i / 4
      const int e = 16 * (i / 4) + 4 * (i % 4);
      qb[t][i][0] = pack_half2(v[e] * down, v[e + 1] * down);
      qb[t][i][1] = pack_half2(v[e + 2] * down, v[e + 3] * down);
    }
    factor[t][0] = p.scale * kUnit * __shfl_sync(0xffffffffu, up, 8 * j);
    factor[t][1] = p.scale * kUnit * __shfl_sync(0xffffffffu, up, 8 * j + 4);
  }

  float m[NT][2], l[NT][2], o[NT][kSteps][4];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t][0] = m[t][1] = -INFINITY;
    l[t][0] = l[t][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.0f;
  }
  int vref_exponent = 0;  // biased; 0: none so far
  float inverse_vref = 0.0f;
  bool timed_out = false;
  const int my_token = S::token(g);
  float mask_next[kEach];
  auto fetch_mask = [&](int it) {
    if constexpr (kMask) {
#pragma unroll
      for (int r = 0; r < kEach; ++r) {
        const int token = (my_first + it * stride) * kTile + 8 * r + my_token;
        mask_next[r] = it < mine && token < length ? load_mask(p, b * p.mask_batch_stride + token) : 0.0f;
      }
    }
  };
  fetch_mask(0);
  // phases: a stage completes only where a copy was issued, so a tile without a block does not turn its parity
  uint32_t phase = 0;

  int it = 0, stage = 0;
  for (; it < mine; ++it, stage = stage + 1 == kStages ? 0 : stage + 1) {
    if (it - base == 32) {
      now = next;
      base = it;
      next = look_up(base + 32 + lane);
    }
    const int slab = __shfl_sync(0xffffffffu, now.slab, it & 31);
    const float ks = __shfl_sync(0xffffffffu, now.ks, it & 31), vs = __shfl_sync(0xffffffffu, now.vs, it & 31);
    if (slab >= 0) {
      if (!__all_sync(0xffffffffu, mbarrier_wait_ready_first(bars + stage * 8, (phase >> stage) & 1, p.wait_limit))) {
        timed_out = true;
        break;
      }
      phase ^= 1u << stage;
    }
    __syncwarp();  // every lane is done with the stage that is filled next
    if (issued < mine) issue();
    float extra[kEach];
#pragma unroll
    for (int r = 0; r < kEach; ++r) extra[r] = kMask ? mask_next[r] : 0.0f;
    fetch_mask(it + 1);
    if (slab < 0) continue;
    const uint32_t keys = ring + stage * 2 * S::kTileBytes, values = keys + S::kTileBytes;
    const int valid = min(length - (my_first + it * stride) * kTile, kTile);

    // ---- scores of the tile ----
    float s[NT][kParts][4];
#pragma unroll
    for (int mt = 0; mt < kParts; ++mt) {
#pragma unroll
      for (int t = 0; t < NT; ++t) s[t][mt][0] = s[t][mt][1] = s[t][mt][2] = s[t][mt][3] = 0.0f;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        uint32_t w0[4], w1[4];
        const int row = 16 * mt + my_token;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w0[0]), "=r"(w0[1]), "=r"(w0[2]), "=r"(w0[3])
                     : "r"(keys + S::at(row, 4 * c + j)));
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w1[0]), "=r"(w1[1]), "=r"(w1[2]), "=r"(w1[3])
                     : "r"(keys + S::at(row + 8, 4 * c + j)));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t a[4];
          Convert<Code>::neighbours(w0[i], a[0], a[2]);
          Convert<Code>::neighbours(w1[i], a[1], a[3]);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_f16_16816(s[t][mt], a, qb[t][4 * c + i][0], qb[t][4 * c + i][1]);
        }
      }
    }
    auto highest = [&](int t, int h) {
      float top = fmaxf(s[t][0][h], s[t][0][2 + h]);
#pragma unroll
      for (int mt = 1; mt < kParts; ++mt) top = fmaxf(top, fmaxf(s[t][mt][h], s[t][mt][2 + h]));
      return top;
    };
    bool over = false;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float f = ks * factor[t][h];
#pragma unroll
        for (int r = 0; r < kEach; ++r) {  // token 8 r + my_token
          float& x = s[t][r >> 1][2 * (r & 1) + h];
          x = kMask ? fmaf(x, f, extra[r]) : x * f;
        }
      }
    if (valid < kTile) {
#pragma unroll
      for (int r = 0; r < kEach; ++r)
        if (8 * r + my_token >= valid) {
#pragma unroll
          for (int t = 0; t < NT; ++t) s[t][r >> 1][2 * (r & 1)] = s[t][r >> 1][2 * (r & 1) + 1] = -INFINITY;
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        over = over || highest(t, h) > m[t][h] + kSlack / kToLog2;
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float top = highest(t, h);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          top = fmaxf(top, m[t][h]);
          const float keep = top == -INFINITY ? 1.0f : exp2_fast((m[t][h] - top) * kToLog2);
          m[t][h] = top;
          l[t][h] *= keep;
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            o[t][i][h] *= keep;
            o[t][i][2 + h] *= keep;
          }
        }
    }
    float weight = vs * inverse_vref;
    if (vs != 0.0f && fabsf(vs) <= FLT_MAX && !(fabsf(weight) >= 0.25f && fabsf(weight) <= 2.0f)) {
      // (only heads that are there count: a column without one weighs every token)
      bool seen = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) seen = seen || (8 * t + 2 * j + h < heads && highest(t, h) > m[t][h] - kUnseen / kToLog2);
      if (__any_sync(0xffffffffu, seen)) {
        int to = min(max(static_cast<int>((__float_as_uint(vs) >> 23) & 255u), 1), 253);
        if (to < vref_exponent) {
          // O grows by as much as leaves its largest element below 2^96, and never by more than one factor can
          float most = 0.0f;
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (8 * t + 2 * j + h < heads)
#pragma unroll
                for (int i = 0; i < kSteps; ++i) most = fmaxf(most, fmaxf(fabsf(o[t][i][h]), fabsf(o[t][i][2 + h])));
#pragma unroll
          for (int x = 1; x < 32; x *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));
          if (most > 0.0f) to = max(to, vref_exponent - max(min(223 - static_cast<int>(__float_as_uint(most) >> 23), 127), 0));
        }
        const int turn = 127 + vref_exponent - to;  // 2^(old - new); beyond one factor's range O is 0, or nothing of it is seen
        const float keep = vref_exponent == 0 || turn > 254 ? 1.0f : turn < 1 ? 0.0f : __uint_as_float(static_cast<uint32_t>(turn) << 23);
        vref_exponent = to;
        inverse_vref = __uint_as_float(static_cast<uint32_t>(254 - to) << 23);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            o[t][i][0] *= keep; o[t][i][1] *= keep; o[t][i][2] *= keep; o[t][i][3] *= keep;
          }
      }
      weight = vs * inverse_vref;
      if (fabsf(weight) >= 4.0f) weight = 0.0f;  // (unseen)
    }
    weight *= kLift;

    // ---- probabilities, transposed into B operands ----
    uint32_t pb[NT][kParts][2], rest[NT][kParts][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float m0 = m[t][0] == -INFINITY ? 0.0f : m[t][0], m1 = m[t][1] == -INFINITY ? 0.0f : m[t][1];
#pragma unroll
      for (int r = 0; r < kEach; ++r) {
        const float p0 = exp2_fast((s[t][r >> 1][2 * (r & 1)] - m0) * kToLog2);
        const float p1 = exp2_fast((s[t][r >> 1][2 * (r & 1) + 1] - m1) * kToLog2);
        l[t][0] += p0;
        l[t][1] += p1;
        const float w0 = p0 * weight, w1 = p1 * weight;
        const uint32_t both = pack_half2(w0, w1);
        pb[t][r >> 1][r & 1] = transpose_8x8(both);
        if constexpr (IsHalf<T>::value)
          rest[t][r >> 1][r & 1] = transpose_8x8(pack_half2(w0 - Elem<__half>::lo(both), w1 - Elem<__half>::hi(both)));
      }
    }
    if constexpr (std::is_same<Code, E4m3Code>::value) {
      if (valid < kTile) {  // codes behind the end may be NaN, which a weight of zero does not silence
        constexpr int kChunks = D / 16;
        for (int i = lane; i < (kTile - valid) * kChunks; i += 32)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(values + S::at(valid + i / kChunks, i % kChunks)),
                       "r"(0u) : "memory");
        __syncwarp();
      }
    }
    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int mt = 0; mt < kParts; ++mt)
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[4];
        ldmatrix_x4_trans(r, values + S::at(16 * mt + ((lane >> 3) & 1) * 8 + S::token(lane & 7), 2 * c + (lane >> 4)));
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t a[4];
          Convert<Code>::every_other(r[2 * half], a[0], a[1]);
          Convert<Code>::every_other(r[2 * half + 1], a[2], a[3]);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma_f16_16816(o[t][2 * c + half], a, pb[t][mt][0], pb[t][mt][1]);
            if constexpr (IsHalf<T>::value) mma_f16_16816(o[t][2 * c + half], a, rest[t][mt][0], rest[t][mt][1]);
          }
        }
      }
  }
  if (bad) atomicOr(p.status, B200_STATUS_BAD_POSITION);
  if (timed_out) {  // copies in flight still write to this CTA's memory: wait for them, with the same limit
    for (; it < issued; ++it) mbarrier_wait_bounded(bars + it % kStages * 8, (phase >> it % kStages) & 1, p.wait_limit);
    if (lane == 0) atomicOr(p.status, B200_STATUS_WAIT_TIMEOUT);
  }

  // ---- the four warps' parts, through the ring's memory: means, since the sum of a long sequence's values may leave fp32
  // where they do not ----
  float share[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float sum = l[t][h];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if (g == 0) {
        merge_m[warp][8 * t + 2 * j + h] = m[t][h];
        merge_l[warp][8 * t + 2 * j + h] = sum;
      }
      share[t][h] = inverse_of(kLift * sum);
    }
  __syncthreads();  // every ring is done with
  if (!S::kBeside(NT) && p.cluster && !alone) cluster_arrive();
  float* parts = reinterpret_cast<float*>(smem);  // [warp][head][D]
  const float vref = __uint_as_float(static_cast<uint32_t>(vref_exponent) << 23);
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int head = 8 * t + 2 * j + h;
        *reinterpret_cast<float2*>(parts + (warp * kHeads + head) * D + 16 * i + 2 * g) =
            make_float2(o[t][i][h] * share[t][h] * vref, o[t][i][2 + h] * share[t][h] * vref);
      }
  __syncthreads();
  const int64_t item = b * gridDim.y + item_head;
  // merged by a thread for a whole row of four; NaN in a part stays (a weight of zero does not silence it)
  auto put_out = [&](int head, int d, float4 value, float sum) {
    const int64_t at = (b * p.q_heads + head0 + head) * D + d;
    if (sum == 0.0f) value = make_float4(NAN, NAN, NAN, NAN);  // (a sequence without tokens, or with none left by its mask)
    *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at) = make_uint2(Elem<T>::pack(value.x, value.y), Elem<T>::pack(value.z, value.w));
  };
  auto add_part = [](float share, const float4& part, float4& value) {
    value.x = fmaf(share, part.x, value.x); value.y = fmaf(share, part.y, value.y);
    value.z = fmaf(share, part.z, value.z); value.w = fmaf(share, part.w, value.w);
  };
  auto weight_of = [&](float one, float top) { return one == -INFINITY ? 0.0f : exp2_fast((one - top) * kToLog2); };
  // In a cluster each CTA finishes every `active`-th run of four, and is given the others' parts of those: stores to another
  // SM are over sooner than loads from it, and nobody reads from a CTA that would like to leave (1 x 1000: 5.3 us with loads).
  float4* given = reinterpret_cast<float4*>(smem + S::kGivenAt(NT));  // [CTA][runs of this one]
  const int runs = heads * (D / 4), own_runs = (runs + active - 1) / active;
  if (p.cluster && !alone) {
    __syncwarp();
    cluster_wait();  // the others' memory is there
  }
  for (int e = threadIdx.x; e < heads * (D / 4); e += kThreads) {
    const int head = e / (D / 4), d = e % (D / 4) * 4;
    float top = -INFINITY, sum = 0.0f, part_l[kWarps];
    float4 value = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, merge_m[w][head]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      part_l[w] = weight_of(merge_m[w][head], top) * merge_l[w][head];
      sum += part_l[w];
    }
    const float inverse = inverse_of(sum);
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      add_part(part_l[w] * inverse, *reinterpret_cast<const float4*>(parts + (w * kHeads + head) * D + d), value);
    if (alone) {
      if (split == 0) put_out(head, d, value, sum);
    } else if (p.cluster) {
      const int local = e / active;
      store_cluster_f32x4(smem_u32(given + split * own_runs + local), e - local * active, value);
      if (d == 0)
        for (int i = 0; i < active; ++i) store_cluster_f32x2(smem_u32(&joined[split][head]), i, make_float2(top, sum));
    } else {
      const int64_t part = (item * p.num_splits + split) * p.block_heads + head;
      *reinterpret_cast<float4*>(p.ws_o + part * D + d) = value;
      if (d == 0) {
        p.ws_ml[2 * part] = top;
        p.ws_ml[2 * part + 1] = sum;
      }
    }
  }
  if (p.cluster) {
    if (alone) return;
    __syncwarp();
    cluster_sync();
    for (int local = threadIdx.x; local * active + split < runs; local += kThreads) {
      const int e = local * active + split, head = e / (D / 4), d = e % (D / 4) * 4;
      float top = -INFINITY, sum = 0.0f;
      float4 value = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float2 ml[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ml[i] = i < active ? joined[i][head] : make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, ml[i].x);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ml[i].y *= weight_of(ml[i].x, top);
        sum += ml[i].y;
      }
      const float inverse = inverse_of(sum);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < active) add_part(ml[i].y * inverse, given[i * own_runs + local], value);
      put_out(head, d, value, sum);
    }
    return;
  }
  if (alone) return;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();  // (behind the barrier: the partials of all threads)
    last_flag = atomicAdd(p.counters + item, 1) == active - 1;
    __threadfence();
  }
  __syncthreads();
  if (!last_flag) return;
  for (int e = threadIdx.x; e < heads * (D / 4); e += kThreads) {
    const int head = e / (D / 4), d = e % (D / 4) * 4;
    const int64_t first = item * p.num_splits * p.block_heads + head;
    float top = -INFINITY, sum = 0.0f;
    float4 value = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = 0; s0 < active; s0 += 16) {  // sixteen loads in flight
      float2 ml[16];
      float4 part[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int64_t at = first + static_cast<int64_t>(min(s0 + i, active - 1)) * p.block_heads;
        ml[i] = __ldcg(reinterpret_cast<const float2*>(p.ws_ml) + at);
        part[i] = __ldcg(reinterpret_cast<const float4*>(p.ws_o + at * D + d));
      }
      float over_all = top;
#pragma unroll
      for (int i = 0; i < 16; ++i) over_all = fmaxf(over_all, ml[i].x);  // (the last one again does no harm)
      const float before = sum * weight_of(top, over_all);
      top = over_all;
      sum = before;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (s0 + i < active) {
          ml[i].y *= weight_of(ml[i].x, top);
          sum += ml[i].y;
        }
      const float inverse = inverse_of(sum), keep = before * inverse;
      value.x *= keep; value.y *= keep; value.z *= keep; value.w *= keep;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (s0 + i < active) add_part(ml[i].y * inverse, part[i], value);
    }
    put_out(head, d, value, sum);
  }
  if (threadIdx.x == 0) p.counters[item] = 0;
}

// [slabs, block_size, D] codes of one (block, head) after another, in boxes of 32 tokens x one swizzle span.
template <int D>
bool make_pool_map(CUtensorMap* map, const void* base, int64_t slabs, int64_t block_size) {
  EncodeTiledFn encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  const cuuint64_t dims[3] = {D, static_cast<cuuint64_t>(block_size), static_cast<cuuint64_t>(slabs)};
  const cuuint64_t strides[2] = {D, static_cast<cuuint64_t>(D * block_size)};
  const cuuint32_t box[3] = {Shape<D>::kRowBytes, Shape<D>::kTile, 1}, element_strides[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, element_strides,
                CU_TENSOR_MAP_INTERLEAVE_NONE, D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, typename Code, int D, int NT, bool kMask>
int launch_shape(const Params& p, const void* keys, const void* values, int64_t batch, cudaStream_t stream) {
  CUtensorMap key_map, value_map;
  if (!make_pool_map<D>(&key_map, keys, p.num_blocks * p.kv_heads, p.block_size) ||
      !make_pool_map<D>(&value_map, values, p.num_blocks * p.kv_heads, p.block_size))
    return B200_ERR_UNSUPPORTED;
  constexpr int smem = std::max(Shape<D>::kBytes(NT), Shape<D>::kPartBytes(NT));
  auto kernel = cache_attention_kernel<T, Code, D, NT, kMask>;
  static std::atomic<uint64_t> allowed{0};
  if (!allow_shared_memory(kernel, smem, allowed)) return B200_ERR_LAUNCH;
  const dim3 grid(static_cast<unsigned>(p.num_splits), static_cast<unsigned>(p.kv_heads * p.head_blocks),
                  static_cast<unsigned>(batch));
  return launch_chained_cluster(kernel, grid, dim3(kThreads), smem, stream, p.cluster ? static_cast<unsigned>(p.num_splits) : 1u,
                                p, key_map, value_map) == cudaSuccess ? launch_status() : B200_ERR_LAUNCH;
}
template <typename T, typename Code, int D, int NT>
int launch_mask(const Params& p, const void* keys, const void* values, int64_t batch, cudaStream_t stream) {
  return p.mask != nullptr ? launch_shape<T, Code, D, NT, true>(p, keys, values, batch, stream)
                           : launch_shape<T, Code, D, NT, false>(p, keys, values, batch, stream);
}
// n-tiles of heads: one up to eight heads of a block, else two (head_dim 256: one, its accumulators fill the registers)
template <typename T, typename Code>
int launch_code(const Params& p, const void* keys, const void* values, int64_t batch, int64_t dim, cudaStream_t stream) {
  const bool one = p.block_heads <= 8;
  if (dim == 64)
    return one ? launch_mask<T, Code, 64, 1>(p, keys, values, batch, stream) : launch_mask<T, Code, 64, 2>(p, keys, values, batch, stream);
  if (dim == 128)
    return one ? launch_mask<T, Code, 128, 1>(p, keys, values, batch, stream) : launch_mask<T, Code, 128, 2>(p, keys, values, batch, stream);
  return launch_mask<T, Code, 256, 1>(p, keys, values, batch, stream);
}

// instances, in a file each
int launch_int8_bf16(const Params& p, const void* keys, const void* values, int64_t batch, int64_t dim, cudaStream_t stream);
int launch_int8_f16(const Params& p, const void* keys, const void* values, int64_t batch, int64_t dim, cudaStream_t stream);
int launch_e4m3_bf16(const Params& p, const void* keys, const void* values, int64_t batch, int64_t dim, cudaStream_t stream);
int launch_e4m3_f16(const Params& p, const void* keys, const void* values, int64_t batch, int64_t dim, cudaStream_t stream);

}  // namespace cache_attention
}  // namespace b200
