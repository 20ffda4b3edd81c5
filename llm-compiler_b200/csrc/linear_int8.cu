// Projections in 8-bit integers on the tensor cores: y = (c_x . c_w) s_x s_w + bias, then SwiGLU or a residual, rounded once.
//
// c_x [M, K] and c_w [N, K] are codes with a scale per row (token) and per output column. tcgen05.mma kind::i8 multiplies
// 32 of them along K in the time of 16 bf16 and sums in 32-bit integers, which is exact (K is at most 131056: 131056 * 128 *
// 128 is below 2^31): the result does not depend on the order or on the split of a sum, and a projection may be cut
// anywhere along K. Both operands are K-major; a stage of the rings holds 128 codes of K, one 128-byte swizzled row each,
// copied by TMA with zeros beyond M, N and K. Two kernels:
//
// linear_int8_stream_kernel, few rows (decode, short prompts): bound by the read of the weight. The WEIGHT's columns
//   lie along the product's M (128 of them a tile) and all rows of x along its N, so every weight byte is read once and no
//   row of x is padded beyond the next multiple of 16. (More rows against a narrow weight go in chunks of up to 256, where
//   that keeps more SMs busy than the other kernel's tiles.) A CTA per SM takes whole tiles in turn; where there are fewer tiles
//   than SMs, the K slices of a tile are the CTAs of a cluster, which add their sums through distributed shared memory
//   (4.0 us less than integer additions in global memory at 64 x 384 x 512, where the slices then wait for one another there).
//   48 x 3584 x 37888 SwiGLU: 25 us, 5.5 TB/s, 0.85 of a copy's rate; a call of a few tiles takes 4 to 5 us whatever its size.
// linear_int8_pair_kernel, more rows: bound by the tensor cores. Two SMs work on one tile of 256 rows x up to 256 columns
//   (cta_group::2): each holds half of both operands, which halves the bytes that shared memory and L2 deliver per product
//   (at 128 x 256 a CTA they are what limits it: 96 of 128 bytes a cycle in, as many out). Two accumulators alternate, so
//   the epilogue of a tile runs under the products of the next; where there are few tiles and K is long, two to four pairs of a
//   cluster take slices of K and add their sums through distributed shared memory (512 x 4864 x 896: 8.9 us, 10.9 without).
//   4096 x 3584 x 37888 SwiGLU: 324 us, 3.4 POP/s, the tensor pipe busy 97 % of the time; below K of some 1000 the epilogue
//   (2.8 us a tile) is what is seen: 16384 x 896 x 9728 SwiGLU 124 us where the products alone take 79.
#include <algorithm>
#include <type_traits>

#include "quantized.cuh"
#include "tcgen05.cuh"
#include "tensor_map.cuh"

namespace b200 {
namespace {

constexpr int kMaxK = 131056;
constexpr int kBK = 128;          // codes of a k-block: one 128-byte row
constexpr int kEpilogueWarps = 4;
constexpr int kThreads = (kEpilogueWarps + 2) * 32;  // and a producer and a product warp
constexpr int kRowsAtMost = 256;  // of the stream kernel
constexpr int kRingBytes = 192 * 1024;

struct Int8LinearParams {
  const float* x_scales;
  const float* w_scales;
  const void* bias;
  const void* residual;
  void* out;
  int32_t* status;
  int m, k, n, epilogue;
  int cols;     // stream: rows of x, rounded up to 16, the product's N. pair: columns of a tile
  int stages;   // stream
  int slices;   // stream: of K, the CTAs of a cluster
  int n_fastest;  // pair: order of the tiles
  int ahead;      // stream: the weight may be read while what is in front of the kernel still runs
  uint32_t wait_limit;
  int drop_loads;
};

// Instruction descriptor of kind::i8: 32-bit integer accumulator, both operands signed, K-major.
__host__ __device__ constexpr uint32_t instruction_descriptor_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
template <int CTAS>
__device__ __forceinline__ void umma_i8_if(uint32_t leader, uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  if constexpr (CTAS == 1)
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
  else
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
}
// The products so far arrive on the barrier at this offset in both CTAs of the pair, whose first has rank `first`.
__device__ __forceinline__ void umma_commit_pair_if(uint32_t leader, uint32_t bar, int first) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
               "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}"
               ::"r"(bar), "r"(leader), "h"(static_cast<uint16_t>(3 << first)) : "memory");
}
// A box into this CTA's memory whose bytes count on a barrier of the pair's first CTA.
__device__ __forceinline__ void tma_load_pair_if(uint32_t leader, uint32_t dst, const void* tensor_map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tensor_map)), "r"(bar), "r"(c0), "r"(c1), "r"(leader)
      : "memory");
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, int rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  return remote;
}

// A producer that gives up at stage s of turn `turn`: the copies that it has asked for still write to shared memory.
__device__ __forceinline__ void wait_for_copies(uint64_t* full, int stages, int s, int turn, uint32_t limit) {
  for (int i = 0; i < stages; ++i) {
    const int last = i < s ? turn : turn - 1;
    if (last >= 0) mbarrier_wait_warp(smem_u32(&full[i]), last & 1, limit);
  }
}

// gate / (1 + e^-gate) * up on the special-function unit: 2^x and 1 / x there are good to two units of 2^-23, and the
// exponent's rounding adds |gate| of them. (Below -88 the sum is infinite and its reciprocal 0: the right answer.)
__device__ __forceinline__ float silu_times(float gate, float up) {
  float power, inverse;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(power) : "f"(-1.4426950408889634f * gate));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(1.0f + power));
  return gate * inverse * up;
}

// a = a row t.x + t.z and b = b row t.y + t.w, each product and sum of the two in one instruction
__device__ __forceinline__ void scale_two(float& a, float& b, float row, const float4& t) {
  asm("{\n\t.reg .b64 v, r, s, c;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 r, {%2, %2};\n\tmov.b64 s, {%3, %4};\n\t"
      "mov.b64 c, {%5, %6};\n\tmul.rn.f32x2 v, v, r;\n\tfma.rn.f32x2 v, v, s, c;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "+f"(a), "+f"(b) : "f"(row), "f"(t.x), "f"(t.y), "f"(t.z), "f"(t.w));
}

__device__ __forceinline__ int4 load_cluster_i32x4(uint32_t remote) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(remote)
               : "memory");
  return v;
}

// Four columns of a row whose sums are in shared memory of the cluster's CTAs at `addr`, CTAs `step` apart from `first`: the
// epilogue, behind the slices of K.
template <typename T>
struct FourColumns {
  int col, width;  // the first, and how many of the four there are
  float w_scale[4], bias[4];
  __device__ FourColumns(const Int8LinearParams& p, int col_) : col(col_), width(min(p.n - col_, 4)) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      w_scale[c] = c < width ? p.w_scales[col + c] : 0.0f;
      bias[c] = c < width && p.bias != nullptr ? Elem<T>::load(static_cast<const T*>(p.bias) + col + c) : 0.0f;
    }
  }
  template <int kSlices>
  __device__ void finish(uint32_t addr, int first, int step, int slices, float scale, const T* residual, T* out, bool swiglu) const {
    int4 part[kSlices];
#pragma unroll
    for (int i = 0; i < kSlices; ++i)
      part[i] = i < slices ? load_cluster_i32x4(map_to_rank(addr, first + i * step)) : make_int4(0, 0, 0, 0);
    float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (residual != nullptr) {
      const T* from = residual + col;
      if (width == 4) {
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = Elem<T>::load(from + c);
      } else {
        for (int c = 0; c < width; ++c) y[c] = Elem<T>::load(from + c);
      }
    }
#pragma unroll
    for (int i = 1; i < kSlices; ++i) {
      part[0].x += part[i].x; part[0].y += part[i].y; part[0].z += part[i].z; part[0].w += part[i].w;
    }
    y[0] += static_cast<float>(part[0].x) * scale * w_scale[0] + bias[0];
    y[1] += static_cast<float>(part[0].y) * scale * w_scale[1] + bias[1];
    y[2] += static_cast<float>(part[0].z) * scale * w_scale[2] + bias[2];
    y[3] += static_cast<float>(part[0].w) * scale * w_scale[3] + bias[3];
    T* to = out + (swiglu ? col / 2 : col);
    if (swiglu) {
      if (width > 0) Elem<T>::store(to, silu_times(y[0], y[1]));
      if (width > 2) Elem<T>::store(to + 1, silu_times(y[2], y[3]));
    } else if (width == 4) {
#pragma unroll
      for (int c = 0; c < 4; ++c) Elem<T>::store(to + c, y[c]);
    } else {
      for (int c = 0; c < width; ++c) Elem<T>::store(to + c, y[c]);
    }
  }
};

// ------------------------------------------------------------------------------------------------------------ stream ----
template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
linear_int8_stream_kernel(const Int8LinearParams p, const __grid_constant__ CUtensorMap w_map,
                          const __grid_constant__ CUtensorMap x_map) {
  constexpr int kMaxStages = 10;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
  __shared__ float scales[kRowsAtMost];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;

  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stages = p.stages, stage_bytes = (128 + p.cols) * 128;
  int acc_columns = 16;  // of an accumulator, a power of two
  while (acc_columns < p.cols) acc_columns *= 2;
  const int tmem_columns = 2 * acc_columns;
  const uint32_t smem_base = smem_u32(smem);
  const int all_kb = (p.k + kBK - 1) / kBK, tiles = (p.n + 127) / 128;
  const int rank = p.slices > 1 ? cluster_cta_rank() : 0;
  const int kb_first = all_kb * rank / p.slices, nkb = all_kb * (rank + 1) / p.slices - kb_first;  // this slice: two at least
  const int tile_first = blockIdx.x / p.slices, tile_step = gridDim.x / p.slices;
  const int row_first = blockIdx.y * p.cols, rows = min(p.cols, p.m - row_first);  // this CTA's chunk of x

  if (threadIdx.x == 0) {
    failed = 0;
    for (int s = 0; s < stages; ++s) {
      mbarrier_init(smem_u32(&full[s]), 1);
      mbarrier_init(smem_u32(&empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbarrier_init(smem_u32(&acc_full[a]), 1);
      mbarrier_init(smem_u32(&acc_empty[a]), kEpilogueWarps);
    }
    fence_mbarrier_init();
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&w_map)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&x_map)) : "memory");
  }
  if (warp == kEpilogueWarps + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_slot)), "r"(static_cast<uint32_t>(tmem_columns)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_slot;
  // Where the weight may be read ahead (a step's projections, launched while the kernel in front still runs), the ring's
  // stages are asked for before the wait, all but their rows of x.
  int ahead = 0;
  if (p.ahead && warp == kEpilogueWarps && !p.drop_loads) {
    const uint32_t leader = elect_one();
    ahead = min(stages, nkb * ((tiles - tile_first + tile_step - 1) / tile_step));
    for (int s = 0, tile = tile_first, kb = 0; s < ahead; ++s) {
      mbarrier_arrive_expect_tx_if(leader, smem_u32(&full[s]), stage_bytes);
      tma_load_2d_if(leader, smem_base + s * stage_bytes, &w_map, smem_u32(&full[s]), (kb_first + kb) * kBK, tile * 128);
      if (++kb == nkb) { kb = 0; tile += tile_step; }
    }
  }
  grid_dependency_wait();
  const bool swiglu = p.epilogue == B200_EPILOGUE_SWIGLU;
  const int64_t out_cols = swiglu ? p.n / 2 : p.n;
  T* out = static_cast<T*>(p.out) + row_first * out_cols;
  const T* residual = p.residual ? static_cast<const T*>(p.residual) + row_first * out_cols : nullptr;

  if (warp == kEpilogueWarps && !p.drop_loads) {
    // ---- producer: the ring runs on across tile ends ----
    const uint32_t leader = elect_one();
    int s = 0, turn = 0;
    bool ok = true;
    for (int tile = tile_first; ok && tile < tiles; tile += tile_step)
      for (int kb = 0; kb < nkb; ++kb) {
        if (turn > 0 && !mbarrier_wait_warp(smem_u32(&empty[s]), (turn - 1) & 1, p.wait_limit)) {
          failed = 1;
          wait_for_copies(full, stages, s, turn, p.wait_limit);
          ok = false;
          break;
        }
        const uint32_t bar = smem_u32(&full[s]), dst = smem_base + s * stage_bytes;
        if (ahead > 0) {
          --ahead;
        } else {
          mbarrier_arrive_expect_tx_if(leader, bar, stage_bytes);
          tma_load_2d_if(leader, dst, &w_map, bar, (kb_first + kb) * kBK, tile * 128);
        }
        tma_load_2d_if(leader, dst + 128 * 128, &x_map, bar, (kb_first + kb) * kBK, row_first);
        if (++s == stages) { s = 0; ++turn; }
      }
  } else if (warp == kEpilogueWarps + 1) {
    // ---- products ----
    const uint32_t leader = elect_one();
    const uint32_t idesc = instruction_descriptor_i8(128, p.cols);
    int s = 0, turn = 0, done = 0;
    bool ok = true;
    for (int tile = tile_first; ok && tile < tiles; tile += tile_step, ++done) {
      const int acc = done & 1;
      if (done >= 2 && !mbarrier_wait_warp(smem_u32(&acc_empty[acc]), ((done >> 1) - 1) & 1, p.wait_limit)) { ok = false; break; }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t d = tmem_base + acc * acc_columns;
      for (int kb = 0; kb < nkb; ++kb) {
        if (!mbarrier_wait_warp(smem_u32(&full[s]), turn & 1, p.wait_limit)) { ok = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t a_desc = smem_descriptor(smem_base + s * stage_bytes), b_desc = descriptor_advance(a_desc, 128 * 128);
#pragma unroll
        for (int q = 0; q < kBK / 32; ++q)
          umma_i8_if<1>(leader, d, descriptor_advance(a_desc, q * 32), descriptor_advance(b_desc, q * 32), idesc,
                        (kb > 0 || q > 0) ? 1u : 0u);
        umma_commit_if(leader, smem_u32(&empty[s]));
        if (++s == stages) { s = 0; ++turn; }
      }
      if (ok) umma_commit_if(leader, smem_u32(&acc_full[acc]));
    }
    if (!ok) failed = 1;
  } else if (warp < kEpilogueWarps) {
    // ---- epilogue: lanes of the accumulator are columns of y, its columns are rows ----
    for (int r = threadIdx.x; r < p.cols; r += kEpilogueWarps * 32) scales[r] = r < rows ? p.x_scales[row_first + r] : 0.0f;
    asm volatile("bar.sync 1, 128;" ::: "memory");
    bool ok = true;
    int done = 0;
    for (int tile = tile_first; tile < tiles; tile += tile_step, ++done) {
      const int acc = done & 1;
      // a thread owns a column; 16 rows at a time: all operands before all stores, which the compiler may not swap, and
      // what comes from memory before the wait for the products or beside the rows in front
      const int col = tile * 128 + warp * 32 + lane;
      const bool there = col < p.n && p.slices == 1;
      const float w_scale = there ? p.w_scales[col] : 0.0f;
      const float bias = there && p.bias != nullptr ? Elem<T>::load(static_cast<const T*>(p.bias) + col) : 0.0f;
      float near[16], far[16];  // the residual of the next 16 rows and of those behind them
      auto fetch = [&](int r0, float (&other)[16]) {
        if (residual == nullptr || !there) return;
        const T* from = residual + r0 * out_cols + col;
        if (r0 + 16 <= rows) {
#pragma unroll
          for (int r = 0; r < 16; ++r) other[r] = Elem<T>::load(from + r * out_cols);
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) other[r] = r0 + r < rows ? Elem<T>::load(from + r * out_cols) : 0.0f;
        }
      };
      fetch(0, near);
      fetch(16, far);
      ok = __all_sync(0xffffffffu, mbarrier_wait_bounded(smem_u32(&acc_full[acc]), (done >> 1) & 1, p.wait_limit));
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t t_addr = tmem_base + acc * acc_columns + (static_cast<uint32_t>(warp * 32) << 16);
      if (p.slices > 1) {
        // (one tile a CTA: every stage has been read, the sums take the ring's place: [row][128])
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += 16) {
          float v[16];
          tmem_load_32x32(t_addr + r0, v);
          const uint32_t to = smem_base + r0 * 512 + (warp * 32 + lane) * 4;
#pragma unroll
          for (int r = 0; r < 16; ++r) asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + r * 512), "f"(v[r]) : "memory");
        }
        break;
      }
      const bool writes = there && !(swiglu && (lane & 1) != 0);
      T* to = out + (swiglu ? col / 2 : col);
      auto sixteen = [&](int r0, float (&other)[16]) {
        float v[16];
        tmem_load_32x32(t_addr + r0, v);
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = static_cast<float>(__float_as_int(v[r])) * scales[r0 + r] * w_scale + bias;
        if (residual != nullptr) {
#pragma unroll
          for (int r = 0; r < 16; ++r) v[r] += other[r];
          if (r0 + 32 < rows) fetch(r0 + 32, other);
        } else if (swiglu) {
#pragma unroll
          for (int r = 0; r < 16; ++r) v[r] = silu_times(v[r], __shfl_xor_sync(0xffffffffu, v[r], 1));
        }
        if (writes) {
          T* at = to + r0 * out_cols;
          if (r0 + 16 <= rows) {
#pragma unroll
            for (int r = 0; r < 16; ++r) Elem<T>::store(at + r * out_cols, v[r]);
          } else {
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (r0 + r < rows) Elem<T>::store(at + r * out_cols, v[r]);
          }
        }
      };
#pragma unroll 1
      for (int r0 = 0; r0 < rows; r0 += 32) {
        sixteen(r0, near);
        if (r0 + 16 < rows) sixteen(r0 + 16, far);
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&acc_empty[acc])) : "memory");
    }
    if (!ok) failed = 1;
  }
  __syncwarp();
  if (p.slices > 1) {
    // ---- the slices' sums: this CTA finishes rows rank, rank + slices, ...; a lane takes four columns ----
    cluster_sync();
    const FourColumns<T> four(p, tile_first * 128 + 4 * lane);
    for (int row = rank + warp * p.slices; row < rows; row += kThreads / 32 * p.slices)
      four.template finish<8>(smem_base + row * 512 + lane * 16, 0, 1, p.slices, scales[row],
                              residual != nullptr ? residual + row * out_cols : nullptr, out + row * out_cols, swiglu);
    __syncwarp();
    cluster_sync();  // (the others may still read this CTA's sums)
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0 && failed) atomicOr(p.status, B200_STATUS_WAIT_TIMEOUT);
  if (warp == kEpilogueWarps + 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                 ::"r"(tmem_base), "r"(static_cast<uint32_t>(tmem_columns)) : "memory");
}

// -------------------------------------------------------------------------------------------------------------- pair ----
// A stage: half of 256 rows of x, half of a tile's columns of the weight.
__host__ __device__ constexpr int pair_stage_bytes(int bn) { return (128 + bn / 2) * 128; }
constexpr int kPairStagesAtMost = 8;
constexpr int kPairWarps = 8;      // of the epilogue, for each quarter of the accumulator's lanes
constexpr int kAcross = kPairWarps / 4, kStep = kAcross * 32, kChunksAtMost = (8 + kAcross - 1) / kAcross;  // a quarter's warps share the columns
constexpr int kPairThreads = (kPairWarps + 2) * 32;

// Staging tiles of 32 x 32 a warp of the epilogue has, and what that leaves of the ring.
template <typename T, typename Piece>
__host__ __device__ constexpr int pair_tiles() { return sizeof(Piece) < 16 ? 1 : sizeof(T) == 4 ? 2 : 3; }
template <typename T, typename Piece>
__host__ __device__ constexpr int pair_ring() { return ((sizeof(Piece) < 16 ? 6 : 5) - (sizeof(T) == 4 ? 1 : 0)) * pair_stage_bytes(256); }
template <typename T, typename Piece>
constexpr int pair_smem() {
  return pair_ring<T, Piece>() +
         kPairWarps * (pair_tiles<T, Piece>() * 32 * 32 * static_cast<int>(sizeof(T)) + kChunksAtMost * 32 * 8);
}

// A box of shared memory to memory, if `leader`; a group of its own (an empty one for the other lanes: no branch, which would
// cost as much as the store).
__device__ __forceinline__ void tma_store_2d_if(uint32_t leader, const void* tensor_map, uint32_t from, int c0, int c1) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %4, 0;\n\t"
               "@q cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];\n\t}\n\t"
               "cp.async.bulk.commit_group;"
               ::"l"(reinterpret_cast<uint64_t>(tensor_map)), "r"(from), "r"(c0), "r"(c1), "r"(leader) : "memory");
}
// All but the thread's last `kLeft` stores have read shared memory.
template <int kLeft>
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kLeft) : "memory"); }

// Piece: uint4 where rows of y start on multiples of 16 bytes: chunks of y leave, and those of a residual come, by TMA (with
// the warps' own loads and stores of 16 bytes 16384 x 128 x 9728 with a residual takes 204 us, so 139). Else what a lane moves
// of a row at a time, 4 bytes or 2.
// kSplit: K in slices, pairs of one cluster; they add their sums through distributed shared memory (a tile a cluster).
template <typename T, typename Piece, bool kSplit>
__global__ void __launch_bounds__(kPairThreads, 1)
linear_int8_pair_kernel(const Int8LinearParams p, const __grid_constant__ CUtensorMap x_map,
                        const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap y_map,
                        const __grid_constant__ CUtensorMap residual_map) {
  constexpr bool kBulk = sizeof(Piece) == 16;
  constexpr int kRing = pair_ring<T, Piece>(), kTiles = pair_tiles<T, Piece>();
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ __align__(8) uint64_t full[kPairStagesAtMost], empty[kPairStagesAtMost], acc_full[2], acc_empty[2];
  __shared__ __align__(8) uint64_t arrived[kPairWarps * kTiles];  // a residual's chunks
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;

  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int place_in_cluster = cluster_cta_rank(), rank = place_in_cluster & 1, first_rank = kSplit ? place_in_cluster & ~1 : 0;
  const int bn = p.cols, half = bn / 2, stage_bytes = pair_stage_bytes(bn), stages = min(kRing / stage_bytes, kPairStagesAtMost);
  const uint32_t smem_base = smem_u32(smem);
  const int slices = kSplit ? p.slices : 1, slice = first_rank >> 1, all_kb = (p.k + kBK - 1) / kBK;
  const int kb_first = kSplit ? all_kb * slice / slices : 0, nkb = kSplit ? all_kb * (slice + 1) / slices - kb_first : all_kb;
  const int tiles_n = (p.n + bn - 1) / bn, tiles_m = (p.m + 255) / 256, tiles = tiles_n * tiles_m;
  const int pair = blockIdx.x / (2 * slices), pairs = gridDim.x / (2 * slices);  // (kSplit: as many as tiles)
  // a pair's tiles, one after another without a division each
  struct Place {
    int tile, slow, fast, step, step_slow, step_fast, along;
    bool n_fastest;
    __device__ Place(int first, int step_, int along_, bool n_fastest_)
        : tile(first), slow(first / along_), fast(first % along_), step(step_), step_slow(step_ / along_), step_fast(step_ % along_),
          along(along_), n_fastest(n_fastest_) {}
    __device__ void next() {
      tile += step; slow += step_slow; fast += step_fast;
      if (fast >= along) { fast -= along; ++slow; }
    }
    __device__ int m() const { return n_fastest ? slow : fast; }
    __device__ int n() const { return n_fastest ? fast : slow; }
  };
  const Place start(pair, pairs, p.n_fastest ? tiles_n : tiles_m, p.n_fastest);

  if (threadIdx.x == 0) {
    failed = 0;
    for (int s = 0; s < stages; ++s) {
      mbarrier_init(smem_u32(&full[s]), 1);
      mbarrier_init(smem_u32(&empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbarrier_init(smem_u32(&acc_full[a]), 1);
      mbarrier_init(smem_u32(&acc_empty[a]), 2 * kPairWarps);  // (the first CTA's counts: both CTAs' warps)
    }
    if constexpr (kBulk)
      for (int i = 0; i < kPairWarps * kTiles; ++i) mbarrier_init(smem_u32(&arrived[i]), 1);
    fence_mbarrier_init();
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&x_map)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&w_map)) : "memory");
  }
  if (warp == kPairWarps + 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();  // the other CTA's barriers are ready
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_slot;
  grid_dependency_wait();

  if (warp == kPairWarps && !p.drop_loads) {
    // ---- producer: this CTA's halves; all bytes of a stage count on the first CTA's barrier ----
    const uint32_t leader = elect_one();
    bool ok = true;
    int s = 0, turn = 0;
    for (Place at = start; ok && at.tile < tiles; at.next()) {
      const int tile_m = at.m(), tile_n = at.n();
      for (int kb = 0; kb < nkb; ++kb) {
        if (turn > 0 && !mbarrier_wait_warp(smem_u32(&empty[s]), (turn - 1) & 1, p.wait_limit)) {
          ok = false;
          if (rank == 0) wait_for_copies(full, stages, s, turn, p.wait_limit);
          break;
        }
        const uint32_t dst = smem_base + s * stage_bytes;
        if (rank == 0) mbarrier_arrive_expect_tx_if(leader, smem_u32(&full[s]), 2 * (128 + half) * 128);
        const uint32_t bar = map_to_rank(smem_u32(&full[s]), first_rank);
        tma_load_pair_if(leader, dst, &x_map, bar, (kb_first + kb) * kBK, tile_m * 256 + rank * 128);
        tma_load_pair_if(leader, dst + 128 * 128, &w_map, bar, (kb_first + kb) * kBK, tile_n * bn + rank * half);
        if (++s == stages) { s = 0; ++turn; }
      }
    }
    if (!ok) failed = 1;
  } else if (warp == kPairWarps + 1 && rank == 0) {
    // ---- products of both CTAs, issued by the first ----
    const uint32_t leader = elect_one();
    const uint32_t idesc = instruction_descriptor_i8(256, bn);
    bool ok = true;
    int s = 0, turn = 0, done = 0;
    for (int tile = pair; ok && tile < tiles; tile += pairs, ++done) {
      const int acc = done & 1;
      if (done >= 2 && !mbarrier_wait_warp(smem_u32(&acc_empty[acc]), ((done >> 1) - 1) & 1, p.wait_limit)) { ok = false; break; }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t d = tmem_base + acc * 256;
      for (int kb = 0; kb < nkb; ++kb) {
        if (!mbarrier_wait_warp(smem_u32(&full[s]), turn & 1, p.wait_limit)) { ok = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t a_desc = smem_descriptor(smem_base + s * stage_bytes), b_desc = descriptor_advance(a_desc, 128 * 128);
#pragma unroll
        for (int q = 0; q < kBK / 32; ++q)
          umma_i8_if<2>(leader, d, descriptor_advance(a_desc, q * 32), descriptor_advance(b_desc, q * 32), idesc,
                        (kb > 0 || q > 0) ? 1u : 0u);
        umma_commit_pair_if(leader, smem_u32(&empty[s]), first_rank);
        if (++s == stages) { s = 0; ++turn; }
      }
      if (ok) umma_commit_pair_if(leader, smem_u32(&acc_full[acc]), first_rank);
    }
    if (!ok) failed = 1;
  } else if (kSplit && warp < kPairWarps) {
    // ---- this slice's sums, in the place of the ring, whose stages have all been read: [row][bn], the 16-byte units of
    // eight rows in different banks ----
    const bool ok = __all_sync(0xffffffffu, mbarrier_wait_bounded(smem_u32(&acc_full[0]), 0, p.wait_limit));
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const int quarter = warp & 3, row = quarter * 32 + lane;
    if (!ok) failed = 1;
#pragma unroll 1
    for (int c0 = (warp >> 2) * 32; ok && c0 < bn; c0 += kStep) {
      float v[32];
      tmem_load_32x32(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + c0, v);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};"
                     ::"r"(smem_base + row * bn * 4 + (((c0 / 4 + u) ^ (row & 7)) << 4)), "f"(v[4 * u]), "f"(v[4 * u + 1]),
                       "f"(v[4 * u + 2]), "f"(v[4 * u + 3]) : "memory");
    }
    __syncwarp();
  } else if (!kSplit && warp < kPairWarps) {
    // ---- epilogue: this CTA's 128 rows; lanes 32 (warp % 4) .., every other chunk of 32 columns ----
    // What comes from memory is asked for ahead: scales and bias during the tile before, a residual one chunk or two. A
    // chunk leaves through a staging tile, by TMA where rows allow it; where their length does not, the warp writes whole rows
    // of it in pieces of 4 bytes or 2 (2008 x 512 x 3890: 110 us with a thread for each row).
    const bool swiglu = p.epilogue == B200_EPILOGUE_SWIGLU;
    const int out_cols = swiglu ? p.n / 2 : p.n;
    T* out = static_cast<T*>(p.out);
    const T* residual = static_cast<const T*>(p.residual);
    constexpr int kVec = 16 / static_cast<int>(sizeof(T)), kUnits = 32 / kVec;  // of 16 bytes: a row of a chunk
    const int quarter = warp & 3, turn0 = warp >> 2;
    constexpr int kStageTile = 32 * 32 * static_cast<int>(sizeof(T));
    const uint32_t stage_tiles = smem_base + kRing + warp * kTiles * kStageTile;
    float* column_terms = reinterpret_cast<float*>(smem + kRing + kPairWarps * kTiles * kStageTile) + warp * kChunksAtMost * 64;
    const uint32_t acc_empty_first = map_to_rank(smem_u32(&acc_empty[0]), 0);
    uint32_t stage_tile = stage_tiles;
    // 16-byte unit `unit` of row r of a chunk with `units` of them: 128 bytes of rows side by side never share a bank (the
    // swizzle of a tensor map whose boxes have rows of 32, 64 or 128 bytes)
    auto unit_at = [&](int r, int unit, int units) {
      return stage_tile + r * units * 16 + ((unit ^ ((r * units >> 3) & (units - 1))) << 4);
    };
    // use(i, address in the staging tile, row, element of the row) of this lane's i-th piece of a chunk: pieces side by side
    // over the lanes, whole rows one after another
    auto some_pieces = [&](auto units_tag, int first, auto many_tag, auto&& use) {
      constexpr int kBytes = sizeof(Piece), units = decltype(units_tag)::value, kEach = units * 16 / kBytes;
#pragma unroll
      for (int i = 0; i < decltype(many_tag)::value; ++i) {
        const int at = (first + i) * 32 + lane, r = at / kEach, byte = at % kEach * kBytes;
        use(i, unit_at(r, byte >> 4, units) + (byte & 15), r, byte / static_cast<int>(sizeof(T)));
      }
    };
    auto each_piece = [&](auto units_tag, auto&& use) {
      some_pieces(units_tag, 0, std::integral_constant<int, decltype(units_tag)::value * 16 / static_cast<int>(sizeof(Piece))>{}, use);
    };
    auto first_row = [&](int tile_m) { return tile_m * 256 + rank * 128 + quarter * 32; };
    // scales and bias of a tile's columns that this warp works on
    float next_row_scale = 0.0f, next_scale[kChunksAtMost], next_bias[kChunksAtMost];
    auto ask_terms = [&](const Place& at) {
      if (at.tile >= tiles) return;
      const int tile_n = at.n(), row = first_row(at.m()) + lane, n_end = min(p.n, (tile_n + 1) * bn);
      next_row_scale = row < p.m ? p.x_scales[row] : 0.0f;
#pragma unroll
      for (int q = 0; q < kChunksAtMost; ++q) {
        const int col = tile_n * bn + turn0 * 32 + q * kStep + lane;
        next_scale[q] = col < n_end ? p.w_scales[col] : 0.0f;
        next_bias[q] = col < n_end && p.bias != nullptr ? Elem<T>::load(static_cast<const T*>(p.bias) + col) : 0.0f;
      }
    };
    // kBulk: the residual's chunks in the order in which they are used, each into the staging tile that it leaves through
    Place asked_at = start;
    int asked = 0, asked_slot = 0, asked_c0 = turn0 * 32;
    const uint32_t arrivals = smem_u32(&arrived[kBulk ? warp * kTiles : 0]);
    auto ask_residual = [&]() {
      while (asked_at.tile < tiles) {
        const int col0 = asked_at.n() * bn + asked_c0;
        const bool there = asked_c0 < bn && col0 < p.n;
        if (there) {
          const uint32_t bar = arrivals + asked_slot * 8;
          mbarrier_arrive_expect_tx_if(lane == 0, bar, kStageTile);
          tma_load_2d_if(lane == 0, stage_tiles + asked_slot * kStageTile, &residual_map, bar, col0, first_row(asked_at.m()));
          ++asked;
          asked_slot = asked_slot + 1 == kTiles ? 0 : asked_slot + 1;
          asked_c0 += kStep;
          return;
        }
        asked_at.next();
        asked_c0 = turn0 * 32;
      }
    };
    const bool bulk_residual = kBulk && residual != nullptr;
    bool ok = true;
    int done = 0, chunks = 0, slot = 0;  // slot, phase: chunks % kTiles, chunks / kTiles & 1
    uint32_t phase = 0;
    if constexpr (kBulk) ask_terms(start);  // (else no registers are left for them)
    if (bulk_residual)
      for (int i = 0; i + 1 < kTiles; ++i) ask_residual();
    for (Place at = start; at.tile < tiles; ++done) {
      const int tile_m = at.m(), tile_n = at.n();
      if constexpr (!kBulk) ask_terms(at);
      at.next();
      const int acc = done & 1, row0 = first_row(tile_m);
      const int n_end = min(p.n, (tile_n + 1) * bn);
      const float row_scale = next_row_scale;
      __syncwarp();  // (the tile before is done with the terms)
#pragma unroll
      for (int q = 0; q < kChunksAtMost; ++q) {
        float* to = column_terms + q * 64 + (lane >> 1) * 4 + (lane & 1);
        to[0] = next_scale[q];
        to[2] = next_bias[q];
      }
      __syncwarp();
      if constexpr (kBulk) ask_terms(at);
      constexpr int kWords = sizeof(Piece) < 4 ? 1 : sizeof(Piece) / 4;
      uint32_t ahead[kBulk ? 1 : kUnits * 16 / sizeof(Piece) * kWords];  // the next chunk's residual
      auto fetch = [&](int c0) {
        if constexpr (!kBulk) {
          const int col0 = tile_n * bn + c0;
          if (residual == nullptr || col0 >= n_end) return;
          constexpr int kRows = 32 / (kUnits * 16 / static_cast<int>(sizeof(Piece)));  // that the lanes cover at a time
          const T* from = nullptr;
          each_piece(std::integral_constant<int, kUnits>{}, [&](int i, uint32_t, int r, int element) {
            from = i == 0 ? residual + static_cast<int64_t>(row0 + r) * p.n + col0 + element : from + kRows * static_cast<int64_t>(p.n);
            Piece value = {};
            if (row0 + r < p.m && col0 + element < n_end) value = *reinterpret_cast<const Piece*>(from);
            ahead[i] = value;
          });
        }
      };
      fetch(turn0 * 32);
      ok = ok && __all_sync(0xffffffffu, mbarrier_wait_bounded(smem_u32(&acc_full[acc]), (done >> 1) & 1, p.wait_limit));
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t t_addr = tmem_base + acc * 256 + (static_cast<uint32_t>(quarter * 32) << 16);
      // (relaxed: what has to be over are the reads of tensor memory, which the fence orders. A release would wait for the
      // stores of the tile to reach L2, 1 us of it: 16384 x 896 x 9728 144 us with it)
      auto sums_read = [&]() {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        asm volatile("{\n\t.reg .pred q;\n\tsetp.eq.s32 q, %1, 0;\n\t@q mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n\t}"
                     ::"r"(acc_empty_first + acc * 8), "r"(lane) : "memory");
      };
      uint32_t raw[32];  // kBulk: the next chunk's sums, on their way while a chunk is worked on
      if (tile_n * bn + turn0 * 32 >= n_end) sums_read();
      else if constexpr (kBulk) tmem_load_32x32_issue(t_addr + turn0 * 32, raw);
#pragma unroll 1
      for (int c0 = turn0 * 32, q = 0; c0 < bn; c0 += kStep, ++q, ++chunks) {
        const int col0 = tile_n * bn + c0;
        if (col0 >= n_end) break;  // (warp-uniform)
        if constexpr (!kBulk) tmem_load_32x32_issue(t_addr + c0, raw);
        tmem_load_wait(raw);
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = static_cast<float>(static_cast<int>(raw[i]));
        const bool more = c0 + kStep < bn && col0 + kStep < n_end;
        if (!more) sums_read();
        else if constexpr (kBulk) tmem_load_32x32_issue(t_addr + c0 + kStep, raw);
        const float4* terms = reinterpret_cast<const float4*>(column_terms + q * 64);  // two columns' scales, their bias
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float4 t = terms[i];
          scale_two(v[2 * i], v[2 * i + 1], row_scale, t);
        }
        if constexpr (kBulk) {
          stage_tile = stage_tiles + slot * kStageTile;
          if (residual != nullptr) {
            ok = __all_sync(0xffffffffu, mbarrier_wait_bounded(arrivals + slot * 8, phase, p.wait_limit));
            if (!ok) break;
          } else {
            stores_read<kTiles - 1>();  // the tile's chunk before
            __syncwarp();
          }
        } else {
          __syncwarp();  // the chunk before has been read
        }
        if (++slot == kTiles) { slot = 0; phase ^= 1; }
        // the staged rows to y: `width` columns of them exist
        auto rows_out = [&](auto units_tag, int to_col, int width) {
          if constexpr (kBulk) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            tma_store_2d_if(lane == 0 && row0 < p.m, &y_map, stage_tile, to_col, row0);
          } else {
            __syncwarp();
            T* to = nullptr;
            constexpr int kRows = 32 / (decltype(units_tag)::value * 16 / static_cast<int>(sizeof(Piece)));
            auto next_row = [&](int piece, int r, int element) {
              to = piece == 0 ? out + static_cast<int64_t>(row0 + r) * out_cols + to_col + element : to + kRows * static_cast<int64_t>(out_cols);
            };
            const bool whole = row0 + 32 <= p.m && col0 + 32 <= n_end;  // (a chunk that lies in y needs no questions)
            constexpr int kEach = decltype(units_tag)::value * 16 / static_cast<int>(sizeof(Piece));
            std::integral_constant<int, (kEach < 8 ? kEach : 8)> many;
#pragma unroll
            for (int first = 0; first < kEach; first += 8) {
              Piece values[8];
              some_pieces(units_tag, first, many, [&](int i, uint32_t from, int, int) {
                if constexpr (sizeof(Piece) == 4)
                  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(values[i]) : "r"(from));
                else
                  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(values[i]) : "r"(from));
              });
              if (whole) {
                some_pieces(units_tag, first, many, [&](int i, uint32_t, int r, int element) {
                  next_row(first + i, r, element);
                  *reinterpret_cast<Piece*>(to) = values[i];
                });
              } else {
                some_pieces(units_tag, first, many, [&](int i, uint32_t, int r, int element) {
                  next_row(first + i, r, element);
                  if (row0 + r < p.m && element < width) *reinterpret_cast<Piece*>(to) = values[i];
                });
              }
            }
          }
        };
        if (swiglu) {
          constexpr int kHalf = kUnits / 2;
#pragma unroll
          for (int unit = 0; unit < kHalf; ++unit) {
            Vec16<T> t;
#pragma unroll
            for (int e = 0; e < kVec; ++e) t.v[e] = silu_times(v[2 * (unit * kVec + e)], v[2 * (unit * kVec + e) + 1]);
            uint4 packed;
            t.store(reinterpret_cast<T*>(&packed));
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(unit_at(lane, unit, kHalf)), "r"(packed.x), "r"(packed.y),
                         "r"(packed.z), "r"(packed.w) : "memory");
          }
          rows_out(std::integral_constant<int, kHalf>{}, col0 / 2, (n_end - col0) / 2);
          continue;
        }
        if constexpr (!kBulk) {
          if (residual != nullptr) {
            each_piece(std::integral_constant<int, kUnits>{}, [&](int i, uint32_t to, int, int) {
              if constexpr (sizeof(Piece) == 4)
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(to), "r"(ahead[i]) : "memory");
              else
                asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"(static_cast<uint16_t>(ahead[i])) : "memory");
            });
            if (c0 + kStep < bn) fetch(c0 + kStep);
            __syncwarp();
          }
        }
#pragma unroll
        for (int unit = 0; unit < kUnits; ++unit) {
          Vec16<T> t;
          uint4 packed;
          if (residual != nullptr) {
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(packed.x), "=r"(packed.y), "=r"(packed.z), "=r"(packed.w)
                         : "r"(unit_at(lane, unit, kUnits)));
            t.load(reinterpret_cast<const T*>(&packed));
#pragma unroll
            for (int e = 0; e < kVec; ++e) t.v[e] += v[unit * kVec + e];
          } else {
#pragma unroll
            for (int e = 0; e < kVec; ++e) t.v[e] = v[unit * kVec + e];
          }
          t.store(reinterpret_cast<T*>(&packed));
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(unit_at(lane, unit, kUnits)), "r"(packed.x), "r"(packed.y),
                       "r"(packed.z), "r"(packed.w) : "memory");
        }
        rows_out(std::integral_constant<int, kUnits>{}, col0, n_end - col0);
        if (bulk_residual) {
          stores_read<1>();  // the chunk before this one has left its tile
          __syncwarp();
          ask_residual();
        }
      }
      if (!ok) break;
    }
    if constexpr (kBulk) {
      if (bulk_residual)  // (after a failure: copies still on their way)
        for (; chunks < asked; ++chunks) mbarrier_wait_bounded(arrivals + chunks % kTiles * 8, chunks / kTiles & 1, p.wait_limit);
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      __syncwarp();
    }
    if (!ok) failed = 1;
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  if constexpr (kSplit) {
    // ---- the slices' sums: this CTA finishes rows slice, slice + slices, ... of its half; a lane takes four columns ----
    __syncwarp();
    cluster_sync();
    const bool swiglu = p.epilogue == B200_EPILOGUE_SWIGLU;
    const int64_t out_cols = swiglu ? p.n / 2 : p.n;
    const int tile_m = start.m(), tile_n = start.n(), row0 = tile_m * 256 + rank * 128, rows = min(128, p.m - row0);
    const T* residual = static_cast<const T*>(p.residual);
    for (int unit = lane; unit < bn / 4; unit += 32) {
      const FourColumns<T> four(p, tile_n * bn + 4 * unit);
      if (four.width <= 0) break;
      for (int row = slice + warp * slices; row < rows; row += kPairThreads / 32 * slices)
        four.template finish<4>(smem_base + row * bn * 4 + ((unit ^ (row & 7)) << 4), rank, 2, slices, p.x_scales[row0 + row],
                                residual != nullptr ? residual + (row0 + row) * out_cols : nullptr,
                                static_cast<T*>(p.out) + (row0 + row) * out_cols, swiglu);
    }
    __syncwarp();
  }
  __syncthreads();
  if (threadIdx.x == 0 && failed) atomicOr(p.status, B200_STATUS_WAIT_TIMEOUT);
  cluster_sync();  // neither CTA leaves while the other may still signal it
  if (warp == kPairWarps + 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
}

// y or a residual [m, cols] in boxes of 32 rows of `width` columns, 32, 64 or 128 bytes of them, swizzled as the warps write.
template <typename T>
bool make_chunk_map(CUtensorMap* map, const void* base, int64_t m, int64_t cols, int width) {
  EncodeTiledFn encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(m)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols) * sizeof(T)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(width), 32}, element_strides[2] = {1, 1};
  const int bytes = width * static_cast<int>(sizeof(T));
  return encode(map, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), dims,
                strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                bytes == 32 ? CU_TENSOR_MAP_SWIZZLE_32B : bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// [rows, K] codes in boxes of box_rows x 128 (128-byte rows, 128B swizzle); zeros beyond both.
bool make_code_map(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int box_rows) {
  EncodeTiledFn encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(k)};
  const cuuint32_t box[2] = {kBK, static_cast<cuuint32_t>(box_rows)}, element_strides[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, element_strides,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What either kernel takes, to a few microseconds, from what was measured. Stream: a k-block 0.2 us and 0.42 more at 256 rows,
// the epilogue 2.5 us at 256 rows (256 x 18944 x 3584: 27.9 us in 112 CTAs of 37 k-blocks; 256 x 512 x 18944: 8.4 in 4) behind
// the products, and where a CTA has several tiles 4.5 us each, 7 with SwiGLU, 15 with a residual (6065 x 128 x 15736: 323 us
// there, 110 in pairs). Pair: a k-block 0.25 us at 128 columns and 0.345 at 256 (1407 x 3488 x 25: 10.6 in 28), the epilogue
// 2.8 us a tile beside the products of the next; 4 where rows of y do not start on multiples of 16 bytes, and 2.5 for the last
// tile (910 x 288 x 577 fp32: 9.6 us, 4.5 in the stream kernel); slices of K 6 us at 256 columns (256 x 18944 x 3584 22 us in four,
// 512 x 18944 x 3584 36 in two, 40 in one). Wide tiles need fewer bytes for a product and narrow ones fewer rounds: 5632 x 1280 x
// 18432 97 us at 256 columns, 127 at 128; 4096 x 18944 x 3584 194 at 256, 217 at 160.
// Slices of K are clusters, and more of them than the GPU holds at once cost a second round: 256 x 18944 x 3584 in 16 clusters of
// 8 37 us, in 14 22; 8 x 3584 x 4608 in 36 of 4 9.8, in 36 of 2 6.3, in 36 of 3 5.6.
constexpr double kStreamEpilogue[] = {4.5, 15.0, 7.0};  // none, residual, SwiGLU
struct StreamPlan { int cols, chunks, slices; double us; };
StreamPlan plan_stream(int64_t m, int64_t k, int64_t n, int epilogue) {
  const int64_t tiles = ceil_div(n, 128), blocks = ceil_div(k, kBK);
  StreamPlan best = {0, 0, 0, 1e30};
  for (int64_t chunks = ceil_div(m, kRowsAtMost); chunks <= std::max<int64_t>(16, ceil_div(m, kRowsAtMost)); ++chunks) {
    const int64_t cols = ceil_div(ceil_div(m, chunks), 16) * 16, units = tiles * ceil_div(m, cols);
    // slices of K that fill the GPU where the tiles do not, two k-blocks a slice at least
    int64_t slices = 8;
    while (slices > 1 && (units > clusters_at_once(1, slices) || blocks < 2 * slices)) --slices;
    const double share = cols / 256.0;
    const int64_t across = std::max<int64_t>(1, kNumSMs / chunks), rounds = slices > 1 ? 1 : ceil_div(tiles, across);
    const double products = ceil_div(blocks, slices) * (0.2 + 0.42 * share);
    const double us = 4.0 + products + 2.5 * share + (rounds - 1) * std::max(products, kStreamEpilogue[epilogue] * share);
    if (us < 0.9 * best.us) best = {static_cast<int>(cols), static_cast<int>(ceil_div(m, cols)), static_cast<int>(slices), us};
    if (cols == 16) break;  // (no chunk is smaller)
  }
  return best;
}
struct PairPlan { int cols, slices; double us; };  // whole_rows: rows of y start on multiples of 16 bytes
PairPlan plan_pair(int64_t m, int64_t k, int64_t n, bool whole_rows) {
  const int64_t tiles_m = ceil_div(m, 256), blocks = ceil_div(k, kBK);
  PairPlan best = {0, 0, 1e30};
  for (int bn = 256; bn >= 128; bn -= 32) {
    const int64_t tiles = tiles_m * ceil_div(n, bn);
    const double share = bn / 256.0, block = 0.155 + 0.19 * share;
    // slices of K where the tiles leave pairs idle: clusters of 4, 6 or 8 CTAs
    for (int64_t slices = 1; slices <= 4 && (slices == 1 || (tiles <= clusters_at_once(1, 2 * slices) && blocks >= 4 * slices)); ++slices) {
      const int64_t rounds = slices > 1 ? 1 : ceil_div(tiles, kNumSMs / 2);
      const double products = ceil_div(blocks, slices) * block;
      const double us = 3.5 + std::max(products, 2.0) + (rounds - 1) * std::max(products, (whole_rows ? 2.8 : 4.0) * share) +
                        (slices > 1 ? 1.5 + 4.5 * share : whole_rows ? 0.0 : 2.5 * std::min<int64_t>(n, bn) / 256.0);
      if (us < 0.99 * best.us) best = {bn, static_cast<int>(slices), us};
    }
  }
  return best;
}

template <typename T>
int launch_stream(Int8LinearParams p, const StreamPlan& plan, const void* x, const void* w, cudaStream_t stream) {
  p.cols = plan.cols;
  p.slices = plan.slices;
  p.stages = std::min(10, kRingBytes / ((128 + p.cols) * 128));
  // (a decode step of 6 layers of 896, 64 rows: 315 -> 304 us; 4 layers of 3584: 8 rows 393 -> 378, 64 494 -> 484, 256 868 -> 871)
  constexpr int kAhead = B200_LAUNCH_PROGRAMMATIC | B200_LAUNCH_CONSTANT_WEIGHTS;
  p.ahead = (launch_mode() & kAhead) == kAhead && p.cols <= 128;
  CUtensorMap w_map, x_map;
  if (!make_code_map(&w_map, w, p.n, p.k, 128) || !make_code_map(&x_map, x, p.m, p.k, p.cols)) return B200_ERR_UNSUPPORTED;
  const int64_t tiles = ceil_div(p.n, 128);
  // (whole tiles in turn: chunks side by side share the SMs)
  const int64_t across = std::max<int64_t>(1, kNumSMs / plan.chunks);
  const dim3 grid(static_cast<unsigned>(p.slices > 1 ? tiles * p.slices : std::min(across, tiles)), static_cast<unsigned>(plan.chunks));
  auto kernel = linear_int8_stream_kernel<T>;
  static_assert(tensor_memory_fits(512, kRingBytes), "tensor memory under programmatic launches");
  static std::atomic<uint64_t> allowed{0};
  if (!allow_shared_memory(kernel, kRingBytes, allowed)) return B200_ERR_LAUNCH;
  return launch_chained_cluster(kernel, grid, dim3(kThreads), kRingBytes, stream, static_cast<unsigned>(p.slices), p,
                                w_map, x_map) == cudaSuccess ? launch_status() : B200_ERR_LAUNCH;
}

template <typename T>
int launch_pair(Int8LinearParams p, const PairPlan& plan, const void* x, const void* w, cudaStream_t stream) {
  p.cols = plan.cols;
  p.slices = plan.slices;
  p.n_fastest = p.n <= p.m;
  CUtensorMap x_map, w_map, y_map = {}, residual_map = {};
  if (!make_code_map(&x_map, x, p.m, p.k, 128) || !make_code_map(&w_map, w, p.n, p.k, p.cols / 2)) return B200_ERR_UNSUPPORTED;
  const int64_t tiles = ceil_div(p.m, 256) * ceil_div(p.n, p.cols);
  const unsigned pairs = static_cast<unsigned>(plan.slices > 1 ? tiles * plan.slices : std::min<int64_t>(kNumSMs / 2, tiles));
  // what every row of y and of the residual starts on a multiple of
  const uint64_t starts = static_cast<uint64_t>(p.epilogue == B200_EPILOGUE_SWIGLU ? p.n / 2 : p.n) * sizeof(T) |
                          reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.residual);
  const auto launch = [&](auto piece, auto split) {
    using Piece = decltype(piece);
    auto kernel = linear_int8_pair_kernel<T, Piece, decltype(split)::value>;
    constexpr int kSmem = pair_smem<T, Piece>();
    static_assert(tensor_memory_fits(512, kSmem) && kSmem + 1024 <= 227 * 1024, "tensor memory under programmatic launches");
    static std::atomic<uint64_t> allowed{0};
    if (!allow_shared_memory(kernel, kSmem, allowed)) return B200_ERR_LAUNCH;
    return launch_chained_cluster(kernel, dim3(2 * pairs), dim3(kPairThreads), kSmem, stream, 2u * static_cast<unsigned>(plan.slices), p,
                                  x_map, w_map, y_map, residual_map) == cudaSuccess ? launch_status() : B200_ERR_LAUNCH;
  };
  if (plan.slices > 1) return launch(uint32_t{}, std::true_type{});  // (rows of any alignment)
  if (starts % 16 == 0) {
    const bool swiglu = p.epilogue == B200_EPILOGUE_SWIGLU;
    if (!make_chunk_map<T>(&y_map, p.out, p.m, swiglu ? p.n / 2 : p.n, swiglu ? 16 : 32) ||
        (p.residual && !make_chunk_map<T>(&residual_map, p.residual, p.m, p.n, 32)))
      return B200_ERR_UNSUPPORTED;
    return launch(uint4{}, std::false_type{});
  }
  if constexpr (sizeof(T) == 2) {
    if (starts % 4 != 0) return launch(uint16_t{}, std::false_type{});
  }
  return launch(uint32_t{}, std::false_type{});
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_linear_int8(const b200_linear_int8_call* call, void* stream) {
  if (!call) return B200_ERR_BAD_ARGUMENT;
  const b200_linear_int8_call& c = *call;
  const int dtype = static_cast<int>(c.dtype);
  const int64_t m = c.m, k = c.k, n = c.n;
  if (!c.x || !c.x_scales || !c.weight || !c.weight_scales || !c.output || !c.status || m < 0 || k <= 0 || n <= 0 ||
      c.dtype != dtype || !known_dtype(dtype) || c.epilogue < B200_EPILOGUE_NONE || c.epilogue > B200_EPILOGUE_SWIGLU ||
      (c.epilogue == B200_EPILOGUE_RESIDUAL) != (c.residual != nullptr))
    return B200_ERR_BAD_ARGUMENT;
  if (k % 16 != 0 || (c.epilogue == B200_EPILOGUE_SWIGLU && n % 2 != 0)) return B200_ERR_UNSUPPORTED;
  if (!aligned16(c.x) || !aligned16(c.weight)) return B200_ERR_ALIGNMENT;
  if (k > kMaxK || m > (1 << 22) || n > (1 << 22)) return B200_ERR_TOO_LARGE;
  if (m == 0) return B200_OK;
  Int8LinearParams p = {};
  p.x_scales = c.x_scales; p.w_scales = c.weight_scales;
  p.bias = c.bias; p.residual = c.residual; p.out = c.output; p.status = c.status;
  p.m = static_cast<int>(m); p.k = static_cast<int>(k); p.n = static_cast<int>(n); p.epilogue = static_cast<int>(c.epilogue);
  p.wait_limit = wait_limit(); p.drop_loads = drop_loads();
  const StreamPlan stream_plan = plan_stream(m, k, n, p.epilogue);
  const int64_t row_bytes = (p.epilogue == B200_EPILOGUE_SWIGLU ? n / 2 : n) * (dtype == B200_F32 ? 4 : 2);
  const PairPlan pair_plan = m > kRowsAtMost / 2 ? plan_pair(m, k, n, row_bytes % 16 == 0) : PairPlan{0, 0, 1e30};
  // (beyond 256 rows the stream kernel reads the weight more than once, which other work on the GPU would feel)
  const bool streamed = stream_plan.us < (m <= kRowsAtMost ? 1.0 : 0.95) * pair_plan.us && stream_plan.chunks <= 64;
  int code = B200_ERR_UNSUPPORTED;
  with_element_type(dtype, [&](auto tag) {
    using T = typename decltype(tag)::type;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    code = streamed ? launch_stream<T>(p, stream_plan, c.x, c.weight, s) : launch_pair<T>(p, pair_plan, c.x, c.weight, s);
  });
  return code;
}
