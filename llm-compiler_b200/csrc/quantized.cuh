// Shared pieces of the operators in 8 bits: code types, their largest values, conversions.
#pragma once

#include <cuda_fp8.h>

#include <atomic>

#include "common.cuh"

namespace b200 {

// Codes of a cache: signed integers or e4m3. Both formats stand for code * scale.
struct Int8Code {
  static constexpr float kTop = 127.0f;
  // Nearest integer, ties to even, of a value that the scale brings to [-127, 127]; infinities saturate, NaN gives 0.
  __device__ static uint32_t encode(float v) {
    return static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(v == v ? v : 0.0f, -kTop), kTop))) & 0xffu;
  }
  __device__ static float decode(uint32_t code) { return static_cast<float>(static_cast<int8_t>(code)); }
  // Four codes of finite values that the scale brings to [-127.4, 127.4]: v + 1.5 * 2^23 rounds to the nearest integer, ties
  // to even, and leaves it in the low byte.
  __device__ static uint32_t encode_four(float a, float b, float c, float d) {
    const auto byte = [](float v) { return __float_as_uint(__fadd_rn(v, 12582912.0f)); };
    return __byte_perm(__byte_perm(byte(a), byte(b), 0x0040), __byte_perm(byte(c), byte(d), 0x0040), 0x5410);
  }
};
struct E4m3Code {
  static constexpr float kTop = 448.0f;
  // Nearest e4m3 number, ties to even; what is beyond 448 saturates, NaN stays NaN.
  __device__ static uint32_t encode(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
  __device__ static float decode(uint32_t code) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(code), __NV_E4M3)));
  }
  __device__ static uint32_t encode_four(float a, float b, float c, float d) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) |
           (static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3)) << 16);
  }
};

constexpr float kSmallestScale = 1.17549435e-38f;  // the smallest normal number: 1 / scale stays finite

__device__ __forceinline__ bool is_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

// Clusters of `size` CTAs that the GPU holds at once, with 4, 3 or 1 CTAs an SM: fewer than its CTAs divided by `size`, for a
// cluster stays within a GPC. (As counted on a B200; where one holds fewer, the last few wait for a second round.)
inline int64_t clusters_at_once(int64_t resident, int64_t size) {
  constexpr int kOfFour[] = {592, 296, 187, 142, 112, 93, 78, 71}, kOfThree[] = {444, 222, 142, 104, 82, 71, 56, 48},
                kOfOne[] = {148, 74, 45, 33, 26, 22, 15, 15};
  return (resident == 4 ? kOfFour : resident == 3 ? kOfThree : kOfOne)[size - 1];
}

// Opt-in to `bytes` of dynamic shared memory of a kernel, asked of the runtime once per device (a third of a microsecond a
// call otherwise). `done`: a bit per device, of this kernel and size.
template <typename Kernel>
inline bool allow_shared_memory(Kernel kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return false;
  const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
  if ((done.load(std::memory_order_relaxed) & bit) != 0) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

}  // namespace b200
