// Rows quantised to 8-bit integers with one scale each: plain, or behind a residual sum and an RMS norm.
//
//     r = round(x + residual),  y_i = r_i w_i / sqrt(mean(r^2) + eps),  scale = max|y| / 127,  code_i = round(y_i / scale).
// The row factor 1 / sqrt(..) is common to max|y| and to every y_i, so code_i = round(r_i w_i * (127 / max|r w|)) does not
// need it: the sum of squares and the maximum come out of ONE pass and one reduction, and only the scale carries the factor.
// max|r w| / 127 is at least the smallest normal number (as in a cache's store): below it neither it nor its inverse would
// keep their bits, and such a row's codes stay below 127 instead.
// A row is read once, held in registers, and written as codes (and as r where there is a residual).
#include <algorithm>
#include <type_traits>

#include "quantized.cuh"

namespace b200 {
namespace {

struct QuantParams {
  const void* x;
  const void* residual;  // NULL: r = x
  const void* weight;    // NULL: no norm, y = r
  void* sum;             // where r goes (residual only)
  int8_t* codes;
  float* scales;
  int64_t rows, hidden, x_stride, residual_stride;
  float epsilon;
};

// One row per CTA. kVector: rows in 16-byte loads, kKept of them a thread in registers; what is longer is read again.
// What bounds it is memory: a thread asks for all it keeps of x, the residual and the weight before it uses any (four loads
// of each at 512 bytes a warp; 16384 x 3584 bf16 with a residual: 168 us with one each, 61 with four, 6.7 TB/s). Without
// a residual a CTA takes rows in turn and asks for the next one before it reduces this one (16384 x 3584: 36.8 -> 35.6 us, 4.9
// TB/s; 2048 x 16384 fp16 30.3 -> 21.4; what is left are the registers that hold a row twice). A code is the low byte of
// y * inverse + 1.5 * 2^23, which rounds to the nearest integer, ties to even: one operation instead of clamps and a
// conversion (|y * inverse| <= 127 (1 + 2^-22) by construction).
__device__ __forceinline__ float max_or_nan(float a, float b) {  // (NaN if either is)
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t code_of(float y, float inverse) {  // in the low byte
  return __float_as_uint(fmaf(y, inverse, 12582912.0f));
}
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d, float inverse) {
  const uint32_t ab = __byte_perm(code_of(a, inverse), code_of(b, inverse), 0x0040);
  const uint32_t cd = __byte_perm(code_of(c, inverse), code_of(d, inverse), 0x0040);
  return __byte_perm(ab, cd, 0x5410);
}

template <typename T, bool kVector, bool kResidual, bool kNorm, int kKept>
__global__ void __launch_bounds__(512) quantize_rows_kernel(const QuantParams p) {
  constexpr int per = kVector ? Elem<T>::kPerVec : 1;
  grid_launch_dependents();
  constexpr bool kLoop = kVector && !kResidual;
  __shared__ float parts[2][2][16];
  const int threads = blockDim.x, warps = threads >> 5;
  int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const T* residual = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_stride : nullptr;
  const T* weight = static_cast<const T*>(p.weight);
  T* sum = p.sum ? static_cast<T*>(p.sum) + row * p.hidden : nullptr;
  int8_t* codes = p.codes + row * p.hidden;
  const int items = static_cast<int>(p.hidden / per);
  grid_dependency_wait();

  struct Item { T v[per]; };  // as loaded
  auto load = [&](const T* from, int i, Item& item) {
    if constexpr (kVector) *reinterpret_cast<uint4*>(&item) = *(reinterpret_cast<const uint4*>(from) + i);
    else item.v[0] = from[i];
  };
  auto values = [&](const Item& item, float (&v)[per]) {
    if constexpr (kVector) {
      Vec16<T> t;
      t.load(item.v);
#pragma unroll
      for (int e = 0; e < per; ++e) v[e] = t.v[e];
    } else {
      v[0] = Elem<T>::load(item.v);
    }
  };
  // r (stored where there is a residual) times the weight; its squares and its largest magnitude on the way
  float squares, most;
  auto weighted = [&](const Item& w, float (&y)[per]) {
    if constexpr (kNorm) {
      float f[per];
      values(w, f);
#pragma unroll
      for (int e = 0; e < per; ++e) y[e] *= f[e];
    }
  };
  auto work = [&](int i, Item& in, const Item& other, const Item& w, float (&y)[per]) {
    values(in, y);
    if constexpr (kResidual) {
      float r[per];
      values(other, r);
#pragma unroll
      for (int e = 0; e < per; ++e) y[e] = Elem<T>::round(__fadd_rn(y[e], r[e]));
      if constexpr (kVector) {
        Vec16<T> t;
#pragma unroll
        for (int e = 0; e < per; ++e) t.v[e] = y[e];
        t.store(in.v);
        *reinterpret_cast<uint4*>(sum + i * per) = *reinterpret_cast<const uint4*>(&in);
      } else {
        Elem<T>::store(in.v, y[0]);
        sum[i] = in.v[0];
      }
    }
#pragma unroll
    for (int e = 0; e < per; ++e)
      if constexpr (kNorm) squares = fmaf(y[e], y[e], squares);
    weighted(w, y);
#pragma unroll
    for (int e = 0; e < per; ++e) most = max_or_nan(most, fabsf(y[e]));
  };
  // What a thread keeps. With a residual r, as narrow as it came (y is one product away): registers for more CTAs, which
  // wait for three operands (16384 x 3584: 67 us with y kept, 61 with r). Without one y: there the instructions count
  // (37 us with y kept, 40 with r, 47 with two floats an instruction).
  constexpr bool kNarrow = kResidual && per == 8;
  Item in[kKept], other[kKept], weights[kKept];
  auto load_kept = [&](const T* from, Item (&items_of)[kKept]) {
#pragma unroll
    for (int j = 0; j < kKept; ++j) {
      const int i = threadIdx.x + j * threads;
      if (i < items) load(from, i, items_of[j]);
    }
  };
  load_kept(x, in);
  if constexpr (kResidual) load_kept(residual, other);
  if constexpr (kNorm) load_kept(weight, weights);
  for (int turn = 0;; turn ^= 1) {
    squares = most = 0.0f;
    float kept[kNarrow ? 1 : kKept][per];
#pragma unroll
    for (int j = 0; j < kKept; ++j) {
      const int i = threadIdx.x + j * threads;
      if (i < items) work(i, in[j], other[j], weights[j], kept[kNarrow ? 0 : j]);
    }
    if constexpr (kLoop)
      if (row + gridDim.x < p.rows) load_kept(x + gridDim.x * p.x_stride, in);
    for (int i = threadIdx.x + kKept * threads; i < items; i += threads) {
      Item more, other, w;
      load(x, i, more);
      if constexpr (kResidual) load(residual, i, other);
      if constexpr (kNorm) load(weight, i, w);
      float y[per];
      work(i, more, other, w, y);
    }
    squares = warp_sum(squares);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max_or_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (warps > 1) {
      if ((threadIdx.x & 31) == 0) {
        parts[turn][0][threadIdx.x >> 5] = squares;
        parts[turn][1][threadIdx.x >> 5] = most;
      }
      __syncthreads();
      squares = 0.0f;
      for (int w = 0; w < warps; ++w) {
        squares += parts[turn][0][w];
        most = max_or_nan(most, parts[turn][1][w]);
      }
    }
    const bool fine = most < INFINITY;
    const float inverse = fine && most > 0.0f ? fminf(__fdiv_rn(127.0f, most), 1.0f / kSmallestScale) : 0.0f;
    if (threadIdx.x == 0) {
      float scale = most > 0.0f ? fmaxf(most * (1.0f / 127.0f), kSmallestScale) : 0.0f;
      if (kNorm && most > 0.0f) scale *= rsqrtf(squares / static_cast<float>(p.hidden) + p.epsilon);
      p.scales[row] = fine ? scale : NAN;
    }
    auto put = [&](const float (&y)[per], int i) {
      if constexpr (kVector) {
        uint32_t packed[per / 4];
#pragma unroll
        for (int q = 0; q < per / 4; ++q)
          packed[q] = fine ? four_codes(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3], inverse) : 0u;
        if constexpr (per == 8) *reinterpret_cast<uint2*>(codes + i * 8) = make_uint2(packed[0], packed[1]);
        else *reinterpret_cast<uint32_t*>(codes + i * 4) = packed[0];
      } else {
        codes[i] = fine ? static_cast<int8_t>(code_of(y[0], inverse)) : int8_t(0);
      }
    };
    auto put_again = [&](const Item& r, int i) {
      float y[per];
      Item w;
      values(r, y);
      if constexpr (kNorm) load(weight, i, w);
      weighted(w, y);
      put(y, i);
    };
#pragma unroll
    for (int j = 0; j < kKept; ++j) {
      const int i = threadIdx.x + j * threads;
      if (i < items) {
        if constexpr (kNarrow) put_again(in[j], i);
        else put(kept[j], i);
      }
    }
    for (int i = threadIdx.x + kKept * threads; i < items; i += threads) {
      Item r;
      load(kResidual ? sum : x, i, r);  // (this thread's own store)
      put_again(r, i);
    }
    row += gridDim.x;
    if (!kLoop || row >= p.rows) return;
    x += gridDim.x * p.x_stride;
    codes += gridDim.x * p.hidden;
  }
}

template <typename T>
cudaError_t quantize_typed(const QuantParams& p, cudaStream_t stream) {
  constexpr int per = Elem<T>::kPerVec;
  const bool vector = p.hidden % per == 0 && p.x_stride % per == 0 && aligned16(p.x) && aligned16(p.codes) &&
                      (!p.weight || aligned16(p.weight)) &&
                      (!p.residual || (aligned16(p.residual) && p.residual_stride % per == 0 && aligned16(p.sum)));
  const int64_t items = vector ? p.hidden / per : p.hidden;
  // A thread keeps four loads (of 16 bytes, or eight elements); with few rows there are threads to spare, and one each is
  // over sooner.
  const int64_t each = p.rows > 2 * kNumSMs ? (vector ? 4 : 8) : 1;
  const int threads = static_cast<int>(std::min<int64_t>(512, ceil_div(ceil_div(items, each), 32) * 32));
  const dim3 block(static_cast<unsigned>(threads));
  const auto launch = [&](auto with_residual, auto with_norm) {
    constexpr bool kResidual = decltype(with_residual)::value, kNorm = decltype(with_norm)::value;
    dim3 grid(static_cast<unsigned>(p.rows));
    if (!vector) return launch_chained(quantize_rows_kernel<T, false, kResidual, kNorm, 8>, grid, block, 0, stream, p);
    auto kernel = quantize_rows_kernel<T, true, kResidual, kNorm, 4>;
    if (!kResidual && p.rows > 2 * kNumSMs) {  // CTAs that take rows in turn: as many as there is room for
      int resident = 0;
      const cudaError_t error = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, threads, 0);
      if (error != cudaSuccess) return error;
      grid.x = static_cast<unsigned>(std::min<int64_t>(p.rows, static_cast<int64_t>(kNumSMs) * std::max(resident, 1)));
    }
    return launch_chained(kernel, grid, block, 0, stream, p);
  };
  if (p.residual != nullptr)
    return p.weight != nullptr ? launch(std::true_type{}, std::true_type{}) : launch(std::true_type{}, std::false_type{});
  return p.weight != nullptr ? launch(std::false_type{}, std::true_type{}) : launch(std::false_type{}, std::false_type{});
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_quantize_rows_int8(const b200_quantize_rows_call* call, void* stream) {
  if (!call) return B200_ERR_BAD_ARGUMENT;
  const b200_quantize_rows_call& c = *call;
  const int dtype = static_cast<int>(c.dtype);
  if (!c.input || !c.codes || !c.scales || c.rows < 0 || c.hidden <= 0 || c.input_row_stride < c.hidden ||
      (c.residual && (!c.sum || c.residual_row_stride < c.hidden)) || c.dtype != dtype || !known_dtype(dtype))
    return B200_ERR_BAD_ARGUMENT;
  if (c.rows > 0x7fffffff || c.hidden > (1 << 30)) return B200_ERR_TOO_LARGE;
  if (c.rows == 0) return B200_OK;
  QuantParams p = {};
  p.x = c.input; p.residual = c.residual; p.weight = c.norm_weight; p.sum = c.residual ? c.sum : nullptr;
  p.codes = static_cast<int8_t*>(c.codes); p.scales = c.scales;
  p.rows = c.rows; p.hidden = c.hidden; p.x_stride = c.input_row_stride; p.residual_stride = c.residual_row_stride;
  p.epsilon = static_cast<float>(c.epsilon);
  cudaError_t error = cudaSuccess;
  with_element_type(dtype, [&](auto tag) {
    error = quantize_typed<typename decltype(tag)::type>(p, static_cast<cudaStream_t>(stream));
  });
  return error == cudaSuccess ? launch_status() : B200_ERR_LAUNCH;
}
