// Rows quantised to 8-bit integers with one scale each: plain, or behind a residual sum and an RMS norm.
//
//     r = round(x + residual),  y_i = r_i w_i / sqrt(mean(r^2) + eps),  scale = max|y| / 127,  code_i = round(y_i / scale).
// The row factor 1 / sqrt(..) is common to max|y| and to every y_i, so code_i = round(r_i w_i * (127 / max|r w|)) does not
// need it: the sum of squares and the maximum come out of ONE pass and one reduction, and only the scale carries the factor.
// A row is read once, held in registers, and written as codes (and as r where there is a residual).
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

// One row per CTA. kVector: rows in 16-byte loads, up to kKept of them a thread in registers; what is longer is read again.
template <typename T, bool kVector, int kKept>
__global__ void quantize_rows_kernel(const QuantParams p) {
  constexpr int per = kVector ? Elem<T>::kPerVec : 1;
  grid_launch_dependents();
  __shared__ float parts[2][32];
  const int threads = blockDim.x, warps = threads >> 5;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const T* residual = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_stride : nullptr;
  const T* weight = static_cast<const T*>(p.weight);
  T* sum = p.sum ? static_cast<T*>(p.sum) + row * p.hidden : nullptr;
  int8_t* codes = p.codes + row * p.hidden;
  const int64_t items = p.hidden / per;
  grid_dependency_wait();

  auto load = [&](const T* from, int64_t i, float (&v)[per]) {
    if constexpr (kVector) {
      Vec16<T> t;
      t.load(from + i * per);
#pragma unroll
      for (int e = 0; e < per; ++e) v[e] = t.v[e];
    } else {
      v[0] = Elem<T>::load(from + i);
    }
  };
  // r of item i, times the weight; the sum of squares of r on the way
  auto row_item = [&](int64_t i, bool first, float& squares, float (&y)[per]) {
    load(x, i, y);
    if (residual != nullptr) {
      if (first) {
        float other[per];
        load(residual, i, other);
#pragma unroll
        for (int e = 0; e < per; ++e) y[e] = Elem<T>::round(__fadd_rn(y[e], other[e]));
        if constexpr (kVector) {
          Vec16<T> t;
#pragma unroll
          for (int e = 0; e < per; ++e) t.v[e] = y[e];
          t.store(sum + i * per);
        } else {
          Elem<T>::store(sum + i, y[0]);
        }
      } else {
        load(sum, i, y);  // (this thread's own store)
      }
    }
#pragma unroll
    for (int e = 0; e < per; ++e) squares = fmaf(y[e], y[e], squares);
    if (weight != nullptr) {
      float w[per];
      load(weight, i, w);
#pragma unroll
      for (int e = 0; e < per; ++e) y[e] *= w[e];
    }
  };
  float kept[kKept][per];
  float squares = 0.0f, most = 0.0f;
  bool nan = false;
  auto look = [&](const float (&y)[per]) {
#pragma unroll
    for (int e = 0; e < per; ++e) {
      most = fmaxf(most, fabsf(y[e]));
      nan = nan || y[e] != y[e];
    }
  };
#pragma unroll
  for (int j = 0; j < kKept; ++j) {
    const int64_t i = threadIdx.x + static_cast<int64_t>(j) * threads;
#pragma unroll
    for (int e = 0; e < per; ++e) kept[j][e] = 0.0f;
    if (i < items) row_item(i, true, squares, kept[j]);
    look(kept[j]);
  }
  for (int64_t i = threadIdx.x + static_cast<int64_t>(kKept) * threads; i < items; i += threads) {
    float y[per];
    row_item(i, true, squares, y);
    look(y);
  }
  if (nan) most = INFINITY;  // (a row with NaN: the maximum alone would drop it)
  squares = warp_sum(squares);
  most = warp_max(most);
  if ((threadIdx.x & 31) == 0) {
    parts[0][threadIdx.x >> 5] = squares;
    parts[1][threadIdx.x >> 5] = most;
  }
  __syncthreads();
  squares = 0.0f;
  for (int w = 0; w < warps; ++w) {
    squares += parts[0][w];
    most = fmaxf(most, parts[1][w]);
  }
  const bool fine = most < INFINITY;
  const float inverse = fine && most > 0.0f ? fminf(__fdiv_rn(127.0f, most), 3.0e38f) : 0.0f;
  if (threadIdx.x == 0) {
    float scale = most * (1.0f / 127.0f);
    if (weight != nullptr && most > 0.0f) scale *= rsqrtf(squares / static_cast<float>(p.hidden) + p.epsilon);
    p.scales[row] = fine ? scale : NAN;
  }
  auto put = [&](const float (&y)[per], int64_t i) {
    if constexpr (kVector) {
      uint32_t packed[per / 4];
#pragma unroll
      for (int q = 0; q < per / 4; ++q) {
        packed[q] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) packed[q] |= (fine ? Int8Code::encode(y[4 * q + e] * inverse) : 0u) << (8 * e);
      }
      if constexpr (per == 8) *reinterpret_cast<uint2*>(codes + i * 8) = make_uint2(packed[0], packed[1]);
      else *reinterpret_cast<uint32_t*>(codes + i * 4) = packed[0];
    } else {
      codes[i] = fine ? static_cast<int8_t>(Int8Code::encode(y[0] * inverse)) : int8_t(0);
    }
  };
#pragma unroll
  for (int j = 0; j < kKept; ++j) {
    const int64_t i = threadIdx.x + static_cast<int64_t>(j) * threads;
    if (i < items) put(kept[j], i);
  }
  for (int64_t i = threadIdx.x + static_cast<int64_t>(kKept) * threads; i < items; i += threads) {
    float y[per], unused = 0.0f;
    row_item(i, false, unused, y);
    put(y, i);
  }
}

template <typename T>
cudaError_t quantize_typed(const QuantParams& p, cudaStream_t stream) {
  constexpr int per = Elem<T>::kPerVec;
  const bool vector = p.hidden % per == 0 && p.x_stride % per == 0 && aligned16(p.x) && aligned16(p.codes) &&
                      (!p.weight || aligned16(p.weight)) &&
                      (!p.residual || (aligned16(p.residual) && p.residual_stride % per == 0 && aligned16(p.sum)));
  const int64_t items = vector ? p.hidden / per : p.hidden;
  const int threads = static_cast<int>(items >= 512 ? 512 : ceil_div(items, 32) * 32);
  const dim3 grid(static_cast<unsigned>(p.rows)), block(static_cast<unsigned>(threads));
  return vector ? launch_chained(quantize_rows_kernel<T, true, 4>, grid, block, 0, stream, p)
                : launch_chained(quantize_rows_kernel<T, false, 8>, grid, block, 0, stream, p);
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
  if (c.rows > 0x7fffffff) return B200_ERR_TOO_LARGE;
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
