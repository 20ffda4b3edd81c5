// Projections in 8-bit integers: y = (c_x . c_w) s_x s_w + bias, then SwiGLU or a residual, rounded once.
//
// c_x [M, K] and c_w [N, K] are codes with a scale per row (token) and per output column; their products are summed in
// 32-bit integers, which is exact, so a result does not depend on the order or the split of the sum. K is at most
// 131056: 131056 * 128 * 128 is below 2^31.
#include "quantized.cuh"

namespace b200 {
namespace {

constexpr int kMaxK = 131056;

struct Int8LinearParams {
  const int8_t* x;
  const float* x_scales;
  const int8_t* w;
  const float* w_scales;
  const void* bias;
  const void* residual;
  void* out;
  int32_t* status;
  int m, k, n, epilogue;
};

// 64 x 64 outputs a CTA of 256 threads, 4 x 4 each, K in steps of 64 codes through shared memory.
template <typename T>
__global__ void __launch_bounds__(256) linear_int8_kernel(const Int8LinearParams p) {
  __shared__ uint32_t xs[64][17], ws[64][17];
  grid_launch_dependents();
  grid_dependency_wait();
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int n0 = blockIdx.x * 64, m0 = blockIdx.y * 64;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < p.k; k0 += 64) {
    const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;  // K is a multiple of 16
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    const uint4 a = m0 + r < p.m && k0 + c < p.k
        ? *reinterpret_cast<const uint4*>(p.x + static_cast<int64_t>(m0 + r) * p.k + k0 + c) : zero;
    const uint4 b = n0 + r < p.n && k0 + c < p.k
        ? *reinterpret_cast<const uint4*>(p.w + static_cast<int64_t>(n0 + r) * p.k + k0 + c) : zero;
    __syncthreads();
    xs[r][c / 4] = a.x; xs[r][c / 4 + 1] = a.y; xs[r][c / 4 + 2] = a.z; xs[r][c / 4 + 3] = a.w;
    ws[r][c / 4] = b.x; ws[r][c / 4 + 1] = b.y; ws[r][c / 4 + 2] = b.z; ws[r][c / 4 + 3] = b.w;
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 16; ++kk) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __dp4a(static_cast<int>(xs[ty * 4 + i][kk]), static_cast<int>(ws[tx * 4 + j][kk]), acc[i][j]);
    }
  }
  const bool swiglu = p.epilogue == B200_EPILOGUE_SWIGLU;
  const int out_cols = swiglu ? p.n / 2 : p.n;
  for (int i = 0; i < 4; ++i) {
    const int row = m0 + ty * 4 + i;
    if (row >= p.m) break;
    float y[4];
    for (int j = 0; j < 4; ++j) {
      const int col = n0 + tx * 4 + j;
      y[j] = 0.0f;
      if (col >= p.n) continue;
      y[j] = static_cast<float>(acc[i][j]) * p.x_scales[row] * p.w_scales[col];
      if (p.bias) y[j] += Elem<T>::load(static_cast<const T*>(p.bias) + col);
    }
    for (int j = 0; j < 4; ++j) {
      const int col = n0 + tx * 4 + j;
      if (col >= p.n) continue;
      T* out = static_cast<T*>(p.out) + static_cast<int64_t>(row) * out_cols;
      if (swiglu) {
        if (j % 2 == 0) Elem<T>::store(out + col / 2, y[j] / (1.0f + expf(-y[j])) * y[j + 1]);
      } else {
        const float more = p.epilogue == B200_EPILOGUE_RESIDUAL
            ? Elem<T>::load(static_cast<const T*>(p.residual) + static_cast<int64_t>(row) * p.n + col) : 0.0f;
        Elem<T>::store(out + col, y[j] + more);
      }
    }
  }
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_linear_int8(const void* x, const float* x_scales, const void* weight, const float* weight_scales,
                                const void* bias, const void* residual, void* output, int64_t m, int64_t k, int64_t n,
                                int dtype, int epilogue, int32_t* status, void* stream) {
  if (!x || !x_scales || !weight || !weight_scales || !output || !status || m < 0 || k <= 0 || n <= 0 || !known_dtype(dtype) ||
      epilogue < B200_EPILOGUE_NONE || epilogue > B200_EPILOGUE_SWIGLU ||
      (epilogue == B200_EPILOGUE_RESIDUAL) != (residual != nullptr))
    return B200_ERR_BAD_ARGUMENT;
  if (k % 16 != 0 || (epilogue == B200_EPILOGUE_SWIGLU && n % 2 != 0)) return B200_ERR_UNSUPPORTED;
  if (!aligned16(x) || !aligned16(weight)) return B200_ERR_ALIGNMENT;
  if (k > kMaxK || m > (1 << 22) || n > (1 << 22)) return B200_ERR_TOO_LARGE;
  if (m == 0) return B200_OK;
  Int8LinearParams p = {};
  p.x = static_cast<const int8_t*>(x); p.x_scales = x_scales;
  p.w = static_cast<const int8_t*>(weight); p.w_scales = weight_scales;
  p.bias = bias; p.residual = residual; p.out = output; p.status = status;
  p.m = static_cast<int>(m); p.k = static_cast<int>(k); p.n = static_cast<int>(n); p.epilogue = epilogue;
  if (ceil_div(m, 64) > 65535) return B200_ERR_TOO_LARGE;
  const dim3 grid(static_cast<unsigned>(ceil_div(n, 64)), static_cast<unsigned>(ceil_div(m, 64)));
  cudaError_t error = cudaSuccess;
  with_element_type(dtype, [&](auto tag) {
    error = launch_chained(linear_int8_kernel<typename decltype(tag)::type>, grid, dim3(256), 0,
                           static_cast<cudaStream_t>(stream), p);
  });
  return error == cudaSuccess ? launch_status() : B200_ERR_LAUNCH;
}
