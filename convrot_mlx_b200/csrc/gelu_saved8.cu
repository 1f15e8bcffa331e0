// Tanh GELU of a training step whose saved input is held in 8 bits: the
// forward pass writes y and, instead of keeping x for the backward pass, int8
// codes of x with one float32 scale for each 128 features of a row; the
// backward pass restores x from them.
//   y = x s(x),  s(x) = 1 / (1 + exp(-2 u)),  u = c (x + 0.044715 x^3), c = sqrt(2 / pi)
// (0.5 (1 + tanh u) = s, without the cancellation of 1 + tanh u for negative
// u), and with x^ the restored input
//   dx = dy (s + x^ s (1 - s) 2 c (1 + 3 * 0.044715 x^2)).
//
// Memory-bound: forward e + e + 1 + 4 / 128 bytes an element, backward the
// same, for e bytes in the type of x.
#include "rows.cuh"

namespace convrot {
namespace {

constexpr int kGroup = 128;
constexpr float kC2 = 1.5957691216057308f;  // 2 c
constexpr float kA = 0.044715f;

// x^2, bounded so that it stays finite: from |x| = 100 on the gate is exactly
// 0 or 1 and its slope exactly 0 whatever the square.
__device__ __forceinline__ float square(float x) { return fminf(x * x, 1.0e4f); }

__device__ __forceinline__ float gate(float x, float x2) {
  return __fdividef(1.0f, 1.0f + __expf(-kC2 * x * (1.0f + kA * x2)));
}

// One warp for each group of 128 features of a row.
template <typename T>
__global__ void __launch_bounds__(256) gelu_fwd_kernel(const T* __restrict__ x, int64_t rows, int64_t features,
                                                       T* __restrict__ y, int8_t* __restrict__ codes,
                                                       float* __restrict__ scales) {
  const int lane = threadIdx.x & 31;
  const int64_t groups = (features + kGroup - 1) / kGroup;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * 8;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); i < rows * groups; i += warps) {
    const int64_t row = i / groups, c0 = i % groups * kGroup;
    float v[4];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = c0 + lane + 32 * j;
      v[j] = c < features ? Elem<T>::to_f(x[row * features + c]) : 0.0f;
      top = max(top, abs_bits(v[j]));
    }
    top = warp_max(top);
    const Quant8 quant(top);
    if (lane == 0 && scales) scales[i] = Quant8::scale(top);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = c0 + lane + 32 * j;
      if (c >= features) break;
      y[row * features + c] = Elem<T>::from_f(v[j] * gate(v[j], square(v[j])));
      if (codes) codes[row * features + c] = top < kInfBits ? static_cast<int8_t>(quant.code(v[j])) : 0;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) gelu_bwd_kernel(const T* __restrict__ dy, int64_t rows, int64_t features,
                                                       const int8_t* __restrict__ codes,
                                                       const float* __restrict__ scales, T* __restrict__ dx) {
  const int64_t groups = (features + kGroup - 1) / kGroup;
  const int64_t total = rows * features;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const float x = static_cast<float>(codes[i]) * scales[i / features * groups + i % features / kGroup];
    const float x2 = square(x), s = gate(x, x2);
    const float slope = s + x * s * (1.0f - s) * kC2 * (1.0f + 3.0f * kA * x2);
    dx[i] = Elem<T>::from_f(Elem<T>::to_f(dy[i]) * slope);
  }
}

int check_shape(int dtype, int64_t rows, int64_t features) {
  CONVROT_REQUIRE(valid_dtype(dtype), CONVROT_ERR_INVALID, "unknown dtype %d", dtype);
  CONVROT_REQUIRE(rows >= 0 && features > 0, CONVROT_ERR_INVALID, "invalid shape (%lld, %lld)",
                  static_cast<long long>(rows), static_cast<long long>(features));
  return CONVROT_OK;
}

unsigned grid_of(int64_t items) {
  const int64_t most = 8LL * device_sm_count();
  return static_cast<unsigned>(items < most ? items : most);
}

template <typename T>
int forward(const void* x, int64_t rows, int64_t features, void* y, int8_t* codes, float* scales, cudaStream_t s) {
  const int64_t groups = rows * ((features + kGroup - 1) / kGroup);
  gelu_fwd_kernel<T><<<grid_of((groups + 7) / 8), 256, 0, s>>>(static_cast<const T*>(x), rows, features,
                                                              static_cast<T*>(y), codes, scales);
  return check_launch("convrot_gelu_saved8");
}

template <typename T>
int backward(const void* dy, int64_t rows, int64_t features, const int8_t* codes, const float* scales, void* dx,
             cudaStream_t s) {
  gelu_bwd_kernel<T><<<grid_of((rows * features + 255) / 256), 256, 0, s>>>(
      static_cast<const T*>(dy), rows, features, codes, scales, static_cast<T*>(dx));
  return check_launch("convrot_gelu_saved8_backward");
}

}  // namespace
}  // namespace convrot

extern "C" {

int convrot_gelu_saved8(const void* x, int dtype, int64_t rows, int64_t features, void* y, int8_t* codes,
                        float* scales, void* stream) {
  using namespace convrot;
  const int rc = check_shape(dtype, rows, features);
  if (rc != CONVROT_OK || rows == 0) return rc;
  CONVROT_REQUIRE(x && y && (codes != nullptr) == (scales != nullptr), CONVROT_ERR_INVALID, "null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CONVROT_BF16: return forward<__nv_bfloat16>(x, rows, features, y, codes, scales, s);
    case CONVROT_F16: return forward<__half>(x, rows, features, y, codes, scales, s);
    default: return forward<float>(x, rows, features, y, codes, scales, s);
  }
}

int convrot_gelu_saved8_backward(const void* dy, int dtype, int64_t rows, int64_t features, const int8_t* codes,
                                 const float* scales, void* dx, void* stream) {
  using namespace convrot;
  const int rc = check_shape(dtype, rows, features);
  if (rc != CONVROT_OK || rows == 0) return rc;
  CONVROT_REQUIRE(dy && dx && codes && scales, CONVROT_ERR_INVALID, "null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CONVROT_BF16: return backward<__nv_bfloat16>(dy, rows, features, codes, scales, dx, s);
    case CONVROT_F16: return backward<__half>(dy, rows, features, codes, scales, dx, s);
    default: return backward<float>(dy, rows, features, codes, scales, dx, s);
  }
}

}  // extern "C"
