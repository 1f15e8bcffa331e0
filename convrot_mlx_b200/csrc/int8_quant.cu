// Row quantizer of the 8-bit linear: int8 codes and one float32 scale for
// each row (token), optionally after a product with one factor for each
// column (the gradient of the 8-bit linear folds the weight scales in).
//
// Memory-bound: a row is read once from HBM and its codes are written once.
#include "rows.cuh"

namespace convrot {
namespace {

template <typename T>
__device__ __forceinline__ float scaled(const T* x, const float* col_scale, int64_t c) {
  const float v = Elem<T>::to_f(x[c]);
  return col_scale ? __fmul_rn(v, col_scale[c]) : v;
}

template <typename T>
__global__ void __launch_bounds__(256) quantize_i8_kernel(const T* __restrict__ x, int64_t rows, int64_t features,
                                                          int64_t x_stride, const float* __restrict__ col_scale,
                                                          int8_t* __restrict__ q, int64_t q_stride,
                                                          float* __restrict__ scales) {
  __shared__ uint32_t red[8];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * x_stride;
    uint32_t top = 0;
    for (int64_t c = threadIdx.x; c < features; c += 256) top = max(top, abs_bits(scaled(xr, col_scale, c)));
    top = warp_max(top);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    top = red[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) top = max(top, red[w]);
    const Quant8 quant(top);
    if (threadIdx.x == 0) scales[row] = Quant8::scale(top);
    for (int64_t c = threadIdx.x; c < features; c += 256)
      q[row * q_stride + c] = top < kInfBits ? static_cast<int8_t>(quant.code(scaled(xr, col_scale, c))) : 0;
  }
}

template <typename T>
int launch(const void* x, int64_t rows, int64_t features, int64_t x_stride, const float* col_scale, int8_t* q,
           int64_t q_stride, float* scales, cudaStream_t stream) {
  const int64_t ctas = 8LL * device_sm_count();
  const int64_t grid = rows < ctas ? rows : ctas;
  quantize_i8_kernel<T><<<static_cast<unsigned>(grid), 256, 0, stream>>>(static_cast<const T*>(x), rows, features,
                                                                        x_stride, col_scale, q, q_stride, scales);
  return check_launch("convrot_quantize_i8");
}

}  // namespace
}  // namespace convrot

extern "C" {

int convrot_quantize_i8(const void* x, int dtype, int64_t rows, int64_t features, int64_t x_stride,
                        const float* col_scale, int8_t* q, int64_t q_stride, float* scales, void* stream) {
  using namespace convrot;
  CONVROT_REQUIRE(valid_dtype(dtype), CONVROT_ERR_INVALID, "unknown dtype %d", dtype);
  CONVROT_REQUIRE(rows >= 0 && features > 0, CONVROT_ERR_INVALID, "invalid shape (%lld, %lld)",
                  static_cast<long long>(rows), static_cast<long long>(features));
  CONVROT_REQUIRE(x_stride >= features && q_stride >= features, CONVROT_ERR_INVALID,
                  "row strides must cover the features (%lld, %lld)", static_cast<long long>(x_stride),
                  static_cast<long long>(q_stride));
  if (rows == 0) return CONVROT_OK;
  CONVROT_REQUIRE(x && q && scales, CONVROT_ERR_INVALID, "null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CONVROT_BF16: return launch<__nv_bfloat16>(x, rows, features, x_stride, col_scale, q, q_stride, scales, s);
    case CONVROT_F16: return launch<__half>(x, rows, features, x_stride, col_scale, q, q_stride, scales, s);
    default: return launch<float>(x, rows, features, x_stride, col_scale, q, q_stride, scales, s);
  }
}

}  // extern "C"
