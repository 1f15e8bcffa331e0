// Row quantizer of the 8-bit linear: int8 codes and one float32 scale for
// each row (token), optionally after a product with one factor for each
// column (the gradient of the 8-bit linear folds the weight scales in).
//
// Memory-bound: a row is read once from HBM and its codes are written once.
// One CTA for each row, which stays in registers between the maximum and the
// codes; wide loads where address and pitch allow, else one element a lane
// (consecutive lanes on consecutive elements).  Rows that do not fit the
// registers are read a second time, through L2.
#include "rows.cuh"

namespace convrot {
namespace {

// Most threads of a CTA: more for single elements, which are narrow loads.
template <int VEC> constexpr int kThreads = VEC == 1 ? 1024 : 512;

struct QuantParams {
  const void* x;
  const float* col_scale;
  int8_t* q;
  float* scales;
  int64_t rows, x_stride, q_stride;
  int features;
};

__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = warp_max(v);
  if (blockDim.x > 32) {
    __syncthreads();  // red may still be read by the previous row
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < (blockDim.x >> 5) ? red[threadIdx.x & 31] : 0u;
    v = warp_max(v);
  }
  return v;
}

// VEC consecutive elements at column c as float32; columns past the end read 0.
template <typename T, int VEC>
__device__ __forceinline__ void load(const QuantParams& p, int64_t row, int c, float (&v)[VEC]) {
  const T* src = static_cast<const T*>(p.x) + row * p.x_stride + c;
  if (c + VEC <= p.features) {
    Pack<T, VEC> pk;
    pk.load(src);
    pk.get(v);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = c + i < p.features ? Elem<T>::to_f(src[i]) : 0.0f;
  }
  if (p.col_scale) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = c + i < p.features ? __fmul_rn(v[i], __ldg(p.col_scale + c + i)) : 0.0f;
  }
}

template <int VEC>
__device__ __forceinline__ void store(const QuantParams& p, int64_t row, int c, const Quant8& quant,
                                      const float (&v)[VEC]) {
  int8_t* dst = p.q + row * p.q_stride + c;
  uint32_t code[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) code[i] = quant.code(v[i]);
  if constexpr (VEC % 4 == 0) {
    if (c + VEC <= p.features) {
      store_codes<VEC>(dst, code, quant.mask);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    if (c + i < p.features) dst[i] = static_cast<int8_t>(code[i] & quant.mask);
}

// NV vectors of VEC elements a thread in registers; NV = 0: any length, in
// two passes over the row.
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(kThreads<VEC>) quantize_i8_kernel(const QuantParams p) {
  __shared__ uint32_t red[32];
  grid_dependency_wait();  // x may come from the previous kernel of the stream
  grid_dependents_launch();
  const int step = blockDim.x * VEC;
  const int c0 = threadIdx.x * VEC;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    uint32_t top = 0;
    if constexpr (NV > 0) {
      float v[NV][VEC];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = c0 + j * step;
        if (c < p.features) {
          load<T, VEC>(p, row, c, v[j]);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[j][i] = 0.0f;
        }
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) top = max(top, abs_bits(v[j][i]));
      top = block_max(top, red);
      const Quant8 quant(top);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = c0 + j * step;
        if (c < p.features) store<VEC>(p, row, c, quant, v[j]);
      }
    } else {
      for (int c = c0; c < p.features; c += step) {
        float v[VEC];
        load<T, VEC>(p, row, c, v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) top = max(top, abs_bits(v[i]));
      }
      top = block_max(top, red);
      const Quant8 quant(top);
      for (int c = c0; c < p.features; c += step) {
        float v[VEC];
        load<T, VEC>(p, row, c, v);
        store<VEC>(p, row, c, quant, v);
      }
    }
    if (threadIdx.x == 0) p.scales[row] = Quant8::scale(top);
  }
}

template <typename T, int VEC, int NV>
int launch_nv(const QuantParams& p, int threads, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows < (1LL << 30) ? p.rows : (1LL << 30)), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, quantize_i8_kernel<T, VEC, NV>, p));
  return check_launch("convrot_quantize_i8");
}

template <typename T, int VEC>
int launch_vec(const QuantParams& p, cudaStream_t stream) {
  // two vectors (four single elements) a thread, more where the CTA is full
  constexpr int kLeast = VEC == 1 ? 4 : 2;
  const int vectors = (p.features + VEC - 1) / VEC;
  int nv = kLeast;
  while (nv < 4 * kLeast && vectors > nv * kThreads<VEC>) nv *= 2;
  const int64_t per = (vectors + nv - 1) / nv;
  if (per > kThreads<VEC>) return launch_nv<T, VEC, 0>(p, kThreads<VEC>, stream);
  const int threads = static_cast<int>((per + 31) / 32 * 32);
  if (nv == kLeast) return launch_nv<T, VEC, kLeast>(p, threads, stream);
  if (nv == 2 * kLeast) return launch_nv<T, VEC, 2 * kLeast>(p, threads, stream);
  return launch_nv<T, VEC, 4 * kLeast>(p, threads, stream);
}

template <typename T>
int launch(const QuantParams& p, cudaStream_t stream) {
  constexpr int kWide = 16 / sizeof(T);
  const bool wide = aligned_to(p.x, 16) && p.x_stride * static_cast<int64_t>(sizeof(T)) % 16 == 0 &&
                    aligned_to(p.q, 8) && p.q_stride % 8 == 0;
  return wide ? launch_vec<T, kWide>(p, stream) : launch_vec<T, 1>(p, stream);
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
  CONVROT_REQUIRE(features <= (1 << 30), CONVROT_ERR_UNSUPPORTED, "too many features");
  CONVROT_REQUIRE(x_stride >= features && q_stride >= features, CONVROT_ERR_INVALID,
                  "row strides must cover the features (%lld, %lld)", static_cast<long long>(x_stride),
                  static_cast<long long>(q_stride));
  if (rows == 0) return CONVROT_OK;
  CONVROT_REQUIRE(x && q && scales, CONVROT_ERR_INVALID, "null pointer");
  const QuantParams p{x, col_scale, q, scales, rows, x_stride, q_stride, static_cast<int>(features)};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CONVROT_BF16: return launch<__nv_bfloat16>(p, s);
    case CONVROT_F16: return launch<__half>(p, s);
    default: return launch<float>(p, s);
  }
}

}  // extern "C"
