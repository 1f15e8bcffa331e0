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

// The type whose quantizer applies: that of x, or float32 after the product
// with the column scales.
template <typename T, bool SCALED>
using Quantized = Quant8<typename std::conditional<SCALED, float, T>::type>;

// One thread's share of a row: NV vectors of VEC elements, `step` apart.
template <typename T, int VEC, int NV, bool SCALED>
struct Share {
  Pack<T, VEC> raw[NV];
  Pack<float, VEC> factor[SCALED ? NV : 1];

  __device__ __forceinline__ void load(const QuantParams& p, int64_t row, int c0, int step) {
    const T* src = static_cast<const T*>(p.x) + row * p.x_stride;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = c0 + j * step;
      raw[j].clear();
      if (c + VEC <= p.features) {
        raw[j].load_nc(src + c);
      } else if (VEC > 1 && c < p.features) {
        raw[j].load_part(src + c, p.features - c);
      }
    }
    if constexpr (SCALED) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = c0 + j * step;
        factor[j].clear();
        if (c + VEC <= p.features) {
          factor[j].load_nc(p.col_scale + c);
        } else if (VEC > 1 && c < p.features) {
          factor[j].load_part(p.col_scale + c, p.features - c);
        }
      }
    }
  }
  __device__ __forceinline__ void get(int j, float (&v)[VEC]) const {
    raw[j].get(v);
    if constexpr (SCALED) {
      float f[VEC];
      factor[j].get(f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = __fmul_rn(v[i], f[i]);
    }
  }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if constexpr (SCALED) {
        float v[VEC];
        get(j, v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) m = max(m, abs_bits(v[i]));
      } else {
        m = max(m, raw[j].top());
      }
    }
    return m;
  }
  __device__ __forceinline__ void store(const QuantParams& p, int64_t row, int c0, int step,
                                        const Quantized<T, SCALED>& quant) const {
    int8_t* dst = p.q + row * p.q_stride;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = c0 + j * step;
      if (c < p.features) {
        float v[VEC];
        uint32_t code[VEC];
        get(j, v);
        quant.codes(v, code);
        if (c + VEC <= p.features) {
          store_codes<VEC>(dst + c, code, quant.mask());
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (c + i < p.features) dst[c + i] = static_cast<int8_t>(code[i] & quant.mask());
        }
      }
    }
  }
};

template <typename T, int VEC, int NV, bool SCALED>
__global__ void __launch_bounds__(kThreads<VEC>) quantize_i8_kernel(const QuantParams p) {
  __shared__ uint32_t red[2][32];
  grid_dependency_wait();  // x may come from the previous kernel of the stream
  grid_dependents_launch();
  const int c0 = threadIdx.x * VEC, step = blockDim.x * VEC, lane = threadIdx.x & 31;
  int turn = 0;
  Share<T, VEC, NV, SCALED> x, next;
  next.load(p, blockIdx.x, c0, step);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    x = next;
    if (row + gridDim.x < p.rows) next.load(p, row + gridDim.x, c0, step);  // in flight while this row is worked on
    uint32_t top = warp_max(x.top());
    if (blockDim.x > 32) {
      if (lane == 0) red[turn][threadIdx.x >> 5] = top;
      __syncthreads();
      top = warp_max(lane < (blockDim.x >> 5) ? red[turn][lane] : 0u);
      turn ^= 1;
    }
    x.store(p, row, c0, step, Quantized<T, SCALED>(top));
    if (threadIdx.x == 0) p.scales[row] = scale8(top);
  }
}

// Rows too long for the registers: two passes, the second through L2.
template <typename T, int VEC, bool SCALED>
__global__ void __launch_bounds__(kThreads<VEC>) quantize_i8_long_kernel(const QuantParams p) {
  __shared__ uint32_t red[32];
  grid_dependency_wait();
  grid_dependents_launch();
  const int step = blockDim.x * VEC;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    uint32_t top = 0;
    for (int c = threadIdx.x * VEC; c < p.features; c += 4 * step) {
      Share<T, VEC, 4, SCALED> x;
      x.load(p, row, c, step);
      top = max(top, x.top());
    }
    top = block_max(top, red);
    const Quantized<T, SCALED> quant(top);
    for (int c = threadIdx.x * VEC; c < p.features; c += 4 * step) {
      Share<T, VEC, 4, SCALED> x;
      x.load(p, row, c, step);
      x.store(p, row, c, step, quant);
    }
    if (threadIdx.x == 0) p.scales[row] = scale8(top);
  }
}

// As many CTAs as rows, up to about 1536 threads for each SM.
int enqueue(void (*kernel)(QuantParams), const QuantParams& p, int threads, cudaStream_t stream) {
  const int per_sm = threads > 768 ? 1 : threads < 64 ? 24 : 1536 / threads;
  const int64_t most = static_cast<int64_t>(device_sm_count()) * per_sm;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows < most ? p.rows : most), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p));
  return check_launch("convrot_quantize_i8");
}

template <typename T, int VEC, bool SCALED>
int launch_vec(const QuantParams& p, cudaStream_t stream) {
  // two vectors (four single elements) a thread, more where the CTA is full
  constexpr int kLeast = VEC == 1 ? 4 : 2;
  const int vectors = (p.features + VEC - 1) / VEC;
  int nv = kLeast;
  while (nv < 4 * kLeast && vectors > nv * kThreads<VEC>) nv *= 2;
  const int64_t per = (vectors + nv - 1) / nv;
  if (per > kThreads<VEC>) return enqueue(quantize_i8_long_kernel<T, VEC, SCALED>, p, kThreads<VEC>, stream);
  const int threads = static_cast<int>((per + 31) / 32 * 32);
  if (nv == kLeast) return enqueue(quantize_i8_kernel<T, VEC, kLeast, SCALED>, p, threads, stream);
  if (nv == 2 * kLeast) return enqueue(quantize_i8_kernel<T, VEC, 2 * kLeast, SCALED>, p, threads, stream);
  return enqueue(quantize_i8_kernel<T, VEC, 4 * kLeast, SCALED>, p, threads, stream);
}

template <typename T>
int launch(const QuantParams& p, cudaStream_t stream) {
  constexpr int kWide = 16 / sizeof(T);
  const bool wide = aligned_to(p.x, 16) && p.x_stride * static_cast<int64_t>(sizeof(T)) % 16 == 0 &&
                    aligned_to(p.q, 8) && p.q_stride % 8 == 0 && aligned_to(p.col_scale, 16);
  if (p.col_scale) return wide ? launch_vec<T, kWide, true>(p, stream) : launch_vec<T, 1, true>(p, stream);
  return wide ? launch_vec<T, kWide, false>(p, stream) : launch_vec<T, 1, false>(p, stream);
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
