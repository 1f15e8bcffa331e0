// Row quantizer of the 8-bit linear: int8 codes and one float32 scale for
// each row (token), optionally after a product with one factor for each
// column (the gradient of the 8-bit linear folds the weight scales in).
//
// Memory-bound: a row is read once from HBM and its codes are written once.
// A row stays in the registers of a warp or a CTA between the maximum and the
// codes, with the next row's loads in flight; accesses of 16 bytes, or of one
// or two elements where addresses and pitch allow no more.  What limits beside
// the memory is the number of instructions: a thread has up to 32 values of a
// row, so that the exchange of the maximum and the division are little beside
// them.  Rows that do not fit the registers are read twice, through L2.
// bf16 rows from HBM: 4096 x 12288 in 27.6 us (0.84 of a copy's bandwidth),
// 4096 x 3072 in 9.6 (0.61), 16 x 4096 in 1.6 (a launch); with column scales
// 33.6 and 11.2, 1536 x 3072 5.1 (floor 2.2); 4096 x 3071, whose rows start at any
// byte pair, 14 to 16.  At 4096 x 3072 64% of the issue slots are used by 45% of
// the warps that an SM holds: the codes' instructions, and only one row ahead to
// cover the memory's latency, rather than its bandwidth.
#include "rows.cuh"

namespace convrot {
namespace {

struct QuantParams {
  const void* x;
  const float* col_scale;
  int8_t* q;
  float* scales;
  int64_t rows, x_stride, q_stride;
  int features;
};

constexpr int kWarps = 4;  // of a CTA whose warps each have rows of their own

// The maximum over the T threads of a row, for all of them.  red holds two
// sets of a CTA's warps' values, used in turn, so that one barrier is enough.
template <int T>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t (*red)[32], int& turn) {
  v = warp_max(v);
  if constexpr (T > 32) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) red[turn][threadIdx.x >> 5] = v;
    __syncthreads();
    v = warp_max(lane < T / 32 ? red[turn][lane] : 0u);
    turn ^= 1;
  }
  return v;
}

// The type whose quantizer applies: that of x, or float32 after the product
// with the column scales.
template <typename E, bool SCALED>
using Quantized = Quant8<typename std::conditional<SCALED, float, E>::type>;

// One thread's share of a row: NV vectors of VEC elements, T vectors apart,
// from column c0 = VEC * (thread of the row) on; left: columns from there on.
// Absent elements are 0.
template <typename E, int VEC, int NV, int T, bool SCALED>
struct Share {
  Pack<E, VEC> raw[NV];
  Pack<float, VEC> factor[SCALED ? NV : 1];

  template <typename F>
  static __device__ __forceinline__ void load_one(Pack<F, VEC>& pk, const F* src, int at, int left) {
    pk.clear();
    if (at + VEC <= left) pk.load_ahead(src + at);
    else if (VEC > 1 && at < left) pk.load_part(src + at, left - at);
  }
  __device__ __forceinline__ void load(const E* row, int left) {
#pragma unroll
    for (int j = 0; j < NV; ++j) load_one(raw[j], row, j * T * VEC, left);
  }
  __device__ __forceinline__ void load_factors(const float* col_scale, int left) {
    if constexpr (SCALED)
#pragma unroll
      for (int j = 0; j < NV; ++j) load_one(factor[j], col_scale, j * T * VEC, left);
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
  __device__ __forceinline__ void store(int8_t* dst, int left, const Quantized<E, SCALED>& quant) const {
    if (quant.tiny()) store_as(dst, left, Quant8<float>(quant.bits));
    else store_as(dst, left, quant);
  }
  template <typename Q>
  __device__ __forceinline__ void store_as(int8_t* dst, int left, const Q& quant) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = j * T * VEC;
      if (at < left) {
        float v[VEC];
        uint32_t code[VEC];
        get(j, v);
        quant.codes(v, code);
        if (at + VEC <= left) {
          store_codes<VEC>(dst + at, code, quant.mask());
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (at + i < left) dst[at + i] = static_cast<int8_t>(code[i] & quant.mask());
        }
      }
    }
  }
};

// T threads share a row: 32 (each warp of the CTA rows of its own), or the CTA.
template <typename E, int VEC, int NV, int T, bool SCALED>
__global__ void __launch_bounds__(T == 32 ? 32 * kWarps : T, 1024 / (T == 32 ? 32 * kWarps : T))
    quantize_i8_kernel(const QuantParams p) {
  __shared__ uint32_t red[2][32];
  grid_dependency_wait();  // x may come from the previous kernel of the stream
  grid_dependents_launch();
  const int c0 = (T == 32 ? threadIdx.x & 31 : threadIdx.x) * VEC, left = p.features - c0;
  const int64_t first = T == 32 ? static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t stride = T == 32 ? static_cast<int64_t>(gridDim.x) * kWarps : gridDim.x;
  int turn = 0;
  const E* src = static_cast<const E*>(p.x) + first * p.x_stride + c0;
  int8_t* dst = p.q + first * p.q_stride + c0;
  Share<E, VEC, NV, T, SCALED> x, next;
  if (first < p.rows) next.load(src, left);
  next.load_factors(p.col_scale + c0, left);
  for (int64_t row = first; row < p.rows; row += stride) {
    x = next;
    src += stride * p.x_stride;
    if (row + stride < p.rows) next.load(src, left);
    const uint32_t top = row_max<T>(x.top(), red, turn);
    x.store(dst, left, Quantized<E, SCALED>(top));
    if (c0 == 0) p.scales[row] = scale8(top);
    dst += stride * p.q_stride;
  }
}

// Rows too long for the registers: two passes, the second through L2.
template <typename E, int VEC, bool SCALED>
__global__ void __launch_bounds__(512) quantize_i8_long_kernel(const QuantParams p) {
  __shared__ uint32_t red[2][32];
  grid_dependency_wait();
  grid_dependents_launch();
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const E* src = static_cast<const E*>(p.x) + row * p.x_stride;
    Share<E, VEC, 4, 512, SCALED> x;
    uint32_t top = 0;
    for (int c = threadIdx.x * VEC; c < p.features; c += 4 * 512 * VEC) {
      x.load(src + c, p.features - c);
      x.load_factors(p.col_scale + c, p.features - c);
      top = max(top, x.top());
    }
    top = row_max<512>(top, red, turn);
    const Quantized<E, SCALED> quant(top);
    for (int c = threadIdx.x * VEC; c < p.features; c += 4 * 512 * VEC) {
      x.load(src + c, p.features - c);
      x.load_factors(p.col_scale + c, p.features - c);
      x.store(p.q + row * p.q_stride + c, p.features - c, quant);
    }
    if (threadIdx.x == 0) p.scales[row] = scale8(top);
  }
}

// As many CTAs as rows need, up to about 1024 threads for each SM.
int enqueue(void (*kernel)(QuantParams), const QuantParams& p, int threads, cudaStream_t stream) {
  const int64_t at_once = threads == 32 ? kWarps : 1;
  const int cta = threads == 32 ? 32 * kWarps : threads;
  const int64_t want = (p.rows + at_once - 1) / at_once, most = static_cast<int64_t>(device_sm_count()) * (1024 / cta);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(want < most ? want : most), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(cta), 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p));
  return check_launch("convrot_quantize_i8");
}

// U vectors a thread: four of 16 bytes (two beside column scales, which take
// registers too), or eight of one or two elements; one
// or two for the shortest rows.
template <typename E, int VEC, bool SCALED>
int launch_vec(const QuantParams& p, cudaStream_t stream) {
  constexpr int U = VEC > 2 ? (SCALED ? 2 : 4) : 8;
  constexpr int kShort = (U + 3) / 4;
  const int vectors = (p.features + VEC - 1) / VEC;
#define CONVROT_QUANT(NV, T) enqueue(quantize_i8_kernel<E, VEC, NV, T, SCALED>, p, T, stream)
  if (vectors <= 32 * kShort) return CONVROT_QUANT(kShort, 32);
  if (vectors <= 32 * U) return CONVROT_QUANT(U, 32);
  if (vectors <= 64 * U) return CONVROT_QUANT(U, 64);
  if (vectors <= 128 * U) return CONVROT_QUANT(U, 128);
  if (vectors <= 256 * U) return CONVROT_QUANT(U, 256);
  if (vectors <= 512 * U) return CONVROT_QUANT(U, 512);
  if (vectors <= 1024 * U) return CONVROT_QUANT(U, 1024);
  if constexpr (VEC == 1)
    if (vectors <= 1024 * 2 * U) return CONVROT_QUANT(2 * U, 1024);
#undef CONVROT_QUANT
  return enqueue(quantize_i8_long_kernel<E, VEC, SCALED>, p, 512, stream);
}

template <typename E, bool SCALED>
int launch_scaled(const QuantParams& p, cudaStream_t stream) {
  constexpr int W = 16 / sizeof(E);
  auto aligned_for = [&](int vec) {
    const int64_t bytes = vec * static_cast<int64_t>(sizeof(E));
    return aligned_to(p.x, bytes) && p.x_stride % vec == 0 && aligned_to(p.q, vec) && p.q_stride % vec == 0 &&
           aligned_to(p.col_scale, vec * 4 < 16 ? vec * 4 : 16);
  };
  if (aligned_for(W)) return launch_vec<E, W, SCALED>(p, stream);
  if (aligned_for(2)) return launch_vec<E, 2, SCALED>(p, stream);
  return launch_vec<E, 1, SCALED>(p, stream);
}

template <typename E>
int launch(const QuantParams& p, cudaStream_t stream) {
  return p.col_scale ? launch_scaled<E, true>(p, stream) : launch_scaled<E, false>(p, stream);
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
