// Tanh GELU of a training step whose saved input is held in 8 bits: the
// forward pass writes y and, instead of keeping x for the backward pass, int8
// codes of x with one float32 scale for each 128 features of a row; the
// backward pass restores x from them.
//   y = x s(x),  s(x) = 1 / (1 + exp(-2 u)),  u = c (x + 0.044715 x^3), c = sqrt(2 / pi)
// (0.5 (1 + tanh u) = s, without the cancellation of 1 + tanh u for negative
// u), and with x^ the restored input
//   dx = dy (s + x^ s (1 - s) 2 c (1 + 3 * 0.044715 x^2)).
//
// Memory-bound: forward 2 e + 1 + 4 / 128 bytes an element, backward the same,
// for e bytes in the type of x.  A group never leaves the lanes that loaded
// it, so x is read once, and four groups a lane set are in flight to cover the
// latency.  12288 x 12288 bf16: forward 120 us (0.97 of a copy's bandwidth),
// backward 111 (1.05); 500 x 4100 float16, both ways, 11 us, of which about 6
// are two launches and two trips to memory.  Widths that 16 bytes do not divide
// take narrower accesses, down to one element and one code: 4096 rows of bf16,
// forward and backward, 12288 wide 42 and 40 us, 12284 67 and 60, 12286 74 and
// 67, 12287 94 and 100; float32 68 and 68, 12287 95 and 98.
// A group of 128, a quarter of a 16-bit row of the smallest widths, costs 3%
// of the saved bytes in scales; one scale for a whole row would let a single
// outlier take the precision of all other values.
#include "rows.cuh"

namespace convrot {
namespace {

constexpr int kGroup = 128;
constexpr float kC2 = 1.5957691216057308f;  // 2 c
constexpr float kA = 0.044715f;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// s(x) from x and x^2: 1 / (1 + 2^(-x (k + k a x^2))), k = 2 c log2(e).  Where
// the power overflows s is 0, and where x^2 does it is 0 or 1, as it should.
__device__ __forceinline__ float gate(float x, float x2) {
  return rcp(1.0f + ex2(x * fmaf(-kC2 * kLog2e * kA, x2, -kC2 * kLog2e)));
}

// A group is spread over LANES lanes, NV vectors of VEC elements each; a CTA
// of 256 threads takes kUnroll groups for each of its 256 / LANES lane sets,
// all loaded before the first is used.
template <int VEC>
struct Spread {
  static constexpr int kLanes = kGroup / VEC < 32 ? kGroup / VEC : 32;
  static constexpr int kVectors = kGroup / (VEC * kLanes);
  static constexpr int kSets = 256 / kLanes;
};
constexpr int kUnroll = 4;

struct GeluParams {
  const void* in;  // x, or dy
  void* out;       // y, or dx
  int8_t* codes;
  float* scales;
  uint32_t total, groups;  // groups of all rows, and of a row
  int64_t features;
};

// Element offset of a group's first value and its length (0 past the last
// group).  FULL: the features are whole groups, which then follow one another
// in memory.
template <bool FULL>
__device__ __forceinline__ void locate(const GeluParams& p, uint32_t group, int64_t& base, int& length) {
  base = 0;
  length = 0;
  if (group >= p.total) return;
  if constexpr (FULL) {
    base = static_cast<int64_t>(group) * kGroup;
    length = kGroup;
  } else {
    const uint32_t row = group / p.groups, g = group - row * p.groups;
    base = static_cast<int64_t>(row) * p.features + static_cast<int64_t>(g) * kGroup;
    const int64_t left = p.features - static_cast<int64_t>(g) * kGroup;
    length = left < kGroup ? static_cast<int>(left) : kGroup;
  }
}

template <typename T, int VEC, bool FULL>
__global__ void __launch_bounds__(256) gelu_fwd_kernel(const GeluParams p) {
  using S = Spread<VEC>;
  grid_dependency_wait();
  grid_dependents_launch();
  const int lane = threadIdx.x % S::kLanes;
  const uint32_t first = blockIdx.x * (S::kSets * kUnroll) + threadIdx.x / S::kLanes;
  const T* x = static_cast<const T*>(p.in);
  Pack<T, VEC> raw[kUnroll][S::kVectors];
  int64_t base[kUnroll];
  int length[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t group = first + u * S::kSets;
    locate<FULL>(p, group, base[u], length[u]);
#pragma unroll
    for (int j = 0; j < S::kVectors; ++j) {
      const int c = (lane + j * S::kLanes) * VEC;
      if (FULL ? length[u] > 0 : c < length[u]) raw[u][j].load_ahead(x + base[u] + c);
    }
  }
  if (p.codes) {
    // The groups' maxima; then lane u of a set forms the quantizer of group u,
    // so that its divisions are done once, and the set takes it from there.
    uint32_t mine = 0;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < S::kVectors; ++j)
        if (FULL ? length[u] > 0 : (lane + j * S::kLanes) * VEC < length[u]) top = max(top, raw[u][j].top());
      if constexpr (S::kLanes == 32) {
        top = warp_max(top);
      } else {
#pragma unroll
        for (int o = S::kLanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
      }
      if (lane == u) mine = top;
    }
    const Quant8<T> own(mine);
    if (lane < kUnroll && first + lane * S::kSets < p.total) p.scales[first + lane * S::kSets] = scale8(mine);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const Quant8<T> quant = own.from_lane(u, S::kLanes);
#pragma unroll
      for (int j = 0; j < S::kVectors; ++j) {
        const int c = (lane + j * S::kLanes) * VEC;
        if (FULL ? length[u] > 0 : c < length[u]) {
          float v[VEC];
          uint32_t code[VEC];
          raw[u][j].get(v);
          if (quant.tiny()) Quant8<float>(quant.bits).codes(v, code);
          else quant.codes(v, code);
          store_codes<VEC>(p.codes + base[u] + c, code, quant.mask());
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
#pragma unroll
    for (int j = 0; j < S::kVectors; ++j) {
      const int c = (lane + j * S::kLanes) * VEC;
      if (FULL ? length[u] > 0 : c < length[u]) {
        float v[VEC];
        raw[u][j].get(v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] *= gate(v[i], v[i] * v[i]);
        Pack<T, VEC> out;
        out.set(v);
        out.store(static_cast<T*>(p.out) + base[u] + c);
      }
    }
}

template <typename T, int VEC, bool FULL>
__global__ void __launch_bounds__(256) gelu_bwd_kernel(const GeluParams p) {
  using S = Spread<VEC>;
  grid_dependency_wait();
  grid_dependents_launch();
  const int lane = threadIdx.x % S::kLanes;
  const uint32_t first = blockIdx.x * (S::kSets * kUnroll) + threadIdx.x / S::kLanes;
  const T* dy = static_cast<const T*>(p.in);
  Pack<T, VEC> raw[kUnroll][S::kVectors];
  Pack<uint8_t, VEC> codes[kUnroll][S::kVectors];
  float scale[kUnroll];
  int64_t base[kUnroll];
  int length[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t group = first + u * S::kSets;
    locate<FULL>(p, group, base[u], length[u]);
    scale[u] = length[u] > 0 ? ld_f32(p.scales + group) : 0.0f;
#pragma unroll
    for (int j = 0; j < S::kVectors; ++j) {
      const int c = (lane + j * S::kLanes) * VEC;
      if (FULL ? length[u] > 0 : c < length[u]) {
        raw[u][j].load_ahead(dy + base[u] + c);
        codes[u][j].load_ahead(reinterpret_cast<const uint8_t*>(p.codes) + base[u] + c);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
#pragma unroll
    for (int j = 0; j < S::kVectors; ++j) {
      const int c = (lane + j * S::kLanes) * VEC;
      if (FULL ? length[u] > 0 : c < length[u]) {
        float d[VEC];
        raw[u][j].get(d);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float x = signed_byte(codes[u][j].w[i / 4], i % 4) * scale[u];
          // x^2 bounded so that it stays finite: from |x| = 100 on s is
          // exactly 0 or 1, and s - s^2 exactly 0 whatever it is multiplied by
          const float x2 = fminf(x * x, 1.0e4f), s = gate(x, x2);
          d[i] *= fmaf(x * fmaf(-s, s, s), fmaf(3.0f * kC2 * kA, x2, kC2), s);
        }
        Pack<T, VEC> out;
        out.set(d);
        out.store(static_cast<T*>(p.out) + base[u] + c);
      }
    }
}

int check_shape(int dtype, int64_t rows, int64_t features) {
  CONVROT_REQUIRE(valid_dtype(dtype), CONVROT_ERR_INVALID, "unknown dtype %d", dtype);
  CONVROT_REQUIRE(rows >= 0 && features > 0, CONVROT_ERR_INVALID, "invalid shape (%lld, %lld)",
                  static_cast<long long>(rows), static_cast<long long>(features));
  CONVROT_REQUIRE(features <= (1LL << 31) && rows <= (1LL << 31) / ((features + kGroup - 1) / kGroup),
                  CONVROT_ERR_UNSUPPORTED, "more than 2^31 groups of %d", kGroup);
  return CONVROT_OK;
}

template <int VEC>
int enqueue(void (*kernel)(GeluParams), const GeluParams& p, const char* what, cudaStream_t s) {
  constexpr uint32_t kPerCta = Spread<VEC>::kSets * kUnroll;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.total + kPerCta - 1) / kPerCta, 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p));
  return check_launch(what);
}

// Elements of a vector: 16 bytes' worth, or the most for which every row's
// start is aligned in all three arrays.
template <typename T>
int vector_of(const GeluParams& p) {
  for (int vec = 16 / sizeof(T); vec > 1; vec /= 2)
    if (p.features % vec == 0 && aligned_to(p.in, vec * sizeof(T)) && aligned_to(p.out, vec * sizeof(T)) &&
        aligned_to(p.codes, vec))
      return vec;
  return 1;
}

template <typename T>
int forward(const GeluParams& p, cudaStream_t s) {
  const char* what = "convrot_gelu_saved8";
  const int vec = vector_of<T>(p);
  constexpr int W = 16 / sizeof(T);
  if (vec == W && p.features % kGroup == 0) return enqueue<W>(gelu_fwd_kernel<T, W, true>, p, what, s);
  if constexpr (W == 8)
    if (vec == 8) return enqueue<8>(gelu_fwd_kernel<T, 8, false>, p, what, s);
  if (vec == 4) return enqueue<4>(gelu_fwd_kernel<T, 4, false>, p, what, s);
  if (vec == 2) return enqueue<2>(gelu_fwd_kernel<T, 2, false>, p, what, s);
  return enqueue<1>(gelu_fwd_kernel<T, 1, false>, p, what, s);
}

template <typename T>
int backward(const GeluParams& p, cudaStream_t s) {
  const char* what = "convrot_gelu_saved8_backward";
  const int vec = vector_of<T>(p);
  constexpr int W = 16 / sizeof(T);
  if (vec == W && p.features % kGroup == 0) return enqueue<W>(gelu_bwd_kernel<T, W, true>, p, what, s);
  if constexpr (W == 8)
    if (vec == 8) return enqueue<8>(gelu_bwd_kernel<T, 8, false>, p, what, s);
  if (vec == 4) return enqueue<4>(gelu_bwd_kernel<T, 4, false>, p, what, s);
  if (vec == 2) return enqueue<2>(gelu_bwd_kernel<T, 2, false>, p, what, s);
  return enqueue<1>(gelu_bwd_kernel<T, 1, false>, p, what, s);
}

GeluParams params(const void* in, void* out, int8_t* codes, float* scales, int64_t rows, int64_t features) {
  const int64_t groups = (features + kGroup - 1) / kGroup;
  return {in, out, codes, scales, static_cast<uint32_t>(rows * groups), static_cast<uint32_t>(groups), features};
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
  CONVROT_REQUIRE(aligned_to(x, dtype_size(dtype)) && aligned_to(y, dtype_size(dtype)) && aligned_to(scales, 4),
                  CONVROT_ERR_INVALID, "tensors must be aligned to their elements");
  const GeluParams p = params(x, y, codes, scales, rows, features);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CONVROT_BF16: return forward<__nv_bfloat16>(p, s);
    case CONVROT_F16: return forward<__half>(p, s);
    default: return forward<float>(p, s);
  }
}

int convrot_gelu_saved8_backward(const void* dy, int dtype, int64_t rows, int64_t features, const int8_t* codes,
                                 const float* scales, void* dx, void* stream) {
  using namespace convrot;
  const int rc = check_shape(dtype, rows, features);
  if (rc != CONVROT_OK || rows == 0) return rc;
  CONVROT_REQUIRE(dy && dx && codes && scales, CONVROT_ERR_INVALID, "null pointer");
  CONVROT_REQUIRE(aligned_to(dy, dtype_size(dtype)) && aligned_to(dx, dtype_size(dtype)) && aligned_to(scales, 4),
                  CONVROT_ERR_INVALID, "tensors must be aligned to their elements");
  const GeluParams p =
      params(dy, dx, const_cast<int8_t*>(codes), const_cast<float*>(scales), rows, features);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CONVROT_BF16: return backward<__nv_bfloat16>(p, s);
    case CONVROT_F16: return backward<__half>(p, s);
    default: return backward<float>(p, s);
  }
}

}  // extern "C"
