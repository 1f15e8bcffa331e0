// The AdamW step over many tensors in one launch, and the sum of squares of
// many tensors (the gradient norm).
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps),
// all in float32, each operation rounded; p rounded once to its type.
// Moments in 32 bits are kept as they are.  In 8 bits m and r = sqrt(v) are
// kept as e4m3 codes with a float32 scale for each 256 values of a tensor,
// max|m| / 448 and max r / 448: a square would need twice the range, and a block
// whose gradients grow or fade together follows its scale exactly, however small
// a step changes it.  A root above 0 keeps a code above 0, since it divides.
//
// Memory-bound.  The tensors' addresses and sizes are kernel parameters, so a
// step needs no table on the device and can be captured.  A warp has 256
// values at a time, 8 a lane, so the maximum over a block of 8-bit moments is one
// exchange in the warp.  CTAs take contiguous shares of all tensors' blocks.
#include "rows.cuh"

namespace convrot {
namespace optim {

constexpr int kBlock = 256;  // values of a warp's turn; of a scale
constexpr int kLane = kBlock / 32;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr float kTop = 448.0f;         // the largest e4m3 value
constexpr float kLeast = 0.001953125f;  // the smallest above 0, 2^-9

struct Entry {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* scales;
  int64_t n;
  uint32_t first;    // of the blocks of all tensors, in the order of the table
  uint32_t aligned;  // vector accesses may be used
};

struct Scalars {
  int count;
  int64_t blocks;
  float decay, beta1, beta2, rest1, rest2, eps, step_size, root;  // root: 1 / sqrt(1 - b2^t)
  // the step and the learning rate where they are on the device
  const float* step;
  const float* lr;
  double log1, log2, wd;  // log of b1 and b2
  float host_lr, host_step;
  // clipping by the norm: sums of squares of the gradients
  const double* sums;
  int sums_count;
  float max_norm;
  float* norm;
};

// A table that kernel parameters hold: 32 tensors in 2 KB for the launch's
// sake, 512 in 28 KB (of the 32 KB that there are).
template <int CAP>
struct Table {
  Scalars s;
  Entry e[CAP];
};

template <typename T>
__device__ __forceinline__ void load(const T* src, int count, bool vec, float (&v)[kLane]) {
  if (vec) {
    Pack<T, kLane> p;
    p.load_ahead(src);
    p.get(v);
  } else {
#pragma unroll
    for (int i = 0; i < kLane; ++i) v[i] = i < count ? Elem<T>::to_f(src[i]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store(T* dst, int count, bool vec, const float (&v)[kLane]) {
  if (vec) {
    Pack<T, kLane> p;
    p.set(v);
    p.store(dst);
  } else {
#pragma unroll
    for (int i = 0; i < kLane; ++i)
      if (i < count) dst[i] = cvt_out<T>(v[i]);
  }
}

__device__ __forceinline__ uint2 load_codes(const uint8_t* src, int count, bool vec) {
  if (vec) return ld_64(src);
  uint32_t w[2] = {};
#pragma unroll
  for (int i = 0; i < kLane; ++i)
    if (i < count) w[i / 4] |= static_cast<uint32_t>(src[i]) << (8 * (i & 3));
  return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ void store_codes8(uint8_t* dst, int count, bool vec, uint2 w) {
  if (vec) {
    *reinterpret_cast<uint2*>(dst) = w;
  } else {
#pragma unroll
    for (int i = 0; i < kLane; ++i)
      if (i < count) dst[i] = static_cast<uint8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
  }
}

__device__ __forceinline__ void decode(uint2 w, float (&v)[kLane]) {
#pragma unroll
  for (int i = 0; i < kLane / 2; ++i) {
    const uint16_t pair = static_cast<uint16_t>((i < 2 ? w.x : w.y) >> (16 * (i & 1)));
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(pair));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ uint2 encode(const float (&v)[kLane]) {
  uint32_t w[2] = {};
#pragma unroll
  for (int i = 0; i < kLane / 2; ++i) {
    uint16_t pair;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(pair) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
    w[i / 2] |= static_cast<uint32_t>(pair) << (16 * (i & 1));
  }
  return make_uint2(w[0], w[1]);
}

// Codes of the block's values, whose largest magnitude has the bits `top`, and
// their scale: 0 for a block of zeros, NaN (codes 0) for one that is not finite.
template <bool ROOT>
__device__ __forceinline__ uint2 quantize(float (&v)[kLane], uint32_t top, float& scale) {
  scale = top < kInfBits ? __fdiv_rn(__uint_as_float(top), kTop) : __uint_as_float(0x7FC00000u);
  const bool live = scale > 0.0f;
#pragma unroll
  for (int i = 0; i < kLane; ++i) {
    const float q = live ? __fdiv_rn(v[i], scale) : 0.0f;
    v[i] = ROOT && live && v[i] > 0.0f ? fmaxf(q, kLeast) : q;
  }
  return encode(v);
}

// The sum of `count` values in an order that depends on count alone, for all
// threads of the CTA.
__device__ __forceinline__ double sum_all(const double* sums, int count, double* red) {
  double v = 0.0;
  for (int i = threadIdx.x; i < count; i += kThreads) v += sums[i];
#pragma unroll
  for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) v += red[w];
  return v;
}

// The last tensor whose first block is not behind `block`; one with no values
// is never it, since the next begins at the same block.
template <int CAP>
__device__ __forceinline__ int find(const Table<CAP>& t, int64_t block) {
  int lo = 0, hi = t.s.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.e[mid].first <= block) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename T, int BITS, int CAP>
__global__ void __launch_bounds__(kThreads, 3) adamw_kernel(const __grid_constant__ Table<CAP> t) {
  __shared__ double red[kWarps];
  __shared__ float how[3];
  const Scalars& s = t.s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  grid_dependents_launch();
  float step_size = s.step_size, root = s.root, decay = s.decay, coef = 1.0f;
  if (s.step || s.lr) {
    if (threadIdx.x == 0) {
      const double step = s.step ? *s.step : s.host_step, lr = s.lr ? *s.lr : s.host_lr;
      how[0] = static_cast<float>(lr / -expm1(step * s.log1));
      how[1] = static_cast<float>(rsqrt(-expm1(step * s.log2)));
      how[2] = static_cast<float>(1.0 - lr * s.wd);
    }
    __syncthreads();
    step_size = how[0], root = how[1], decay = how[2];
  }
  if (s.sums) {
    const float norm = static_cast<float>(sqrt(sum_all(s.sums, s.sums_count, red)));
    const float c = __fdiv_rn(s.max_norm, __fadd_rn(norm, 1e-6f));
    coef = c >= 1.0f ? 1.0f : c;  // NaN stays
    if (s.norm && blockIdx.x == 0 && threadIdx.x == 0) *s.norm = norm;
  }
  const int64_t per = (s.blocks + gridDim.x - 1) / gridDim.x;
  const int64_t begin = per * blockIdx.x, end = begin + per < s.blocks ? begin + per : s.blocks;
  int64_t block = begin + warp;
  if (block >= end) return;
  int at = find(t, block);
  for (; block < end; block += kWarps) {
    while (at + 1 < s.count && t.e[at + 1].first <= block) ++at;
    const Entry& e = t.e[at];
    const int64_t i0 = (block - e.first) * kBlock + lane * kLane, left = e.n - i0;
    const int count = left >= kLane ? kLane : (left > 0 ? static_cast<int>(left) : 0);
    const bool vec = e.aligned && count == kLane;
    T* p_at = static_cast<T*>(e.p) + i0;
    float p[kLane], g[kLane], m[kLane], v[kLane];
    load(static_cast<const T*>(e.g) + i0, count, vec, g);
    load(p_at, count, vec, p);
    if constexpr (BITS == 32) {
      load(static_cast<const float*>(e.m) + i0, count, vec, m);
      load(static_cast<const float*>(e.v) + i0, count, vec, v);
    } else {
      const uint2 mc = load_codes(static_cast<const uint8_t*>(e.m) + i0, count, vec);
      const uint2 rc = load_codes(static_cast<const uint8_t*>(e.v) + i0, count, vec);
      const float* scales = e.scales + 2 * (block - e.first);
      const float ms = ld_f32(scales), rs = ld_f32(scales + 1);
      decode(mc, m);
      decode(rc, v);
#pragma unroll
      for (int i = 0; i < kLane; ++i) {
        m[i] = __fmul_rn(m[i], ms);
        const float r = __fmul_rn(v[i], rs);
        v[i] = __fmul_rn(r, r);
      }
    }
    float r[kLane];
#pragma unroll
    for (int i = 0; i < kLane; ++i) {
      if (s.sums) g[i] = __fmul_rn(g[i], coef);
      m[i] = __fadd_rn(__fmul_rn(m[i], s.beta1), __fmul_rn(g[i], s.rest1));
      v[i] = __fadd_rn(__fmul_rn(v[i], s.beta2), __fmul_rn(__fmul_rn(g[i], g[i]), s.rest2));
      r[i] = __fsqrt_rn(v[i]);
      p[i] = __fsub_rn(__fmul_rn(p[i], decay),
                       __fdividef(__fmul_rn(step_size, m[i]), __fadd_rn(__fmul_rn(r[i], root), s.eps)));
    }
    store(p_at, count, vec, p);
    if constexpr (BITS == 32) {
      store(static_cast<float*>(e.m) + i0, count, vec, m);
      store(static_cast<float*>(e.v) + i0, count, vec, v);
    } else {
      uint32_t m_top = 0, r_top = 0;
#pragma unroll
      for (int i = 0; i < kLane; ++i) {
        m_top = max(m_top, i < count ? abs_bits(m[i]) : 0u);
        r_top = max(r_top, i < count ? abs_bits(r[i]) : 0u);
      }
      float ms, rs;
      const uint2 mc = quantize<false>(m, warp_max(m_top), ms), rc = quantize<true>(r, warp_max(r_top), rs);
      store_codes8(static_cast<uint8_t*>(e.m) + i0, count, vec, mc);
      store_codes8(static_cast<uint8_t*>(e.v) + i0, count, vec, rc);
      if (lane == 0) {
        float* scales = e.scales + 2 * (block - e.first);
        scales[0] = ms;
        scales[1] = rs;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Sums of squares.  Eight squares are added in float32 and their sum to a
// 64-bit one; where eight squares leave the range of float32 (a sum that is not
// finite, or so small that squares may have been lost) they are formed in 64
// bits.  Each CTA writes one sum, of a share that depends on the sizes alone.

struct NormEntry {
  const void* g;
  int64_t n;
  uint32_t first;
  uint32_t aligned;
};

template <int CAP>
struct NormTable {
  int count, add;  // add: to what an earlier launch has left
  int64_t blocks;
  double* sums;
  NormEntry e[CAP];
};

template <typename T, int CAP>
__global__ void __launch_bounds__(kThreads) square_sums(const __grid_constant__ NormTable<CAP> t) {
  __shared__ double red[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  grid_dependents_launch();
  const int64_t per = (t.blocks + gridDim.x - 1) / gridDim.x;
  const int64_t begin = per * blockIdx.x, end = begin + per < t.blocks ? begin + per : t.blocks;
  int64_t block = begin + warp;
  double acc = 0.0;
  if (block < end) {
    int at = 0, hi = t.count - 1;
    while (at < hi) {
      const int mid = (at + hi + 1) / 2;
      if (t.e[mid].first <= block) at = mid;
      else hi = mid - 1;
    }
    for (; block < end; block += kWarps) {
      while (at + 1 < t.count && t.e[at + 1].first <= block) ++at;
      const NormEntry& e = t.e[at];
      const int64_t i0 = (block - e.first) * kBlock + lane * kLane, left = e.n - i0;
      const int count = left >= kLane ? kLane : (left > 0 ? static_cast<int>(left) : 0);
      float g[kLane];
      load(static_cast<const T*>(e.g) + i0, count, e.aligned && count == kLane, g);
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kLane; ++i) sum = __fmaf_rn(g[i], g[i], sum);
      double part = sum;
      if (!(sum < 0x1p120f && sum > 0x1p-90f)) {
        part = 0.0;
#pragma unroll
        for (int i = 0; i < kLane; ++i) part += static_cast<double>(g[i]) * static_cast<double>(g[i]);
      }
      acc += part;
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d /= 2) acc += __shfl_xor_sync(0xFFFFFFFFu, acc, d);
  if (lane == 0) red[warp] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double v = t.add ? t.sums[blockIdx.x] : 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += red[w];
    t.sums[blockIdx.x] = v;
  }
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double* sums, int count, float* norm) {
  __shared__ double red[kWarps];
  grid_dependency_wait();
  grid_dependents_launch();
  const double v = sum_all(sums, count, red);
  if (threadIdx.x == 0) *norm = static_cast<float>(sqrt(v));
}

// ---------------------------------------------------------------------------
// host side

namespace {

constexpr int kSmall = 32, kLarge = 512;        // tensors of a launch
constexpr int kNormSmall = 64, kNormLarge = 1024;

template <typename K, typename A>
int launch(K kernel, int64_t ctas, const A& args, cudaStream_t s, const char* what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args));
  return check_launch(what);
}

int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

template <typename T, int BITS, int CAP>
int adamw_part(const Scalars& s, const convrot_adamw_tensor* tensors, int count, cudaStream_t stream) {
  Table<CAP> t;
  t.s = s;
  t.s.count = count;
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) {
    const convrot_adamw_tensor& c = tensors[i];
    const uintptr_t moments = BITS == 8 ? 8 : 16;
    const bool aligned = aligned_to(c.param, 16) && aligned_to(c.grad, 16) && aligned_to(c.exp_avg, moments) &&
                         aligned_to(c.exp_avg_sq, moments);
    Entry& e = t.e[i];
    e.p = c.param, e.g = c.grad, e.m = c.exp_avg, e.v = c.exp_avg_sq, e.scales = c.scales, e.n = c.numel;
    e.first = static_cast<uint32_t>(blocks), e.aligned = aligned;
    blocks += blocks_of(c.numel);
  }
  if (blocks == 0) return CONVROT_OK;
  CONVROT_REQUIRE(blocks < (1LL << 32), CONVROT_ERR_UNSUPPORTED, "tensors too large");
  t.s.blocks = blocks;
  const int64_t ctas = (blocks + kWarps - 1) / kWarps, most = 3 * static_cast<int64_t>(device_sm_count());
  return launch(adamw_kernel<T, BITS, CAP>, ctas < most ? ctas : most, t, stream, "adamw step");
}

template <typename T, int BITS>
int adamw_all(const Scalars& s, const convrot_adamw_tensor* tensors, int64_t count, cudaStream_t stream) {
  for (int64_t at = 0; at < count; at += kLarge) {
    const int n = static_cast<int>(count - at < kLarge ? count - at : kLarge);
    const int rc = n <= kSmall ? adamw_part<T, BITS, kSmall>(s, tensors + at, n, stream)
                               : adamw_part<T, BITS, kLarge>(s, tensors + at, n, stream);
    if (rc != CONVROT_OK) return rc;
  }
  return CONVROT_OK;
}

template <typename T>
int adamw_bits(int bits, const Scalars& s, const convrot_adamw_tensor* tensors, int64_t count, cudaStream_t stream) {
  return bits == 8 ? adamw_all<T, 8>(s, tensors, count, stream) : adamw_all<T, 32>(s, tensors, count, stream);
}

template <typename T, int CAP>
int sums_part(const convrot_grad_tensor* tensors, int count, int64_t ctas, double* sums, bool add, cudaStream_t stream) {
  NormTable<CAP> t;
  t.count = count, t.add = add, t.sums = sums;
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) {
    t.e[i].g = tensors[i].grad, t.e[i].n = tensors[i].numel;
    t.e[i].first = static_cast<uint32_t>(blocks), t.e[i].aligned = aligned_to(tensors[i].grad, 16);
    blocks += blocks_of(tensors[i].numel);
  }
  CONVROT_REQUIRE(blocks < (1LL << 32), CONVROT_ERR_UNSUPPORTED, "tensors too large");
  t.blocks = blocks;
  return launch(square_sums<T, CAP>, ctas, t, stream, "sums of squares");
}

template <typename T>
int sums_all(const convrot_grad_tensor* tensors, int64_t count, int64_t ctas, double* sums, cudaStream_t stream) {
  for (int64_t at = 0; at < count || at == 0; at += kNormLarge) {
    const int n = static_cast<int>(count - at < kNormLarge ? count - at : kNormLarge);
    const int rc = n <= kNormSmall ? sums_part<T, kNormSmall>(tensors + at, n, ctas, sums, at > 0, stream)
                                   : sums_part<T, kNormLarge>(tensors + at, n, ctas, sums, at > 0, stream);
    if (rc != CONVROT_OK) return rc;
  }
  return CONVROT_OK;
}

}  // namespace
}  // namespace optim
}  // namespace convrot

extern "C" {

int64_t convrot_square_sums_count(int64_t count, const convrot_grad_tensor* tensors) {
  using namespace convrot;
  if (count < 0 || (count > 0 && !tensors)) return 1;
  int64_t blocks = 0;
  for (int64_t i = 0; i < count; ++i) blocks += tensors[i].numel > 0 ? optim::blocks_of(tensors[i].numel) : 0;
  const int64_t ctas = (blocks + optim::kWarps - 1) / optim::kWarps, most = 4 * static_cast<int64_t>(device_sm_count());
  return ctas < 1 ? 1 : (ctas < most ? ctas : most);
}

int convrot_square_sums(int64_t count, const convrot_grad_tensor* tensors, int dtype, double* sums, int64_t sums_count,
                        void* stream) {
  using namespace convrot;
  CONVROT_REQUIRE(valid_dtype(dtype), CONVROT_ERR_INVALID, "unknown dtype %d", dtype);
  CONVROT_REQUIRE(count >= 0 && (count == 0 || tensors) && sums && aligned_to(sums, 8) && sums_count > 0 &&
                      sums_count <= (1 << 20),
                  CONVROT_ERR_INVALID, "invalid tensor list or sums");
  for (int64_t i = 0; i < count; ++i)
    CONVROT_REQUIRE(tensors[i].numel >= 0 &&
                        (tensors[i].numel == 0 || (tensors[i].grad && aligned_to(tensors[i].grad, dtype_size(dtype)))),
                    CONVROT_ERR_INVALID, "tensor %lld: null or misaligned pointer, or negative size", static_cast<long long>(i));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CONVROT_BF16: return optim::sums_all<__nv_bfloat16>(tensors, count, sums_count, sums, s);
    case CONVROT_F16: return optim::sums_all<__half>(tensors, count, sums_count, sums, s);
    default: return optim::sums_all<float>(tensors, count, sums_count, sums, s);
  }
}

int convrot_norm_of_sums(const double* sums, int64_t sums_count, float* norm, void* stream) {
  using namespace convrot;
  CONVROT_REQUIRE(sums && norm && sums_count > 0 && sums_count <= (1 << 24), CONVROT_ERR_INVALID, "invalid sums");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1, 1, 1);
  cfg.blockDim = dim3(optim::kThreads, 1, 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, optim::norm_kernel, sums, static_cast<int>(sums_count), norm));
  return check_launch("norm of sums");
}

int convrot_adamw(int64_t count, const convrot_adamw_tensor* tensors, int dtype, int state_bits,
                  const convrot_adamw_options* o, void* stream) {
  using namespace convrot;
  CONVROT_REQUIRE(valid_dtype(dtype), CONVROT_ERR_INVALID, "unknown dtype %d", dtype);
  CONVROT_REQUIRE(state_bits == 8 || state_bits == 32, CONVROT_ERR_INVALID, "moments are kept in 8 or 32 bits, not %d",
                  state_bits);
  CONVROT_REQUIRE(count >= 0 && (count == 0 || tensors) && o, CONVROT_ERR_INVALID, "null tensor list or options");
  CONVROT_REQUIRE(o->beta1 >= 0 && o->beta1 < 1 && o->beta2 >= 0 && o->beta2 < 1 && o->eps >= 0 && o->weight_decay >= 0,
                  CONVROT_ERR_INVALID, "betas must be in [0, 1), eps and weight decay non-negative");
  CONVROT_REQUIRE((o->step_device || o->step >= 1) && (o->lr_device || o->lr >= 0), CONVROT_ERR_INVALID,
                  "the step counts from 1 and the learning rate is non-negative");
  CONVROT_REQUIRE(!o->sums || (o->sums_count > 0 && o->sums_count <= (1 << 24) && o->max_norm >= 0), CONVROT_ERR_INVALID,
                  "clipping needs sums of squares and a non-negative norm");
  for (int64_t i = 0; i < count; ++i) {
    const convrot_adamw_tensor& t = tensors[i];
    const uintptr_t e = dtype_size(dtype), moment = state_bits == 8 ? 1 : 4;
    CONVROT_REQUIRE(t.numel >= 0 && (t.numel == 0 || (t.param && t.grad && t.exp_avg && t.exp_avg_sq && aligned_to(t.param, e) &&
                                                      aligned_to(t.grad, e) && aligned_to(t.exp_avg, moment) &&
                                                      aligned_to(t.exp_avg_sq, moment))),
                    CONVROT_ERR_INVALID, "tensor %lld: null or misaligned pointer, or negative size", static_cast<long long>(i));
    CONVROT_REQUIRE(state_bits == 32 || t.numel == 0 || (t.scales && aligned_to(t.scales, 4)), CONVROT_ERR_INVALID,
                    "tensor %lld: 8-bit moments need their scales", static_cast<long long>(i));
  }
  const double c1 = 1.0 - pow(o->beta1, o->step), c2 = 1.0 - pow(o->beta2, o->step);
  optim::Scalars s = {};
  s.decay = static_cast<float>(1.0 - o->lr * o->weight_decay);
  s.beta1 = static_cast<float>(o->beta1);
  s.beta2 = static_cast<float>(o->beta2);
  s.rest1 = static_cast<float>(1.0 - o->beta1);
  s.rest2 = static_cast<float>(1.0 - o->beta2);
  s.eps = static_cast<float>(o->eps);
  s.step_size = static_cast<float>(o->lr / c1);
  s.root = static_cast<float>(1.0 / sqrt(c2));
  s.step = o->step_device;
  s.lr = o->lr_device;
  s.log1 = log(o->beta1);
  s.log2 = log(o->beta2);
  s.wd = o->weight_decay;
  s.host_lr = static_cast<float>(o->lr);
  s.host_step = static_cast<float>(o->step);
  s.sums = o->sums;
  s.sums_count = static_cast<int>(o->sums_count);
  s.max_norm = static_cast<float>(o->max_norm);
  s.norm = o->norm;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CONVROT_BF16: return optim::adamw_bits<__nv_bfloat16>(state_bits, s, tensors, count, st);
    case CONVROT_F16: return optim::adamw_bits<__half>(state_bits, s, tensors, count, st);
    default: return optim::adamw_bits<float>(state_bits, s, tensors, count, st);
  }
}

}  // extern "C"
