// Layer norm over the features of a row, forward and backward, with the
// reduction of the gradients of its weight and bias.
//   mean = E[x], r = (E[(x - mean)^2] + eps)^-1/2, h = (x - mean) r
//   y  = h w + b                         (w = 1 + weight with add_one)
//   g  = dy w
//   dx = r (g - E[g] - h E[g h])
//   dweight = sum dy h,  dbias = sum dy  (over the rows that share a weight)
// Rows come in segments of rows_per_weight rows; segment s reads its weight
// and bias at s * weight_stride, so one kernel serves the affine norm (one
// segment) and the modulated norm of a DiT block (a scale and a shift for
// each sample).  All arithmetic is float32; each output is rounded once.
//
// Memory-bound: forward reads and writes a row once; backward reads x and dy
// and writes dx.
#include "rows.cuh"

namespace convrot {
namespace {

struct NormParams {
  const void* x;
  const void* dy;
  const void* weight;
  const void* bias;
  void* y;   // dx in the backward pass
  float* mean;
  float* rstd;
  void* dweight;
  void* dbias;
  float* partial;  // (segments, chunks, 2, features)
  int64_t rows, rows_per_weight, weight_stride;
  int features, chunks, add_one;
  float eps;
};

__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += red[w];
  return s;
}

template <typename TW>
__device__ __forceinline__ float weight_at(const NormParams& p, int64_t segment, int c) {
  const float w = p.weight ? Elem<TW>::to_f(static_cast<const TW*>(p.weight)[segment * p.weight_stride + c])
                           : (p.add_one ? 0.0f : 1.0f);
  return p.add_one ? 1.0f + w : w;
}

template <typename T, typename TW>
__global__ void __launch_bounds__(256) norm_fwd_kernel(const NormParams p) {
  __shared__ float red[8];
  const int F = p.features;
  const float inv = 1.0f / static_cast<float>(F);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * F;
    T* y = static_cast<T*>(p.y) + row * F;
    const int64_t seg = row / p.rows_per_weight;
    float s = 0.0f;
    for (int c = threadIdx.x; c < F; c += 256) s += Elem<T>::to_f(x[c]);
    const float mean = block_sum(s, red) * inv;
    s = 0.0f;
    for (int c = threadIdx.x; c < F; c += 256) {
      const float d = Elem<T>::to_f(x[c]) - mean;
      s = fmaf(d, d, s);
    }
    const float rstd = rsqrtf(block_sum(s, red) * inv + p.eps);
    if (threadIdx.x == 0 && p.mean) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    for (int c = threadIdx.x; c < F; c += 256) {
      const float b = p.bias ? Elem<TW>::to_f(static_cast<const TW*>(p.bias)[seg * p.weight_stride + c]) : 0.0f;
      y[c] = Elem<T>::from_f(fmaf((Elem<T>::to_f(x[c]) - mean) * rstd, weight_at<TW>(p, seg, c), b));
    }
  }
}

template <typename T, typename TW>
__global__ void __launch_bounds__(256) norm_dx_kernel(const NormParams p) {
  __shared__ float red[8];
  const int F = p.features;
  const float inv = 1.0f / static_cast<float>(F);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * F;
    const T* dy = static_cast<const T*>(p.dy) + row * F;
    T* dx = static_cast<T*>(p.y) + row * F;
    const int64_t seg = row / p.rows_per_weight;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float sg = 0.0f, sgh = 0.0f;
    for (int c = threadIdx.x; c < F; c += 256) {
      const float g = Elem<T>::to_f(dy[c]) * weight_at<TW>(p, seg, c);
      sg += g;
      sgh = fmaf(g, (Elem<T>::to_f(x[c]) - mean) * rstd, sgh);
    }
    const float mg = block_sum(sg, red) * inv, mgh = block_sum(sgh, red) * inv;
    for (int c = threadIdx.x; c < F; c += 256) {
      const float g = Elem<T>::to_f(dy[c]) * weight_at<TW>(p, seg, c);
      const float h = (Elem<T>::to_f(x[c]) - mean) * rstd;
      dx[c] = Elem<T>::from_f(rstd * (g - mg - h * mgh));
    }
  }
}

// Partial sums of one chunk of a segment's rows, one thread for a column.
template <typename T>
__global__ void __launch_bounds__(256) norm_partial_kernel(const NormParams p) {
  const int F = p.features;
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= F) return;
  const int64_t part = blockIdx.y, seg = part / p.chunks, chunk = part % p.chunks;
  const int64_t r0 = seg * p.rows_per_weight + p.rows_per_weight * chunk / p.chunks;
  const int64_t r1 = seg * p.rows_per_weight + p.rows_per_weight * (chunk + 1) / p.chunks;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = r0; row < r1; ++row) {
    const float d = Elem<T>::to_f(static_cast<const T*>(p.dy)[row * F + c]);
    dw = fmaf(d, (Elem<T>::to_f(static_cast<const T*>(p.x)[row * F + c]) - p.mean[row]) * p.rstd[row], dw);
    db += d;
  }
  p.partial[(part * 2) * F + c] = dw;
  p.partial[(part * 2 + 1) * F + c] = db;
}

template <typename TW>
__global__ void __launch_bounds__(256) norm_reduce_kernel(const NormParams p) {
  const int F = p.features;
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= F) return;
  const int64_t seg = blockIdx.y;
  float dw = 0.0f, db = 0.0f;
  for (int chunk = 0; chunk < p.chunks; ++chunk) {
    const float* part = p.partial + ((seg * p.chunks + chunk) * 2) * F;
    dw += part[c];
    db += part[F + c];
  }
  if (p.dweight) static_cast<TW*>(p.dweight)[seg * F + c] = Elem<TW>::from_f(dw);
  if (p.dbias) static_cast<TW*>(p.dbias)[seg * F + c] = Elem<TW>::from_f(db);
}

// Row chunks that share one partial sum: enough for the whole GPU.
int chunks_of(int64_t rows_per_weight, int64_t segments) {
  int64_t chunks = (2LL * device_sm_count() + segments - 1) / segments;
  if (chunks > rows_per_weight) chunks = rows_per_weight;
  return static_cast<int>(chunks < 1 ? 1 : chunks);
}

template <typename T, typename TW>
int forward(const NormParams& p, cudaStream_t s) {
  const int64_t most = 8LL * device_sm_count();
  norm_fwd_kernel<T, TW><<<static_cast<unsigned>(p.rows < most ? p.rows : most), 256, 0, s>>>(p);
  return check_launch("convrot_layer_norm");
}

template <typename T, typename TW>
int backward(const NormParams& p, cudaStream_t s) {
  const int64_t most = 8LL * device_sm_count();
  norm_dx_kernel<T, TW><<<static_cast<unsigned>(p.rows < most ? p.rows : most), 256, 0, s>>>(p);
  if (p.dweight || p.dbias) {
    const unsigned cols = (p.features + 255) / 256;
    const unsigned segments = static_cast<unsigned>(p.rows / p.rows_per_weight);
    norm_partial_kernel<T><<<dim3(cols, segments * p.chunks), 256, 0, s>>>(p);
    norm_reduce_kernel<TW><<<dim3(cols, segments), 256, 0, s>>>(p);
  }
  return check_launch("convrot_layer_norm_backward");
}

int check_shape(int dtype, int64_t rows, int64_t features, int weight_dtype, int64_t rows_per_weight,
                int64_t weight_stride) {
  CONVROT_REQUIRE(valid_dtype(dtype), CONVROT_ERR_INVALID, "unknown dtype %d", dtype);
  CONVROT_REQUIRE(weight_dtype == dtype || weight_dtype == CONVROT_F32, CONVROT_ERR_INVALID,
                  "the weight's dtype must be float32 or that of x");
  CONVROT_REQUIRE(rows >= 0 && features > 0 && features <= (1 << 20), CONVROT_ERR_INVALID, "invalid shape (%lld, %lld)",
                  static_cast<long long>(rows), static_cast<long long>(features));
  CONVROT_REQUIRE(rows_per_weight > 0 && rows % rows_per_weight == 0 && rows / rows_per_weight <= 65535,
                  CONVROT_ERR_INVALID, "%lld rows are not 0 to 65535 segments of %lld", static_cast<long long>(rows),
                  static_cast<long long>(rows_per_weight));
  CONVROT_REQUIRE(weight_stride >= features || rows <= rows_per_weight, CONVROT_ERR_INVALID,
                  "the weight stride %lld must cover the features", static_cast<long long>(weight_stride));
  return CONVROT_OK;
}

}  // namespace
}  // namespace convrot

#define CONVROT_NORM_DISPATCH(FN)                                                      \
  switch (dtype) {                                                                     \
    case CONVROT_BF16:                                                                 \
      return weight_dtype == CONVROT_F32 ? FN<__nv_bfloat16, float>(p, s)              \
                                         : FN<__nv_bfloat16, __nv_bfloat16>(p, s);     \
    case CONVROT_F16:                                                                  \
      return weight_dtype == CONVROT_F32 ? FN<__half, float>(p, s) : FN<__half, __half>(p, s); \
    default: return FN<float, float>(p, s);                                            \
  }

extern "C" {

int convrot_layer_norm(const void* x, int dtype, int64_t rows, int64_t features, const void* weight, const void* bias,
                       int weight_dtype, int64_t rows_per_weight, int64_t weight_stride, int add_one, float eps,
                       void* y, float* mean, float* rstd, void* stream) {
  using namespace convrot;
  const int rc = check_shape(dtype, rows, features, weight_dtype, rows_per_weight, weight_stride);
  if (rc != CONVROT_OK || rows == 0) return rc;
  CONVROT_REQUIRE(eps >= 0.0f, CONVROT_ERR_INVALID, "eps must be non-negative");
  CONVROT_REQUIRE(x && y && (mean != nullptr) == (rstd != nullptr), CONVROT_ERR_INVALID, "null pointer");
  NormParams p = {};
  p.x = x;
  p.weight = weight;
  p.bias = bias;
  p.y = y;
  p.mean = mean;
  p.rstd = rstd;
  p.rows = rows;
  p.rows_per_weight = rows_per_weight;
  p.weight_stride = weight_stride;
  p.features = static_cast<int>(features);
  p.add_one = add_one;
  p.eps = eps;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  CONVROT_NORM_DISPATCH(forward)
}

int64_t convrot_layer_norm_workspace(int64_t rows, int64_t features, int64_t rows_per_weight) {
  using namespace convrot;
  if (rows <= 0 || features <= 0 || rows_per_weight <= 0) return 0;
  const int64_t segments = rows / rows_per_weight;
  return segments * chunks_of(rows_per_weight, segments) * 2 * features * static_cast<int64_t>(sizeof(float));
}

int convrot_layer_norm_backward(const void* x, const void* dy, int dtype, int64_t rows, int64_t features,
                                const void* weight, int weight_dtype, int64_t rows_per_weight, int64_t weight_stride,
                                int add_one, const float* mean, const float* rstd, void* dx, void* dweight,
                                void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace convrot;
  const int rc = check_shape(dtype, rows, features, weight_dtype, rows_per_weight, weight_stride);
  if (rc != CONVROT_OK || rows == 0) return rc;
  CONVROT_REQUIRE(x && dy && dx && mean && rstd, CONVROT_ERR_INVALID, "null pointer");
  const bool sums = dweight || dbias;
  CONVROT_REQUIRE(!sums || (workspace && aligned_to(workspace, 16) &&
                            workspace_bytes >= convrot_layer_norm_workspace(rows, features, rows_per_weight)),
                  CONVROT_ERR_INVALID, "the workspace is too small or not 16-byte aligned");
  NormParams p = {};
  p.x = x;
  p.dy = dy;
  p.weight = weight;
  p.y = dx;
  p.mean = const_cast<float*>(mean);
  p.rstd = const_cast<float*>(rstd);
  p.dweight = dweight;
  p.dbias = dbias;
  p.partial = static_cast<float*>(workspace);
  p.rows = rows;
  p.rows_per_weight = rows_per_weight;
  p.weight_stride = weight_stride;
  p.features = static_cast<int>(features);
  p.chunks = chunks_of(rows_per_weight, rows / rows_per_weight);
  p.add_one = add_one;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  CONVROT_NORM_DISPATCH(backward)
}

}  // extern "C"
