// Layer norm over the features of a row, forward and backward, with the
// reduction of the gradients of its weight and bias (kernels and formulas in
// layer_norm.cuh).  Rows come in segments of rows_per_weight rows; segment s
// reads its weight and bias at s * weight_stride, so one kernel serves the
// affine norm (one segment) and the modulated norm of a DiT block (a scale and
// a shift for each sample).  All arithmetic is float32; each output is rounded
// once.
#include "layer_norm.cuh"

namespace convrot {
namespace norm {
namespace {

// dweight and dbias: the chunks' sums added up, COLS columns a CTA, 512 / COLS
// threads for each column that take every so many-th chunk, then a tree.
template <typename TW, int COLS>
__global__ void __launch_bounds__(512) norm_reduce_kernel(const NormParams p) {
  constexpr int kWays = 512 / COLS;
  __shared__ float sw[kWays][COLS + 1], sb[kWays][COLS + 1];
  grid_dependency_wait();
  grid_dependents_launch();
  const int F = p.features;
  const int x = threadIdx.x % COLS, y = threadIdx.x / COLS;
  const int c = blockIdx.x * COLS + x;
  const int64_t seg = blockIdx.y;
  float dw = 0.0f, db = 0.0f;
  if (c < F) {
    const float* part = p.partial + seg * p.chunks * 2 * F + c;
#pragma unroll 4
    for (int chunk = y; chunk < p.chunks; chunk += kWays) {
      dw += ld_f32(part + static_cast<int64_t>(chunk) * 2 * F);
      db += ld_f32(part + static_cast<int64_t>(chunk) * 2 * F + F);
    }
  }
  sw[y][x] = dw;
  sb[y][x] = db;
  __syncthreads();
#pragma unroll
  for (int o = kWays / 2; o > 0; o >>= 1) {
    if (y < o) {
      sw[y][x] += sw[y + o][x];
      sb[y][x] += sb[y + o][x];
    }
    __syncthreads();
  }
  if (y == 0 && c < F) {
    if (p.dweight) static_cast<TW*>(p.dweight)[seg * F + c] = Elem<TW>::from_f(sw[0][x]);
    if (p.dbias) static_cast<TW*>(p.dbias)[seg * F + c] = Elem<TW>::from_f(sb[0][x]);
  }
}

// CTAs that share a segment's rows, each with one partial sum: as many as the
// GPU holds at once (fewer for wide rows, whose CTAs and sums are large), and
// two rows each at least.
int chunks_of(int64_t rows_per_weight, int64_t segments, int64_t features) {
  const int64_t per_sm = features <= 3072 ? 3 : features <= 8192 ? 2 : 1;
  int64_t chunks = per_sm * device_sm_count() / segments;
  if (chunks > rows_per_weight / 2) chunks = rows_per_weight / 2;
  return static_cast<int>(chunks < 1 ? 1 : chunks);
}

// Many chunks: few columns a CTA, so that there are CTAs and threads enough.
template <typename TW>
int reduce(const NormParams& p, cudaStream_t s) {
  const bool many = p.chunks > 64;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.features + (many ? 7 : 31)) / (many ? 8 : 32),
                     static_cast<unsigned>(p.rows / p.rows_per_weight), 1);
  cfg.blockDim = dim3(512, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, many ? norm_reduce_kernel<TW, 8> : norm_reduce_kernel<TW, 32>, p));
  return check_launch("layer norm reduction");
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
}  // namespace norm
}  // namespace convrot

extern "C" {

int convrot_layer_norm(const void* x, int dtype, int64_t rows, int64_t features, const void* weight, const void* bias,
                       int weight_dtype, int64_t rows_per_weight, int64_t weight_stride, int add_one, float eps,
                       void* y, float* mean, float* rstd, void* stream) {
  using namespace convrot;
  using namespace convrot::norm;
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
  p.wide_weight = dtype != CONVROT_F32 && weight_dtype == CONVROT_F32;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CONVROT_BF16: return forward<__nv_bfloat16>(p, s);
    case CONVROT_F16: return forward<__half>(p, s);
    default: return forward<float>(p, s);
  }
}

int64_t convrot_layer_norm_workspace(int64_t rows, int64_t features, int64_t rows_per_weight) {
  using namespace convrot;
  using namespace convrot::norm;
  if (rows <= 0 || features <= 0 || rows_per_weight <= 0) return 0;
  const int64_t segments = rows / rows_per_weight;
  return segments * chunks_of(rows_per_weight, segments, features) * 2 * features * static_cast<int64_t>(sizeof(float));
}

int convrot_layer_norm_backward(const void* x, const void* dy, int dtype, int64_t rows, int64_t features,
                                const void* weight, int weight_dtype, int64_t rows_per_weight, int64_t weight_stride,
                                int add_one, const float* mean, const float* rstd, void* dx, void* dweight,
                                void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace convrot;
  using namespace convrot::norm;
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
  p.partial = sums ? static_cast<float*>(workspace) : nullptr;
  p.rows = rows;
  p.rows_per_weight = rows_per_weight;
  p.weight_stride = weight_stride;
  p.features = static_cast<int>(features);
  p.chunks = chunks_of(rows_per_weight, rows / rows_per_weight, features);
  p.add_one = add_one;
  p.wide_weight = dtype != CONVROT_F32 && weight_dtype == CONVROT_F32;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int launched = dtype == CONVROT_BF16  ? backward<__nv_bfloat16>(p, s)
                       : dtype == CONVROT_F16 ? backward<__half>(p, s)
                                              : backward<float>(p, s);
  if (launched != CONVROT_OK || !sums) return launched;
  switch (weight_dtype) {
    case CONVROT_BF16: return reduce<__nv_bfloat16>(p, s);
    case CONVROT_F16: return reduce<__half>(p, s);
    default: return reduce<float>(p, s);
  }
}

}  // extern "C"
