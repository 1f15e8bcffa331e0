// Quantizers of the 8-bit floating-point linear.  A block of values shares one
// scale 2^e, e the least exponent with max|x| <= 448 * 2^e (448 is the largest
// e4m3 value), kept as the biased byte e + 127 (e >= -127); a value's code is
// e4m3(x * 2^-e), to nearest even.  The scale is a power of two, so the
// multiplication is exact and codes do not depend on how they are computed;
// e4m3 has its own exponent, so nothing of its precision is lost to it.
// A zero block has scale 2^-127 and codes 0; a block that holds an infinity or
// a NaN has the scale byte 255, which stands for NaN, and codes 0.
//
// Activations: blocks of 128 consecutive values of a row.  Eight threads a
// block, 16 values a thread: 16 codes are one 16-byte store, and the maximum
// is three exchanges.  Memory-bound: 7800 x 5120 bf16 in 18.6 us (6.4 TB/s, a
// copy's 6.6; 23.9 with a select and a product for each value instead of paired
// products), 1536 x 5120 in 3.9, 451 x 2203, whose rows start at any byte pair and
// are read value by value, in 2.5.  Weights: blocks of 128 x 128, a CTA each, once
// for a layer (13824 x 5120 in 32.5 us, 6.5 TB/s).
#include "fp8.cuh"

namespace convrot {
namespace fp8 {

constexpr int kThreads = 256;

struct QuantParams {
  const void* x;
  uint8_t* codes;
  uint8_t* scales;
  int64_t rows, x_stride, codes_stride, scales_stride;
  int features, spans;
};

// WHOLE: rows start on multiples of 16 bytes.
template <typename T, bool WHOLE>
__global__ void __launch_bounds__(kThreads) quantize_rows(const QuantParams p) {
  grid_dependency_wait();
  grid_dependents_launch();
  const uint32_t unit = blockIdx.x * (kThreads / kSpanThreads) + threadIdx.x / kSpanThreads;
  const uint32_t row = unit / static_cast<uint32_t>(p.spans), span = unit - row * p.spans;
  const bool live = row < p.rows;
  const int c = static_cast<int>(span) * kSpan + static_cast<int>(threadIdx.x % kSpanThreads) * kChunk;
  Pack<T, kChunk> w;
  w.clear();
  if (live) load_chunk<T, WHOLE>(static_cast<const T*>(p.x) + static_cast<int64_t>(row) * p.x_stride, c, p.features, w);
  const uint32_t top = span_max(w.top());
  if (!live) return;
  const uint32_t byte = scale_byte(top);
  // rows of codes are on a pitch of a multiple of 16 bytes: a chunk that begins inside a row ends inside its pitch
  P2 v[kChunk / 2];
  w.get_lanes(v);
  if (c < p.features)
    *reinterpret_cast<uint4*>(p.codes + static_cast<int64_t>(row) * p.codes_stride + c) = codes_of(v, byte);
  if (threadIdx.x % kSpanThreads == 0)
    p.scales[static_cast<int64_t>(row) * p.scales_stride + span] = static_cast<uint8_t>(byte);
}

template <typename T, bool WHOLE>
__global__ void __launch_bounds__(kThreads) quantize_blocks(const QuantParams p) {
  constexpr int kRowsAt = kThreads / kSpanThreads, kTurns = kSpan / kRowsAt;
  __shared__ uint32_t red[kThreads / 32];
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * kSpan + threadIdx.x / kSpanThreads;
  const int c = blockIdx.x * kSpan + static_cast<int>(threadIdx.x % kSpanThreads) * kChunk;
  Pack<T, kChunk> w[kTurns];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int64_t row = row0 + i * kRowsAt;
    w[i].clear();
    if (row < p.rows) load_chunk<T, WHOLE>(static_cast<const T*>(p.x) + row * p.x_stride, c, p.features, w[i]);
  }
#pragma unroll
  for (int i = 0; i < kTurns; ++i) top = max(top, w[i].top());
  top = warp_max(top);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = top;
  __syncthreads();
  top = warp_max(red[threadIdx.x % (kThreads / 32)]);
  const uint32_t byte = scale_byte(top);
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int64_t row = row0 + i * kRowsAt;
    P2 v[kChunk / 2];
    w[i].get_lanes(v);
    if (row < p.rows && c < p.features)
      *reinterpret_cast<uint4*>(p.codes + row * p.codes_stride + c) = codes_of(v, byte);
  }
  if (threadIdx.x == 0) p.scales[blockIdx.y * p.scales_stride + blockIdx.x] = static_cast<uint8_t>(byte);
}

namespace {

int check(const void* x, int dtype, int64_t rows, int64_t features, int64_t x_stride, const uint8_t* codes,
          int64_t codes_stride, const uint8_t* scales, int64_t scales_stride) {
  CONVROT_REQUIRE(valid_dtype(dtype), CONVROT_ERR_INVALID, "unknown dtype %d", dtype);
  CONVROT_REQUIRE(rows >= 0 && features > 0, CONVROT_ERR_INVALID, "invalid shape rows=%lld features=%lld",
                  static_cast<long long>(rows), static_cast<long long>(features));
  const int64_t spans = (features + kSpan - 1) / kSpan;
  CONVROT_REQUIRE(features < (1LL << 30) && rows < (1LL << 30) && rows * spans < (1LL << 31), CONVROT_ERR_UNSUPPORTED,
                  "shape too large");
  CONVROT_REQUIRE(x_stride >= features && codes_stride >= features && codes_stride % 16 == 0 && scales_stride >= spans,
                  CONVROT_ERR_INVALID, "row strides must cover the rows, those of codes in multiples of 16 bytes");
  if (rows == 0) return CONVROT_OK;
  CONVROT_REQUIRE(x && codes && scales, CONVROT_ERR_INVALID, "null pointer");
  CONVROT_REQUIRE(aligned_to(codes, 16) && aligned_to(x, dtype_size(dtype)), CONVROT_ERR_INVALID,
                  "codes must be 16-byte aligned, the input aligned to its elements");
  return CONVROT_OK;
}

template <typename T>
bool whole(const QuantParams& p) {
  return aligned_to(p.x, 16) && p.x_stride * sizeof(T) % 16 == 0;
}

template <typename T>
int launch_rows(const QuantParams& p, cudaStream_t s) {
  const int64_t units = p.rows * p.spans, per = kThreads / kSpanThreads;
  auto kernel = whole<T>(p) ? quantize_rows<T, true> : quantize_rows<T, false>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((units + per - 1) / per), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p));
  return check_launch("8-bit float quantizer");
}

template <typename T>
int launch_blocks(const QuantParams& p, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(p.spans), static_cast<unsigned>((p.rows + kSpan - 1) / kSpan));
  if (whole<T>(p)) quantize_blocks<T, true><<<grid, kThreads, 0, s>>>(p);
  else quantize_blocks<T, false><<<grid, kThreads, 0, s>>>(p);
  return check_launch("8-bit float weight quantizer");
}

}  // namespace
}  // namespace fp8
}  // namespace convrot

extern "C" {

int convrot_quantize_fp8(const void* x, int dtype, int64_t rows, int64_t features, int64_t x_stride, uint8_t* codes,
                         int64_t codes_stride, uint8_t* scales, int64_t scales_stride, void* stream) {
  using namespace convrot;
  const int rc = fp8::check(x, dtype, rows, features, x_stride, codes, codes_stride, scales, scales_stride);
  if (rc != CONVROT_OK || rows == 0) return rc;
  const fp8::QuantParams p{x, codes, scales, rows, x_stride, codes_stride, scales_stride, static_cast<int>(features),
                           static_cast<int>((features + fp8::kSpan - 1) / fp8::kSpan)};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CONVROT_BF16: return fp8::launch_rows<__nv_bfloat16>(p, s);
    case CONVROT_F16: return fp8::launch_rows<__half>(p, s);
    default: return fp8::launch_rows<float>(p, s);
  }
}

int convrot_quantize_fp8_weight(const void* w, int dtype, int64_t rows, int64_t features, int64_t w_stride,
                                uint8_t* codes, int64_t codes_stride, uint8_t* scales, int64_t scales_stride,
                                void* stream) {
  using namespace convrot;
  const int rc = fp8::check(w, dtype, rows, features, w_stride, codes, codes_stride, scales, scales_stride);
  if (rc != CONVROT_OK || rows == 0) return rc;
  CONVROT_REQUIRE(rows <= 65535 * fp8::kSpan, CONVROT_ERR_UNSUPPORTED, "shape too large");
  const fp8::QuantParams p{w, codes, scales, rows, w_stride, codes_stride, scales_stride, static_cast<int>(features),
                           static_cast<int>((features + fp8::kSpan - 1) / fp8::kSpan)};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CONVROT_BF16: return fp8::launch_blocks<__nv_bfloat16>(p, s);
    case CONVROT_F16: return fp8::launch_blocks<__half>(p, s);
    default: return fp8::launch_blocks<float>(p, s);
  }
}

}  // extern "C"
