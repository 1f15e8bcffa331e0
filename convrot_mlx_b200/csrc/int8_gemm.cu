// 8-bit integer matrix product with one scale for each token (row of the
// activation) and one for each channel (row of the weight):
//   out[m, n] = T(fl(fl(float(sum_k a[m, k] w[n, k]) * xs[m]) * ws[n]) + bias[n]),
// with an exact int32 dot (K <= 131072: |dot| <= 127 * 127 K < 2^31).
// Layout NK reads w as (n, k) rows, the forward product; layout KN reads it
// as (k, n) rows: the same weight matrix contracted over its rows, the
// product of the input's gradient.
#include "rows.cuh"

namespace convrot {
namespace {

constexpr int kMaxK = 131072;
constexpr int kTile = 64;   // rows and columns of a tile
constexpr int kStep = 64;   // K bytes of a step

struct I8Params {
  const int8_t* act;
  const int8_t* weight;
  const float* xscales;
  const float* wscales;
  const float* bias;
  void* out;
  int64_t act_stride, weight_stride;
  int m, n, k;
};

// 256 threads, 4 x 4 outputs each; both operands as words of 4 consecutive k
// in shared memory.
template <int LAYOUT, typename TOut>
__global__ void __launch_bounds__(256) i8_gemm_kernel(const I8Params p) {
  __shared__ int8_t sa[kTile][kStep + 4];
  __shared__ int8_t sb[kTile][kStep + 4];
  const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < p.k; k0 += kStep) {
    for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
      const int r = i / kStep, c = i % kStep;
      sa[r][c] = m0 + r < p.m && k0 + c < p.k ? p.act[(m0 + r) * p.act_stride + k0 + c] : 0;
      if (LAYOUT == CONVROT_LAYOUT_NK) {
        sb[r][c] = n0 + r < p.n && k0 + c < p.k ? p.weight[(n0 + r) * p.weight_stride + k0 + c] : 0;
      } else {  // row r of the step is k, column c of the tile is n
        sb[c][r] = n0 + c < p.n && k0 + r < p.k ? p.weight[(k0 + r) * p.weight_stride + n0 + c] : 0;
      }
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < kStep; kk += 4) {
      int a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = *reinterpret_cast<const int*>(&sa[ty + 16 * i][kk]);
        b[i] = *reinterpret_cast<const int*>(&sb[tx + 16 * i][kk]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
  TOut* out = static_cast<TOut*>(p.out);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m < p.m && n < p.n) {
        float v = __fmul_rn(__int2float_rn(acc[i][j]), p.xscales[m]);
        if (p.wscales) v = __fmul_rn(v, p.wscales[n]);
        if (p.bias) v = __fadd_rn(v, p.bias[n]);
        out[static_cast<int64_t>(m) * p.n + n] = cvt_out<TOut>(v);
      }
    }
}

template <int LAYOUT, typename TOut>
int launch(const I8Params& p, cudaStream_t stream) {
  const dim3 grid((p.n + kTile - 1) / kTile, (p.m + kTile - 1) / kTile);
  i8_gemm_kernel<LAYOUT, TOut><<<grid, 256, 0, stream>>>(p);
  return check_launch("convrot_i8_gemm");
}

}  // namespace
}  // namespace convrot

extern "C" {

int convrot_i8_gemm(const int8_t* act, int64_t act_stride, const int8_t* weight, int64_t weight_stride, int layout,
                    const float* xscales, const float* wscales, const float* bias, void* out, int out_dtype, int64_t m,
                    int64_t n, int64_t k, void* stream) {
  using namespace convrot;
  CONVROT_REQUIRE(layout == CONVROT_LAYOUT_NK || layout == CONVROT_LAYOUT_KN, CONVROT_ERR_INVALID, "unknown layout %d",
                  layout);
  CONVROT_REQUIRE(valid_dtype(out_dtype), CONVROT_ERR_INVALID, "unknown output dtype %d", out_dtype);
  CONVROT_REQUIRE(m >= 0 && n > 0 && k > 0, CONVROT_ERR_INVALID, "invalid shape m=%lld n=%lld k=%lld",
                  static_cast<long long>(m), static_cast<long long>(n), static_cast<long long>(k));
  CONVROT_REQUIRE(k <= kMaxK, CONVROT_ERR_UNSUPPORTED, "k %lld can overflow the int32 dot (at most %d)",
                  static_cast<long long>(k), kMaxK);
  CONVROT_REQUIRE(m < (1LL << 21) && n < (1LL << 21), CONVROT_ERR_UNSUPPORTED, "shape too large");
  CONVROT_REQUIRE(act_stride >= k && weight_stride >= (layout == CONVROT_LAYOUT_NK ? k : n) && act_stride % 16 == 0 &&
                      weight_stride % 16 == 0,
                  CONVROT_ERR_INVALID, "row strides must cover the rows and be multiples of 16 bytes (%lld, %lld)",
                  static_cast<long long>(act_stride), static_cast<long long>(weight_stride));
  if (m == 0) return CONVROT_OK;
  CONVROT_REQUIRE(act && weight && xscales && out, CONVROT_ERR_INVALID, "null pointer");
  CONVROT_REQUIRE(aligned_to(act, 16) && aligned_to(weight, 16) && aligned_to(out, 16), CONVROT_ERR_INVALID,
                  "activation, weight and output must be 16-byte aligned");
  const I8Params p{act,        weight,        xscales,           wscales,          bias,
                   out,        act_stride,    weight_stride,     static_cast<int>(m), static_cast<int>(n),
                   static_cast<int>(k)};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (layout == CONVROT_LAYOUT_NK) {
    switch (out_dtype) {
      case CONVROT_BF16: return launch<CONVROT_LAYOUT_NK, __nv_bfloat16>(p, s);
      case CONVROT_F16: return launch<CONVROT_LAYOUT_NK, __half>(p, s);
      default: return launch<CONVROT_LAYOUT_NK, float>(p, s);
    }
  }
  switch (out_dtype) {
    case CONVROT_BF16: return launch<CONVROT_LAYOUT_KN, __nv_bfloat16>(p, s);
    case CONVROT_F16: return launch<CONVROT_LAYOUT_KN, __half>(p, s);
    default: return launch<CONVROT_LAYOUT_KN, float>(p, s);
  }
}

}  // extern "C"
