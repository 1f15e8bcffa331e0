// Rotary positions with several axes (time, height, width) for the queries
// and keys of an attention, forward and backward in one kernel.
//
// The first sum(widths) values of a head form pairs, adjacent (x[2i],
// x[2i + 1]) or sum(widths) / 2 apart; axis a owns widths[a] / 2 consecutive
// pairs, and its pair j turns by t = position_a * theta^(-2 j / widths[a]):
//   y0 = x0 cos t - x1 sin t,   y1 = x0 sin t + x1 cos t;
// what follows the pairs is copied.  The rotation is orthogonal, so the
// gradient of the input is the rotation by -t of the gradient of the output.
//
// The angle is formed in 64 bits as a number of turns and reduced to less
// than half a turn there, so that large positions lose nothing; sine and
// cosine are 32-bit.
#include "rows.cuh"

#include <cmath>

namespace convrot {
namespace {

constexpr int kMaxPairs = 128;  // head dimension at most 256
constexpr int kMaxAxes = 8;

struct RotaryTensor {
  const void* in;
  void* out;
  int64_t in_b, in_h, in_t;     // element strides of batch, head and token
  int64_t out_b, out_h, out_t;
  int heads;
};

struct RotaryParams {
  RotaryTensor t[2];  // queries and keys
  const float* positions;  // (tokens, axes), for each sample pos_b apart
  int64_t pos_b;
  int64_t tokens;
  int batch, dim, pairs, axes, adjacent;
  float sign;  // 1, or -1 for the gradient
  double turns[kMaxPairs];  // frequency of each pair in turns a position
  uint8_t axis[kMaxPairs];
};

// One thread for each pair (or pair of copied values) of a head.
template <typename T>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryParams p) {
  const int half = (p.dim + 1) / 2;
  const int heads = p.t[0].heads + p.t[1].heads;
  const int64_t total = static_cast<int64_t>(p.batch) * p.tokens * heads * half;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int j = static_cast<int>(i % half);
    int h = static_cast<int>(i / half % heads);
    const int64_t bt = i / half / heads, token = bt % p.tokens, b = bt / p.tokens;
    const int which = h >= p.t[0].heads;
    h -= which ? p.t[0].heads : 0;
    const RotaryTensor& t = p.t[which];
    const T* in = static_cast<const T*>(t.in) + b * t.in_b + h * t.in_h + token * t.in_t;
    T* out = static_cast<T*>(t.out) + b * t.out_b + h * t.out_h + token * t.out_t;
    if (j < p.pairs) {
      const double turn = static_cast<double>(p.positions[b * p.pos_b + token * p.axes + p.axis[j]]) * p.turns[j];
      float s, c;
      sincospif(2.0f * static_cast<float>(turn - rint(turn)), &s, &c);
      s *= p.sign;
      const int i0 = p.adjacent ? 2 * j : j, i1 = p.adjacent ? 2 * j + 1 : j + p.pairs;
      const float x0 = Elem<T>::to_f(in[i0]), x1 = Elem<T>::to_f(in[i1]);
      out[i0] = Elem<T>::from_f(x0 * c - x1 * s);
      out[i1] = Elem<T>::from_f(x0 * s + x1 * c);
    } else {
      out[2 * j] = in[2 * j];
      if (2 * j + 1 < p.dim) out[2 * j + 1] = in[2 * j + 1];
    }
  }
}

template <typename T>
int launch(const RotaryParams& p, cudaStream_t stream) {
  const int64_t total =
      static_cast<int64_t>(p.batch) * p.tokens * (p.t[0].heads + p.t[1].heads) * ((p.dim + 1) / 2);
  const int64_t blocks = (total + 255) / 256, most = 16LL * device_sm_count();
  rotary_kernel<T><<<static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, stream>>>(p);
  return check_launch("convrot_axial_rotary");
}

}  // namespace
}  // namespace convrot

extern "C" {

int convrot_axial_rotary(int dtype, int64_t batch, int64_t tokens, int64_t dim, const void* q, int64_t q_heads,
                         const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, const void* k,
                         int64_t k_heads, const int64_t* k_strides, void* k_out, const int64_t* k_out_strides,
                         const float* positions, int64_t position_batch_stride, int axes, const int32_t* widths,
                         double theta, int interleaved, int inverse, void* stream) {
  using namespace convrot;
  CONVROT_REQUIRE(valid_dtype(dtype), CONVROT_ERR_INVALID, "unknown dtype %d", dtype);
  CONVROT_REQUIRE(batch >= 0 && tokens >= 0 && q_heads >= 0 && k_heads >= 0, CONVROT_ERR_INVALID, "negative size");
  CONVROT_REQUIRE(dim > 0 && dim <= 2 * kMaxPairs, CONVROT_ERR_UNSUPPORTED, "head dimension %lld is not in 1..%d",
                  static_cast<long long>(dim), 2 * kMaxPairs);
  CONVROT_REQUIRE(axes >= 1 && axes <= kMaxAxes && widths != nullptr, CONVROT_ERR_INVALID,
                  "the number of axes must be 1..%d, got %d", kMaxAxes, axes);
  CONVROT_REQUIRE(theta > 0.0 && std::isfinite(theta), CONVROT_ERR_INVALID, "theta must be positive and finite");
  CONVROT_REQUIRE(batch < (1LL << 31) && tokens < (1LL << 31) && q_heads + k_heads < (1LL << 20),
                  CONVROT_ERR_UNSUPPORTED, "shape too large");
  RotaryParams p = {};
  int pairs = 0;
  for (int a = 0; a < axes; ++a) {
    CONVROT_REQUIRE(widths[a] > 0 && widths[a] % 2 == 0 && 2 * pairs + widths[a] <= dim, CONVROT_ERR_INVALID,
                    "axis widths must be positive, even and sum to at most the head dimension %lld",
                    static_cast<long long>(dim));
    for (int j = 0; j < widths[a] / 2; ++j, ++pairs) {
      p.turns[pairs] = std::exp2(-2.0 * j / widths[a] * std::log2(theta)) * 0.15915494309189533577;  // 1 / (2 pi)
      p.axis[pairs] = static_cast<uint8_t>(a);
    }
  }
  if (batch == 0 || tokens == 0 || q_heads + k_heads == 0) return CONVROT_OK;
  CONVROT_REQUIRE(positions != nullptr && (q_heads == 0 || (q && q_out && q_strides && q_out_strides)) &&
                      (k_heads == 0 || (k && k_out && k_strides && k_out_strides)),
                  CONVROT_ERR_INVALID, "null pointer");
  if (q_heads > 0)
    p.t[0] = RotaryTensor{q,           q_out, q_strides[0], q_strides[1], q_strides[2], q_out_strides[0], q_out_strides[1],
                          q_out_strides[2], static_cast<int>(q_heads)};
  if (k_heads > 0)
    p.t[1] = RotaryTensor{k,           k_out, k_strides[0], k_strides[1], k_strides[2], k_out_strides[0], k_out_strides[1],
                          k_out_strides[2], static_cast<int>(k_heads)};
  p.positions = positions;
  p.pos_b = position_batch_stride;
  p.tokens = tokens;
  p.batch = static_cast<int>(batch);
  p.dim = static_cast<int>(dim);
  p.pairs = pairs;
  p.axes = axes;
  p.adjacent = interleaved != 0;
  p.sign = inverse ? -1.0f : 1.0f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CONVROT_BF16: return launch<__nv_bfloat16>(p, s);
    case CONVROT_F16: return launch<__half>(p, s);
    default: return launch<float>(p, s);
  }
}

}  // extern "C"
