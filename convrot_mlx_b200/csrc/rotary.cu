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
// The angle is formed as a number of turns, position times frequency, with the
// frequency in two floats: the product with the first is exact in two floats
// (its rounding error by one FMA), so that whole turns can be taken off
// exactly and large positions lose nothing; sine and cosine are 32-bit.
//
// Memory-bound: every head is read and written once, the sines are formed once
// for all heads of a token.  12288 tokens of 48 heads of 128 (adjacent, bf16):
// 50 us, 0.92 of a copy's bandwidth; 17627 tokens of 24 heads (half apart,
// float16, forward and backward): 87 us, 0.76; one token of 32 heads: 3.0 us.
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
  int units;       // threads that a head's values are spread over
  uint32_t slots;  // tokens of a CTA
  uint32_t groups; // of heads in a CTA
  float sign;  // 1, or -1 for the gradient
  float2 turns[kMaxPairs];  // frequency of each pair in turns a position, high and low part
  uint8_t axis[kMaxPairs];
};

// A CTA has some tokens; its threads first form the sines and cosines of all
// their pairs, once for all heads, in shared memory.  Then a thread has one
// unit of a head's values, of one token and one group of the heads, keeps the
// unit's sines and cosines in registers and turns its heads, kHeads of them at
// a time.  Units of a head,
// adjacent pairs: unit u is the VEC values from VEC u on (values past the
// pairs are copied).  Pairs half apart: unit u is the VEC values from VEC u on
// and the VEC from pairs + VEC u on; further units copy VEC values each.
// WIDE: VEC values move in one access; else one value an access.
// 128 bytes of a thread in flight; with 64 and as many ahead in registers 53 us
// instead of 50 for 12288 tokens of 48 heads of 128.
template <bool ADJACENT> constexpr int kHeads = ADJACENT ? 8 : 4;
constexpr int kThreads = 256;

template <typename T, int VEC, bool WIDE>
struct Unit {
  Pack<T, VEC> raw;
  __device__ __forceinline__ void load(const T* src, int left) {
    if constexpr (WIDE) {
      raw.load(src);
    } else if constexpr (VEC == 1) {
      raw.load(src);
    } else {
      raw.load_part(src, left < VEC ? left : VEC);
    }
  }
  __device__ __forceinline__ void store(T* dst, int left) const {
    if constexpr (WIDE || VEC == 1) {
      raw.store(dst);
    } else {
      float v[VEC];
      raw.get(v);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (i < left) dst[i] = Elem<T>::from_f(v[i]);
    }
  }
};

template <typename T, int VEC, bool WIDE, bool ADJACENT>
__global__ void __launch_bounds__(kThreads, 3) rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int NP = ADJACENT ? VEC / 2 : VEC;  // pairs of a unit
  constexpr int kUnroll = kHeads<ADJACENT>;
  // tokens x pairs: at most one unit of NP pairs for each thread
  __shared__ float2 turned[kThreads * NP];
  // the frequencies, since threads of a warp would read different ones from
  // the parameters one after another
  __shared__ float2 freq[kMaxPairs];
  __shared__ uint8_t axis[kMaxPairs];
  for (int j = threadIdx.x; j < p.pairs; j += kThreads) {
    freq[j] = p.turns[j];
    axis[j] = p.axis[j];
  }
  __syncthreads();
  grid_dependency_wait();
  grid_dependents_launch();
  const uint32_t all = p.batch * static_cast<uint32_t>(p.tokens);
  const uint32_t bt0 = blockIdx.x * p.slots;
  for (uint32_t i = threadIdx.x; i < p.slots * p.pairs; i += kThreads) {
    const uint32_t s = i / p.pairs, j = i - s * p.pairs, bt = bt0 + s;
    if (bt < all) {
      const uint32_t sample = bt / static_cast<uint32_t>(p.tokens);
      const int64_t token = bt - sample * static_cast<uint32_t>(p.tokens);
      const float pos = ld_f32(p.positions + sample * p.pos_b + token * p.axes + axis[j]);
      const float whole = __fmul_rn(pos, freq[j].x);
      const float rest = __fmaf_rn(pos, freq[j].y, __fmaf_rn(pos, freq[j].x, -whole));
      float2 cs;
      sincospif(2.0f * (__fsub_rn(whole, rintf(whole)) + rest), &cs.y, &cs.x);
      cs.y *= p.sign;
      turned[i] = cs;
    }
  }
  __syncthreads();
  // thread = (group of heads, token, unit)
  const uint32_t per_group = p.slots * p.units;
  const uint32_t group = threadIdx.x / per_group, at = threadIdx.x - group * per_group;
  const uint32_t slot = at / static_cast<uint32_t>(p.units), bt = bt0 + slot;
  const int u = static_cast<int>(at - slot * p.units);
  if (group >= p.groups || bt >= all) return;
  const uint32_t sample = bt / static_cast<uint32_t>(p.tokens);
  const int64_t b = sample, token = bt - sample * static_cast<uint32_t>(p.tokens);
  const int turning = ADJACENT ? p.units : p.pairs / VEC;  // units that turn
  const bool turns = u < turning;
  const int e0 = ADJACENT || turns ? u * VEC : 2 * p.pairs + (u - turning) * VEC;  // first value of the unit
  const int left = p.dim - e0;
  const int count = turns ? min(NP, max(0, p.pairs - u * NP)) : 0;  // pairs of the unit

  float cs[NP], sn[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const float2 v = i < count ? turned[slot * p.pairs + u * NP + i] : make_float2(1.0f, 0.0f);
    cs[i] = v.x;
    sn[i] = v.y;
  }
  const int heads = p.t[0].heads + p.t[1].heads;
  const int share = static_cast<int>(blockIdx.y * p.groups + group), shares = static_cast<int>(gridDim.y * p.groups);
  const int h0 = static_cast<int>(static_cast<int64_t>(heads) * share / shares);
  const int h1 = static_cast<int>(static_cast<int64_t>(heads) * (share + 1) / shares);
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const RotaryTensor& t = p.t[which];
    const int lo = which ? p.t[0].heads : 0, hi = min(h1, lo + t.heads);
    const T* in = static_cast<const T*>(t.in) + b * t.in_b + token * t.in_t + e0;
    T* out = static_cast<T*>(t.out) + b * t.out_b + token * t.out_t + e0;
    Unit<T, VEC, WIDE> x[kUnroll], y[ADJACENT ? 1 : kUnroll];
    const int begin = max(h0, lo);
    const T* src = in + (begin - lo) * t.in_h;
    T* dst = out + (begin - lo) * t.out_h;
    const int64_t src_step = t.in_h, dst_step = t.out_h;
#pragma unroll 1
    for (int h = begin; h < hi; h += kUnroll) {
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        if (h + k < hi) {
          x[k].load(src, left);
          if constexpr (!ADJACENT)
            if (turns) y[k].load(src + p.pairs, VEC);
        }
        src += src_step;
      }
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        if (h + k < hi) {
          if constexpr (ADJACENT) {
            if (count > 0) {  // values past the pairs keep their bits
              float v[VEC];
              x[k].raw.get(v);
              const bool full = count == NP;
#pragma unroll
              for (int i = 0; i < NP; ++i)
                if (full || i < count) {
                  const float x0 = v[2 * i], x1 = v[2 * i + 1];
                  v[2 * i] = x0 * cs[i] - x1 * sn[i];
                  v[2 * i + 1] = x0 * sn[i] + x1 * cs[i];
                }
              x[k].raw.set(v);
            }
          } else if (turns) {
            float v[VEC], w[VEC];
            x[k].raw.get(v);
            y[k].raw.get(w);
#pragma unroll
            for (int i = 0; i < NP; ++i) {
              const float x0 = v[i], x1 = w[i];
              v[i] = x0 * cs[i] - x1 * sn[i];
              w[i] = x0 * sn[i] + x1 * cs[i];
            }
            x[k].raw.set(v);
            y[k].raw.set(w);
            y[k].store(dst + p.pairs, VEC);
          }
          x[k].store(dst, left);
        }
        dst += dst_step;
      }
    }
  }
}

template <typename T, int VEC, bool WIDE, bool ADJACENT>
int launch(RotaryParams& p, cudaStream_t stream) {
  p.units = ADJACENT ? (p.dim + VEC - 1) / VEC : p.pairs / VEC + (p.dim - 2 * p.pairs + VEC - 1) / VEC;
  // Several groups of heads in a CTA, so that the sines are formed by as many
  // threads as use them, of eight heads at least (with three or four a thread
  // only starts and ends: 17627 tokens of 24 heads took 70 us instead of 51).
  const int heads = p.t[0].heads + p.t[1].heads;
  const int most = (heads + kHeads<ADJACENT> - 1) / kHeads<ADJACENT>;
  const int room = kThreads / (4 * p.units), wanted = heads / 12;
  const int groups = room < wanted ? room : wanted;
  p.groups = static_cast<uint32_t>(groups < 1 ? 1 : groups);
  p.slots = kThreads / (p.units * p.groups);
  const int64_t blocks = (static_cast<int64_t>(p.batch) * p.tokens + p.slots - 1) / p.slots;
  // Few tokens: more CTAs for the same tokens, until there are about 4 for
  // each SM.
  int64_t shares = (4LL * device_sm_count() + blocks - 1) / blocks;
  const int64_t limit = (most + p.groups - 1) / p.groups;
  if (shares > limit) shares = limit;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(shares), 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, rotary_kernel<T, VEC, WIDE, ADJACENT>, p));
  return check_launch("convrot_axial_rotary");
}

// Whether every vector of `vec` values is aligned: addresses, strides, and
// for pairs half apart the second half's start and the copied tail's.
template <typename T>
bool aligned_for(const RotaryParams& p, int vec) {
  if (p.dim % vec || (!p.adjacent && p.pairs % vec)) return false;
  const int64_t bytes = vec * static_cast<int64_t>(sizeof(T));
  for (const RotaryTensor& t : p.t) {
    if (t.heads == 0) continue;
    const int64_t strides = t.in_b | t.in_h | t.in_t | t.out_b | t.out_h | t.out_t;
    if (strides % vec || !aligned_to(t.in, bytes) || !aligned_to(t.out, bytes)) return false;
  }
  return true;
}

template <typename T>
int launch_type(RotaryParams& p, cudaStream_t s) {
  constexpr int W = 16 / sizeof(T);
  if (p.adjacent) {
    if (aligned_for<T>(p, W)) return launch<T, W, true, true>(p, s);
    if (aligned_for<T>(p, 2)) return launch<T, 2, true, true>(p, s);
    return launch<T, 2, false, true>(p, s);
  }
  if (aligned_for<T>(p, W)) return launch<T, W, true, false>(p, s);
  if constexpr (W == 8)
    if (aligned_for<T>(p, 4)) return launch<T, 4, true, false>(p, s);
  if (aligned_for<T>(p, 2)) return launch<T, 2, true, false>(p, s);
  return launch<T, 1, false, false>(p, s);
}

}  // namespace
}  // namespace convrot

extern "C" {

int convrot_axial_rotary(int dtype, int64_t batch, int64_t tokens, int64_t dim, const void* q, void* q_out,
                         int64_t q_heads, const void* k, void* k_out, int64_t k_heads, const int64_t* strides,
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
  CONVROT_REQUIRE(batch < (1LL << 31) && tokens < (1LL << 31) && batch * tokens < (1LL << 31) &&
                      q_heads + k_heads < (1LL << 20),
                  CONVROT_ERR_UNSUPPORTED, "shape too large");
  RotaryParams p = {};
  int pairs = 0;
  for (int a = 0; a < axes; ++a) {
    CONVROT_REQUIRE(widths[a] > 0 && widths[a] % 2 == 0 && 2 * pairs + widths[a] <= dim, CONVROT_ERR_INVALID,
                    "axis widths must be positive, even and sum to at most the head dimension %lld",
                    static_cast<long long>(dim));
    const double ratio = std::pow(theta, -2.0 / widths[a]);
    double turns = 0.15915494309189533577;  // 1 / (2 pi): pair 0 turns by one radian a position
    for (int j = 0; j < widths[a] / 2; ++j, ++pairs, turns *= ratio) {
      const float high = static_cast<float>(turns);
      p.turns[pairs] = make_float2(high, static_cast<float>(turns - high));
      p.axis[pairs] = static_cast<uint8_t>(a);
    }
  }
  if (batch == 0 || tokens == 0 || q_heads + k_heads == 0) return CONVROT_OK;
  CONVROT_REQUIRE(positions && strides && (q_heads == 0 || (q && q_out)) && (k_heads == 0 || (k && k_out)),
                  CONVROT_ERR_INVALID, "null pointer");
  if (q_heads > 0)
    p.t[0] = RotaryTensor{q,          q_out,      strides[0], strides[1], strides[2], strides[3], strides[4],
                          strides[5], static_cast<int>(q_heads)};
  if (k_heads > 0)
    p.t[1] = RotaryTensor{k,           k_out,       strides[6], strides[7], strides[8], strides[9], strides[10],
                          strides[11], static_cast<int>(k_heads)};
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
    case CONVROT_BF16: return launch_type<__nv_bfloat16>(p, s);
    case CONVROT_F16: return launch_type<__half>(p, s);
    default: return launch_type<float>(p, s);
  }
}

}  // extern "C"
