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
// exactly; sine and cosine are 32-bit.  Of the angle's n turns 2^-46 n are lost
// to the second float and the rounding of the two products' rests, and at most
// 2^-25 of a turn to the rounding of what is left of them: 3.4 units of 2^-24
// radians up to position 2^20, twice that at 2^24.
//
// Memory-bound: every head is read and written once, the sines are formed once
// for all heads of a token.  12288 tokens of 48 heads of 128 (adjacent, bf16):
// 49 us, 0.94 of a copy's bandwidth; 17627 tokens of 24 heads (half apart,
// float16, forward and backward): 82 us, 0.81, and adjacent 77; one token of 32
// heads: 2.7 us.
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

constexpr int kThreads = 256;

// A CTA has some tokens; its threads first form the sines and cosines of all
// their pairs, once for all heads, in shared memory.  Then a thread has some
// values of a head, of one token and one group of the heads, keeps their sines
// and cosines in registers and turns its heads, a batch of them at a time; the
// first batch is on its way while the sines are formed (one token of 32 heads:
// 2.7 us, 3.0 with its loads after the sines).

// The frequencies, since threads of a warp would read different ones from the
// parameters one after another.
struct Frequencies {
  float2 turns[kMaxPairs];
  uint8_t axis[kMaxPairs];
  __device__ __forceinline__ void fill(const RotaryParams& p) {
    for (int j = threadIdx.x; j < p.pairs; j += kThreads) {
      turns[j] = p.turns[j];
      axis[j] = p.axis[j];
    }
  }
};

// Cosines and sines of a CTA's tokens from bt0 on: (token, pair).
__device__ __forceinline__ void form_sines(const RotaryParams& p, const Frequencies& f, uint32_t bt0, uint32_t all,
                                           float2* turned) {
  for (uint32_t i = threadIdx.x; i < p.slots * p.pairs; i += kThreads) {
    const uint32_t s = i / p.pairs, j = i - s * p.pairs, bt = bt0 + s;
    if (bt < all) {
      const uint32_t sample = bt / static_cast<uint32_t>(p.tokens);
      const int64_t token = bt - sample * static_cast<uint32_t>(p.tokens);
      const float pos = ld_f32(p.positions + sample * p.pos_b + token * p.axes + f.axis[j]);
      const float whole = __fmul_rn(pos, f.turns[j].x);
      const float rest = __fmaf_rn(pos, f.turns[j].y, __fmaf_rn(pos, f.turns[j].x, -whole));
      float2 cs;
      sincospif(2.0f * (__fsub_rn(whole, rintf(whole)) + rest), &cs.y, &cs.x);
      cs.y *= p.sign;
      turned[i] = cs;
    }
  }
}

// A thread's heads, those of share `group` of the CTA's, in batches of up to N
// that hold only queries or only keys.
struct Heads {
  int64_t b, token;
  int which, h, end, last;
  __device__ __forceinline__ Heads(const RotaryParams& p, uint32_t bt, uint32_t group) {
    const uint32_t sample = bt / static_cast<uint32_t>(p.tokens);
    b = sample;
    token = bt - sample * static_cast<uint32_t>(p.tokens);
    const int heads = p.t[0].heads + p.t[1].heads;
    const int share = static_cast<int>(blockIdx.y * p.groups + group), shares = static_cast<int>(gridDim.y * p.groups);
    h = static_cast<int>(static_cast<int64_t>(heads) * share / shares);
    last = static_cast<int>(static_cast<int64_t>(heads) * (share + 1) / shares);
    which = h < p.t[0].heads ? 0 : 1;
    end = which ? last : min(last, p.t[0].heads);
  }
  // The next batch; false past the last.
  __device__ __forceinline__ bool next(int count) {
    h += count;
    if (h < end) return true;
    if (end == last) return false;
    which = 1;
    h = end;
    end = last;
    return true;
  }
  template <typename T>
  __device__ __forceinline__ const T* in(const RotaryParams& p) const {
    const RotaryTensor& t = p.t[which];
    return static_cast<const T*>(t.in) + b * t.in_b + token * t.in_t + (h - (which ? p.t[0].heads : 0)) * t.in_h;
  }
  template <typename T>
  __device__ __forceinline__ T* out(const RotaryParams& p) const {
    const RotaryTensor& t = p.t[which];
    return static_cast<T*>(t.out) + b * t.out_b + token * t.out_t + (h - (which ? p.t[0].heads : 0)) * t.out_h;
  }
};

template <typename T, int VEC, bool WIDE>
struct Unit {
  Pack<T, VEC> raw;
  __device__ __forceinline__ void load(const T* src, int left) {
    if constexpr (WIDE || VEC == 1) {
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

// Units of a head, adjacent pairs: unit u is the VEC values from VEC u on
// (values past the pairs are copied).  Pairs half apart: unit u is the VEC
// values from VEC u on and the VEC from pairs + VEC u on; further units copy
// VEC values each.  WIDE: VEC values move in one access; else one value an
// access.  kHeads: 128 bytes of a thread in flight; with 64 and as many ahead
// in registers 53 us instead of 50 for 12288 tokens of 48 heads of 128.
constexpr int kHeads = 8;

template <typename T, int VEC, bool WIDE, bool ADJACENT>
__global__ void __launch_bounds__(kThreads, 3) rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int NP = ADJACENT ? VEC / 2 : VEC;  // pairs of a unit
  // tokens x pairs: at most one unit of NP pairs for each thread
  __shared__ float2 turned[kThreads * NP];
  __shared__ Frequencies freq;
  freq.fill(p);
  __syncthreads();
  grid_dependency_wait();
  grid_dependents_launch();
  const uint32_t all = p.batch * static_cast<uint32_t>(p.tokens);
  const uint32_t bt0 = blockIdx.x * p.slots;
  // thread = (group of heads, token, unit)
  const uint32_t per_group = p.slots * p.units;
  const uint32_t group = threadIdx.x / per_group, at = threadIdx.x - group * per_group;
  const uint32_t slot = at / static_cast<uint32_t>(p.units), bt = bt0 + slot;
  const int u = static_cast<int>(at - slot * p.units);
  const bool active = group < p.groups && bt < all;
  const int turning = ADJACENT ? p.units : p.pairs / VEC;  // units that turn
  const bool turns = u < turning;
  const int e0 = ADJACENT || turns ? u * VEC : 2 * p.pairs + (u - turning) * VEC;  // first value of the unit
  const int left = p.dim - e0;
  const int count = turns ? min(NP, max(0, p.pairs - u * NP)) : 0;  // pairs of the unit

  Heads heads(p, bt, group);
  Unit<T, VEC, WIDE> x[kHeads], y[ADJACENT ? 1 : kHeads];
  auto load = [&] {
    const T* src = heads.in<T>(p) + e0;
    const int64_t step = p.t[heads.which].in_h;
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
      if (heads.h + k < heads.end) {
        x[k].load(src, left);
        if constexpr (!ADJACENT)
          if (turns) y[k].load(src + p.pairs, VEC);
      }
      src += step;
    }
  };
  if (active) load();
  form_sines(p, freq, bt0, all, turned);
  __syncthreads();
  if (!active) return;
  float cs[NP], sn[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const float2 v = i < count ? turned[slot * p.pairs + u * NP + i] : make_float2(1.0f, 0.0f);
    cs[i] = v.x;
    sn[i] = v.y;
  }
  bool here = true;
#pragma unroll 1
  do {
    if (!here) load();
    here = false;
    T* dst = heads.out<T>(p) + e0;
    const int64_t step = p.t[heads.which].out_h;
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
      if (heads.h + k < heads.end) {
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
      dst += step;
    }
  } while (heads.next(kHeads));
}

// Pairs half apart in heads of whole 16-byte vectors.  A head is spread over
// `units` lanes of one warp, lane u with the vectors u and, NJ = 2, u + units,
// so that all accesses are of whole vectors and whole sectors wherever the
// pairs' halves lie (each half read and written where it lies, 17627 tokens of
// 24 heads of 128 with 56 pairs, float16, take 43.3 us instead of 41.7; value
// by value, as 25 pairs in heads of 64 need it, 10359 tokens of 48 heads 123
// instead of 28).  The partners of a vector's values, `pairs` further on
// or back, come through shared memory: as a vector (EVEN: pairs are a multiple
// of the vector), or value by value, for which every eight lanes' vectors are a
// bank off the last eight's, so that neither the stores nor the loads conflict.
// Four vectors of a thread in flight and four CTAs for each SM; with eight and
// three 43.5 us, with partners by shuffles 42.0.
constexpr int kHalfVectors = 4;

template <typename T, int NJ, bool EVEN>
__global__ void __launch_bounds__(kThreads, 4) rotary_half_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int W = 16 / static_cast<int>(sizeof(T));
  constexpr int kBatch = kHalfVectors / NJ;
  constexpr int kWarpBytes = 32 * 16 + 16;
  __shared__ float2 turned[kThreads * 4];  // slots x pairs: pairs are at most 4 for each lane of a head
  __shared__ Frequencies freq;
  __shared__ __align__(16) uint8_t exchange[kThreads / 32][kBatch * NJ][kWarpBytes];
  freq.fill(p);
  __syncthreads();
  grid_dependency_wait();
  grid_dependents_launch();
  const uint32_t all = p.batch * static_cast<uint32_t>(p.tokens);
  const uint32_t bt0 = blockIdx.x * p.slots;
  // rows of lanes, p.units each, warp by warp; row = (group of heads, token)
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, rows = 32 / p.units, in_warp = lane / p.units;
  const uint32_t row = warp * rows + in_warp, group = row / p.slots, slot = row - group * p.slots, bt = bt0 + slot;
  const int first = static_cast<int>(in_warp * p.units), u = static_cast<int>(lane) - first;
  const bool active = in_warp < rows && group < p.groups && bt < all;

  Heads heads(p, bt, group);
  Pack<T, W> x[kBatch][NJ];
  auto load = [&] {
    const T* src = heads.in<T>(p) + u * W;
    const int64_t step = p.t[heads.which].in_h;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (heads.h + k < heads.end)
#pragma unroll
        for (int j = 0; j < NJ; ++j) x[k][j].load(src + j * p.units * W);
      src += step;
    }
  };
  if (active) load();
  form_sines(p, freq, bt0, all, turned);
  __syncthreads();

  // Per value: the turn, with the sine's sign for the pair's first or second
  // value, and where the partner lies.  Values past the pairs are copied.
  const uint32_t base = smem_u32(exchange[warp]);
  auto place = [&](int e) -> uint32_t {  // of value e of this row
    const int v = e / W, j = NJ == 2 && v >= p.units, l = first + v - (j ? p.units : 0);
    return base + j * kWarpBytes + l * 16 + (EVEN ? 0 : l / 8 * 4) + e % W * static_cast<int>(sizeof(T));
  };
  float cs[NJ][W], sn[NJ][W];
  uint32_t from[NJ][EVEN ? 1 : W], to[NJ];
  uint32_t turning = 0;  // bit j W + i
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e0 = (u + j * p.units) * W;
    to[j] = base + j * kWarpBytes + lane * 16 + (EVEN ? 0 : lane / 8 * 4);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int e = e0 + i;
      const bool second = e >= p.pairs, in = active && e < 2 * p.pairs;
      const float2 v = in ? turned[slot * p.pairs + (second ? e - p.pairs : e)] : make_float2(1.0f, 0.0f);
      cs[j][i] = v.x;
      sn[j][i] = second ? v.y : -v.y;
      if (in) turning |= 1u << (j * W + i);
      if (!EVEN || i == 0) from[j][EVEN ? 0 : i] = in ? place(second ? e - p.pairs : e + p.pairs) : to[j];
    }
  }
  // every lane of a warp takes part as long as any has a batch
  bool more = active, here = true;
#pragma unroll 1
  while (__any_sync(0xFFFFFFFFu, more)) {
    if (!here && more) load();
    here = false;
    __syncwarp();  // the last batch's partners have been read
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (more && heads.h + k < heads.end)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const uint32_t at = to[j] + k * NJ * kWarpBytes;
          const uint32_t(&w)[4] = x[k][j].w;
          if constexpr (EVEN) {
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + 4 * i), "r"(w[i]) : "memory");
          }
        }
    }
    __syncwarp();
    if (more) {
      T* dst = heads.out<T>(p) + u * W;
      const int64_t step = p.t[heads.which].out_h;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (heads.h + k < heads.end)
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            constexpr uint32_t kAll = (1u << W) - 1;
            const uint32_t turn = turning >> (j * W) & kAll;
            if (turn) {
              float v[W], w[W];
              x[k][j].get(v);
              if constexpr (EVEN) {
                Pack<T, W> other;
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(other.w[0]), "=r"(other.w[1]), "=r"(other.w[2]), "=r"(other.w[3])
                             : "r"(from[j][0] + k * NJ * kWarpBytes)
                             : "memory");
                other.get(w);
              } else {
#pragma unroll
                for (int i = 0; i < W; ++i) {
                  Pack<T, 1> other;
                  const uint32_t at = from[j][i] + k * NJ * kWarpBytes;
                  if constexpr (sizeof(T) == 4) {
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(other.w[0]) : "r"(at) : "memory");
                  } else {
                    uint16_t half;
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(half) : "r"(at) : "memory");
                    other.w[0] = half;
                  }
                  float one[1];
                  other.get(one);
                  w[i] = one[0];
                }
              }
#pragma unroll
              for (int i = 0; i < W; ++i)
                if (turn == kAll || (turn >> i & 1)) v[i] = v[i] * cs[j][i] + w[i] * sn[j][i];
              x[k][j].set(v);
            }
            x[k][j].store(dst + j * p.units * W);
          }
        dst += step;
      }
      more = heads.next(kBatch);
    }
  }
}

// Tokens and groups of heads of a CTA whose rows of p.units threads are
// `rows`, and the launch.  Several groups of heads, so that the sines are
// formed by as many threads as use them, of twelve heads at least (with three
// or four a thread only starts and ends: 17627 tokens of 24 heads took 70 us
// instead of 51).
int launch(void (*kernel)(RotaryParams), RotaryParams& p, int rows, int batch, cudaStream_t stream) {
  const int heads = p.t[0].heads + p.t[1].heads;
  const int most = (heads + batch - 1) / batch;
  const int room = rows / 4, wanted = heads / 12;
  const int groups = room < wanted ? room : wanted;
  p.groups = static_cast<uint32_t>(groups < 1 ? 1 : groups);
  p.slots = static_cast<uint32_t>(rows) / p.groups;
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
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p));
  return check_launch("convrot_axial_rotary");
}

template <typename T, int VEC, bool WIDE, bool ADJACENT>
int launch_units(RotaryParams& p, cudaStream_t stream) {
  p.units = ADJACENT ? (p.dim + VEC - 1) / VEC : p.pairs / VEC + (p.dim - 2 * p.pairs + VEC - 1) / VEC;
  return launch(rotary_kernel<T, VEC, WIDE, ADJACENT>, p, kThreads / p.units, kHeads, stream);
}

template <typename T, int NJ>
int launch_half(RotaryParams& p, cudaStream_t stream) {
  constexpr int W = 16 / sizeof(T);
  p.units = p.dim / (W * NJ);
  return launch(p.pairs % W ? rotary_half_kernel<T, NJ, false> : rotary_half_kernel<T, NJ, true>, p,
                kThreads / 32 * (32 / p.units), kHalfVectors / NJ, stream);
}

// Whether every vector of `vec` values is aligned: addresses and strides.
template <typename T>
bool aligned_for(const RotaryParams& p, int vec) {
  if (p.dim % vec) return false;
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
    if (aligned_for<T>(p, W)) return launch_units<T, W, true, true>(p, s);
    if (aligned_for<T>(p, 2)) return launch_units<T, 2, true, true>(p, s);
    return launch_units<T, 2, false, true>(p, s);
  }
  if (aligned_for<T>(p, W) && p.dim <= 32 * W) return launch_half<T, 1>(p, s);
  if constexpr (W == 4)
    if (aligned_for<T>(p, 4) && p.dim % 8 == 0) return launch_half<T, 2>(p, s);
  if (aligned_for<T>(p, 2) && p.pairs % 2 == 0) return launch_units<T, 2, true, false>(p, s);
  return launch_units<T, 1, false, false>(p, s);
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
