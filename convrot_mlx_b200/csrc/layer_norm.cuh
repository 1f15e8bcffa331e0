// Layer norm kernels (layer_norm.cu), instantiated for one type of x in each
// of layer_norm_{bf16,f16,f32}.cu.
//   mean = E[x], r = (E[(x - mean)^2] + eps)^-1/2, h = (x - mean) r
//   y  = h w + b                         (w = 1 + weight with add_one)
//   g  = dy w
//   dx = r (g - E[g] - h E[g h])
//   dweight = sum dy h,  dbias = sum dy  (over the rows that share a weight)
// A row far from zero would lose its values to the rounding of the mean: that of
// 1664 times 30000, by sum * (1 / F) in float32, is off by 0.002, which eps =
// 1e-6 makes 0.9 of h.  So where the mean is beyond twice the deviation the
// centred values d are summed once more, and h = (d - E[d]) r with variance
// E[d^2] - E[d]^2 (E[d] is a rounding error, so nothing cancels).  Other rows'
// h is off by at most 2 + max|h| of a row sum's relative error, and they pay
// one comparison: d summed for every row took 10 to 14% longer where one CTA
// fills an SM (2048 x 16384 bf16 28.7 us instead of 27.3).  The backward pass
// subtracts the mean before it multiplies, as the forward pass does.
// Memory-bound: forward reads and writes a row once; backward reads x and dy
// and writes dx, once each.  A thread keeps the same columns for all rows of
// its CTA: a row stays in registers between its statistics and its output,
// the weights are loaded once for a CTA, and the column sums of the backward
// pass stay in registers too (a second small kernel adds up the CTAs' sums in
// a fixed order).  What limits beside the memory is the number of
// instructions and, with few rows for each CTA, the chain of a row's two
// reductions: a thread has up to 24 values of a row, so that the exchange
// between the threads of a row is little beside them, the arithmetic is in
// paired float32, sizes are compile-time, and the next rows' loads are in
// flight while a row is worked on.
// us (fraction of a copy's bandwidth), bf16, backward with all three gradients:
//   rows x features   65536 x 512  12288 x 1024  12288 x 3072  8192 x 4096  4096 x 8192  2048 x 16384
//   forward           25 (0.82)    11 (0.71)     27 (0.86)     27 (0.76)    30 (0.69)    27 (0.75)
//   backward          38 (0.80)    19 (0.61)     44 (0.79)     40 (0.77)    51 (0.60)    75 (0.41)
// (inputs and outputs rotated beyond L2; with one output, which L2 holds,
// forward 22, 9.1 and 25 for the first three).  Rows far from zero 12288 x 3072:
// forward 27.0 instead of 25.5.
// Rows of odd length, whose elements are moved one by one: 5003 x 1153 float32
// 13.1 and 21.5 us (1152: 9.7 and 16.8), 4096 x 6143 bf16 42 and 83 (6142: 37 and
// 56).  16-byte pieces copied to shared memory across the rows' ends and read
// back by element took a fifth longer forward and as long backward, for the
// barrier that each row then needs.
#pragma once

#include <algorithm>

#include "rows.cuh"

namespace convrot {
namespace norm {

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
  int wide_weight;  // the vectors are float32 beside a 16-bit x
  int keep;         // long rows: shared memory holds them between the passes
  float eps;
};

// Launches for x of type T; definitions in layer_norm_<type>.cu.
template <typename T> int forward(const NormParams& p, cudaStream_t s);
template <typename T> int backward(const NormParams& p, cudaStream_t s);

#ifdef CONVROT_NORM_KERNELS
namespace {

constexpr int kWarps = 4;  // of a CTA whose warps each have rows of their own

// CTAs of T threads that the registers of an SM are shared out to.
constexpr int ctas_of(int threads) {
  return threads == 64 ? 6 : threads == 32 || threads == 128 ? 3 : threads <= 256 ? 2 : 1;
}

// Adds up each of N values (1 or 2) over a warp: two are exchanged so that
// each half of the lanes goes on with one.  Afterwards v[0] of lane l is the
// sum of value l / (32 / N).
template <int N>
__device__ __forceinline__ void warp_sums(float (&v)[N]) {
  if constexpr (N == 2) {
    const bool high = threadIdx.x & 16;
    const float send = high ? v[0] : v[1];
    v[0] = (high ? v[1] : v[0]) + __shfl_xor_sync(0xFFFFFFFFu, send, 16);
  } else {
    v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], 16);
  }
#pragma unroll
  for (int o = 8; o > 0; o /= 2) v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], o);
}

// Sums of N values over the T threads of a row, for all of them.  red holds
// two sets of a CTA's warps' values, used in turn, so that one barrier for
// each call is enough.
template <int T, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*red)[16][N], int& turn) {
  warp_sums<N>(v);
  const float mine = v[0];
  if constexpr (T == 32) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xFFFFFFFFu, mine, i * (32 / N));
  } else {
    const int lane = threadIdx.x & 31;
    if (lane % (32 / N) == 0) red[turn][threadIdx.x >> 5][lane / (32 / N)] = mine;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = red[turn][0][i];
#pragma unroll
    for (int w = 1; w < T / 32; ++w)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += red[turn][w][i];
    turn ^= 1;
  }
}

// Whether a row's first mean has to be corrected, from its variance about it
// (false for NaN); and the variance less the square of the correction.
__device__ __forceinline__ bool far_from_zero(float mean, float var, float eps) { return mean * mean > 4.0f * (var + eps); }
__device__ __forceinline__ float corrected(float var, float off) { return fmaxf(fma(-off, off, var), 0.0f); }

// One thread's share of a row: NV vectors of VEC elements, T vectors apart,
// from column c0 = VEC * (thread of the row) on.  Columns past the end are
// never touched.
template <typename E, int VEC, int NV, int T>
struct Share {
  Pack<E, VEC> v[NV];
  // row: of column c0; left: columns from there to the end
  __device__ __forceinline__ void load(const E* row, int left) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * T * VEC < left) v[j].load_ahead(row + j * T * VEC);
  }
};

template <int VEC, int NV>
using Lanes = Lane<VEC>[NV][kLanes<VEC>];

// Rows ahead of the one in work: each thread copies its own columns of ARRAYS
// arrays asynchronously into places of shared memory that only it reads, so
// that no barrier is needed and no register is held.  kDepth places, of which
// one is being read.
template <typename E, int VEC, int NV, int T, int ARRAYS>
struct Ahead {
  static constexpr int kBytes = VEC * static_cast<int>(sizeof(E));
  static constexpr bool kAsync = kBytes >= 4;  // the copies' least size
  static constexpr int kDepth = 3;
  static constexpr int kThreads = T == 32 ? 32 * kWarps : T;
  static constexpr int kPlace = ARRAYS * NV * kThreads * kBytes;
  static constexpr int kSmem = kAsync ? kDepth * kPlace : 0;

  uint32_t base;
  int write = 0, read = 0;
  __device__ __forceinline__ explicit Ahead(const void* smem) : base(smem_u32(smem) + threadIdx.x * kBytes) {}

  // A row of each array into the next place (`there`: whether the row exists).
  template <typename... P>
  __device__ __forceinline__ void issue(bool there, int left, const P*... rows) {
    if (there) {
      uint32_t dst = base + write * kPlace;
      (copy(dst, rows, left), ...);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    write = write + 1 == kDepth ? 0 : write + 1;
  }
  __device__ __forceinline__ void copy(uint32_t& dst, const E* row, int left) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j * T * VEC < left) {
        const E* src = row + j * T * VEC;
        if constexpr (kBytes == 16)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + j * kThreads * kBytes), "l"(src) : "memory");
        else if constexpr (kBytes == 8)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst + j * kThreads * kBytes), "l"(src) : "memory");
        else
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + j * kThreads * kBytes), "l"(src) : "memory");
      }
    }
    dst += NV * kThreads * kBytes;
  }
  // The oldest row, once it has landed.
  template <typename... S>
  __device__ __forceinline__ void take(int left, S&... shares) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
    uint32_t src = base + read * kPlace;
    (fetch(src, shares, left), ...);
    read = read + 1 == kDepth ? 0 : read + 1;
  }
  __device__ __forceinline__ void fetch(uint32_t& src, Share<E, VEC, NV, T>& share, int left) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j * T * VEC < left) {
        uint32_t(&w)[Pack<E, VEC>::kWords] = share.v[j].w;
        const uint32_t at = src + j * kThreads * kBytes;
        if constexpr (kBytes == 16)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                       : "r"(at)
                       : "memory");
        else if constexpr (kBytes == 8)
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
        else
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
      }
    }
    src += NV * kThreads * kBytes;
  }
};

// A segment's vector: loaded as it lies in memory (of x's type or float32),
// and turned into float32 plus a constant once everything else a thread needs
// first is on its way too.
template <typename E, int VEC, int NV, int T>
struct Vector {
  Pack<float, VEC> raw[NV];
  __device__ __forceinline__ void load(const void* base, bool wide, int64_t at, int left) {
    if (base == nullptr) return;
    if (wide) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j * T * VEC < left) raw[j].load_ahead(static_cast<const float*>(base) + at + j * T * VEC);
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j * T * VEC < left) {
          Pack<E, VEC> pk;
          pk.load_ahead(static_cast<const E*>(base) + at + j * T * VEC);
#pragma unroll
          for (int i = 0; i < Pack<E, VEC>::kWords; ++i) raw[j].w[i] = pk.w[i];
        }
    }
  }
  __device__ __forceinline__ void get(const void* base, bool wide, float absent, float plus, Lanes<VEC, NV>& out) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float f[VEC];
      if (base == nullptr) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = absent;
      } else if (wide) {
        raw[j].get(f);
      } else {
        unpack<E, VEC>(raw[j].w, f);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[i] += plus;
      Pack<float, VEC> pk;
      pk.set(f);
      pk.get_lanes(out[j]);
    }
  }
};

// The rows of a CTA: those of chunk blockIdx % chunks of its segment.
struct Rows {
  int64_t segment, begin, end;
  __device__ __forceinline__ explicit Rows(const NormParams& p) {
    segment = blockIdx.x / p.chunks;
    const int64_t chunk = blockIdx.x % p.chunks, base = segment * p.rows_per_weight;
    begin = base + p.rows_per_weight * chunk / p.chunks;
    end = base + p.rows_per_weight * (chunk + 1) / p.chunks;
  }
};

// VEC values of a segment's vector plus a constant, or `absent` ones.
template <typename E, int VEC>
__device__ __forceinline__ void vector_at(const NormParams& p, const void* base, int64_t at, float absent, float plus,
                                          float (&v)[VEC]) {
  if (base == nullptr) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = absent;
    return;
  }
  if (p.wide_weight) {
    Pack<float, VEC> pk;
    pk.load_ahead(static_cast<const float*>(base) + at);
    pk.get(v);
  } else {
    Pack<E, VEC> pk;
    pk.load_ahead(static_cast<const E*>(base) + at);
    pk.get(v);
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] += plus;
}

// ---------------------------------------------------------------------------
// forward

// Least CTAs of an SM that the registers are shared out to; 0: the compiler's
// choice.  With 1 it spends more registers on loads ahead: 4096 x 6142 bf16 37 us
// instead of 47, but 4096 x 3072 float32 23.6 instead of 18.7.  Two vectors of
// eight values for each lane of a warp would lose the sixth CTA by it (65536 x
// 512 bf16 22.7 us instead of 21.6).
constexpr int fwd_ctas(int size, int vec, int nv, int threads) {
  return size == 4 ? 0 : vec == 8 && nv == 2 && threads == 32 ? 6 : 1;
}

// T threads share a row: 32 (each warp of the CTA rows of its own), or the CTA.
template <typename E, int VEC, int NV, int T>
__global__ void __launch_bounds__(T == 32 ? 32 * kWarps : T, fwd_ctas(sizeof(E), VEC, NV, T))
    norm_fwd_kernel(const NormParams p) {
  constexpr int L = kLanes<VEC>;
  using A = Lane<VEC>;
  __shared__ float red[2][16][1];
  int turn = 0;
  grid_dependency_wait();
  grid_dependents_launch();
  const int F = p.features;
  const float inv = 1.0f / static_cast<float>(F);
  const int c0 = (T == 32 ? threadIdx.x & 31 : threadIdx.x) * VEC, left = F - c0;
  const Rows rows(p);
  const int64_t first = rows.begin + (T == 32 ? threadIdx.x >> 5 : 0), stride = T == 32 ? kWarps : 1;
  const E* src = static_cast<const E*>(p.x) + first * F + c0;
  E* dst = static_cast<E*>(p.y) + first * F + c0;
  const int64_t step = stride * F;
  Share<E, VEC, NV, T> x;
  using Next = Ahead<E, VEC, NV, T, 1>;
  extern __shared__ __align__(16) uint8_t smem[];
  Next next(smem);
  if constexpr (Next::kAsync) {
    next.issue(first < rows.end, left, src);
    next.issue(first + stride < rows.end, left, src + step);
  } else {
    if (first < rows.end) x.load(src, left);
  }
  Lanes<VEC, NV> weight, bias;
  {
    const int64_t offset = rows.segment * p.weight_stride + c0;
    Vector<E, VEC, NV, T> w, b;
    w.load(p.weight, p.wide_weight, offset, left);
    b.load(p.bias, p.wide_weight, offset, left);
    w.get(p.weight, p.wide_weight, p.add_one ? 0.0f : 1.0f, p.add_one ? 1.0f : 0.0f, weight);
    b.get(p.bias, p.wide_weight, 0.0f, 0.0f, bias);
  }
  for (int64_t row = first; row < rows.end; row += stride) {
    Lanes<VEC, NV> v;
    A sum = splat<VEC>(0.0f);
    if constexpr (Next::kAsync) {
      next.take(left, x);
      next.issue(row + 2 * stride < rows.end, left, src + 2 * step);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * T * VEC < left) {
        x.v[j].get_lanes(v[j]);
#pragma unroll
        for (int i = 0; i < L; ++i) sum = add(sum, v[j][i]);
      }
    src += step;
    if (!Next::kAsync && row + stride < rows.end) x.load(src, left);
    float s[1] = {total(sum)};
    row_sums<T>(s, red, turn);
    const float mean = s[0] * inv;
    const A minus = splat<VEC>(-mean);
    sum = splat<VEC>(0.0f);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * T * VEC < left) {
#pragma unroll
        for (int i = 0; i < L; ++i) {
          v[j][i] = add(v[j][i], minus);
          sum = fma(v[j][i], v[j][i], sum);
        }
      }
    s[0] = total(sum);
    row_sums<T>(s, red, turn);
    float var = s[0] * inv, off = 0.0f;
    if (far_from_zero(mean, var, p.eps)) {  // the same for all threads of the row
      sum = splat<VEC>(0.0f);
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j * T * VEC < left) {
#pragma unroll
          for (int i = 0; i < L; ++i) sum = add(sum, v[j][i]);
        }
      s[0] = total(sum);
      row_sums<T>(s, red, turn);
      off = s[0] * inv;
      var = corrected(var, off);
    }
    const float rstd = rsqrtf(var + p.eps);
    const A scale = splat<VEC>(rstd), rest = splat<VEC>(-off * rstd);
    if (c0 == 0 && p.mean) {
      p.mean[row] = mean + off;
      p.rstd[row] = rstd;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * T * VEC < left) {
#pragma unroll
        for (int i = 0; i < L; ++i) v[j][i] = fma(fma(v[j][i], scale, rest), weight[j][i], bias[j][i]);
        Pack<E, VEC> out;
        out.set_lanes(v[j]);
        out.store(dst + j * T * VEC);
      }
    dst += step;
  }
}

// Rows too long for the registers: three passes over the row in shared memory
// (in L2 where even that is too small).  The threads copy the 16-byte pieces
// of memory that a row lies in, wherever it starts, and with room for two rows
// the next one is on its way while a row is worked on.  2048 x 12288 float32:
// forward 44 us (55 with the later passes through L2), dx 65 (106); rows that
// start at any element, 2048 x 16383 bf16: 73 and 95 (80 and 177).
constexpr int kLong = 512;              // threads of a long row
constexpr int kLongSmem = 208 * 1024;  // most bytes of rows that are kept

// ARRAYS rows in shared memory, p.keep (1 or 2) times.
template <typename E, int ARRAYS>
struct Kept {
  uint32_t pitch;  // bytes of a row's place
  int bytes, places;
  const uint8_t* smem;
  __host__ __device__ static int64_t pitch_of(int features) {
    return (static_cast<int64_t>(features) * sizeof(E) + 15) / 16 * 16 + 16;
  }
  // Sets of rows: two where two CTAs for each SM have room for them, else one
  // (2048 x 12288 float32, dx: 65 us, 88 with two sets and one CTA).
  static int fitting(int features) {
    const int64_t bytes = ARRAYS * pitch_of(features);
    return 2 * bytes <= kLongSmem / 2 ? 2 : bytes <= kLongSmem ? 1 : 0;
  }
  __device__ __forceinline__ Kept(const NormParams& p, const uint8_t* smem)
      : pitch(static_cast<uint32_t>(pitch_of(p.features))), bytes(p.features * static_cast<int>(sizeof(E))),
        places(p.keep), smem(smem) {}
  // Copies row `row` of array `a` into place `place`, asynchronously.
  __device__ __forceinline__ void issue(const E* array, int64_t row, int a, int place) const {
    const uint64_t start = reinterpret_cast<uint64_t>(array) + static_cast<uint64_t>(row) * bytes;
    const int shift = static_cast<int>(start & 15), end = shift + bytes;
    const uint32_t dst = smem_u32(smem) + (place * ARRAYS + a) * pitch;
    for (int i = threadIdx.x * 16; i < end; i += kLong * 16) {
      // a row's last piece ends with the row; its first may begin in the rows
      // before, but not before the first row of all
      if (i == 0 && shift > row * bytes) {
        for (int e = shift; e < (end < 16 ? end : 16); e += sizeof(E)) {
          const void* src = reinterpret_cast<const void*>(start - shift + e);
          if constexpr (sizeof(E) == 4)
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst + e), "r"(ld_32(src)) : "memory");
          else
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + e), "h"(static_cast<uint16_t>(ld_16(src))) : "memory");
        }
      } else {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + i), "l"(start - shift + i),
                     "r"(end - i < 16 ? end - i : 16)
                     : "memory");
      }
    }
  }
  __device__ __forceinline__ const E* at(const E* array, int64_t row, int a, int place) const {
    const uint64_t start = reinterpret_cast<uint64_t>(array) + static_cast<uint64_t>(row) * bytes;
    return reinterpret_cast<const E*>(smem + (place * ARRAYS + a) * pitch + (start & 15));
  }
};

// Brings row `row` to its place; fetch starts a row's copies.
template <typename F>
__device__ __forceinline__ void bring(const NormParams& p, int64_t row, int64_t next, int place, F&& fetch) {
  if (p.keep == 1) {
    __syncthreads();  // the last row has been read
    fetch(row, 0);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();  // with two places this also says that the other one has been read
  if (p.keep == 2 && next < p.rows) fetch(next, place ^ 1);
}

template <typename E, int VEC, bool KEPT>
__global__ void __launch_bounds__(kLong, 2) norm_fwd_long_kernel(const NormParams p) {
  __shared__ float red[2][16][1];
  extern __shared__ __align__(16) uint8_t smem[];
  int turn = 0, place = 0;
  grid_dependency_wait();
  grid_dependents_launch();
  const int F = p.features, c0 = threadIdx.x * VEC;
  constexpr int kStep = kLong * VEC;
  const float inv = 1.0f / static_cast<float>(F);
  const Kept<E, 1> kept(p, smem);
  const E* xs = static_cast<const E*>(p.x);
  auto fetch = [&](int64_t row, int to) { kept.issue(xs, row, 0, to); };
  if (KEPT && p.keep == 2 && blockIdx.x < p.rows) fetch(blockIdx.x, 0);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, place ^= 1) {
    if constexpr (KEPT) bring(p, row, row + gridDim.x, place, fetch);
    const E* x = KEPT ? kept.at(xs, row, 0, p.keep == 2 ? place : 0) : xs + row * F;
    E* y = static_cast<E*>(p.y) + row * F;
    float s[1] = {0.0f}, v[VEC];
    Pack<E, VEC> pk;
#pragma unroll 4
    for (int c = c0; c < F; c += kStep) {
      pk.load(x + c);
      pk.get(v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[0] += v[e];
    }
    row_sums<kLong>(s, red, turn);
    const float mean = s[0] * inv;
    s[0] = 0.0f;
#pragma unroll 4
    for (int c = c0; c < F; c += kStep) {
      pk.load(x + c);
      pk.get(v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[0] = fma(v[e] - mean, v[e] - mean, s[0]);
    }
    row_sums<kLong>(s, red, turn);
    float var = s[0] * inv, off = 0.0f;
    if (far_from_zero(mean, var, p.eps)) {  // the same for all threads
      s[0] = 0.0f;
#pragma unroll 4
      for (int c = c0; c < F; c += kStep) {
        pk.load(x + c);
        pk.get(v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[0] += v[e] - mean;
      }
      row_sums<kLong>(s, red, turn);
      off = s[0] * inv;
      var = corrected(var, off);
    }
    const float rstd = rsqrtf(var + p.eps), rest = -off * rstd;
    if (threadIdx.x == 0 && p.mean) {
      p.mean[row] = mean + off;
      p.rstd[row] = rstd;
    }
    const int64_t offset = row / p.rows_per_weight * p.weight_stride;
#pragma unroll 4
    for (int c = c0; c < F; c += kStep) {
      float w[VEC], b[VEC];
      vector_at<E, VEC>(p, p.weight, offset + c, 1.0f, p.add_one ? 1.0f : 0.0f, w);
      vector_at<E, VEC>(p, p.bias, offset + c, 0.0f, 0.0f, b);
      pk.load(x + c);
      pk.get(v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = fma(fma(v[e] - mean, rstd, rest), w[e], b[e]);
      pk.set(v);
      pk.store(y + c);
    }
  }
}

// ---------------------------------------------------------------------------
// backward

// With c = x - mean, t = dy c and per row u = -r^2 E[g h], v = -r E[g]:
//   dw += t r,  E[g h] = r E[t w],  dx = (dy r) w + (c u + v).
// With up to 24 values of a row a thread keeps c in float32; with more it
// keeps the row as it lies in memory and forms c twice.
template <typename E, int VEC, int NV, int T>
__global__ void __launch_bounds__(T == 32 ? 32 * kWarps : T, ctas_of(T))
    norm_bwd_kernel(const NormParams p) {
  constexpr int L = kLanes<VEC>;
  using A = Lane<VEC>;
  // c kept in float32 beside the row, and rows ahead: in shared memory, or, for
  // elements that are too small to be copied (of which there are few), in
  // registers
  constexpr bool kKeep = VEC * NV <= 24;
  using Next = Ahead<E, VEC, NV, T, 2>;
  static_assert(Next::kAsync || kKeep, "room in the registers for the next row");
  __shared__ float red[2][16][2];
  extern __shared__ __align__(16) uint8_t smem[];  // rows ahead; then, T = 32, sums (kWarps, 2, features)
  int turn = 0;
  grid_dependency_wait();
  grid_dependents_launch();
  const int F = p.features;
  const float inv = 1.0f / static_cast<float>(F);
  const int warp = threadIdx.x >> 5;
  const int c0 = (T == 32 ? threadIdx.x & 31 : threadIdx.x) * VEC, left = F - c0;
  const Rows rows(p);
  Lanes<VEC, NV> weight, dw, db;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < L; ++i) dw[j][i] = db[j][i] = splat<VEC>(0.0f);
  const int64_t first = rows.begin + (T == 32 ? warp : 0), stride = T == 32 ? kWarps : 1;
  int64_t at = first * F + c0;
  const int64_t step = stride * F;
  const E* xs = static_cast<const E*>(p.x);
  const E* dys = static_cast<const E*>(p.dy);
  Share<E, VEC, NV, T> x, dy, next_x, next_dy;
  Next next(smem);
  float mean = 0.0f, rstd = 0.0f, next_mean = 0.0f, next_rstd = 0.0f;
  auto issue = [&](int64_t row, int64_t offset) { next.issue(row < rows.end, left, xs + offset, dys + offset); };
  auto fetch = [&](int64_t row, int64_t offset) {
    if (row < rows.end) {
      if constexpr (!Next::kAsync) {
        next_x.load(xs + offset, left);
        next_dy.load(dys + offset, left);
      }
      next_mean = ld_f32(p.mean + row);
      next_rstd = ld_f32(p.rstd + row);
    }
  };
  if constexpr (Next::kAsync) {
    issue(first, at);
    issue(first + stride, at + step);
  }
  fetch(first, at);
  {
    Vector<E, VEC, NV, T> w;
    w.load(p.weight, p.wide_weight, rows.segment * p.weight_stride + c0, left);
    w.get(p.weight, p.wide_weight, p.add_one ? 0.0f : 1.0f, p.add_one ? 1.0f : 0.0f, weight);
  }
  for (int64_t row = first; row < rows.end; row += stride) {
    mean = next_mean;
    rstd = next_rstd;
    if constexpr (Next::kAsync) {
      next.take(left, x, dy);
      issue(row + 2 * stride, at + 2 * step);
    } else {
      x = next_x;
      dy = next_dy;
    }
    fetch(row + stride, at + step);
    const A scale = splat<VEC>(rstd), minus = splat<VEC>(-mean);
    A centred[kKeep ? NV : 1][L], s0 = splat<VEC>(0.0f), s1 = s0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * T * VEC < left) {
        A d[L];
        A(&c)[L] = centred[kKeep ? j : 0];
        x.v[j].get_lanes(c);
        dy.v[j].get_lanes(d);
#pragma unroll
        for (int i = 0; i < L; ++i) {
          c[i] = add(c[i], minus);
          const A t = mul(d[i], c[i]);
          dw[j][i] = fma(t, scale, dw[j][i]);
          db[j][i] = add(db[j][i], d[i]);
          s0 = fma(d[i], weight[j][i], s0);
          s1 = fma(t, weight[j][i], s1);
        }
      }
    float s[2] = {total(s0), total(s1)};
    row_sums<T>(s, red, turn);
    const float gh = s[1] * inv * rstd;  // E[g h]
    const A v = splat<VEC>(-s[0] * inv * rstd), u = splat<VEC>(-gh * rstd * rstd);
    E* dx = static_cast<E*>(p.y) + at;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * T * VEC < left) {
        A d[L];
        A(&c)[L] = centred[kKeep ? j : 0];
        dy.v[j].get_lanes(d);
        if constexpr (!kKeep) {
          x.v[j].get_lanes(c);
#pragma unroll
          for (int i = 0; i < L; ++i) c[i] = add(c[i], minus);
        }
#pragma unroll
        for (int i = 0; i < L; ++i) d[i] = fma(mul(d[i], scale), weight[j][i], fma(c[i], u, v));
        Pack<E, VEC> out;
        out.set_lanes(d);
        out.store(dx + j * T * VEC);
      }
    at += step;
  }
  if (!p.partial) return;
  float* part = p.partial + static_cast<int64_t>(blockIdx.x) * 2 * F;
  float* sums = reinterpret_cast<float*>(smem);
  float* to = T == 32 ? sums + warp * 2 * F : part;
  if constexpr (T == 32) __syncthreads();  // every warp is done with its rows
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = c0 + j * T * VEC;
    if (c < F) {
      Pack<float, VEC> out;
      out.set_lanes(dw[j]);
      out.store(to + c);
      out.set_lanes(db[j]);
      out.store(to + F + c);
    }
  }
  if constexpr (T == 32) {
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * F; c += 32 * kWarps)
      part[c] = (sums[c] + sums[2 * F + c]) + (sums[4 * F + c] + sums[6 * F + c]);
  }
}

// Rows too long for the registers: dx alone, in two passes over the row in
// shared memory or L2 ...
template <typename E, int VEC, bool KEPT>
__global__ void __launch_bounds__(kLong, 2) norm_dx_long_kernel(const NormParams p) {
  __shared__ float red[2][16][2];
  extern __shared__ __align__(16) uint8_t smem[];
  int turn = 0, place = 0;
  grid_dependency_wait();
  grid_dependents_launch();
  const int F = p.features, c0 = threadIdx.x * VEC;
  constexpr int kStep = kLong * VEC;
  const float inv = 1.0f / static_cast<float>(F), plus = p.add_one ? 1.0f : 0.0f;
  const Kept<E, 2> kept(p, smem);
  const E* xs = static_cast<const E*>(p.x);
  const E* dys = static_cast<const E*>(p.dy);
  auto fetch = [&](int64_t row, int to) {
    kept.issue(xs, row, 0, to);
    kept.issue(dys, row, 1, to);
  };
  if (KEPT && p.keep == 2 && blockIdx.x < p.rows) fetch(blockIdx.x, 0);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, place ^= 1) {
    const float mean = ld_f32(p.mean + row), rstd = ld_f32(p.rstd + row);
    if constexpr (KEPT) bring(p, row, row + gridDim.x, place, fetch);
    const E* x = KEPT ? kept.at(xs, row, 0, p.keep == 2 ? place : 0) : xs + row * F;
    const E* dy = KEPT ? kept.at(dys, row, 1, p.keep == 2 ? place : 0) : dys + row * F;
    E* dx = static_cast<E*>(p.y) + row * F;
    const int64_t offset = row / p.rows_per_weight * p.weight_stride;
    float s[2] = {0.0f, 0.0f}, h[VEC], g[VEC], w[VEC];
    Pack<E, VEC> px, pd;
#pragma unroll 4
    for (int c = c0; c < F; c += kStep) {
      vector_at<E, VEC>(p, p.weight, offset + c, 1.0f, plus, w);
      px.load(x + c);
      pd.load(dy + c);
      px.get(h);
      pd.get(g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        g[e] *= w[e];
        s[0] += g[e];
        s[1] = fma(g[e], (h[e] - mean) * rstd, s[1]);
      }
    }
    row_sums<kLong>(s, red, turn);
    const float mg = s[0] * inv, mgh = s[1] * inv;
#pragma unroll 4
    for (int c = c0; c < F; c += kStep) {
      vector_at<E, VEC>(p, p.weight, offset + c, 1.0f, plus, w);
      px.load(x + c);
      pd.load(dy + c);
      px.get(h);
      pd.get(g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) g[e] = rstd * (g[e] * w[e] - mg - (h[e] - mean) * rstd * mgh);
      pd.set(g);
      pd.store(dx + c);
    }
  }
}

// ... and the sums of a chunk of rows, one thread for VEC columns.
template <typename E, int VEC>
__global__ void __launch_bounds__(256) norm_partial_long_kernel(const NormParams p) {
  const int F = p.features;
  const int c = (blockIdx.x * 256 + threadIdx.x) * VEC;
  grid_dependency_wait();
  grid_dependents_launch();
  if (c >= F) return;
  const int64_t part = blockIdx.y, seg = part / p.chunks, chunk = part % p.chunks;
  const int64_t r0 = seg * p.rows_per_weight + p.rows_per_weight * chunk / p.chunks;
  const int64_t r1 = seg * p.rows_per_weight + p.rows_per_weight * (chunk + 1) / p.chunks;
  const E* x = static_cast<const E*>(p.x) + c;
  const E* dy = static_cast<const E*>(p.dy) + c;
  float dw[VEC] = {}, db[VEC] = {};
  constexpr int kRows = VEC > 2 ? 2 : 4;  // rows loaded at a time
  for (int64_t row = r0; row < r1; row += kRows) {
    Pack<E, VEC> px[kRows], pd[kRows];
    float mean[kRows], rstd[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (row + i < r1) {
        px[i].load_ahead(x + (row + i) * F);
        pd[i].load_ahead(dy + (row + i) * F);
        mean[i] = ld_f32(p.mean + row + i);
        rstd[i] = ld_f32(p.rstd + row + i);
      }
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (row + i < r1) {
        float h[VEC], d[VEC];
        px[i].get(h);
        pd[i].get(d);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          dw[e] = fma(d[e], (h[e] - mean[i]) * rstd[i], dw[e]);
          db[e] += d[e];
        }
      }
  }
  // F is a multiple of VEC, but the sums' rows may start at any float
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    p.partial[(part * 2) * F + c + e] = dw[e];
    p.partial[(part * 2 + 1) * F + c + e] = db[e];
  }
}

// ---------------------------------------------------------------------------
// launches

int enqueue(void (*kernel)(NormParams), dim3 grid, int threads, size_t smem, const NormParams& p, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (smem > 40 * 1024)
    CONVROT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p));
  return check_launch("layer norm kernel");
}

// CTAs of a kernel that an SM holds at once.
template <auto Kernel>
int resident(int threads, int smem) {
  static const int ctas = [&] {
    int n = 0;
    if (smem > 40 * 1024) cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kernel, threads, smem) != cudaSuccess) cudaGetLastError();
    return n < 1 ? 1 : n;
  }();
  return ctas;
}

// A CTA for each long row, as many as the GPU holds at once.
template <auto Kernel>
int longest_rows(const NormParams& p, int64_t smem, cudaStream_t s) {
  int n = 0;
  if (smem > 40 * 1024)
    CONVROT_CUDA_CHECK(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  CONVROT_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kernel, kLong, static_cast<size_t>(smem)));
  const int64_t most = static_cast<int64_t>(n < 1 ? 1 : n) * device_sm_count();
  return enqueue(Kernel, dim3(static_cast<unsigned>(p.rows < most ? p.rows : most)), kLong, static_cast<size_t>(smem), p, s);
}

// Whether every vector of `vec` elements of the rows and of the weights is
// aligned for its accesses.
template <typename E>
bool aligned_for(const NormParams& p, int vec) {
  const int64_t bytes = vec * sizeof(E) < 16 ? vec * sizeof(E) : 16;
  const int64_t wsize = p.wide_weight ? 4 : sizeof(E);
  const int64_t wbytes = vec * wsize < 16 ? vec * wsize : 16;
  return p.features % vec == 0 && aligned_to(p.x, bytes) && aligned_to(p.y, bytes) && aligned_to(p.dy, bytes) &&
         aligned_to(p.weight, wbytes) && aligned_to(p.bias, wbytes) && p.weight_stride * wsize % wbytes == 0;
}

// A pass over rows of `vectors` vectors: RUN(NV, T) launches with NV vectors
// for each of T threads.  U: vectors of a unit, one of 16 bytes or four of one
// or two elements.  Up to four units a lane a warp has a row to itself; then
// CTAs of two or more for each SM, with three or four units a thread, in the
// sizes that keep most of their threads busy; then the largest.
#define CONVROT_NORM_SIZES(RUN, LONG)                   \
  if (vectors <= 32 * U) return RUN(U, 32);             \
  if (vectors <= 32 * 2 * U) return RUN(2 * U, 32);     \
  if (vectors <= 32 * 4 * U) return RUN(4 * U, 32);     \
  if (vectors <= 64 * 3 * U) return RUN(3 * U, 64);     \
  if (vectors <= 128 * 3 * U) return RUN(3 * U, 128);   \
  if (vectors <= 192 * 3 * U) return RUN(3 * U, 192);   \
  if (vectors <= 384 * 3 * U) return RUN(3 * U, 384);   \
  if (vectors <= 512 * 4 * U) return RUN(4 * U, 512);   \
  return LONG();

template <typename E, int VEC, int U>
int forward_rows(NormParams p, int vectors, cudaStream_t s) {
  const int64_t segments = p.rows / p.rows_per_weight;
  // CTAs that share a segment's rows: a CTA for each row (4 rows), until the
  // SMs hold no more (12288 x 1024 bf16: 9.5 us, 13 with more CTAs than fit)
  auto grid = [&](int threads, int64_t resident) {
    const int64_t rows_at = threads == 32 ? kWarps : 1;
    const int64_t chunks = (p.rows_per_weight + rows_at - 1) / rows_at;
    const int64_t limit = resident * device_sm_count() / segments;
    p.chunks = static_cast<int>(chunks < limit ? chunks : (limit < 1 ? 1 : limit));
    return dim3(static_cast<unsigned>(segments * p.chunks));
  };
  auto longest = [&] {
    p.keep = Kept<E, 1>::fitting(p.features);
    const int64_t bytes = p.keep * Kept<E, 1>::pitch_of(p.features);
    return p.keep ? longest_rows<norm_fwd_long_kernel<E, VEC, true>>(p, bytes, s)
                  : longest_rows<norm_fwd_long_kernel<E, VEC, false>>(p, 0, s);
  };
#define CONVROT_RUN(NV, T)                                                                                       \
  enqueue(norm_fwd_kernel<E, VEC, NV, T>,                                                                        \
          grid(T, resident<norm_fwd_kernel<E, VEC, NV, T>>(T == 32 ? 32 * kWarps : T, Ahead<E, VEC, NV, T, 1>::kSmem)), \
          T == 32 ? 32 * kWarps : T, Ahead<E, VEC, NV, T, 1>::kSmem, p, s)
  CONVROT_NORM_SIZES(CONVROT_RUN, longest)
#undef CONVROT_RUN
}

template <typename E, int VEC, int U>
int backward_rows(NormParams p, int vectors, cudaStream_t s) {
  const unsigned ctas = static_cast<unsigned>(p.rows / p.rows_per_weight * p.chunks);
  auto longest = [&] {
    p.keep = Kept<E, 2>::fitting(p.features);
    const int64_t bytes = 2 * p.keep * Kept<E, 2>::pitch_of(p.features);
    int rc = p.keep ? longest_rows<norm_dx_long_kernel<E, VEC, true>>(p, bytes, s)
                    : longest_rows<norm_dx_long_kernel<E, VEC, false>>(p, 0, s);
    if (rc == CONVROT_OK && p.partial)
      rc = enqueue(norm_partial_long_kernel<E, VEC>, dim3((p.features + 256 * VEC - 1) / (256 * VEC), ctas), 256, 0, p, s);
    return rc;
  };
#define CONVROT_RUN(NV, T)                                                 \
  enqueue(norm_bwd_kernel<E, VEC, NV, T>, ctas, T == 32 ? 32 * kWarps : T, \
          std::max<size_t>(Ahead<E, VEC, NV, T, 2>::kSmem, T == 32 ? 2 * kWarps * sizeof(float) * p.features : 0), p, s)
  CONVROT_NORM_SIZES(CONVROT_RUN, longest)
#undef CONVROT_RUN
}

}  // namespace

template <typename E>
int forward(const NormParams& p, cudaStream_t s) {
  constexpr int W = 16 / sizeof(E);
  if (aligned_for<E>(p, W)) return forward_rows<E, W, 1>(p, p.features / W, s);
  if constexpr (W == 8)
    if (aligned_for<E>(p, 2)) return forward_rows<E, 2, 4>(p, p.features / 2, s);
  return forward_rows<E, 1, 4>(p, p.features, s);
}

template <typename E>
int backward(const NormParams& p, cudaStream_t s) {
  constexpr int W = 16 / sizeof(E);
  if (aligned_for<E>(p, W)) return backward_rows<E, W, 1>(p, p.features / W, s);
  if constexpr (W == 8)
    if (aligned_for<E>(p, 2)) return backward_rows<E, 2, 4>(p, p.features / 2, s);
  return backward_rows<E, 1, 4>(p, p.features, s);
}
#endif  // CONVROT_NORM_KERNELS

}  // namespace norm
}  // namespace convrot
