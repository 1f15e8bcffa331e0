// Layer norm kernels (layer_norm.cu), instantiated for one type of x in each
// of layer_norm_{bf16,f16,f32}.cu.
//   mean = E[x], r = (E[(x - mean)^2] + eps)^-1/2, h = (x - mean) r
//   y  = h w + b                         (w = 1 + weight with add_one)
//   g  = dy w
//   dx = r (g - E[g] - h E[g h])
//   dweight = sum dy h,  dbias = sum dy  (over the rows that share a weight)
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
//   forward           22 (0.93)    9.4 (0.82)    26 (0.89)     27 (0.77)    30 (0.68)    26 (0.79)
//   backward          39 (0.79)    17 (0.67)     44 (0.79)     39 (0.78)    50 (0.62)    75 (0.41)
// Rows of odd length, whose elements are moved one by one: 5003 x 1153 float32
// 10.8 and 18.5 us (1152: 7.5 and 14.8).  16-byte pieces copied to shared
// memory across the rows' ends and read back by element took longer, for the
// barrier that each row then needs: 12.9 and 18.6.
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

template <typename E>
__device__ __forceinline__ E ld(const E* p) {
  Pack<E, 1> pk;
  pk.load_ahead(p);
  if constexpr (sizeof(E) == 4) return __uint_as_float(pk.w[0]);
  else {
    const uint16_t h = static_cast<uint16_t>(pk.w[0]);
    return *reinterpret_cast<const E*>(&h);
  }
}

// One value of a segment's vectors.
template <typename E>
__device__ __forceinline__ float vector_at(const NormParams& p, const void* base, int64_t at) {
  return p.wide_weight ? ld_f32(static_cast<const float*>(base) + at) : Elem<E>::to_f(ld(static_cast<const E*>(base) + at));
}
template <typename E>
__device__ __forceinline__ float weight_at(const NormParams& p, int64_t at) {
  const float one = p.add_one ? 1.0f : 0.0f;
  return p.weight ? one + vector_at<E>(p, p.weight, at) : 1.0f;
}
template <typename E>
__device__ __forceinline__ float bias_at(const NormParams& p, int64_t at) {
  return p.bias ? vector_at<E>(p, p.bias, at) : 0.0f;
}

// ---------------------------------------------------------------------------
// forward

// T threads share a row: 32 (each warp of the CTA rows of its own), or the CTA.
template <typename E, int VEC, int NV, int T>
__global__ void __launch_bounds__(T == 32 ? 32 * kWarps : T) norm_fwd_kernel(const NormParams p) {
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
    const float rstd = rsqrtf(s[0] * inv + p.eps);
    const A scale = splat<VEC>(rstd);
    if (c0 == 0 && p.mean) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * T * VEC < left) {
#pragma unroll
        for (int i = 0; i < L; ++i) v[j][i] = fma(mul(v[j][i], scale), weight[j][i], bias[j][i]);
        Pack<E, VEC> out;
        out.set_lanes(v[j]);
        out.store(dst + j * T * VEC);
      }
    dst += step;
  }
}

// Rows too long for the registers: three passes over the row, the later ones
// through L2.
template <typename E>
__global__ void __launch_bounds__(512) norm_fwd_long_kernel(const NormParams p) {
  __shared__ float red[2][16][1];
  int turn = 0;
  grid_dependency_wait();
  grid_dependents_launch();
  const int F = p.features;
  const float inv = 1.0f / static_cast<float>(F);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const E* x = static_cast<const E*>(p.x) + row * F;
    E* y = static_cast<E*>(p.y) + row * F;
    float s[1] = {0.0f};
#pragma unroll 8
    for (int c = threadIdx.x; c < F; c += 512) s[0] += Elem<E>::to_f(ld(x + c));
    row_sums<512>(s, red, turn);
    const float mean = s[0] * inv;
    s[0] = 0.0f;
#pragma unroll 8
    for (int c = threadIdx.x; c < F; c += 512) {
      const float d = Elem<E>::to_f(ld(x + c)) - mean;
      s[0] = fma(d, d, s[0]);
    }
    row_sums<512>(s, red, turn);
    const float rstd = rsqrtf(s[0] * inv + p.eps);
    if (threadIdx.x == 0 && p.mean) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    const int64_t offset = row / p.rows_per_weight * p.weight_stride;
#pragma unroll 4
    for (int c = threadIdx.x; c < F; c += 512)
      y[c] = Elem<E>::from_f(fma((Elem<E>::to_f(ld(x + c)) - mean) * rstd, weight_at<E>(p, offset + c),
                                 bias_at<E>(p, offset + c)));
  }
}

// ---------------------------------------------------------------------------
// backward

// With h = x r - mean r and per row u = -r E[g h], v = -r E[g]:
//   dx = (dy r) w + (h u + v).
// With up to 24 values of a row a thread keeps h in float32; with more it
// keeps the row as it lies in memory and forms h twice.
template <typename E, int VEC, int NV, int T>
__global__ void __launch_bounds__(T == 32 ? 32 * kWarps : T, ctas_of(T))
    norm_bwd_kernel(const NormParams p) {
  constexpr int L = kLanes<VEC>;
  using A = Lane<VEC>;
  // h kept in float32 beside the row, and rows ahead: in shared memory, or in
  // registers for elements that are too small to be copied
  constexpr bool kKeep = VEC * NV <= 24;
  using Next = Ahead<E, VEC, NV, T, 2>;
  constexpr bool kRegs = !Next::kAsync && kKeep;
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
  if (Next::kAsync || kRegs) fetch(first, at);
  {
    Vector<E, VEC, NV, T> w;
    w.load(p.weight, p.wide_weight, rows.segment * p.weight_stride + c0, left);
    w.get(p.weight, p.wide_weight, p.add_one ? 0.0f : 1.0f, p.add_one ? 1.0f : 0.0f, weight);
  }
  for (int64_t row = first; row < rows.end; row += stride) {
    if (!Next::kAsync && !kRegs) fetch(row, at);
    mean = next_mean;
    rstd = next_rstd;
    if constexpr (Next::kAsync) {
      next.take(left, x, dy);
      issue(row + 2 * stride, at + 2 * step);
    } else {
      x = next_x;
      dy = next_dy;
    }
    if (Next::kAsync || kRegs) fetch(row + stride, at + step);
    const A scale = splat<VEC>(rstd), minus = splat<VEC>(-mean * rstd);
    A h[kKeep ? NV : 1][L], s0 = splat<VEC>(0.0f), s1 = s0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * T * VEC < left) {
        A d[L];
        A(&hj)[L] = h[kKeep ? j : 0];
        x.v[j].get_lanes(hj);
        dy.v[j].get_lanes(d);
#pragma unroll
        for (int i = 0; i < L; ++i) {
          hj[i] = fma(hj[i], scale, minus);
          const A t = mul(d[i], hj[i]);
          dw[j][i] = add(dw[j][i], t);
          db[j][i] = add(db[j][i], d[i]);
          s0 = fma(d[i], weight[j][i], s0);
          s1 = fma(t, weight[j][i], s1);
        }
      }
    float s[2] = {total(s0), total(s1)};
    row_sums<T>(s, red, turn);
    const A v = splat<VEC>(-s[0] * inv * rstd), u = splat<VEC>(-s[1] * inv * rstd);
    E* dx = static_cast<E*>(p.y) + at;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * T * VEC < left) {
        A d[L];
        A(&hj)[L] = h[kKeep ? j : 0];
        dy.v[j].get_lanes(d);
        if constexpr (!kKeep) {
          x.v[j].get_lanes(hj);
#pragma unroll
          for (int i = 0; i < L; ++i) hj[i] = fma(hj[i], scale, minus);
        }
#pragma unroll
        for (int i = 0; i < L; ++i) d[i] = fma(mul(d[i], scale), weight[j][i], fma(hj[i], u, v));
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

// Rows too long for the registers: dx alone, in two passes over the row ...
template <typename E>
__global__ void __launch_bounds__(512) norm_dx_long_kernel(const NormParams p) {
  __shared__ float red[2][16][2];
  int turn = 0;
  grid_dependency_wait();
  grid_dependents_launch();
  const int F = p.features;
  const float inv = 1.0f / static_cast<float>(F);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const E* x = static_cast<const E*>(p.x) + row * F;
    const E* dy = static_cast<const E*>(p.dy) + row * F;
    E* dx = static_cast<E*>(p.y) + row * F;
    const int64_t offset = row / p.rows_per_weight * p.weight_stride;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s[2] = {0.0f, 0.0f};
#pragma unroll 4
    for (int c = threadIdx.x; c < F; c += 512) {
      const float g = Elem<E>::to_f(ld(dy + c)) * weight_at<E>(p, offset + c);
      s[0] += g;
      s[1] = fma(g, (Elem<E>::to_f(ld(x + c)) - mean) * rstd, s[1]);
    }
    row_sums<512>(s, red, turn);
    const float mg = s[0] * inv, mgh = s[1] * inv;
#pragma unroll 4
    for (int c = threadIdx.x; c < F; c += 512) {
      const float g = Elem<E>::to_f(ld(dy + c)) * weight_at<E>(p, offset + c);
      const float h = (Elem<E>::to_f(ld(x + c)) - mean) * rstd;
      dx[c] = Elem<E>::from_f(rstd * (g - mg - h * mgh));
    }
  }
}

// ... and the sums of a chunk of rows, one thread for a column.
template <typename E>
__global__ void __launch_bounds__(256) norm_partial_long_kernel(const NormParams p) {
  const int F = p.features;
  const int c = blockIdx.x * 256 + threadIdx.x;
  grid_dependency_wait();
  grid_dependents_launch();
  if (c >= F) return;
  const int64_t part = blockIdx.y, seg = part / p.chunks, chunk = part % p.chunks;
  const int64_t r0 = seg * p.rows_per_weight + p.rows_per_weight * chunk / p.chunks;
  const int64_t r1 = seg * p.rows_per_weight + p.rows_per_weight * (chunk + 1) / p.chunks;
  const E* x = static_cast<const E*>(p.x);
  const E* dy = static_cast<const E*>(p.dy);
  float dw = 0.0f, db = 0.0f;
#pragma unroll 4
  for (int64_t row = r0; row < r1; ++row) {
    const float d = Elem<E>::to_f(ld(dy + row * F + c));
    dw = fma(d, (Elem<E>::to_f(ld(x + row * F + c)) - ld_f32(p.mean + row)) * ld_f32(p.rstd + row), dw);
    db += d;
  }
  p.partial[(part * 2) * F + c] = dw;
  p.partial[(part * 2 + 1) * F + c] = db;
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
    const int64_t most = 4LL * device_sm_count();
    return enqueue(norm_fwd_long_kernel<E>, dim3(static_cast<unsigned>(p.rows < most ? p.rows : most)), 512, 0, p, s);
  };
#define CONVROT_RUN(NV, T)                                                                                       \
  enqueue(norm_fwd_kernel<E, VEC, NV, T>,                                                                        \
          grid(T, resident<norm_fwd_kernel<E, VEC, NV, T>>(T == 32 ? 32 * kWarps : T, Ahead<E, VEC, NV, T, 1>::kSmem)), \
          T == 32 ? 32 * kWarps : T, Ahead<E, VEC, NV, T, 1>::kSmem, p, s)
  CONVROT_NORM_SIZES(CONVROT_RUN, longest)
#undef CONVROT_RUN
}

template <typename E, int VEC, int U>
int backward_rows(const NormParams& p, int vectors, cudaStream_t s) {
  const unsigned ctas = static_cast<unsigned>(p.rows / p.rows_per_weight * p.chunks);
  auto longest = [&] {
    const int64_t most = 4LL * device_sm_count();
    int rc = enqueue(norm_dx_long_kernel<E>, dim3(static_cast<unsigned>(p.rows < most ? p.rows : most)), 512, 0, p, s);
    if (rc == CONVROT_OK && p.partial)
      rc = enqueue(norm_partial_long_kernel<E>, dim3((p.features + 255) / 256, ctas), 256, 0, p, s);
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
