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
// and writes dx, once each.  A row stays in registers between its statistics
// and its output.  In the backward pass a thread keeps the same columns for
// all rows of its CTA, so the column sums stay in registers too; a second
// small kernel adds up the CTAs' sums in a fixed order.
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

// Sums of N values over the rows' threads: a warp (WARP) or the CTA.  red
// holds two sets of 32 warps' values, used in turn, so that one barrier for
// each call is enough.
template <bool WARP, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*red)[32][N], int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if constexpr (!WARP) {
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) red[turn][threadIdx.x >> 5][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < warps ? red[turn][lane][i] : 0.0f);
    turn ^= 1;
  }
}

// A row's share of one thread: NV vectors of VEC elements, `threads` vectors
// apart.  Columns past the end are never touched.
template <typename T, int VEC, int NV>
struct Share {
  Pack<T, VEC> v[NV];
  __device__ __forceinline__ void load(const T* row, int c0, int step, int features) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (c0 + j * step < features) v[j].load_nc(row + c0 + j * step);
  }
};

template <typename TW, int VEC>
__device__ __forceinline__ void weights(const NormParams& p, const TW* w, int c, float (&out)[VEC]) {
  if (w) {
    Pack<TW, VEC> pk;
    pk.load_nc(w + c);
    pk.get(out);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = p.add_one ? 0.0f : 1.0f;
  }
  if (p.add_one)
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] += 1.0f;
}

template <typename TW>
__device__ __forceinline__ const TW* at(const void* base, int64_t offset) {
  return base ? static_cast<const TW*>(base) + offset : nullptr;
}

// ---------------------------------------------------------------------------
// forward

template <typename T, typename TW, int VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 512) norm_fwd_kernel(const NormParams p) {
  __shared__ float red[2][32][1];
  int turn = 0;
  grid_dependency_wait();
  grid_dependents_launch();
  const int F = p.features;
  const float inv = 1.0f / static_cast<float>(F);
  const int c0 = (WARP ? threadIdx.x & 31 : threadIdx.x) * VEC, step = (WARP ? 32 : blockDim.x) * VEC;
  const int64_t first = WARP ? static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t stride = WARP ? static_cast<int64_t>(gridDim.x) * 4 : gridDim.x;
  for (int64_t row = first; row < p.rows; row += stride) {
    Share<T, VEC, NV> x;
    x.load(static_cast<const T*>(p.x) + row * F, c0, step, F);
    float s[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (c0 + j * step < F) {
        float v[VEC];
        x.v[j].get(v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[0] += v[i];
      }
    row_sum<WARP>(s, red, turn);
    const float mean = s[0] * inv;
    s[0] = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (c0 + j * step < F) {
        float v[VEC];
        x.v[j].get(v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[0] = fmaf(v[i] - mean, v[i] - mean, s[0]);
      }
    row_sum<WARP>(s, red, turn);
    const float rstd = rsqrtf(s[0] * inv + p.eps);
    if ((WARP ? threadIdx.x & 31 : threadIdx.x) == 0 && p.mean) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    const int64_t offset = p.rows == p.rows_per_weight ? 0 : row / p.rows_per_weight * p.weight_stride;
    const TW* weight = at<TW>(p.weight, offset);
    const TW* bias = at<TW>(p.bias, offset);
    T* y = static_cast<T*>(p.y) + row * F;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = c0 + j * step;
      if (c < F) {
        float v[VEC], w[VEC], b[VEC];
        x.v[j].get(v);
        weights<TW, VEC>(p, weight, c, w);
        if (bias) {
          Pack<TW, VEC> pk;
          pk.load_nc(bias + c);
          pk.get(b);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = fmaf((v[i] - mean) * rstd, w[i], bias ? b[i] : 0.0f);
        Pack<T, VEC> out;
        out.set(v);
        out.store(y + c);
      }
    }
  }
}

// Rows too long for the registers: three passes over the row, the later ones
// through L2.
template <typename T, typename TW>
__global__ void __launch_bounds__(512) norm_fwd_long_kernel(const NormParams p) {
  __shared__ float red[2][32][1];
  int turn = 0;
  grid_dependency_wait();
  grid_dependents_launch();
  const int F = p.features;
  const float inv = 1.0f / static_cast<float>(F);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * F;
    T* y = static_cast<T*>(p.y) + row * F;
    float s[1] = {0.0f};
    for (int c = threadIdx.x; c < F; c += blockDim.x) s[0] += Elem<T>::to_f(x[c]);
    row_sum<false>(s, red, turn);
    const float mean = s[0] * inv;
    s[0] = 0.0f;
    for (int c = threadIdx.x; c < F; c += blockDim.x) {
      const float d = Elem<T>::to_f(x[c]) - mean;
      s[0] = fmaf(d, d, s[0]);
    }
    row_sum<false>(s, red, turn);
    const float rstd = rsqrtf(s[0] * inv + p.eps);
    if (threadIdx.x == 0 && p.mean) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    const int64_t offset = row / p.rows_per_weight * p.weight_stride;
    const TW* weight = at<TW>(p.weight, offset);
    const TW* bias = at<TW>(p.bias, offset);
    for (int c = threadIdx.x; c < F; c += blockDim.x) {
      float w[1];
      weights<TW, 1>(p, weight, c, w);
      y[c] = Elem<T>::from_f(
          fmaf((Elem<T>::to_f(x[c]) - mean) * rstd, w[0], bias ? Elem<TW>::to_f(bias[c]) : 0.0f));
    }
  }
}

// ---------------------------------------------------------------------------
// backward

// CTA (segment, chunk) walks the rows of its chunk.  WARP: each of 4 warps a
// row of its own; else the CTA one row at a time.
template <typename T, typename TW, int VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 512) norm_bwd_kernel(const NormParams p) {
  __shared__ float red[2][32][2];
  extern __shared__ float sums[];  // WARP: (4, 2, features)
  int turn = 0;
  grid_dependency_wait();
  grid_dependents_launch();
  const int F = p.features;
  const float inv = 1.0f / static_cast<float>(F);
  const int warp = threadIdx.x >> 5;
  const int c0 = (WARP ? threadIdx.x & 31 : threadIdx.x) * VEC, step = (WARP ? 32 : blockDim.x) * VEC;
  const int64_t seg = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
  const int64_t base = seg * p.rows_per_weight;
  const int64_t r0 = base + p.rows_per_weight * chunk / p.chunks;
  const int64_t r1 = base + p.rows_per_weight * (chunk + 1) / p.chunks;
  const TW* weight = at<TW>(p.weight, seg * p.weight_stride);
  const T* xs = static_cast<const T*>(p.x);
  const T* dys = static_cast<const T*>(p.dy);
  T* dxs = static_cast<T*>(p.y);
  float dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[j][i] = db[j][i] = 0.0f;
  const int64_t first = WARP ? r0 + warp : r0, stride = WARP ? 4 : 1;
  // the next row's loads are in flight while this row is worked on, where the
  // registers hold both
  constexpr bool kAhead = NV * Pack<T, VEC>::kWords <= 8;
  Share<T, VEC, NV> x, dy, next_x, next_dy;
  float mean, rstd, next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch = [&](int64_t row) {
    if (row < r1) {
      next_x.load(xs + row * F, c0, step, F);
      next_dy.load(dys + row * F, c0, step, F);
      next_mean = __ldg(p.mean + row);
      next_rstd = __ldg(p.rstd + row);
    }
  };
  if (kAhead) fetch(first);
  for (int64_t row = first; row < r1; row += stride) {
    if (!kAhead) fetch(row);
    x = next_x;
    dy = next_dy;
    mean = next_mean;
    rstd = next_rstd;
    if (kAhead) fetch(row + stride);
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = c0 + j * step;
      if (c < F) {
        float v[VEC], d[VEC], w[VEC];
        x.v[j].get(v);
        dy.v[j].get(d);
        weights<TW, VEC>(p, weight, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float h = (v[i] - mean) * rstd, g = d[i] * w[i];
          dw[j][i] = fmaf(d[i], h, dw[j][i]);
          db[j][i] += d[i];
          s[0] += g;
          s[1] = fmaf(g, h, s[1]);
        }
      }
    }
    row_sum<WARP>(s, red, turn);
    const float mg = s[0] * inv, mgh = s[1] * inv;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = c0 + j * step;
      if (c < F) {
        float v[VEC], d[VEC], w[VEC];
        x.v[j].get(v);
        dy.v[j].get(d);
        weights<TW, VEC>(p, weight, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float h = (v[i] - mean) * rstd, g = d[i] * w[i];
          v[i] = rstd * (g - mg - h * mgh);
        }
        Pack<T, VEC> out;
        out.set(v);
        out.store(dxs + row * F + c);
      }
    }
  }
  if (!p.partial) return;
  float* part = p.partial + static_cast<int64_t>(blockIdx.x) * 2 * F;
  if constexpr (WARP) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = c0 + j * step + i;
        if (c < F) {
          sums[(warp * 2) * F + c] = dw[j][i];
          sums[(warp * 2 + 1) * F + c] = db[j][i];
        }
      }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * F; c += 128)
      part[c] = (sums[c] + sums[2 * F + c]) + (sums[4 * F + c] + sums[6 * F + c]);
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = c0 + j * step;
      if (c < F) {
        if constexpr (VEC % 4 == 0) {
#pragma unroll
          for (int i = 0; i < VEC; i += 4) {
            *reinterpret_cast<float4*>(part + c + i) = make_float4(dw[j][i], dw[j][i + 1], dw[j][i + 2], dw[j][i + 3]);
            *reinterpret_cast<float4*>(part + F + c + i) =
                make_float4(db[j][i], db[j][i + 1], db[j][i + 2], db[j][i + 3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            part[c + i] = dw[j][i];
            part[F + c + i] = db[j][i];
          }
        }
      }
    }
  }
}

// Rows too long for the registers: dx alone, in two passes over the row ...
template <typename T, typename TW>
__global__ void __launch_bounds__(512) norm_dx_long_kernel(const NormParams p) {
  __shared__ float red[2][32][2];
  int turn = 0;
  grid_dependency_wait();
  grid_dependents_launch();
  const int F = p.features;
  const float inv = 1.0f / static_cast<float>(F);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * F;
    const T* dy = static_cast<const T*>(p.dy) + row * F;
    T* dx = static_cast<T*>(p.y) + row * F;
    const TW* weight = at<TW>(p.weight, row / p.rows_per_weight * p.weight_stride);
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s[2] = {0.0f, 0.0f};
    for (int c = threadIdx.x; c < F; c += blockDim.x) {
      float w[1];
      weights<TW, 1>(p, weight, c, w);
      const float g = Elem<T>::to_f(dy[c]) * w[0];
      s[0] += g;
      s[1] = fmaf(g, (Elem<T>::to_f(x[c]) - mean) * rstd, s[1]);
    }
    row_sum<false>(s, red, turn);
    const float mg = s[0] * inv, mgh = s[1] * inv;
    for (int c = threadIdx.x; c < F; c += blockDim.x) {
      float w[1];
      weights<TW, 1>(p, weight, c, w);
      const float g = Elem<T>::to_f(dy[c]) * w[0], h = (Elem<T>::to_f(x[c]) - mean) * rstd;
      dx[c] = Elem<T>::from_f(rstd * (g - mg - h * mgh));
    }
  }
}

// ... and the sums of a chunk of rows, one thread for a column.
template <typename T>
__global__ void __launch_bounds__(256) norm_partial_long_kernel(const NormParams p) {
  const int F = p.features;
  const int c = blockIdx.x * 256 + threadIdx.x;
  grid_dependency_wait();
  grid_dependents_launch();
  if (c >= F) return;
  const int64_t part = blockIdx.y, seg = part / p.chunks, chunk = part % p.chunks;
  const int64_t r0 = seg * p.rows_per_weight + p.rows_per_weight * chunk / p.chunks;
  const int64_t r1 = seg * p.rows_per_weight + p.rows_per_weight * (chunk + 1) / p.chunks;
  float dw = 0.0f, db = 0.0f;
#pragma unroll 4
  for (int64_t row = r0; row < r1; ++row) {
    const float d = Elem<T>::to_f(static_cast<const T*>(p.dy)[row * F + c]);
    dw = fmaf(d, (Elem<T>::to_f(static_cast<const T*>(p.x)[row * F + c]) - p.mean[row]) * p.rstd[row], dw);
    db += d;
  }
  p.partial[(part * 2) * F + c] = dw;
  p.partial[(part * 2 + 1) * F + c] = db;
}

// dweight and dbias: the chunks' sums added up, 32 columns a CTA, 16 threads
// for each column that take every 16th chunk, then a tree over the 16.
template <typename TW>
__global__ void __launch_bounds__(512) norm_reduce_kernel(const NormParams p) {
  __shared__ float sw[16][33], sb[16][33];
  grid_dependency_wait();
  grid_dependents_launch();
  const int F = p.features;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + x;
  const int64_t seg = blockIdx.y;
  float dw = 0.0f, db = 0.0f;
  if (c < F) {
    const float* part = p.partial + seg * p.chunks * 2 * F;
#pragma unroll 4
    for (int chunk = y; chunk < p.chunks; chunk += 16) {
      dw += part[static_cast<int64_t>(chunk) * 2 * F + c];
      db += part[static_cast<int64_t>(chunk) * 2 * F + F + c];
    }
  }
  sw[y][x] = dw;
  sb[y][x] = db;
  __syncthreads();
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
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

// ---------------------------------------------------------------------------
// launches

// CTAs that share a segment's rows, each with one partial sum: about two CTAs
// for each SM in all.
int chunks_of(int64_t rows_per_weight, int64_t segments) {
  int64_t chunks = 2LL * device_sm_count() / segments;
  if (chunks > rows_per_weight) chunks = rows_per_weight;
  return static_cast<int>(chunks < 1 ? 1 : chunks);
}

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
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p));
  return check_launch("layer norm kernel");
}

// How a row is spread over threads: `wide` elements a vector where every row
// and vector is aligned for it, else single elements.
template <typename T>
struct Plan {
  static constexpr int kWide = 16 / sizeof(T);
  bool wide;
  int vectors;
  Plan(const NormParams& p, bool weight_ok) {
    wide = p.features % kWide == 0 && aligned_to(p.x, 16) && aligned_to(p.y, 16) && aligned_to(p.dy, 16) && weight_ok;
    vectors = wide ? p.features / kWide : p.features;
  }
};

template <typename TW>
bool weight_aligned(const NormParams& p, int vec) {
  const int64_t bytes = vec * static_cast<int64_t>(sizeof(TW)) < 16 ? vec * sizeof(TW) : 16;
  return aligned_to(p.weight, bytes) && aligned_to(p.bias, bytes) &&
         p.weight_stride * static_cast<int64_t>(sizeof(TW)) % bytes == 0;
}

inline unsigned rows_grid(int64_t rows, int64_t per_cta, int64_t most) {
  const int64_t ctas = (rows + per_cta - 1) / per_cta;
  return static_cast<unsigned>(ctas < most ? ctas : most);
}

template <typename T, typename TW, int VEC, int E>
int forward_rows(const NormParams& p, int vectors, cudaStream_t s) {
  // E: vectors that make 16 bytes' worth of elements (1 when wide)
  const int64_t most = 64LL * device_sm_count();
  if (vectors <= 32 * 4 * E) return enqueue(norm_fwd_kernel<T, TW, VEC, 4 * E, true>, rows_grid(p.rows, 4, most), 128, 0, p, s);
  if (VEC > 1 && vectors <= 32 * 12 && p.rows >= 4LL * device_sm_count())
    return enqueue(norm_fwd_kernel<T, TW, VEC, (VEC > 1 ? 12 : 4), true>, rows_grid(p.rows, 4, most), 128, 0, p, s);
  const int per = vectors <= 512 * E ? E : 4 * E;
  const int threads = (((vectors + per - 1) / per) + 31) / 32 * 32;
  if (vectors <= 512 * E) return enqueue(norm_fwd_kernel<T, TW, VEC, E, false>, rows_grid(p.rows, 1, most), threads, 0, p, s);
  if (vectors <= 512 * 4 * E)
    return enqueue(norm_fwd_kernel<T, TW, VEC, 4 * E, false>, rows_grid(p.rows, 1, most), threads, 0, p, s);
  return enqueue(norm_fwd_long_kernel<T, TW>, rows_grid(p.rows, 1, most), 512, 0, p, s);
}

template <typename T, typename TW>
int forward(const NormParams& p, cudaStream_t s) {
  constexpr int W = Plan<T>::kWide;
  const Plan<T> plan(p, weight_aligned<TW>(p, W));
  if (plan.wide) return forward_rows<T, TW, W, 1>(p, plan.vectors, s);
  return forward_rows<T, TW, 1, W>(p, plan.vectors, s);
}

template <typename T, typename TW, int VEC, int E>
int backward_rows(const NormParams& p, int vectors, cudaStream_t s) {
  const unsigned ctas = static_cast<unsigned>(p.rows / p.rows_per_weight * p.chunks);
  if (vectors <= 32 * 4 * E)
    return enqueue(norm_bwd_kernel<T, TW, VEC, 4 * E, true>, ctas, 128, 8 * sizeof(float) * p.features, p, s);
  const int most = sizeof(T) == 2 ? 4 : 4;
  const int per = vectors <= 512 * E ? 1 : vectors <= 1024 * E ? 2 : most;
  const int threads = ((vectors + per * E - 1) / (per * E) + 31) / 32 * 32;
  if (vectors <= 512 * E) return enqueue(norm_bwd_kernel<T, TW, VEC, E, false>, ctas, threads, 0, p, s);
  if (vectors <= 1024 * E) return enqueue(norm_bwd_kernel<T, TW, VEC, 2 * E, false>, ctas, threads, 0, p, s);
  if (vectors <= 2048 * E) return enqueue(norm_bwd_kernel<T, TW, VEC, 4 * E, false>, ctas, threads, 0, p, s);
  const unsigned most_rows = rows_grid(p.rows, 1, 8LL * device_sm_count());
  int rc = enqueue(norm_dx_long_kernel<T, TW>, most_rows, 512, 0, p, s);
  if (rc == CONVROT_OK && p.partial)
    rc = enqueue(norm_partial_long_kernel<T>, dim3((p.features + 255) / 256, ctas), 256, 0, p, s);
  return rc;
}

template <typename T, typename TW>
int backward(const NormParams& p, cudaStream_t s) {
  constexpr int W = Plan<T>::kWide;
  const Plan<T> plan(p, weight_aligned<TW>(p, W));
  const int rc = plan.wide ? backward_rows<T, TW, W, 1>(p, plan.vectors, s) : backward_rows<T, TW, 1, W>(p, plan.vectors, s);
  if (rc != CONVROT_OK || !p.partial) return rc;
  const unsigned segments = static_cast<unsigned>(p.rows / p.rows_per_weight);
  return enqueue(norm_reduce_kernel<TW>, dim3((p.features + 31) / 32, segments), 512, 0, p, s);
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
  p.partial = sums ? static_cast<float*>(workspace) : nullptr;
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
