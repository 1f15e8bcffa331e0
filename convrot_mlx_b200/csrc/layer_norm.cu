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
// and writes dx, once each.  A thread keeps the same columns for all rows of
// its CTA: a row stays in registers between its statistics and its output,
// the weights are loaded once for a CTA, and the column sums of the backward
// pass stay in registers too (a second small kernel adds up the CTAs' sums in
// a fixed order).  What costs beside the memory is the exchange between the
// threads of a row, so a thread has 24 values of a row (12 in float32) and a
// CTA exchanges the sums of two rows at once.
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

// Adds up each of N values (1, 2 or 4) over a warp: while there are several,
// lanes exchange halves of the set, so N values take about as many shuffles as
// one.  Afterwards v[0] of lane l is the sum of value l / (32 / N).
template <int N>
__device__ __forceinline__ void warp_sums(float (&v)[N]) {
  const int lane = threadIdx.x & 31;
  int o = 16;
#pragma unroll
  for (int n = N; n > 1; n /= 2, o /= 2) {
    const bool high = lane & o;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float send = high ? v[i] : v[i + n / 2];
      v[i] = (high ? v[i + n / 2] : v[i]) + __shfl_xor_sync(0xFFFFFFFFu, send, o);
    }
  }
#pragma unroll
  for (; o > 0; o /= 2) v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], o);
}

// Sums of N values over the threads of a row, a warp (WARP) or the CTA, for
// all of them.  red holds two sets of 16 warps' values, used in turn, so that
// one barrier for each call is enough.
template <bool WARP, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*red)[16][N], int& turn) {
  warp_sums<N>(v);
  const float mine = v[0];
  if constexpr (WARP) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xFFFFFFFFu, mine, i * (32 / N));
  } else {
    const int lane = threadIdx.x & 31;
    if (lane % (32 / N) == 0) red[turn][threadIdx.x >> 5][lane / (32 / N)] = mine;
    __syncthreads();
    const int warps = blockDim.x >> 5;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = red[turn][0][i];
    for (int w = 1; w < warps; ++w)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += red[turn][w][i];
    turn ^= 1;
  }
}

// One thread's share of a row: NV vectors of VEC elements, `step` apart.
// Columns past the end are never touched.
template <typename T, int VEC, int NV>
struct Share {
  Pack<T, VEC> v[NV];
  __device__ __forceinline__ void load(const T* row, int c0, int step, int features) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (c0 + j * step < features) v[j].load_nc(row + c0 + j * step);
  }
  __device__ __forceinline__ void fill(float value) {
    float f[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = value;
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j].set(f);
  }
};

// The vectors of a segment; an absent weight is 1 (0 with add_one), an absent
// bias 0.
template <typename TW, int VEC, int NV>
__device__ __forceinline__ Share<TW, VEC, NV> vector_of(const TW* base, float absent, int c0, int step, int features) {
  Share<TW, VEC, NV> s;
  if (base) s.load(base, c0, step, features);
  else s.fill(absent);
  return s;
}

template <typename TW>
__device__ __forceinline__ float weight_at(const NormParams& p, const TW* w, int c) {
  const float v = w ? Elem<TW>::to_f(w[c]) : (p.add_one ? 0.0f : 1.0f);
  return p.add_one ? 1.0f + v : v;
}

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

constexpr int kWarps = 4;  // of a CTA whose warps each have rows of their own

template <typename TW>
__device__ __forceinline__ const TW* at(const void* base, int64_t offset) {
  return base ? static_cast<const TW*>(base) + offset : nullptr;
}

// ---------------------------------------------------------------------------
// forward

// R rows at a time; WARP: each warp rows of its own, else the CTA together.
template <typename T, typename TW, int VEC, int NV, int R, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kWarps : (R == 2 ? 256 : 512)) norm_fwd_kernel(const NormParams p) {
  __shared__ float red[2][16][R];
  int turn = 0;
  grid_dependency_wait();
  grid_dependents_launch();
  const int F = p.features;
  const float inv = 1.0f / static_cast<float>(F);
  const int c0 = (WARP ? threadIdx.x & 31 : threadIdx.x) * VEC, step = (WARP ? 32 : blockDim.x) * VEC;
  const Rows rows(p);
  const auto weight = vector_of<TW, VEC, NV>(at<TW>(p.weight, rows.segment * p.weight_stride),
                                             p.add_one ? 0.0f : 1.0f, c0, step, F);
  const auto bias = vector_of<TW, VEC, NV>(at<TW>(p.bias, rows.segment * p.weight_stride), 0.0f, c0, step, F);
  const float one = p.add_one ? 1.0f : 0.0f;
  const int64_t first = rows.begin + (WARP ? (threadIdx.x >> 5) * R : 0);
  for (int64_t row = first; row < rows.end; row += WARP ? kWarps * R : R) {
    Share<T, VEC, NV> x[R];
    float mean[R], s[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (row + r < rows.end) x[r].load(static_cast<const T*>(p.x) + (row + r) * F, c0, step, F);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[r] = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (c0 + j * step < F) {
          float v[VEC];
          x[r].v[j].get(v);
#pragma unroll
          for (int i = 0; i < VEC; ++i) s[r] += v[i];
        }
    }
    row_sums<WARP>(s, red, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = s[r] * inv;
      s[r] = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (c0 + j * step < F) {
          float v[VEC];
          x[r].v[j].get(v);
#pragma unroll
          for (int i = 0; i < VEC; ++i) s[r] = fmaf(v[i] - mean[r], v[i] - mean[r], s[r]);
        }
    }
    row_sums<WARP>(s, red, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (row + r >= rows.end) break;
      const float rstd = rsqrtf(s[r] * inv + p.eps);
      if (c0 == 0 && p.mean) {
        p.mean[row + r] = mean[r];
        p.rstd[row + r] = rstd;
      }
      T* y = static_cast<T*>(p.y) + (row + r) * F;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (c0 + j * step < F) {
          float v[VEC], w[VEC], b[VEC];
          x[r].v[j].get(v);
          weight.v[j].get(w);
          bias.v[j].get(b);
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[i] = fmaf((v[i] - mean[r]) * rstd, one + w[i], b[i]);
          Pack<T, VEC> out;
          out.set(v);
          out.store(y + c0 + j * step);
        }
    }
  }
}

// Rows too long for the registers: three passes over the row, the later ones
// through L2.
template <typename T, typename TW>
__global__ void __launch_bounds__(512) norm_fwd_long_kernel(const NormParams p) {
  __shared__ float red[2][16][1];
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
    row_sums<false>(s, red, turn);
    const float mean = s[0] * inv;
    s[0] = 0.0f;
    for (int c = threadIdx.x; c < F; c += blockDim.x) {
      const float d = Elem<T>::to_f(x[c]) - mean;
      s[0] = fmaf(d, d, s[0]);
    }
    row_sums<false>(s, red, turn);
    const float rstd = rsqrtf(s[0] * inv + p.eps);
    if (threadIdx.x == 0 && p.mean) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    const int64_t offset = row / p.rows_per_weight * p.weight_stride;
    const TW* weight = at<TW>(p.weight, offset);
    const TW* bias = at<TW>(p.bias, offset);
    for (int c = threadIdx.x; c < F; c += blockDim.x) {
      const float w = weight_at<TW>(p, weight, c);
      y[c] = Elem<T>::from_f(
          fmaf((Elem<T>::to_f(x[c]) - mean) * rstd, w, bias ? Elem<TW>::to_f(bias[c]) : 0.0f));
    }
  }
}

// ---------------------------------------------------------------------------
// backward

// R rows at a time, as in the forward pass.
template <typename T, typename TW, int VEC, int NV, int R, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kWarps : (R == 2 ? 256 : 512)) norm_bwd_kernel(const NormParams p) {
  __shared__ float red[2][16][2 * R];
  extern __shared__ float sums[];  // WARP: (kWarps, 2, features)
  int turn = 0;
  grid_dependency_wait();
  grid_dependents_launch();
  const int F = p.features;
  const float inv = 1.0f / static_cast<float>(F);
  const int warp = threadIdx.x >> 5;
  const int c0 = (WARP ? threadIdx.x & 31 : threadIdx.x) * VEC, step = (WARP ? 32 : blockDim.x) * VEC;
  const Rows rows(p);
  const auto weight = vector_of<TW, VEC, NV>(at<TW>(p.weight, rows.segment * p.weight_stride),
                                             p.add_one ? 0.0f : 1.0f, c0, step, F);
  const float one = p.add_one ? 1.0f : 0.0f;
  float dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[j][i] = db[j][i] = 0.0f;
  const int64_t first = rows.begin + (WARP ? warp * R : 0);
  for (int64_t row = first; row < rows.end; row += WARP ? kWarps * R : R) {
    Share<T, VEC, NV> x[R], dy[R];
    float mean[R], rstd[R], s[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = rstd[r] = 0.0f;
      if (row + r < rows.end) {
        x[r].load(static_cast<const T*>(p.x) + (row + r) * F, c0, step, F);
        dy[r].load(static_cast<const T*>(p.dy) + (row + r) * F, c0, step, F);
        mean[r] = __ldg(p.mean + row + r);
        rstd[r] = __ldg(p.rstd + row + r);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[2 * r] = s[2 * r + 1] = 0.0f;
      if (row + r < rows.end) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (c0 + j * step < F) {
            float v[VEC], d[VEC], w[VEC];
            x[r].v[j].get(v);
            dy[r].v[j].get(d);
            weight.v[j].get(w);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float h = (v[i] - mean[r]) * rstd[r], g = d[i] * (one + w[i]);
              dw[j][i] = fmaf(d[i], h, dw[j][i]);
              db[j][i] += d[i];
              s[2 * r] += g;
              s[2 * r + 1] = fmaf(g, h, s[2 * r + 1]);
            }
          }
      }
    }
    row_sums<WARP>(s, red, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (row + r >= rows.end) break;
      const float mg = s[2 * r] * inv, mgh = s[2 * r + 1] * inv;
      T* dx = static_cast<T*>(p.y) + (row + r) * F;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (c0 + j * step < F) {
          float v[VEC], d[VEC], w[VEC];
          x[r].v[j].get(v);
          dy[r].v[j].get(d);
          weight.v[j].get(w);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float h = (v[i] - mean[r]) * rstd[r];
            v[i] = rstd[r] * (fmaf(d[i], one + w[i], -mg) - h * mgh);
          }
          Pack<T, VEC> out;
          out.set(v);
          out.store(dx + c0 + j * step);
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
    for (int c = threadIdx.x; c < 2 * F; c += 32 * kWarps)
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
  __shared__ float red[2][16][2];
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
      const float w = weight_at<TW>(p, weight, c);
      const float g = Elem<T>::to_f(dy[c]) * w;
      s[0] += g;
      s[1] = fmaf(g, (Elem<T>::to_f(x[c]) - mean) * rstd, s[1]);
    }
    row_sums<false>(s, red, turn);
    const float mg = s[0] * inv, mgh = s[1] * inv;
    for (int c = threadIdx.x; c < F; c += blockDim.x) {
      const float w = weight_at<TW>(p, weight, c);
      const float g = Elem<T>::to_f(dy[c]) * w, h = (Elem<T>::to_f(x[c]) - mean) * rstd;
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
#pragma unroll 8
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

// Most CTAs that share a segment's rows, each with one partial sum: about four
// for each SM in all, and at least 16 rows each.
int chunks_of(int64_t rows_per_weight, int64_t segments) {
  int64_t chunks = 4LL * device_sm_count() / segments;
  if (chunks > rows_per_weight / 16) chunks = rows_per_weight / 16;
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

// Whether every vector of `vec` elements of the rows and of the weights is
// aligned for its accesses.
template <typename T, typename TW>
bool aligned_for(const NormParams& p, int vec) {
  const int64_t bytes = vec * sizeof(T) < 16 ? vec * sizeof(T) : 16;
  const int64_t wbytes = vec * sizeof(TW) < 16 ? vec * sizeof(TW) : 16;
  return p.features % vec == 0 && aligned_to(p.x, bytes) && aligned_to(p.y, bytes) && aligned_to(p.dy, bytes) &&
         aligned_to(p.weight, wbytes) && aligned_to(p.bias, wbytes) &&
         p.weight_stride * static_cast<int64_t>(sizeof(TW)) % wbytes == 0;
}

inline unsigned rows_grid(int64_t rows, int64_t per_cta, int64_t most) {
  const int64_t ctas = (rows + per_cta - 1) / per_cta;
  return static_cast<unsigned>(ctas < most ? ctas : most);
}

// Threads that share a row of `vectors` vectors, NV each.
constexpr int threads_of(int vectors, int nv) { return ((vectors + nv - 1) / nv + 31) / 32 * 32; }

// NV counts in units of E vectors: 1 of 16 bytes, or 4 of one or two elements.
template <typename T, typename TW, int VEC, int E>
int forward_rows(NormParams p, int vectors, cudaStream_t s) {
  const int64_t segments = p.rows / p.rows_per_weight;
  // CTAs: for a few rows at a time each, many enough to fill the GPU
  auto grid = [&](int64_t rows_at, int64_t most) {
    int64_t chunks = (p.rows_per_weight + rows_at - 1) / rows_at, limit = (most * device_sm_count() + segments - 1) / segments;
    p.chunks = static_cast<int>(chunks < limit ? chunks : limit);
    return dim3(static_cast<unsigned>(segments * p.chunks));
  };
  if (vectors <= 32 * 4 * E) {
    const dim3 g = grid(kWarps, 8);
    return enqueue(norm_fwd_kernel<T, TW, VEC, 4 * E, 1, true>, g, 32 * kWarps, 0, p, s);
  }
  if (vectors <= 256 * 3 * E) {
    const int threads = threads_of(vectors, 3 * E);
    const dim3 g = grid(1, threads <= 128 ? 8 : 1024 / threads);
    return enqueue(norm_fwd_kernel<T, TW, VEC, 3 * E, 2, false>, g, threads, 0, p, s);
  }
  if (vectors <= 512 * 4 * E) {
    const dim3 g = grid(1, 2);
    return enqueue(norm_fwd_kernel<T, TW, VEC, 4 * E, 1, false>, g, 512, 0, p, s);
  }
  return enqueue(norm_fwd_long_kernel<T, TW>, rows_grid(p.rows, 1, 8LL * device_sm_count()), 512, 0, p, s);
}

template <typename T, typename TW>
int forward(const NormParams& p, cudaStream_t s) {
  constexpr int W = 16 / sizeof(T);
  if (aligned_for<T, TW>(p, W)) return forward_rows<T, TW, W, 1>(p, p.features / W, s);
  if constexpr (W == 8)
    if (aligned_for<T, TW>(p, 2)) return forward_rows<T, TW, 2, 4>(p, p.features / 2, s);
  return forward_rows<T, TW, 1, 4>(p, p.features, s);
}

template <typename T, typename TW, int VEC, int E>
int backward_rows(const NormParams& p, int vectors, cudaStream_t s) {
  const unsigned ctas = static_cast<unsigned>(p.rows / p.rows_per_weight * p.chunks);
  if (vectors <= 32 * 4 * E)
    return enqueue(norm_bwd_kernel<T, TW, VEC, 4 * E, 1, true>, ctas, 32 * kWarps, 2 * kWarps * sizeof(float) * p.features,
                   p, s);
  if (vectors <= 256 * 3 * E)
    return enqueue(norm_bwd_kernel<T, TW, VEC, 3 * E, 2, false>, ctas, threads_of(vectors, 3 * E), 0, p, s);
  if (vectors <= 512 * 4 * E)
    return enqueue(norm_bwd_kernel<T, TW, VEC, 4 * E, 1, false>, ctas, threads_of(vectors, 4 * E), 0, p, s);
  int rc = enqueue(norm_dx_long_kernel<T, TW>, rows_grid(p.rows, 1, 8LL * device_sm_count()), 512, 0, p, s);
  if (rc == CONVROT_OK && p.partial)
    rc = enqueue(norm_partial_long_kernel<T>, dim3((p.features + 255) / 256, ctas), 256, 0, p, s);
  return rc;
}

template <typename T, typename TW>
int backward(const NormParams& p, cudaStream_t s) {
  constexpr int W = 16 / sizeof(T);
  int rc;
  if (aligned_for<T, TW>(p, W)) rc = backward_rows<T, TW, W, 1>(p, p.features / W, s);
  else if (W == 8 && aligned_for<T, TW>(p, 2)) rc = backward_rows<T, TW, (W == 8 ? 2 : 1), 4>(p, p.features / 2, s);
  else rc = backward_rows<T, TW, 1, 4>(p, p.features, s);
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
