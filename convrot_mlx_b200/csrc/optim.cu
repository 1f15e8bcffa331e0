// The AdamW step over many tensors in one launch, and the sum of squares of
// many tensors (the gradient norm).
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps),
// all in float32.  The moments' products and sums are rounded one by one, so
// that codes are what separate operations give; p is rounded once to its type,
// its quotient good to 22 bits.
// Moments in 32 bits are kept as they are.  In 8 bits m and r = sqrt(v) are
// kept as e4m3 codes with a float32 scale for each 256 values of a tensor,
// max|m| / 448 and max r / 448: a square would need twice the range, and a block
// whose gradients grow or fade together follows its scale exactly, however small
// a step changes it.  The update uses the moments before they are rounded; the
// codes are rounded to nearest (2^-4 of a value at most), so a change of a value
// against its block's largest is kept once it is more than half a step, and lost
// below, each step anew.  With b2 up to 0.95 changes of roots and of the scale are
// large enough that no loss adds up (the median root within 1% of its average
// after 200 steps of other gradients); with 0.99 and more, roots of values that
// change against their block lag by a factor of 2 and more.  A root above 0 keeps a
// code above 0, since it divides.
//
// Memory-bound.  The tensors' addresses and sizes are kernel parameters, so a
// step needs no table on the device and can be captured.  A warp has 256
// values at a time, 8 a lane, so the maximum over a block of 8-bit moments is one
// exchange in the warp.  A CTA's 2048 values are of one tensor, so that all that
// depends on the tensor is the same in its threads and costs no instruction of
// theirs.  Times of the step: 246M bf16 values with 8-bit moments 452 us (5.5
// TB/s of a copy's 6.6), 62M float32 ones in 640 tensors with 8-bit moments 185
// (5.5), 113M float32 with 32-bit moments 510 (6.2), six vectors 1.9.  With 8-bit
// moments the instructions weigh as much as the memory (390 a warp and 256
// values, issue 67% active): arithmetic is on pairs, one chunk ahead is in
// registers (a ring in shared memory filled by cp.async: 550 instead of 454 us,
// IEEE division and root: 1210).  Roots of subnormal v are a branch of their own
// (roots_of_any): looking for them takes 1% with 8-bit moments and 16-bit values,
// nothing otherwise.
#include "rows.cuh"

namespace convrot {
namespace optim {

constexpr int kBlock = 256;  // values of a warp's turn; of a scale
constexpr int kLane = kBlock / 32;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kChunk = kThreads * kLane;  // values of a CTA's turn
constexpr float kTop = 448.0f;         // the largest e4m3 value
constexpr float kLeast = 0.001953125f;  // the smallest above 0, 2^-9

struct Entry {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* scales;
  int64_t n;
  uint32_t first;    // of the chunks of all tensors, in the order of the table
  uint32_t aligned;  // vector accesses may be used
};

struct Scalars {
  int count;
  uint32_t chunks;
  uint32_t share, span, step_by;  // a CTA's chunks: from share * its number on, of the next `span` every step_by
  float decay, beta1, beta2, rest1, rest2, eps, step_size, root;  // root: 1 / sqrt(1 - b2^t)
  // the step and the learning rate where they are on the device
  const float* step;
  const float* lr;
  double log1, log2, wd;  // log of b1 and b2
  float host_lr, host_step;
  // clipping by the norm: sums of squares of the gradients
  const double* sums;
  int sums_count;
  float max_norm;
  float* norm;
};

// A table that kernel parameters hold: 32 tensors in 2 KB for the launch's
// sake, 512 in 28 KB (of the 32 KB that there are).
template <int CAP>
struct Table {
  Scalars s;
  Entry e[CAP];
};

// ---------------------------------------------------------------------------
// A thread's 8 values: groups of GROUP consecutive ones, 32 lanes' groups one
// after another, in the 256 of its warp.  Groups of 4 where something is
// float32 (16 bytes), else one of 8.

template <typename T, int BITS> constexpr int kGroup = sizeof(T) == 4 || BITS == 32 ? 4 : 8;

template <int GROUP>
__device__ __forceinline__ int place(int group) {  // the first value of a group in the chunk
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  return warp * kBlock + group * 32 * GROUP + lane * GROUP;
}

// WHOLE: the chunk is all in the tensor and vector accesses may be used.
template <typename T, int GROUP, bool WHOLE>
__device__ __forceinline__ void fetch_values(const T* src, int count, uint32_t (&w)[kLane * sizeof(T) / 4]) {
  constexpr int kWords = GROUP * sizeof(T) / 4;
#pragma unroll
  for (int j = 0; j < kLane / GROUP; ++j) {
    const int at = place<GROUP>(j);
    Pack<T, GROUP> g;
    if constexpr (WHOLE) {
      g.load_ahead(src + at);
    } else {
      g.clear();
#pragma unroll
      for (int i = 0; i < GROUP; ++i)
        if (at + i < count) reinterpret_cast<T*>(g.w)[i] = src[at + i];
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[j * kWords + i] = g.w[i];
  }
}
template <typename T>
__device__ __forceinline__ void pairs_of(const uint32_t (&w)[kLane * sizeof(T) / 4], P2 (&v)[kLane / 2]) {
  float f[kLane];
  unpack<T, kLane>(w, f);
#pragma unroll
  for (int i = 0; i < kLane / 2; ++i) v[i] = p2(f[2 * i], f[2 * i + 1]);
}
template <typename T, int GROUP, bool WHOLE>
__device__ __forceinline__ void store_values(T* dst, int count, const uint32_t (&w)[kLane * sizeof(T) / 4]) {
  constexpr int kWords = GROUP * sizeof(T) / 4;
#pragma unroll
  for (int j = 0; j < kLane / GROUP; ++j) {
    const int at = place<GROUP>(j);
    Pack<T, GROUP> g;
#pragma unroll
    for (int i = 0; i < kWords; ++i) g.w[i] = w[j * kWords + i];
    if constexpr (WHOLE) {
      g.store(dst + at);
    } else {
#pragma unroll
      for (int i = 0; i < GROUP; ++i)
        if (at + i < count) dst[at + i] = reinterpret_cast<const T*>(g.w)[i];
    }
  }
}

constexpr int kPairs = kLane / 2;

__device__ __forceinline__ void decode(const uint32_t (&w)[2], P2 (&v)[kPairs]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t lo, hi;
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w[i]));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    v[2 * i] = p2(a.x, a.y), v[2 * i + 1] = p2(b.x, b.y);
  }
}

__device__ __forceinline__ void encode(const P2 (&v)[kPairs], uint32_t (&w)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 lo = p2_get(v[2 * i]), hi = p2_get(v[2 * i + 1]);
    asm("{\n\t.reg .b16 a, b;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 b, %4, %3;\n\t"
        "mov.b32 %0, {a, b};\n\t}"
        : "=r"(w[i])
        : "f"(lo.x), "f"(lo.y), "f"(hi.x), "f"(hi.y));
  }
}

// One instruction each, good to 22 bits; subnormal numbers count as 0.
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rsqrt_approx(float x) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Square roots of v from 2^-126 on: s = v y with y = 1 / sqrt(v) is what divides;
// an infinite v has an infinite s, no update.  roots_of_any takes the others.
constexpr float kLow = 0x1p-126f, kHigh = 0x1.fffffep127f;
__device__ __forceinline__ P2 root_of(P2 v, P2& y) {
  const float2 f = p2_get(v);
  y = p2(rsqrt_approx(fminf(f.x, kHigh)), rsqrt_approx(fminf(f.y, kHigh)));
  return mul(v, y);
}
// What is kept in 8 bits is s after one step of Newton's iteration on s * s = v,
// the residual in one FMA: rounded as a root is but for a last bit (an infinite
// one becomes NaN).
__device__ __forceinline__ P2 refined_root(P2 v, P2 y, P2 s) {
  const P2 half_residual = mul(fma(mul(s, p2(-1.0f, -1.0f)), s, v), p2(0.5f, 0.5f));
  return fma(half_residual, y, s);
}
// Both of any v: a subnormal one as 2^64 times it, whose root is 2^32 times the
// root; 0 has 0.  Of all others the same bits as above.
__device__ __forceinline__ void roots_of_any(P2 v, P2& s, P2& refined) {
  const float2 f = p2_get(v);
  const bool x = f.x < kLow, y = f.y < kLow;
  const P2 down = p2(x ? 0x1p-32f : 1.0f, y ? 0x1p-32f : 1.0f);
  const float2 up = p2_get(mul(v, p2(x ? 0x1p64f : 1.0f, y ? 0x1p64f : 1.0f)));
  P2 inverse;
  root_of(p2(fmaxf(up.x, kLow), fmaxf(up.y, kLow)), inverse);
  v = p2(up.x, up.y);
  s = mul(v, inverse);
  refined = mul(refined_root(v, inverse, s), down);
  s = mul(s, down);
}
__device__ __forceinline__ float smaller(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A paired product and a paired sum may be compiled to one operation with one
// rounding.  The moments are defined with two, so that 8-bit codes are the same
// however a step is computed; sums of the halves stay sums.
__device__ __forceinline__ P2 sum_of(P2 a, P2 b) {
  const float2 x = p2_get(a), y = p2_get(b);
  return p2(__fadd_rn(x.x, y.x), __fadd_rn(x.y, y.y));
}

// Codes of the block's values, whose largest magnitude has the bits `top`, and
// their scale: 0 for a block of zeros (and of values below 2^-117, whose scale
// is no normal number), NaN for one that is not finite, both with codes 0.
// The quotient by the scale is a product with its reciprocal and one residual
// correction: rounded as a division is.
template <bool ROOT>
__device__ __forceinline__ float quantize(const P2 (&v)[kPairs], uint32_t top, uint32_t (&w)[2]) {
  const float scale = top < kInfBits ? __fmul_rn(__uint_as_float(top), 1.0f / kTop) : __uint_as_float(0x7FC00000u);
  if (!(scale >= 0x1p-126f)) {
    w[0] = w[1] = 0;
    return scale < 0x1p-126f ? 0.0f : scale;
  }
  const float inv = rcp_approx(scale);
  const P2 inv2 = p2(inv, inv), by2 = p2(-scale, -scale);
  P2 q[kPairs];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const P2 a = mul(v[i], inv2);
    q[i] = fma(fma(a, by2, v[i]), inv2, a);
  }
  if constexpr (ROOT) {
    // the least quotient above 0, by its bits less one: seldom one that would become 0
    uint32_t least = 0xFFFFFFFFu;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const float2 f = p2_get(q[i]);
      least = min(least, min(__float_as_uint(f.x) - 1u, __float_as_uint(f.y) - 1u));
    }
    if (least < __float_as_uint(kLeast)) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const float2 f = p2_get(q[i]);
        q[i] = p2(f.x > 0.0f ? fmaxf(f.x, kLeast) : 0.0f, f.y > 0.0f ? fmaxf(f.y, kLeast) : 0.0f);
      }
    }
  }
  encode(q, w);
  return scale;
}

// The bits of the largest magnitude of the warp's values: those of a NaN, if
// there is one.
__device__ __forceinline__ float larger(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t top_of(const P2 (&v)[kPairs]) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const float2 f = p2_get(v[i]);
    top = larger(top, f.x, f.y);
  }
  return warp_max(abs_bits(top));
}

// The sum of `count` values in an order that depends on count alone, for all
// threads of the CTA.
__device__ __forceinline__ double sum_all(const double* sums, int count, double* red) {
  double v = 0.0;
  for (int i = threadIdx.x; i < count; i += kThreads) v += sums[i];
#pragma unroll
  for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) v += red[w];
  return v;
}

// The last tensor whose first chunk is not behind `chunk`; one with no values
// is never it, since the next begins at the same chunk.
template <typename TABLE>
__device__ __forceinline__ int find(const TABLE& t, int count, uint32_t chunk) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.e[mid].first <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <int BITS> using Moment = typename std::conditional<BITS == 32, float, uint8_t>::type;

// A thread's values of a chunk as they lie in memory.
template <typename T, int BITS>
struct Words {
  uint32_t g[kLane * sizeof(T) / 4], p[kLane * sizeof(T) / 4];
  uint32_t m[kLane * sizeof(Moment<BITS>) / 4], v[kLane * sizeof(Moment<BITS>) / 4];
  float2 scales;
};

// CTAs that an SM holds: 80 or 64 registers a thread, as the words of the chunk ahead ask for.
template <typename T, int BITS> constexpr int kCtas = sizeof(T) == 4 || BITS == 32 ? 3 : 4;

template <typename T, int BITS, bool WHOLE>
__device__ __forceinline__ void fetch(const Entry& e, uint32_t in, int count, Words<T, BITS>& w) {
  using M = Moment<BITS>;
  constexpr int G = kGroup<T, BITS>;
  const int64_t base = static_cast<int64_t>(in) * kChunk;
  fetch_values<T, G, WHOLE>(static_cast<const T*>(e.g) + base, count, w.g);
  fetch_values<T, G, WHOLE>(static_cast<const T*>(e.p) + base, count, w.p);
  fetch_values<M, G, WHOLE>(static_cast<const M*>(e.m) + base, count, w.m);
  fetch_values<M, G, WHOLE>(static_cast<const M*>(e.v) + base, count, w.v);
  if constexpr (BITS == 8) {
    // the scales of a warp's block; it may be behind the tensor's end, where all codes are 0
    const int block = threadIdx.x / 32;
    uint2 scales = make_uint2(0u, 0u);
    if (WHOLE || block * kBlock < count) scales = ld_64(e.scales + 2 * (base / kBlock + block));
    w.scales = make_float2(__uint_as_float(scales.x), __uint_as_float(scales.y));
  }
}

template <typename T, int BITS, bool WHOLE>
__device__ __forceinline__ void leave(const Entry& e, uint32_t in, int count, const uint32_t (&p)[kLane * sizeof(T) / 4],
                                      const uint32_t (&m)[kLane * sizeof(Moment<BITS>) / 4],
                                      const uint32_t (&v)[kLane * sizeof(Moment<BITS>) / 4], float2 scales) {
  using M = Moment<BITS>;
  constexpr int G = kGroup<T, BITS>;
  const int64_t base = static_cast<int64_t>(in) * kChunk;
  store_values<T, G, WHOLE>(static_cast<T*>(e.p) + base, count, p);
  store_values<M, G, WHOLE>(static_cast<M*>(e.m) + base, count, m);
  store_values<M, G, WHOLE>(static_cast<M*>(e.v) + base, count, v);
  if constexpr (BITS == 8) {
    const int block = threadIdx.x / 32;
    if (threadIdx.x % 32 == 0 && (WHOLE || block * kBlock < count))
      *reinterpret_cast<float2*>(e.scales + 2 * (base / kBlock + block)) = scales;
  }
}

// Values of the chunk that the tensor has.
__device__ __forceinline__ int count_of(int64_t n, uint32_t in) {
  const int64_t left = n - static_cast<int64_t>(in) * kChunk;
  return left < kChunk ? static_cast<int>(left) : kChunk;
}

template <typename T, int BITS, int CAP>
__global__ void __launch_bounds__(kThreads, kCtas<T, BITS>) adamw_kernel(const __grid_constant__ Table<CAP> t) {
  __shared__ double red[kWarps];
  __shared__ float how[3];
  using M = Moment<BITS>;
  const Scalars& s = t.s;
  grid_dependency_wait();
  grid_dependents_launch();
  uint32_t chunk = s.share * blockIdx.x;
  const uint32_t end = min(chunk + s.span, s.chunks);
  int at = chunk < end ? find(t, s.count, chunk) : 0, ahead_at = at;
  Words<T, BITS> next;
  auto fetch_ahead = [&](uint32_t ahead) {
    if (ahead >= end) return;
    while (ahead_at + 1 < s.count && t.e[ahead_at + 1].first <= ahead) ++ahead_at;
    const Entry& e = t.e[ahead_at];
    const uint32_t in = ahead - e.first;
    const int count = count_of(e.n, in);
    if (e.aligned && count == kChunk) fetch<T, BITS, true>(e, in, count, next);
    else fetch<T, BITS, false>(e, in, count, next);
  };
  fetch_ahead(chunk);
  float step_size = s.step_size, root = s.root, decay = s.decay, coef = 1.0f;
  if (s.step || s.lr) {
    if (threadIdx.x == 0) {
      const double step = s.step ? *s.step : s.host_step, lr = s.lr ? *s.lr : s.host_lr;
      how[0] = static_cast<float>(lr / -expm1(step * s.log1));
      how[1] = static_cast<float>(rsqrt(-expm1(step * s.log2)));
      how[2] = static_cast<float>(1.0 - lr * s.wd);
    }
    __syncthreads();
    step_size = how[0], root = how[1], decay = how[2];
  }
  if (s.sums) {
    const float norm = static_cast<float>(sqrt(sum_all(s.sums, s.sums_count, red)));
    const float c = __fdiv_rn(s.max_norm, __fadd_rn(norm, 1e-6f));
    coef = c >= 1.0f ? 1.0f : c;  // NaN stays
    if (s.norm && blockIdx.x == 0 && threadIdx.x == 0) *s.norm = norm;
  }
  const P2 coef2 = p2(coef, coef), beta1 = p2(s.beta1, s.beta1), beta2 = p2(s.beta2, s.beta2), rest1 = p2(s.rest1, s.rest1),
           rest2 = p2(s.rest2, s.rest2), root2 = p2(root, root), eps = p2(s.eps, s.eps), decay2 = p2(decay, decay),
           minus_step = p2(-step_size, -step_size);
  for (; chunk < end; chunk += s.step_by, at = ahead_at) {
    P2 p[kPairs], g[kPairs], m[kPairs], v[kPairs], r[kPairs];
    pairs_of<T>(next.p, p);
    pairs_of<T>(next.g, g);
    if constexpr (BITS == 32) {
      pairs_of<float>(next.m, m);
      pairs_of<float>(next.v, v);
    } else {
      decode(next.m, m);
      decode(next.v, r);
    }
    float2 scales = next.scales;
    const Entry& e = t.e[at];
    fetch_ahead(chunk + s.step_by);
    if constexpr (BITS == 8) {
      const P2 ms = p2(scales.x, scales.x), rs = p2(scales.y, scales.y);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        m[i] = mul(m[i], ms);
        r[i] = mul(r[i], rs);
        v[i] = mul(r[i], r[i]);
      }
    }
    if (s.sums) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) g[i] = mul(g[i], coef2);
    }
    float least = kHigh;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      m[i] = sum_of(mul(m[i], beta1), mul(g[i], rest1));
      v[i] = sum_of(mul(v[i], beta2), mul(mul(g[i], g[i]), rest2));
      const float2 f = p2_get(v[i]);
      least = smaller(least, f.x, f.y);
    }
    auto update = [&](auto any) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        P2 s, y;
        if constexpr (any.value) {
          roots_of_any(v[i], s, r[i]);
        } else {
          s = root_of(v[i], y);
          if constexpr (BITS == 8) r[i] = refined_root(v[i], y, s);
        }
        const float2 den = p2_get(fma(s, root2, eps));
        p[i] = fma(mul(m[i], minus_step), p2(rcp_approx(den.x), rcp_approx(den.y)), mul(p[i], decay2));
      }
    };
    if (least < kLow) update(std::true_type{});  // zeros too
    else update(std::false_type{});
    Pack<T, kLane> out;
    out.set_lanes(p);
    uint32_t m_words[kLane * sizeof(M) / 4], v_words[kLane * sizeof(M) / 4];
    if constexpr (BITS == 32) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const float2 a = p2_get(m[i]), b = p2_get(v[i]);
        m_words[2 * i] = __float_as_uint(a.x), m_words[2 * i + 1] = __float_as_uint(a.y);
        v_words[2 * i] = __float_as_uint(b.x), v_words[2 * i + 1] = __float_as_uint(b.y);
      }
    } else {
      // values behind the tensor's end have moments of 0
      scales.x = quantize<false>(m, top_of(m), m_words);
      scales.y = quantize<true>(r, top_of(r), v_words);
    }
    const uint32_t in = chunk - e.first;
    const int count = count_of(e.n, in);
    if (e.aligned && count == kChunk) leave<T, BITS, true>(e, in, count, out.w, m_words, v_words, scales);
    else leave<T, BITS, false>(e, in, count, out.w, m_words, v_words, scales);
  }
}

// ---------------------------------------------------------------------------
// Sums of squares: 62M float32 values in 640 tensors in 40.8 us (6.2 TB/s), 246M
// bf16 values in 87 (5.7).  Up to 262144 values the norm is one launch of a
// cluster (a call of 3.9 us, 7.2 as two launches).  A thread adds 32 squares in
// float32, in four sums of eight and these in pairs, and the total to a 64-bit
// one; where a sum of eight leaves the range of float32 (not finite, or so small
// that squares may have been lost, zeros too) the squares are formed in 64 bits.  Each CTA
// writes one sum, of a share that depends on the sizes alone.

struct NormEntry {
  const void* g;
  int64_t n;
  uint32_t first;
  uint32_t aligned;
};

template <int CAP>
struct NormTable {
  int count, add;  // add: to what an earlier launch has left
  uint32_t chunks;
  double* sums;
  float* norm;  // of the sums, where the grid is one cluster
  NormEntry e[CAP];
};

constexpr int kAhead = 4;  // chunks in flight
constexpr int kSumCtas = 4;  // of an SM

template <typename T, int CAP>
__global__ void __launch_bounds__(kThreads) square_sums(const __grid_constant__ NormTable<CAP> t) {
  __shared__ double red[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  grid_dependents_launch();
  const uint32_t per = (t.chunks + gridDim.x - 1) / gridDim.x;
  uint32_t chunk = min(per * blockIdx.x, t.chunks);
  const uint32_t end = min(chunk + per, t.chunks);
  double acc = 0.0;
  if (chunk < end) {
    int at = find(t, t.count, chunk);
    for (; chunk < end; chunk += kAhead) {
      constexpr int G = sizeof(T) == 4 ? 4 : 8;
      Pack<T, G> w[kAhead][kLane / G];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
#pragma unroll
        for (int i = 0; i < kLane / G; ++i) w[j][i].clear();
        if (chunk + j >= end) continue;
        while (at + 1 < t.count && t.e[at + 1].first <= chunk + j) ++at;
        const NormEntry& e = t.e[at];
        const uint32_t in = chunk + j - e.first;
        const T* src = static_cast<const T*>(e.g) + static_cast<int64_t>(in) * kChunk;
        const int count = count_of(e.n, in);
        if (e.aligned && count == kChunk) {
#pragma unroll
          for (int i = 0; i < kLane / G; ++i) w[j][i].load_ahead(src + place<G>(i));
        } else {
#pragma unroll
          for (int i = 0; i < kLane / G; ++i) w[j][i].load_part(src + place<G>(i), count - place<G>(i));
        }
      }
      float sums[kAhead];
      bool fine = true;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        P2 square = p2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < kLane / G; ++i) {
          P2 g[G / 2];
          w[j][i].get_lanes(g);
#pragma unroll
          for (int k = 0; k < G / 2; ++k) square = fma(g[k], g[k], square);
        }
        sums[j] = total(square);
        fine = fine && ((sums[j] < 0x1p120f && sums[j] > 0x1p-90f) || chunk + j >= end);
      }
      if (fine) {
        acc += static_cast<double>(__fadd_rn(__fadd_rn(sums[0], sums[1]), __fadd_rn(sums[2], sums[3])));
      } else {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
#pragma unroll
          for (int i = 0; i < kLane / G; ++i) {
            float g[G];
            w[j][i].get(g);
#pragma unroll
            for (int k = 0; k < G; ++k) acc += static_cast<double>(g[k]) * static_cast<double>(g[k]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d /= 2) acc += __shfl_xor_sync(0xFFFFFFFFu, acc, d);
  if (lane == 0) red[warp] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double v = t.add ? t.sums[blockIdx.x] : 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += red[w];
    if (t.norm) red[0] = v;
    else t.sums[blockIdx.x] = v;
  }
  if (!t.norm) return;
  // few values: the CTAs are one cluster, whose first adds up the sums of all
  cluster_sync();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    double v = 0.0;
    for (uint32_t r = 0; r < gridDim.x; ++r) {
      double part;
      asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(part) : "r"(mapa_shared(&red[0], r)) : "memory");
      v += part;
    }
    *t.norm = static_cast<float>(sqrt(v));
  }
  cluster_sync();  // no CTA leaves while its sum may still be read
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double* sums, int count, float* norm) {
  __shared__ double red[kWarps];
  grid_dependency_wait();
  grid_dependents_launch();
  const double v = sum_all(sums, count, red);
  if (threadIdx.x == 0) *norm = static_cast<float>(sqrt(v));
}

// ---------------------------------------------------------------------------
// host side

namespace {

constexpr int kSmall = 32, kLarge = 512;        // tensors of a launch
constexpr int kNormSmall = 64, kNormLarge = 1024;

template <typename K, typename A>
int launch(K kernel, int64_t ctas, const A& args, cudaStream_t s, const char* what, bool one_cluster = false) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = one_cluster ? 2 : 1;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args));
  return check_launch(what);
}

int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

template <typename T, int BITS, int CAP>
int adamw_part(const Scalars& s, const convrot_adamw_tensor* tensors, int count, cudaStream_t stream) {
  Table<CAP> t;
  t.s = s;
  t.s.count = count;
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    const convrot_adamw_tensor& c = tensors[i];
    const uintptr_t moments = BITS == 8 ? 8 : 16;
    const bool aligned = aligned_to(c.param, 16) && aligned_to(c.grad, 16) && aligned_to(c.exp_avg, moments) &&
                         aligned_to(c.exp_avg_sq, moments);
    Entry& e = t.e[i];
    e.p = c.param, e.g = c.grad, e.m = c.exp_avg, e.v = c.exp_avg_sq, e.scales = c.scales, e.n = c.numel;
    e.first = static_cast<uint32_t>(chunks), e.aligned = aligned;
    chunks += chunks_of(c.numel);
  }
  if (chunks == 0) return CONVROT_OK;
  CONVROT_REQUIRE(chunks < (1LL << 31), CONVROT_ERR_UNSUPPORTED, "tensors too large");
  t.s.chunks = static_cast<uint32_t>(chunks);
  const int64_t most = kCtas<T, BITS> * static_cast<int64_t>(device_sm_count()), ctas = chunks < most ? chunks : most;
  if (chunks > most * count) {
    // large tensors: in the order of the CTAs (246M values in 6 tensors, 8-bit
    // moments: 452 us, 460 in contiguous shares; 113M in 16, 32-bit: 508, 518)
    t.s.share = 1, t.s.span = t.s.chunks, t.s.step_by = static_cast<uint32_t>(ctas);
  } else {
    // tensors that a step over the grid would pass by: in contiguous shares
    // (62M values in 640, 8-bit moments: 185 us, 187)
    t.s.share = t.s.span = static_cast<uint32_t>((chunks + ctas - 1) / ctas), t.s.step_by = 1;
  }
  return launch(adamw_kernel<T, BITS, CAP>, ctas, t, stream, "adamw step");
}

template <typename T, int BITS>
int adamw_all(const Scalars& s, const convrot_adamw_tensor* tensors, int64_t count, cudaStream_t stream) {
  for (int64_t at = 0; at < count; at += kLarge) {
    const int n = static_cast<int>(count - at < kLarge ? count - at : kLarge);
    const int rc = n <= kSmall ? adamw_part<T, BITS, kSmall>(s, tensors + at, n, stream)
                               : adamw_part<T, BITS, kLarge>(s, tensors + at, n, stream);
    if (rc != CONVROT_OK) return rc;
  }
  return CONVROT_OK;
}

template <typename T>
int adamw_bits(int bits, const Scalars& s, const convrot_adamw_tensor* tensors, int64_t count, cudaStream_t stream) {
  return bits == 8 ? adamw_all<T, 8>(s, tensors, count, stream) : adamw_all<T, 32>(s, tensors, count, stream);
}

template <typename T, int CAP>
int sums_part(const convrot_grad_tensor* tensors, int count, int64_t ctas, double* sums, bool add, float* norm,
              cudaStream_t stream) {
  NormTable<CAP> t;
  t.count = count, t.add = add, t.sums = sums, t.norm = norm;
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    t.e[i].g = tensors[i].grad, t.e[i].n = tensors[i].numel;
    t.e[i].first = static_cast<uint32_t>(chunks), t.e[i].aligned = aligned_to(tensors[i].grad, 16);
    chunks += chunks_of(tensors[i].numel);
  }
  CONVROT_REQUIRE(chunks < (1LL << 31), CONVROT_ERR_UNSUPPORTED, "tensors too large");
  t.chunks = static_cast<uint32_t>(chunks);
  return launch(square_sums<T, CAP>, ctas, t, stream, "sums of squares", norm != nullptr);
}

template <typename T>
int sums_all(const convrot_grad_tensor* tensors, int64_t count, int64_t ctas, double* sums, float* norm,
             cudaStream_t stream) {
  for (int64_t at = 0; at < count || at == 0; at += kNormLarge) {
    const int n = static_cast<int>(count - at < kNormLarge ? count - at : kNormLarge);
    const int rc = n <= kNormSmall ? sums_part<T, kNormSmall>(tensors + at, n, ctas, sums, at > 0, norm, stream)
                                   : sums_part<T, kNormLarge>(tensors + at, n, ctas, sums, at > 0, norm, stream);
    if (rc != CONVROT_OK) return rc;
  }
  return CONVROT_OK;
}

}  // namespace
}  // namespace optim
}  // namespace convrot

extern "C" {

int64_t convrot_square_sums_count(int64_t count, const convrot_grad_tensor* tensors) {
  using namespace convrot;
  if (count < 0 || (count > 0 && !tensors)) return 1;
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) chunks += tensors[i].numel > 0 ? optim::chunks_of(tensors[i].numel) : 0;
  const int64_t ctas = chunks, most = optim::kSumCtas * static_cast<int64_t>(device_sm_count());
  return ctas < 1 ? 1 : (ctas < most ? ctas : most);
}

int convrot_square_sums(int64_t count, const convrot_grad_tensor* tensors, int dtype, double* sums, int64_t sums_count,
                        float* norm, void* stream) {
  using namespace convrot;
  CONVROT_REQUIRE(valid_dtype(dtype), CONVROT_ERR_INVALID, "unknown dtype %d", dtype);
  CONVROT_REQUIRE(count >= 0 && (count == 0 || tensors) && (sums || norm) && aligned_to(sums, 8) && aligned_to(norm, 4) &&
                      sums_count > 0 && sums_count <= (1 << 20),
                  CONVROT_ERR_INVALID, "invalid tensor list or sums");
  CONVROT_REQUIRE(!norm || (sums_count <= 8 && count <= optim::kNormLarge), CONVROT_ERR_INVALID,
                  "the norm takes at most 8 sums of at most %d tensors", optim::kNormLarge);
  for (int64_t i = 0; i < count; ++i)
    CONVROT_REQUIRE(tensors[i].numel >= 0 &&
                        (tensors[i].numel == 0 || (tensors[i].grad && aligned_to(tensors[i].grad, dtype_size(dtype)))),
                    CONVROT_ERR_INVALID, "tensor %lld: null or misaligned pointer, or negative size", static_cast<long long>(i));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CONVROT_BF16: return optim::sums_all<__nv_bfloat16>(tensors, count, sums_count, sums, norm, s);
    case CONVROT_F16: return optim::sums_all<__half>(tensors, count, sums_count, sums, norm, s);
    default: return optim::sums_all<float>(tensors, count, sums_count, sums, norm, s);
  }
}

int convrot_norm_of_sums(const double* sums, int64_t sums_count, float* norm, void* stream) {
  using namespace convrot;
  CONVROT_REQUIRE(sums && norm && aligned_to(sums, 8) && aligned_to(norm, 4) && sums_count > 0 && sums_count <= (1 << 24),
                  CONVROT_ERR_INVALID, "invalid sums");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1, 1, 1);
  cfg.blockDim = dim3(optim::kThreads, 1, 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, optim::norm_kernel, sums, static_cast<int>(sums_count), norm));
  return check_launch("norm of sums");
}

int convrot_adamw(int64_t count, const convrot_adamw_tensor* tensors, int dtype, int state_bits,
                  const convrot_adamw_options* o, void* stream) {
  using namespace convrot;
  CONVROT_REQUIRE(valid_dtype(dtype), CONVROT_ERR_INVALID, "unknown dtype %d", dtype);
  CONVROT_REQUIRE(state_bits == 8 || state_bits == 32, CONVROT_ERR_INVALID, "moments are kept in 8 or 32 bits, not %d",
                  state_bits);
  CONVROT_REQUIRE(count >= 0 && (count == 0 || tensors) && o, CONVROT_ERR_INVALID, "null tensor list or options");
  CONVROT_REQUIRE(o->beta1 >= 0 && o->beta1 < 1 && o->beta2 >= 0 && o->beta2 < 1 && o->eps >= 0 && o->weight_decay >= 0,
                  CONVROT_ERR_INVALID, "betas must be in [0, 1), eps and weight decay non-negative");
  CONVROT_REQUIRE((o->step_device || o->step >= 1) && (o->lr_device || o->lr >= 0), CONVROT_ERR_INVALID,
                  "the step counts from 1 and the learning rate is non-negative");
  CONVROT_REQUIRE(!o->sums || (o->sums_count > 0 && o->sums_count <= (1 << 24) && o->max_norm >= 0), CONVROT_ERR_INVALID,
                  "clipping needs sums of squares and a non-negative norm");
  CONVROT_REQUIRE(aligned_to(o->step_device, 4) && aligned_to(o->lr_device, 4) && aligned_to(o->norm, 4) &&
                      aligned_to(o->sums, 8),
                  CONVROT_ERR_INVALID, "step, rate, norm and sums must be aligned to their elements");
  for (int64_t i = 0; i < count; ++i) {
    const convrot_adamw_tensor& t = tensors[i];
    const uintptr_t e = dtype_size(dtype), moment = state_bits == 8 ? 1 : 4;
    CONVROT_REQUIRE(t.numel >= 0 && (t.numel == 0 || (t.param && t.grad && t.exp_avg && t.exp_avg_sq && aligned_to(t.param, e) &&
                                                      aligned_to(t.grad, e) && aligned_to(t.exp_avg, moment) &&
                                                      aligned_to(t.exp_avg_sq, moment))),
                    CONVROT_ERR_INVALID, "tensor %lld: null or misaligned pointer, or negative size", static_cast<long long>(i));
    CONVROT_REQUIRE(state_bits == 32 || t.numel == 0 || (t.scales && aligned_to(t.scales, 8)), CONVROT_ERR_INVALID,
                    "tensor %lld: 8-bit moments need their scales", static_cast<long long>(i));
  }
  const double c1 = 1.0 - pow(o->beta1, o->step), c2 = 1.0 - pow(o->beta2, o->step);
  optim::Scalars s = {};
  s.decay = static_cast<float>(1.0 - o->lr * o->weight_decay);
  s.beta1 = static_cast<float>(o->beta1);
  s.beta2 = static_cast<float>(o->beta2);
  s.rest1 = static_cast<float>(1.0 - o->beta1);
  s.rest2 = static_cast<float>(1.0 - o->beta2);
  s.eps = static_cast<float>(o->eps);
  s.step_size = static_cast<float>(o->lr / c1);
  s.root = static_cast<float>(1.0 / sqrt(c2));
  s.step = o->step_device;
  s.lr = o->lr_device;
  s.log1 = log(o->beta1);
  s.log2 = log(o->beta2);
  s.wd = o->weight_decay;
  s.host_lr = static_cast<float>(o->lr);
  s.host_step = static_cast<float>(o->step);
  s.sums = o->sums;
  s.sums_count = static_cast<int>(o->sums_count);
  s.max_norm = static_cast<float>(o->max_norm);
  s.norm = o->norm;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CONVROT_BF16: return optim::adamw_bits<__nv_bfloat16>(state_bits, s, tensors, count, st);
    case CONVROT_F16: return optim::adamw_bits<__half>(state_bits, s, tensors, count, st);
    default: return optim::adamw_bits<float>(state_bits, s, tensors, count, st);
  }
}

}  // extern "C"
