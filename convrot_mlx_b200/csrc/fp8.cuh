// What the quantizers of the 8-bit floating-point linear (fp8_quant.cu) and the
// product that quantizes for itself (fp8_gemm.cu) share: a thread's 16 values of
// a block of 128 to codes.
#pragma once

#include "rows.cuh"

namespace convrot {
namespace fp8 {

constexpr int kSpan = 128;  // values that share a scale
constexpr int kChunk = 16;  // values of a thread
constexpr int kSpanThreads = kSpan / kChunk;

// The biased exponent of the scale for magnitudes up to the value of `top`.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top >= kInfBits) return 255u;
  // top = 1.f * 2^E with biased exponent E + 127: e = E - 8, one more where 1.f > 1.75
  const int e = static_cast<int>(top >> 23) - 8 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(max(e, 0));
}

// 2^-e for the scale byte e + 127; 0 where the block is not finite.  (Bytes
// are at most 247: 448 * 2^120 is above every float32.)
__device__ __forceinline__ float inverse_of(uint32_t byte) {
  return byte == 255u ? 0.0f : __uint_as_float((254u - byte) << 23);
}

// Two codes, a in the low byte.  The product is exact, at most 448.
__device__ __forceinline__ uint32_t code_pair(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}

__device__ __forceinline__ uint4 codes_of(const float (&v)[kChunk], uint32_t byte) {
  const float f = inverse_of(byte);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = byte == 255u ? 0.0f : __fmul_rn(v[4 * i + j], f);  // inf * 0 is no 0
    w[i] = code_pair(s[0], s[1]) | code_pair(s[2], s[3]) << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 values of a row of `features` values from c on; 0 past its end.
template <typename T, bool WHOLE>
__device__ __forceinline__ void load_chunk(const T* row, int c, int features, float (&v)[kChunk]) {
  if (WHOLE && c + kChunk <= features) {
    Pack<T, kChunk> p;
    p.load_ahead(row + c);
    p.get(v);
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) v[i] = c + i < features ? Elem<T>::to_f(row[c + i]) : 0.0f;
  }
}

// The same of rows that start and end on multiples of 16 bytes, wherever in the
// 16 values a row ends.
template <typename T>
__device__ __forceinline__ void load_pieces(const T* row, int c, int features, float (&v)[kChunk]) {
  constexpr int W = 16 / sizeof(T);
#pragma unroll
  for (int j = 0; j < kChunk / W; ++j) {
    Pack<T, W> w;
    w.clear();
    if (c + j * W < features) w.load_ahead(row + c + j * W);
    float f[W];
    w.get(f);
#pragma unroll
    for (int i = 0; i < W; ++i) v[j * W + i] = c + j * W + i < features ? f[i] : 0.0f;
  }
}

__device__ __forceinline__ uint32_t top_of(const float (&v)[kChunk]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kChunk; ++i) top = max(top, abs_bits(v[i]));
  return top;
}

// The largest of the 8 threads that have a block, for all of them.
__device__ __forceinline__ uint32_t span_max(uint32_t top) {
#pragma unroll
  for (int d = 1; d < kSpanThreads; d *= 2) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
  return top;
}

}  // namespace fp8
}  // namespace convrot
