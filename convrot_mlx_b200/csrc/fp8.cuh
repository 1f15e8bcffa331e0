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

// The codes of 16 values: e4m3(v * 2^-e) for the scale byte e + 127, the first
// in the lowest byte.  (Bytes are at most 247: 448 * 2^120 is above every
// float32; the product is exact, at most 448.)  0 where the block is not finite.
__device__ __forceinline__ uint4 codes_of(const P2 (&v)[kChunk / 2], uint32_t byte) {
  if (byte == 255u) return make_uint4(0u, 0u, 0u, 0u);
  const float inverse = __uint_as_float((254u - byte) << 23);
  const P2 f = p2(inverse, inverse);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = p2_get(mul(v[2 * i], f)), b = p2_get(mul(v[2 * i + 1], f));
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(w[i])
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 values of a row of `features` values from c on; 0 past its end.  WHOLE:
// rows start on multiples of 16 bytes.
template <typename T, bool WHOLE>
__device__ __forceinline__ void load_chunk(const T* row, int c, int features, Pack<T, kChunk>& w) {
  if (WHOLE && c + kChunk <= features) w.load_ahead(row + c);
  else w.load_part(row + c, features - c);
}

// The same of rows that start and end on multiples of 16 bytes, wherever in the
// 16 values a row ends.
template <typename T>
__device__ __forceinline__ void load_pieces(const T* row, int c, int features, Pack<T, kChunk>& w) {
  constexpr int W = 16 / sizeof(T);
#pragma unroll
  for (int j = 0; j < kChunk / W; ++j) {
    Pack<T, W> piece;
    piece.clear();
    if (c + j * W < features) piece.load_ahead(row + c + j * W);
#pragma unroll
    for (int i = 0; i < 4; ++i) w.w[4 * j + i] = piece.w[i];
  }
}

// The largest of the 8 threads that have a block, for all of them.
__device__ __forceinline__ uint32_t span_max(uint32_t top) {
#pragma unroll
  for (int d = 1; d < kSpanThreads; d *= 2) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
  return top;
}

}  // namespace fp8
}  // namespace convrot
