// Helpers shared by the row-wise 8-bit and training kernels (int8_quant.cu,
// layer_norm.cu, gelu_saved8.cu): typed loads, reductions, and the 8-bit
// quantizer's arithmetic.
#pragma once

#include "common.cuh"

namespace convrot {

// Bits of |v|: as unsigned integers they order like the values, infinity
// above every finite value and NaN above infinity, so one integer maximum
// finds a row's largest magnitude and whether the row holds anything that is
// not finite (fmaxf would drop NaN).
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
constexpr uint32_t kInfBits = 0x7F800000u;

__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xFFFFFFFFu, v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Two float32 values rounded to a pair of a 16-bit type, in one conversion.
template <typename T>
__device__ __forceinline__ typename Elem<T>::Pair pair_of(float a, float b);
template <>
__device__ __forceinline__ __nv_bfloat162 pair_of<__nv_bfloat16>(float a, float b) { return __floats2bfloat162_rn(a, b); }
template <>
__device__ __forceinline__ __half2 pair_of<__half>(float a, float b) { return __floats2half2_rn(a, b); }

// VEC packed elements of T to float32.
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const uint32_t* w, float (&v)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[i] = __uint_as_float(w[i]);
    } else {
      const typename Elem<T>::Pair h = *reinterpret_cast<const typename Elem<T>::Pair*>(&w[i / 2]);
      v[i] = Elem<T>::to_f(i % 2 ? Elem<T>::hi(h) : Elem<T>::lo(h));
    }
  }
}

// VEC consecutive elements as they lie in memory, moved in accesses of at
// most 16 bytes (the address is a multiple of that, or of VEC elements where
// those are fewer bytes).
template <typename T, int VEC>
struct Pack {
  static constexpr int kBytes = VEC * static_cast<int>(sizeof(T));
  static constexpr int kWords = kBytes < 4 ? 1 : kBytes / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* src) {
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) {
        const uint4 r = reinterpret_cast<const uint4*>(src)[i];
        w[4 * i] = r.x, w[4 * i + 1] = r.y, w[4 * i + 2] = r.z, w[4 * i + 3] = r.w;
      }
    } else if constexpr (kBytes == 8) {
      const uint2 r = *reinterpret_cast<const uint2*>(src);
      w[0] = r.x, w[1] = r.y;
    } else if constexpr (kBytes == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(src);
    } else if constexpr (kBytes == 2) {
      w[0] = *reinterpret_cast<const uint16_t*>(src);
    } else {
      w[0] = *reinterpret_cast<const uint8_t*>(src);
    }
  }
  __device__ __forceinline__ void store(T* dst) const {
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i)
        reinterpret_cast<uint4*>(dst)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    } else if constexpr (kBytes == 4) {
      *reinterpret_cast<uint32_t*>(dst) = w[0];
    } else {
      *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(w[0]);
    }
  }
  __device__ __forceinline__ void get(float (&v)[VEC]) const { unpack<T, VEC>(w, v); }
  __device__ __forceinline__ void set(const float (&v)[VEC]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = __float_as_uint(v[i]);
    } else if constexpr (VEC == 1) {
      const T h = Elem<T>::from_f(v[0]);
      w[0] = *reinterpret_cast<const uint16_t*>(&h);
    } else {
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        const typename Elem<T>::Pair h = pair_of<T>(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
};

// The low bytes of VEC words as VEC consecutive bytes under `mask` (VEC 1, 2,
// 4 or 8, address a multiple of VEC).
template <int VEC>
__device__ __forceinline__ void store_codes(int8_t* dst, const uint32_t (&code)[VEC], uint32_t mask) {
  if constexpr (VEC == 1) {
    *dst = static_cast<int8_t>(code[0] & mask);
  } else if constexpr (VEC == 2) {
    *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(__byte_perm(code[0], code[1], 0x0040) & mask);
  } else {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i)
      w[i] = __byte_perm(__byte_perm(code[4 * i], code[4 * i + 1], 0x0040),
                         __byte_perm(code[4 * i + 2], code[4 * i + 3], 0x0040), 0x5410) & mask;
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(dst) = w[0];
  }
}

// Byte i of a word as a signed value.
__device__ __forceinline__ float signed_byte(uint32_t w, int i) {
  return static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
}

// Symmetric 8-bit quantizer of values whose largest magnitude is `top`:
//   code = rne(127 x / top) in [-127, 127], scale = top / 127.
// x and top are first scaled by the power of two that brings top near 1, so
// that 127 x cannot overflow; q = p r then misses p / top by at most two
// ulps, and one step of residual correction, q += (p - q top) r with the
// residual exact in one FMA, makes it the correctly rounded quotient.  Ties
// (x = top / 2 gives 63.5 exactly) therefore round as in exact arithmetic.
// Adding 1.5 * 2^23 rounds to the integer (nearest even) in the low bits.
// top = 0: codes 0 and scale 0.  top infinite or NaN: codes 0 (their bits may
// be those of a NaN: `mask` clears them), scale NaN.
struct Quant8 {
  float k127, top, r;
  uint32_t mask;
  __device__ __forceinline__ explicit Quant8(uint32_t top_bits) {
    const bool live = top_bits != 0 && top_bits < kInfBits;
    int e = static_cast<int>(top_bits >> 23) - 127;
    e = e < -100 ? -100 : (e > 126 ? 126 : e);
    const float f = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);  // 2^-e
    mask = live ? 0xFFFFFFFFu : 0u;
    k127 = live ? 127.0f * f : 0.0f;
    top = live ? __uint_as_float(top_bits) * f : 1.0f;
    r = __frcp_rn(top);
  }
  // low byte of the result: the code in two's complement
  __device__ __forceinline__ uint32_t code(float x) const {
    const float p = __fmul_rn(x, k127);
    const float q = __fmul_rn(p, r);
    const float c = __fmaf_rn(__fmaf_rn(-q, top, p), r, q);
    return __float_as_uint(__fadd_rn(c, 12582912.0f));
  }
  static __device__ __forceinline__ float scale(uint32_t top_bits) {
    return top_bits < kInfBits ? __fdiv_rn(__uint_as_float(top_bits), 127.0f) : __uint_as_float(0x7FC00000u);
  }
};

}  // namespace convrot
