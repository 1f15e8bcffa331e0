// Helpers shared by the row-wise 8-bit and training kernels (int8_quant.cu,
// layer_norm.cu, gelu_saved8.cu): typed loads, reductions, and the 8-bit
// quantizer's arithmetic.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace convrot {

// Bits of |v|: as unsigned integers they order like the values, infinity
// above every finite value and NaN above infinity, so one integer maximum
// finds a row's largest magnitude and whether the row holds anything that is
// not finite (fmaxf would drop NaN).
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
constexpr uint32_t kInfBits = 0x7F800000u;

__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xFFFFFFFFu, v); }

// Two float32 values rounded to a pair of a 16-bit type, in one conversion.
template <typename T>
__device__ __forceinline__ typename Elem<T>::Pair pair_of(float a, float b);
template <>
__device__ __forceinline__ __nv_bfloat162 pair_of<__nv_bfloat16>(float a, float b) { return __floats2bfloat162_rn(a, b); }
template <>
__device__ __forceinline__ __half2 pair_of<__half>(float a, float b) { return __floats2half2_rn(a, b); }

// Two float32 values in a register pair, for the paired instructions (one
// issue slot for two operations), and the same operations on one float32.
using P2 = unsigned long long;
__device__ __forceinline__ P2 p2(float lo, float hi) {
  P2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 p2_get(P2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ P2 add(P2 a, P2 b) {
  P2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ P2 mul(P2 a, P2 b) {
  P2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ P2 fma(P2 a, P2 b, P2 c) {
  P2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float mul(float a, float b) { return a * b; }
__device__ __forceinline__ float fma(float a, float b, float c) { return __fmaf_rn(a, b, c); }
__device__ __forceinline__ float total(P2 a) { return p2_get(a).x + p2_get(a).y; }
__device__ __forceinline__ float total(float a) { return a; }

// What a vector of VEC values is calculated in: pairs, or one float32.
template <int VEC> using Lane = typename std::conditional<VEC == 1, float, P2>::type;
template <int VEC> constexpr int kLanes = (VEC + 1) / 2;
template <int VEC>
__device__ __forceinline__ Lane<VEC> splat(float v) {
  if constexpr (VEC == 1) return v;
  else return p2(v, v);
}

// VEC packed elements of T to float32.
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const uint32_t* w, float (&v)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      v[i] = __uint_as_float(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    } else {
      const typename Elem<T>::Pair h = *reinterpret_cast<const typename Elem<T>::Pair*>(&w[i / 2]);
      v[i] = Elem<T>::to_f(i % 2 ? Elem<T>::hi(h) : Elem<T>::lo(h));
    }
  }
}

// Loads that keep their place among themselves and behind the wait for the
// previous kernel (an invariant load, as __ldg is, could be moved above it),
// but that ordinary stores do not hold back: for data that the kernel does not
// write.
__device__ __forceinline__ uint4 ld_128(const void* p) {
  uint4 r;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ uint2 ld_64(const void* p) {
  uint2 r;
  asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ uint32_t ld_32(const void* p) {
  uint32_t r;
  asm volatile("ld.global.u32 %0, [%1];" : "=r"(r) : "l"(p));
  return r;
}
__device__ __forceinline__ uint32_t ld_16(const void* p) {
  uint16_t r;
  asm volatile("ld.global.u16 %0, [%1];" : "=h"(r) : "l"(p));
  return r;
}
__device__ __forceinline__ uint32_t ld_8(const void* p) {
  uint32_t r;
  asm volatile("ld.global.u8 %0, [%1];" : "=r"(r) : "l"(p));
  return r;
}
__device__ __forceinline__ float ld_f32(const float* p) { return __uint_as_float(ld_32(p)); }

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
  // The same by ld_* below: not held back by the stores before it.
  __device__ __forceinline__ void load_ahead(const T* src) {
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) {
        const uint4 r = ld_128(reinterpret_cast<const uint4*>(src) + i);
        w[4 * i] = r.x, w[4 * i + 1] = r.y, w[4 * i + 2] = r.z, w[4 * i + 3] = r.w;
      }
    } else if constexpr (kBytes == 8) {
      const uint2 r = ld_64(src);
      w[0] = r.x, w[1] = r.y;
    } else if constexpr (kBytes == 4) {
      w[0] = ld_32(src);
    } else if constexpr (kBytes == 2) {
      w[0] = ld_16(src);
    } else {
      w[0] = ld_8(src);
    }
  }
  // The first `count` < VEC elements, the rest 0.
  __device__ __forceinline__ void load_part(const T* src, int count) {
    float v[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = i < count ? Elem<T>::to_f(src[i]) : 0.0f;
    set(v);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  // Bits of the largest magnitude, as abs_bits orders them.  16-bit types are
  // compared in pairs, by a maximum that keeps NaN.
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (sizeof(T) == 2 && VEC > 1) {
      using P = typename Elem<T>::Pair;
      uint32_t m = w[0] & 0x7FFF7FFFu;
#pragma unroll
      for (int i = 1; i < kWords; ++i) {
        const uint32_t a = w[i] & 0x7FFF7FFFu;
        const P r = __hmax2_nan(*reinterpret_cast<const P*>(&m), *reinterpret_cast<const P*>(&a));
        m = *reinterpret_cast<const uint32_t*>(&r);
      }
      const P r = *reinterpret_cast<const P*>(&m);
      return max(abs_bits(Elem<T>::to_f(Elem<T>::lo(r))), abs_bits(Elem<T>::to_f(Elem<T>::hi(r))));
    } else {
      float v[VEC];
      unpack<T, VEC>(w, v);
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < VEC; ++i) m = max(m, abs_bits(v[i]));
      return m;
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
  __device__ __forceinline__ void get_lanes(Lane<VEC> (&v)[kLanes<VEC>]) const {
    float f[VEC];
    unpack<T, VEC>(w, f);
    if constexpr (VEC == 1) {
      v[0] = f[0];
    } else {
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) v[i] = p2(f[2 * i], f[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void set_lanes(const Lane<VEC> (&v)[kLanes<VEC>]) {
    if constexpr (VEC == 1) {
      set(v);
    } else {
      float f[VEC];
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        const float2 p = p2_get(v[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
      }
      set(f);
    }
  }
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

// Byte i of a word, a two's complement value, as float32: the byte with its
// sign bit turned over, as the low mantissa bits of 2^23, is 2^23 + 128 above
// the value (no integer conversion, whose rate is a quarter of an addition's).
__device__ __forceinline__ float signed_byte(uint32_t w, int i) {
  return __fsub_rn(__uint_as_float(__byte_perm(w ^ 0x80808080u, 0x4B000000u, 0x7440 | i)), 8388736.0f);
}

// Symmetric 8-bit quantizer of values whose largest magnitude is `top`:
//   code = rne(127 x / top) in [-127, 127], scale = top / 127,
// the quotient rounded as in exact arithmetic: x = top / 2 is a tie (63.5)
// that occurs in earnest.
// * bfloat16 x: one FMA, x * f + 1.5 * 2^23, whose rounding is to the integer
//   (nearest even, in the low bits), with f = 127 / top rounded up.  x f is
//   above 127 x / top by less than 2^-23 of it, while a quotient that is not
//   a half is at least 2^-16 of itself away from one (both significands have
//   8 bits).  A half needs 254 x = (2 j + 1) top: since 127 is prime either
//   2 j + 1 = 127, the tie 63.5, which rounding up sends to 64, the even one;
//   or top's significand is 127, where f is a power of two and x f exact.
//   (top below 2^-120, for which f overflows, goes the other way: tiny().)
// * other types: x and top are first scaled by the power of two that brings
//   top near 1, so that nothing overflows; q = p r with p = 127 x misses p / top by at most two ulps, and
//   one step of residual correction, q += (p - q top) r with the residual
//   exact in one FMA, makes it the correctly rounded quotient.
// top = 0: codes 0 and scale 0.  top infinite or NaN: codes 0 (their bits may
// be those of a NaN: mask() clears them), scale NaN.
template <typename T>
struct Quant8 {
  static constexpr bool kFast = std::is_same<T, __nv_bfloat16>::value;
  static constexpr uint32_t kLeastFast = 7u << 23;  // 2^-120: from here on 127 / top is finite
  uint32_t bits;
  float k, top, r;

  __device__ __forceinline__ explicit Quant8(uint32_t top_bits) : bits(top_bits) {
    const bool live = mask() != 0;
    if constexpr (kFast) {
      top = r = 0.0f;
      k = live ? __fdiv_ru(127.0f, __uint_as_float(bits)) : 0.0f;
    } else {
      int e = static_cast<int>(bits >> 23) - 127;
      e = e < -100 ? -100 : (e > 126 ? 126 : e);
      const float f = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);  // 2^-e
      top = live ? __uint_as_float(bits) * f : 1.0f;
      k = live ? 127.0f * f : 0.0f;
      r = __frcp_rn(top);
    }
  }
  __device__ __forceinline__ uint32_t mask() const { return bits - 1u < kInfBits - 1u ? 0xFFFFFFFFu : 0u; }

  // The quantizer that lane `lane` of each set of `lanes` lanes holds.
  __device__ __forceinline__ Quant8 from_lane(int lane, int lanes) const {
    Quant8 q = *this;
    q.bits = __shfl_sync(0xFFFFFFFFu, bits, lane, lanes);
    q.k = __shfl_sync(0xFFFFFFFFu, k, lane, lanes);
    if constexpr (!kFast) {
      q.top = __shfl_sync(0xFFFFFFFFu, top, lane, lanes);
      q.r = __shfl_sync(0xFFFFFFFFu, r, lane, lanes);
    }
    return q;
  }

  // Whether codes() has to be that of Quant8<float>(bits) instead.
  __device__ __forceinline__ bool tiny() const { return kFast && bits < kLeastFast && bits != 0; }

  // The codes in two's complement in the words' low bytes.
  template <int VEC>
  __device__ __forceinline__ void codes(const float (&x)[VEC], uint32_t (&code)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if constexpr (kFast) {
        code[i] = __float_as_uint(__fmaf_rn(x[i], k, 12582912.0f));
      } else {
        const float p = __fmul_rn(x[i], k);
        const float q = __fmul_rn(p, r);
        code[i] = __float_as_uint(__fadd_rn(__fmaf_rn(__fmaf_rn(-q, top, p), r, q), 12582912.0f));
      }
    }
  }
};

__device__ __forceinline__ float scale8(uint32_t top_bits) {
  return top_bits < kInfBits ? __fdiv_rn(__uint_as_float(top_bits), 127.0f) : __uint_as_float(0x7FC00000u);
}

}  // namespace convrot
