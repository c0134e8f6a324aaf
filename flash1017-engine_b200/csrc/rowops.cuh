// rowops.cuh -- row loads and stores shared by the kernels over activation
// rows of f32, bf16 or f16 (moe_route.cu, block_norm.cu, int8_matmul.cu).
//
// Values are computed in f32; a store to a 16-bit type rounds once, to nearest
// even.  A row is read in pieces of VEC elements: 16 bytes where the pointers
// and row strides allow it, single elements otherwise (odd lengths, slices).
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"

namespace ffn {

constexpr size_t dtype_bytes(int dt) { return dt == FFN_B200_DT_F32 ? 4 : 2; }
inline bool dtype_ok(int dt) {
  return dt == FFN_B200_DT_F32 || dt == FFN_B200_DT_BF16 || dt == FFN_B200_DT_F16;
}

// Loads here are plain ones.  Kernels start before the previous one has finished
// (programmatic dependent launch) and may read what it writes, so the read-only
// path, which wants data that nothing writes while the kernel runs, is not used.
__device__ __forceinline__ uint4 load_once(const void *p) {  // not kept in L1
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p) : "memory");
  return r;
}

template <int BYTES> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<2> { using type = uint16_t; };
template <> struct RawOf<1> { using type = uint8_t; };
template <typename T, int VEC> using Raw = typename RawOf<(int)sizeof(T) * VEC>::type;

template <typename T> struct ToF32;
template <> struct ToF32<float> {
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct ToF32<__nv_bfloat16> {
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <> struct ToF32<__half> {
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Raw<T, VEC> &r, float (&f)[VEC]) {
  union { Raw<T, VEC> raw; T e[VEC]; } u;
  u.raw = r;
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = ToF32<T>::get(u.e[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> pack(const float (&f)[VEC]) {
  union { Raw<T, VEC> raw; T e[VEC]; __nv_bfloat162 b[(VEC + 1) / 2]; __half2 h[(VEC + 1) / 2]; } u;
  if constexpr (VEC % 2 == 0 && sizeof(T) == 2) {  // two roundings an instruction
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      if constexpr (std::is_same<T, __half>::value) u.h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      else u.b[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) u.e[i] = ToF32<T>::put(f[i]);
  }
  return u.raw;
}
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> load_raw(const T *row, size_t vec) {
  return reinterpret_cast<const Raw<T, VEC> *>(row)[vec];
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T *row, size_t vec, const float (&f)[VEC]) {
  reinterpret_cast<Raw<T, VEC> *>(row)[vec] = pack<T, VEC>(f);
}
// VEC consecutive f32 parameters (16-byte aligned when VEC is a multiple of 4)
template <int VEC>
__device__ __forceinline__ void load_param(const float *p, size_t vec, float (&f)[VEC]) {
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float4 v = reinterpret_cast<const float4 *>(p)[vec * (VEC / 4) + i];
      f[4 * i] = v.x, f[4 * i + 1] = v.y, f[4 * i + 2] = v.z, f[4 * i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = p[vec * VEC + i];
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// int8 codes of a row: scale = fl32(max|x| / 127), code = fl32(x / scale)
// rounded to the nearest whole number, ties to even, within +-127.  A row of
// zeros has scale 0 and codes 0; a row with an infinity or a NaN has scale NaN
// and codes 0, so that its products are NaN.
//
// The largest magnitude is taken over the bits without the sign, as unsigned
// numbers: their order is that of the magnitudes, with infinity and then the
// NaNs on top, so no value needs a test of its own.
template <typename T, int VEC>
__device__ __forceinline__ uint32_t abs_bits(const Raw<T, VEC> &r) {
  union { Raw<T, VEC> raw; T e[VEC]; uint16_t h[sizeof(T) * VEC / 2]; uint32_t w[(sizeof(T) * VEC + 3) / 4]; } u;
  u.raw = r;
  if constexpr (sizeof(T) == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) m = max(m, u.w[i] & 0x7fffffffu);
    return m;
  } else if constexpr (VEC == 1) {
    return u.h[0] & 0x7fffu;
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) m = __vmaxu2(m, u.w[i] & 0x7fff7fffu);
    return max(m & 0xffffu, m >> 16);
  }
}
// the magnitude with these bits of type T
template <typename T>
__device__ __forceinline__ float from_abs_bits(uint32_t b) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(b);
  else {
    union { uint16_t u; T t; } v;
    v.u = (uint16_t)b;
    return ToF32<T>::get(v.t);
  }
}
__device__ __forceinline__ float int8_scale(float max_abs) {
  return isfinite(max_abs) ? __fdiv_rn(max_abs, 127.f) : __int_as_float(0x7fffffff);
}

// What a row's codes are computed from: x times 127 / max|x|, by the fast
// division (2 steps, 2^-22 relative).  With the rounding of the scale that is
// within 127 * (2^-22 + 2^-24) < 3.8e-5 of x / scale, and fl32 moves that by
// 3.8e-6 at most; so where the product is not within 1e-4 of a half it rounds to
// the same whole number, and next to a half the true quotients decide.  Magnitudes
// outside the fast division's range always take those.
//
// Rows of 16-bit values need no look at the halves (`sided`).  With significands
// of at most 11 bits, 127 x / m is a half h, or |254 x - (2k + 1) m| is at least
// one unit of x and it is 1 / (254 * 2047) = 1.9e-6 away, relatively.  If 127
// does not divide m's significand, it is a half for x = +-m / 2 alone, 63.5, and
// that has one code in the whole row, 63 or 64 by the scale's rounding.  So the
// reciprocal is moved by 9e-7 to that side: more than the 4.8e-7 that all the
// roundings come to, and together less than 1.9e-6.  (8192 x 4096 normally
// distributed bf16 values, among which m / 2 is a frequent one: 31 us with all 8
// values of a piece divided where one is near a half, 28 us with that one divided
// alone, 23 us like this.)
struct Int8Row {
  float max_abs, inv;
  bool zero, divide, sided = false;
  __device__ __forceinline__ explicit Int8Row(float m) : max_abs(m) {
    zero = !(m > 0.f && m < INFINITY);
    divide = m < 1e-28f || m > 1e37f;
    inv = zero || divide ? 0.f : __fdividef(127.f, m);
  }
  // the row whose largest magnitude has these bits of T
  template <typename T>
  static __device__ __forceinline__ Int8Row of_bits(uint32_t bits) {
    Int8Row s(from_abs_bits<T>(bits));
    if constexpr (sizeof(T) == 2) {
      constexpr int F = std::is_same<T, __half>::value ? 10 : 7;  // bits of the fraction
      const uint32_t frac = bits & ((1u << F) - 1u), sig = bits >> F ? frac | 1u << F : frac;
      s.sided = !s.zero && !s.divide && sig % 127u;
      if (s.sided) {
        // fl32((m / 2) / scale) is below 63.5 where it is so by more than half a step
        const float sc = s.scale();
        s.inv *= fmaf(-63.5f, sc, 0.5f * s.max_abs) < -0x1p-19f * sc ? 1.f - 9e-7f : 1.f + 9e-7f;
      }
    }
    return s;
  }
  __device__ __forceinline__ float scale() const { return int8_scale(max_abs); }
};
template <int VEC>
__device__ __forceinline__ Raw<int8_t, VEC> int8_codes(const float (&f)[VEC], const Int8Row &s) {
  // x * inv + 1.5 * 2^23, rounded once: the whole number sits in the low bits
  constexpr float kWhole = 12582912.f;
  uint32_t c[VEC];
  float off = 0.f;
#pragma unroll
  for (int i = 0; i < VEC; ++i) c[i] = __float_as_uint(fmaf(f[i], s.inv, kWhole));
  if (!s.sided)
#pragma unroll
    for (int i = 0; i < VEC; ++i) off = fmaxf(off, fabsf(fmaf(f[i], s.inv, kWhole - __uint_as_float(c[i]))));
  if (off > 0.4999f || s.divide) {
    const float sc = s.scale();
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (s.divide || fabsf(fmaf(f[i], s.inv, kWhole - __uint_as_float(c[i]))) > 0.4999f)
        c[i] = s.zero ? 0u : (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(f[i], sc)), -127.f), 127.f);
  }
  if (s.zero) {  // also rows that are not finite
#pragma unroll
    for (int i = 0; i < VEC; ++i) c[i] = 0u;
  }
  union { Raw<int8_t, VEC> raw; uint32_t w[(VEC + 3) / 4]; uint8_t b[VEC]; } u;
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i)
      u.w[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040), __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040), 0x5410);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) u.b[i] = (uint8_t)c[i];
  }
  return u.raw;
}
// VEC codes at p (aligned to VEC bytes)
template <int VEC>
__device__ __forceinline__ void store_codes(int8_t *p, const float (&f)[VEC], const Int8Row &s) {
  *reinterpret_cast<Raw<int8_t, VEC> *>(p) = int8_codes<VEC>(f, s);
}

// Whether rows at p, ld elements of es bytes apart, can be read 16 bytes at a time.
inline bool rows16(const void *p, size_t ld, size_t es) {
  return p == nullptr || (((uintptr_t)p | (ld * es)) & 15) == 0;
}

}  // namespace ffn
