// rowops.cuh -- row loads and stores shared by the kernels over activation
// rows of f32, bf16 or f16 (moe_route.cu, block_norm.cu, int8_matmul.cu).
//
// Values are computed in f32; a store to a 16-bit type rounds once, to nearest
// even.  A row is read in pieces of VEC elements: 16 bytes where the pointers
// and row strides allow it, single elements otherwise (odd lengths, slices).
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace ffn {

constexpr size_t dtype_bytes(int dt) { return dt == FFN_B200_DT_F32 ? 4 : 2; }
inline bool dtype_ok(int dt) {
  return dt == FFN_B200_DT_F32 || dt == FFN_B200_DT_BF16 || dt == FFN_B200_DT_F16;
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
  union { Raw<T, VEC> raw; T e[VEC]; } u;
#pragma unroll
  for (int i = 0; i < VEC; ++i) u.e[i] = ToF32<T>::put(f[i]);
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
      const float4 v = __ldg(reinterpret_cast<const float4 *>(p) + vec * (VEC / 4) + i);
      f[4 * i] = v.x, f[4 * i + 1] = v.y, f[4 * i + 2] = v.z, f[4 * i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = __ldg(p + vec * VEC + i);
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
// zeros has scale 0 and codes 0; a row with an infinity or a NaN (max_abs not
// finite) has scale NaN and codes 0, so that its products are NaN.
__device__ __forceinline__ float int8_scale(float max_abs) {
  return isfinite(max_abs) ? __fdiv_rn(max_abs, 127.f) : __int_as_float(0x7fffffff);
}
// The quotient by a reciprocal is within 2^-22 of x / scale in relative terms
// (127 * 2^-22 < 2^-15 in absolute ones), so only values that near a half need
// the true division to be rounded the same way.
__device__ __forceinline__ int int8_code(float x, float scale, float inv) {
  const float q = x * inv;
  float r = rintf(q);
  if (!(fabsf(fabsf(q - r) - 0.5f) > 3.1e-5f)) r = rintf(__fdiv_rn(x, scale));
  return (int)fminf(fmaxf(r, -127.f), 127.f);
}
// VEC codes at p (aligned to VEC bytes, 8 at most)
template <int VEC>
__device__ __forceinline__ void store_codes(int8_t *p, const float (&f)[VEC], float scale) {
  // below 2^-126 the reciprocal overflows or loses bits: divide every value
  const bool ok = scale > 0.f, tiny = scale < 1.2e-38f;
  const float inv = ok ? (tiny ? __int_as_float(0x7fffffff) : __fdiv_rn(1.f, scale)) : 0.f;
  union { Raw<int8_t, VEC> raw; int8_t e[VEC]; } u;
#pragma unroll
  for (int i = 0; i < VEC; ++i) u.e[i] = ok ? (int8_t)int8_code(f[i], scale, inv) : (int8_t)0;
  *reinterpret_cast<Raw<int8_t, VEC> *>(p) = u.raw;
}

// Whether rows at p, ld elements of es bytes apart, can be read 16 bytes at a time.
inline bool rows16(const void *p, size_t ld, size_t es) {
  return p == nullptr || (((uintptr_t)p | (ld * es)) & 15) == 0;
}

}  // namespace ffn
