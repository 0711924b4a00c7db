// The 8-bit form of activations: e4m3 codes with one power-of-two scale per 32 channels of a row.
//
//   amax = max |x| over the finite values of the group;  e = the least exponent with amax <= 448 * 2^e (448 = 1.75 * 2^8 is the
//   largest e4m3 value), at least -127; e = 0 for a group of zeros;  code = e4m3(x * 2^-e), round to nearest even.
// The scale is a power of two, so the product is exact and a code's value, 4 significant bits times 2^e, is exact in bf16 and fp32.
// Values that would round to 2^128 (e = 120, code 256) stay at 240 * 2^120; inf and nan become nan (e4m3 has no inf).
#pragma once
#include "dm_common.h"

#define ACT8_GROUP 32

typedef float act8_f32x2 __attribute__((ext_vector_type(2)));

// element types of the half / float operators (ABI values)
enum { ACT8_F32 = 0, ACT8_BF16 = 1, ACT8_F16 = 2 };

__device__ __forceinline__ float act8_2exp(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

__device__ __forceinline__ bool act8_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

__device__ __forceinline__ float act8_finite_abs(float v) { return act8_finite(v) ? fabsf(v) : 0.f; }

// e of a group with this (finite, non-negative) amax
__device__ __forceinline__ int act8_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  if (b == 0) return 0;
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);   // mantissa > 1.75
  return e < -127 ? -127 : e;                                                       // (subnormal amax: e = -135 or -134 -> -127)
}

// four codes of x * inv (inv = 2^-e), lowest byte first
__device__ __forceinline__ uint32_t act8_encode4(float a, float b, float c, float d, float inv, float limit) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(fminf(fmaxf(a * inv, -limit), limit), fminf(fmaxf(b * inv, -limit), limit), 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(fminf(fmaxf(c * inv, -limit), limit), fminf(fmaxf(d * inv, -limit), limit), r, true);
  uint32_t u = (uint32_t)r;
  if (!act8_finite(a)) u = (u & 0xffffff00u) | 0x7fu;
  if (!act8_finite(b)) u = (u & 0xffff00ffu) | 0x7f00u;
  if (!act8_finite(c)) u = (u & 0xff00ffffu) | 0x7f0000u;
  if (!act8_finite(d)) u = (u & 0x00ffffffu) | 0x7f000000u;
  return u;
}

__device__ __forceinline__ float act8_limit(int e) { return e >= 120 ? 240.f : 448.f; }

// four values code * 2^e; the scale is applied in two exact halves, so that e = -127 needs no subnormal factor
__device__ __forceinline__ void act8_decode4(uint32_t u, int e, float *v) {
  const act8_f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, true);
  const int h = e >> 1;
  const float s0 = act8_2exp(h), s1 = act8_2exp(e - h);
  v[0] = lo[0] * s0 * s1, v[1] = lo[1] * s0 * s1, v[2] = hi[0] * s0 * s1, v[3] = hi[1] * s0 * s1;
}

// ---- 8 consecutive elements of a row, any element type --------------------------------------------------------------
__device__ __forceinline__ float act8_bf16_f32(uint32_t h) { return __uint_as_float(h << 16); }

__device__ __forceinline__ uint16_t act8_f32_bf16(float v) {       // round to nearest even, nan kept
  const uint32_t b = __float_as_uint(v);
  if ((b & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((b >> 16) | 0x40u);
  return (uint16_t)((b + 0x7fffu + ((b >> 16) & 1u)) >> 16);
}

template <int T>
__device__ __forceinline__ float act8_get(const void *p, size_t i) {
  if constexpr (T == ACT8_F32) return ((const float *)p)[i];
  else if constexpr (T == ACT8_BF16) return act8_bf16_f32(((const uint16_t *)p)[i]);
  else return (float)((const _Float16 *)p)[i];
}

template <int T>
__device__ __forceinline__ void act8_put(void *p, size_t i, float v) {
  if constexpr (T == ACT8_F32) ((float *)p)[i] = v;
  else if constexpr (T == ACT8_BF16) ((uint16_t *)p)[i] = act8_f32_bf16(v);
  else ((_Float16 *)p)[i] = (_Float16)v;
}

// n (1 .. 8) elements from p + i on; the rest 0.  vec: i and the row are 16-byte aligned (then n < 8 only at a row's end)
template <int T>
__device__ __forceinline__ void act8_load8(const void *p, size_t i, int n, bool vec, float *v) {
  if (vec && n >= 8) {
    if constexpr (T == ACT8_F32) {
      const float4 a = *(const float4 *)((const float *)p + i), b = *(const float4 *)((const float *)p + i + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      const uint4 a = *(const uint4 *)((const uint16_t *)p + i);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (T == ACT8_BF16) {
          v[2 * k] = __uint_as_float(w[k] << 16), v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
        } else {
          union { uint32_t u; _Float16 h[2]; } c;
          c.u = w[k];
          v[2 * k] = (float)c.h[0], v[2 * k + 1] = (float)c.h[1];
        }
      }
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = k < n ? act8_get<T>(p, i + k) : 0.f;
}

template <int T>
__device__ __forceinline__ void act8_store8(void *p, size_t i, int n, bool vec, const float *v) {
  if (vec && n >= 8) {
    if constexpr (T == ACT8_F32) {
      *(float4 *)((float *)p + i) = make_float4(v[0], v[1], v[2], v[3]);
      *(float4 *)((float *)p + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (T == ACT8_BF16) {
          w[k] = (uint32_t)act8_f32_bf16(v[2 * k]) | ((uint32_t)act8_f32_bf16(v[2 * k + 1]) << 16);
        } else {
          union { uint32_t u; _Float16 h[2]; } c;
          c.h[0] = (_Float16)v[2 * k], c.h[1] = (_Float16)v[2 * k + 1];
          w[k] = c.u;
        }
      }
      *(uint4 *)((uint16_t *)p + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < n) act8_put<T>(p, i + k, v[k]);
}

// largest finite value of an element type: what unpacking saturates at (2^16 is a code's value, but not fp16's)
template <int T>
__device__ __forceinline__ float act8_most() {
  if constexpr (T == ACT8_F32) return 3.402823466e38f;
  else if constexpr (T == ACT8_BF16) return 3.3895313892515355e38f;
  else return 65504.f;
}

// a group is 4 neighbouring threads with 8 elements each: maximum over them, by lane exchange inside the quad
__device__ __forceinline__ float act8_quad_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 1));
  return fmaxf(v, __shfl_xor(v, 2));
}

// 8 values of one thread of a quad -> 8 codes; *e_out = the group's exponent.  All 4 threads of the quad take part.
__device__ __forceinline__ uint2 act8_encode8(const float *v, int *e_out) {
  float m = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = fmaxf(m, act8_finite_abs(v[k]));
  const int e = act8_exponent(act8_quad_max(m));
  const float inv = act8_2exp(-e), limit = act8_limit(e);
  *e_out = e;
  return make_uint2(act8_encode4(v[0], v[1], v[2], v[3], inv, limit), act8_encode4(v[4], v[5], v[6], v[7], inv, limit));
}
