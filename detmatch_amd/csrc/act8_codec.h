// The 8-bit form of activations: e4m3 codes with one power-of-two scale per 32 channels of a row.
//
//   amax = max |x| over the finite values of the group;  e = the least exponent with amax <= 448 * 2^e (448 = 1.75 * 2^8 is the
//   largest e4m3 value), at least -127; e = 0 for a group of zeros;  code = e4m3(x * 2^-e), round to nearest even.
// The scale is a power of two, so the product is exact and a code's value, 4 significant bits times 2^e, is exact in fp32; in bf16 too where it is a multiple
// of 2^-133, bf16's least number: every code from e = -124 on, and every code of a row that was bf16 or fp16.
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

// four codes of x * inv (inv = 2^-e), lowest byte first, whatever the values are
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

// the same where the products are at most 448 or nan: the instruction's own rounding, nan -> nan
__device__ __forceinline__ uint32_t act8_encode4_fast(float a, float b, float c, float d, float inv) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false), true);
}

__device__ __forceinline__ float act8_limit(int e) { return e >= 120 ? 240.f : 448.f; }

// four values code * 2^e, eb = e + 127 (2^-127 is a subnormal number).  (Converting and multiplying: with the converting instructions that take a
// scale the backward pass of the norms took 496 us in place of 343 at 32 768 x 4 096 bf16.)
__device__ __forceinline__ void act8_decode4(uint32_t u, uint32_t eb, float *v) {
  const act8_f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, true);
  const float s = __uint_as_float(eb ? eb << 23 : 0x00400000u);
  v[0] = lo[0] * s, v[1] = lo[1] * s, v[2] = hi[0] * s, v[3] = hi[1] * s;
}

// ---- 8 consecutive elements of a row, any element type --------------------------------------------------------------
// Rows of any pitch: the global loads and stores of gfx950 take 16 bytes at any address of the element's alignment, at full rate
// where it is a multiple of 16.
typedef uint32_t act8_u32x4 __attribute__((ext_vector_type(4)));
typedef act8_u32x4 act8_u32x4_any __attribute__((aligned(2)));
typedef __bf16 act8_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 act8_f16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float act8_bf16_f32(uint32_t h) { return __uint_as_float(h << 16); }

__device__ __forceinline__ uint16_t act8_f32_bf16(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }   // to nearest even

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

// 8 elements as they lie in memory
template <int T>
struct Act8Raw {
  act8_u32x4 w[T == ACT8_F32 ? 2 : 1];
};

// n elements from p + i on (none where n <= 0, 8 where n >= 8); the rest 0
template <int T>
__device__ __forceinline__ Act8Raw<T> act8_load_raw(const void *p, size_t i, int n) {
  Act8Raw<T> r;
  if constexpr (T == ACT8_F32) {
    const float *q = (const float *)p + i;
    if (n >= 8) {
      r.w[0] = *(const act8_u32x4_any *)q, r.w[1] = *(const act8_u32x4_any *)(q + 4);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) r.w[k / 4][k % 4] = k < n ? __float_as_uint(q[k]) : 0u;
    }
  } else {
    const uint16_t *q = (const uint16_t *)p + i;
    if (n >= 8) {
      r.w[0] = *(const act8_u32x4_any *)q;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) r.w[0][k] = (2 * k < n ? (uint32_t)q[2 * k] : 0u) | (2 * k + 1 < n ? (uint32_t)q[2 * k + 1] << 16 : 0u);
    }
  }
  return r;
}

template <int T>
__device__ __forceinline__ void act8_unraw(const Act8Raw<T> &r, float *v) {
  if constexpr (T == ACT8_F32) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(r.w[k / 4][k % 4]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t w = r.w[0][k];
      if constexpr (T == ACT8_BF16) v[2 * k] = __uint_as_float(w << 16), v[2 * k + 1] = __uint_as_float(w & 0xffff0000u);
      else {
        const act8_f16x2 h = __builtin_bit_cast(act8_f16x2, w);
        v[2 * k] = (float)h[0], v[2 * k + 1] = (float)h[1];
      }
    }
  }
}

template <int T>
__device__ __forceinline__ Act8Raw<T> act8_raw(const float *v) {
  Act8Raw<T> r;
  if constexpr (T == ACT8_F32) {
#pragma unroll
    for (int k = 0; k < 8; ++k) r.w[k / 4][k % 4] = __float_as_uint(v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (T == ACT8_BF16) {
        act8_bf16x2 h = {(__bf16)v[2 * k], (__bf16)v[2 * k + 1]};
        r.w[0][k] = __builtin_bit_cast(uint32_t, h);
      } else {
        act8_f16x2 h = {(_Float16)v[2 * k], (_Float16)v[2 * k + 1]};
        r.w[0][k] = __builtin_bit_cast(uint32_t, h);
      }
    }
  }
  return r;
}

template <int T>
__device__ __forceinline__ void act8_store_raw(void *p, size_t i, int n, const Act8Raw<T> &r) {
  if constexpr (T == ACT8_F32) {
    float *q = (float *)p + i;
    if (n >= 8) {
      *(act8_u32x4_any *)q = r.w[0], *(act8_u32x4_any *)(q + 4) = r.w[1];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < n) q[k] = __uint_as_float(r.w[k / 4][k % 4]);
    }
  } else {
    uint16_t *q = (uint16_t *)p + i;
    if (n >= 8) {
      *(act8_u32x4_any *)q = r.w[0];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < n) q[k] = (uint16_t)(r.w[0][k / 2] >> (16 * (k & 1)));
    }
  }
}

template <int T>
__device__ __forceinline__ void act8_load8(const void *p, size_t i, int n, float *v) {
  act8_unraw<T>(act8_load_raw<T>(p, i, n), v);
}

template <int T>
__device__ __forceinline__ void act8_store8(void *p, size_t i, int n, const float *v) {
  act8_store_raw<T>(p, i, n, act8_raw<T>(v));
}

// largest finite value of an element type: what unpacking saturates at (2^16 is a code's value, but not fp16's)
template <int T>
__device__ __forceinline__ float act8_most() {
  if constexpr (T == ACT8_F32) return 3.402823466e38f;
  else if constexpr (T == ACT8_BF16) return 3.3895313892515355e38f;
  else return 65504.f;
}

// lane exchange inside 4 neighbouring lanes
template <int CTRL>
__device__ __forceinline__ float act8_dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

enum { ACT8_DPP_XOR1 = 0xB1, ACT8_DPP_XOR2 = 0x4E, ACT8_DPP_HALF_MIRROR = 0x141, ACT8_DPP_MIRROR = 0x140 };

// a group is 4 neighbouring threads with 8 elements each: maximum over them
__device__ __forceinline__ float act8_quad_max(float v) {
  v = fmaxf(v, act8_dpp<ACT8_DPP_XOR1>(v));
  return fmaxf(v, act8_dpp<ACT8_DPP_XOR2>(v));
}

// 8 values of one thread of a quad -> 8 codes; *e_out = the group's exponent.  All 4 threads of the quad take part.
__device__ __forceinline__ uint2 act8_encode8(const float *v, int *e_out) {
  float m = 0.f;
#pragma unroll
  for (int k = 0; k < 8; k += 2) asm("v_max3_f32 %0, |%1|, |%2|, %0" : "+v"(m) : "v"(v[k]), "v"(v[k + 1]));
  m = act8_quad_max(m);
  int e = act8_exponent(m);
  if (act8_finite(m) && e < 120) {               // (a nan beside finite values does not show in m; it becomes a nan all the same)
    const float inv = act8_2exp(-e);
    *e_out = e;
    return make_uint2(act8_encode4_fast(v[0], v[1], v[2], v[3], inv), act8_encode4_fast(v[4], v[5], v[6], v[7], inv));
  }
  m = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = fmaxf(m, act8_finite_abs(v[k]));
  e = act8_exponent(act8_quad_max(m));
  const float inv = act8_2exp(-e), limit = act8_limit(e);
  *e_out = e;
  return make_uint2(act8_encode4(v[0], v[1], v[2], v[3], inv, limit), act8_encode4(v[4], v[5], v[6], v[7], inv, limit));
}
