// What the two passes of the norms around a residual block share (block_norm.hip, block_norm_bwd.hip).
#pragma once
#include "act8_codec.h"

namespace dm_bn {

struct BnArgs {
  const void *x, *f, *gate, *post_w, *post_b, *pre_w, *pre_b, *scale, *gy, *gh;   // scale: a device number, or NULL: scale_host
  void *y, *h, *dx, *df, *dgate;
  const void *y_in;                              // backward: y (exact) ...
  uint8_t *f_codes, *f_exps, *y_codes, *y_exps;  // ... or codes of f and y
  float *f_mean, *f_rstd, *y_mean, *y_rstd;      // statistics (rows); means only for the layer norm
  float *part;                                   // backward: sums per workgroup [set][blocks][C], then [blocks] of the scale's
  long long ldx, ldf, ldg, ldgy, ldgh;
  uint32_t rows, each, groups;                   // groups of `each` rows
  float eps, scale_host, inv_c;
  int C, T, act, post, w32, s32, by_unit, n_blocks, sets;   // sets: which sums over rows are wanted, a bit each
};

enum { ACT_NONE = 0, ACT_SIGMOID = 1, ACT_TANH = 2 };
// sums over rows, in the order of the workspace
enum { SET_PRE_W = 0, SET_PRE_B = 1, SET_POST_W = 2, SET_POST_B = 3, SET_GATE = 4, SETS = 5 };

// tanh within a few units in the last place: (1 - e) / (1 + e), e = exp(-2 |z|), and its power series where that cancels
__device__ __forceinline__ float tanh_of(float z) {
  const float e = __expf(-2.f * fabsf(z)), q = z * z;
  const float far = copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), z);
  const float near = fmaf(z * q, fmaf(q, fmaf(q, fmaf(q, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), z);
  return fabsf(z) < 0.25f ? near : far;
}

__device__ __forceinline__ float act_of(int act, float z) {
  if (act == ACT_SIGMOID) return __builtin_amdgcn_rcpf(1.f + __expf(-z));
  if (act == ACT_TANH) return tanh_of(z);
  return z;
}

__device__ __forceinline__ float act_slope(int act, float g) {      // from the activated value
  return act == ACT_SIGMOID ? g * (1.f - g) : act == ACT_TANH ? 1.f - g * g : 1.f;
}

__device__ __forceinline__ float rsqrt_of(float v) {                 // (the instruction takes no subnormal numbers)
  return v < 1e-30f ? __builtin_amdgcn_rsqf(v * 0x1p64f) * 0x1p32f : __builtin_amdgcn_rsqf(v);
}

// WAVES: a team is whole waves.  Its number, and with it all that follows from a row's number, is then the same for a wave: addresses are
// scalars and one offset a thread, in place of two registers for each operand.
template <bool WAVES>
__device__ __forceinline__ int team_of(int T) {
  const int team = threadIdx.x / T;
  return WAVES ? __builtin_amdgcn_readfirstlane(team) : team;
}

// sums of NV numbers over a team: lane exchanges inside a wave (every lane ends with the same sum), LDS between waves.  `red` holds two sets of
// partial sums in turn, so one barrier a call is enough: a set is written again only after the barrier of the call in between.
template <int NV>
__device__ __forceinline__ void team_sum(float (&v)[NV], int T, float *red, int &turn) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    v[i] += act8_dpp<ACT8_DPP_XOR1>(v[i]);
    v[i] += act8_dpp<ACT8_DPP_XOR2>(v[i]);
    v[i] += act8_dpp<ACT8_DPP_HALF_MIRROR>(v[i]);
    if (T >= 16) v[i] += act8_dpp<ACT8_DPP_MIRROR>(v[i]);
    if (T >= 32) {
      const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
      v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if (T >= 64) {
      const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
      v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
  }
  if (T > 64) {
    float *r = red + turn * 32;
    turn ^= 1;
    const int wave = threadIdx.x >> 6, per = T >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) r[wave * NV + i] = v[i];
    }
    __syncthreads();
    const int w0 = wave & ~(per - 1);
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = 0.f;
    for (int w = 0; w < per; ++w) {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] += r[(w0 + w) * NV + i];
    }
  }
}

template <int T>
__device__ __forceinline__ void load_param(const BnArgs &a, const void *p, int c, float *v, float absent) {
  if (!p) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = absent;
  } else if (a.w32) act8_load8<ACT8_F32>(p, c, a.C - c, v);
  else act8_load8<T>(p, c, a.C - c, v);
}

template <int T>
__device__ __forceinline__ float load_scale(const BnArgs &a) {
  if (!a.scale) return a.scale_host;
  return a.s32 ? *(const float *)a.scale : act8_get<T>(a.scale, 0);
}

struct BnPlan {
  int T, nch, block;
};

// Threads of a row, chunks of 8 channels of a thread, threads of a workgroup.  The forward pass: 512 threads, twice 8 channels each, serve up to
// 8 192.  The backward pass keeps sums in registers, which twice 8 channels would not leave: 512 threads up to 4 096 channels, 1 024 from there on.
inline bool bn_plan(int C, bool backward, BnPlan *p) {
  const int chunks = dm_ceil_div(C, 8), most = 512;
  int t = 8;
  while (t < chunks && t < most) t <<= 1;
  if (chunks > (backward ? t : 2 * t)) t = 1024;
  p->T = t;
  p->nch = dm_ceil_div(chunks, t);
  p->block = t <= most ? most : t;
  return p->nch <= 2;
}

// Workgroups of the backward kernel: x for one group, y groups (by_unit: all groups in x).  From 65 groups on a team takes whole groups, so that a group's gate
// gradient is complete in its registers.  That suits short groups: a row each, or a few rows.  Long ones leave most of the chip idle, as there are no more teams at
// work than groups: 64 groups of 1 000 x 256 bf16 52 us, 65 groups 2 792.
struct BnGrid {
  int x, y, by_unit;
};

inline BnGrid bn_grid(const BnPlan &p, long long rows, long long groups) {
  const int teams = p.block / p.T, most = p.block == 512 ? 512 : 256;     // what is resident at once: each workgroup leaves sums behind
  BnGrid g;
  g.by_unit = groups > 64;
  const long long units = g.by_unit ? groups : rows / (groups > 0 ? groups : 1);
  g.y = g.by_unit || groups < 1 ? 1 : (int)groups;
  long long x = (units + teams - 1) / teams, cap = most / g.y > 0 ? most / g.y : 1;
  g.x = (int)(x < cap ? x : cap);
  return g;
}

}  // namespace dm_bn

// the backward kernel (block_norm_bwd.hip); returns a DM_ERR_* code
int dm_block_norm_launch_backward(int dtype, bool layer, const dm_bn::BnArgs &a, const dm_bn::BnPlan &p, const dm_bn::BnGrid &g, hipStream_t st);
