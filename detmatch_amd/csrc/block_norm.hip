// The norms around a residual block, fused with the block's gate and its residual scale.  Rows of C channels:
//
//   u = N(f) * post_w + post_b          the block's output, normalised (or u = f)
//   y = x + scale * g * u               g = act(gate), one row of gates for `each` rows
//   h = N(y) * pre_w + pre_b            what the next block reads
//   N(v) = (v - mean) * rstd, rstd = 1 / sqrt(mean((v - mean)^2) + eps);  mean = 0 for the RMS norm
//
// Backward, with a = gh * pre_w, yhat and fhat the normalised values, <.> the mean over a row:
//   dy = gy + rstd_y (a - <a> - yhat <a yhat>)    (<a> for the layer norm only);   dx = dy
//   d = scale * dy;  dgate = sum d u act'(gate);  dscale = sum dy g u;  t = d g;  dpost_w = sum t fhat;  dpost_b = sum t
//   q = t post_w;  df = rstd_f (q - <q> - fhat <q fhat>);  dpre_w = sum gh yhat;  dpre_b = sum gh
// f and y may be kept as 8-bit codes (act8_codec.h): fhat and yhat are then taken from the codes, with the statistics of the exact
// values.  All statistics and sums are fp32.
//
// A team of T threads (a power of two) has a row; a thread has 8 neighbouring channels, NCH times, in registers, so each operand
// is read once and the two norms of a row follow one another without a second pass.  Bound by memory.
// Sums over rows: a thread adds its channels over the rows that its team walks, a workgroup's teams are added in LDS, the
// workgroups' sums go to a workspace and a second kernel adds them in order (no atomics).
#include "act8_codec.h"

namespace {

struct BnArgs {
  const void *x, *f, *gate, *post_w, *post_b, *pre_w, *pre_b, *scale, *gy, *gh;   // scale: a device number, or NULL: scale_host
  void *y, *h, *dx, *df, *dgate;
  const void *y_in;                              // backward: y (exact) ...
  uint8_t *f_codes, *f_exps, *y_codes, *y_exps;  // ... or codes of f and y
  float *f_mean, *f_rstd, *y_mean, *y_rstd;      // statistics (rows); means only for the layer norm
  float *part;                                   // backward: sums per workgroup [set][blocks][C], then [blocks] of the scale's
  long long rows, each, groups, ldx, ldf, ldg, ldgy, ldgh;
  float eps, scale_host;
  int C, T, act, post, w32, s32, vx, vf, vg, vgy, vgh, vw, vo, by_unit, n_blocks;
};

enum { ACT_NONE = 0, ACT_SIGMOID = 1, ACT_TANH = 2 };
// sums over rows, in the order of the workspace
enum { SET_PRE_W = 0, SET_PRE_B = 1, SET_POST_W = 2, SET_POST_B = 3, SET_GATE = 4, SETS = 5 };

__device__ __forceinline__ float act_of(int act, float z) {
  if (act == ACT_SIGMOID) return 1.f / (1.f + expf(-z));
  if (act == ACT_TANH) return tanhf(z);
  return z;
}

__device__ __forceinline__ float act_slope(int act, float g) {      // from the activated value
  return act == ACT_SIGMOID ? g * (1.f - g) : act == ACT_TANH ? 1.f - g * g : 1.f;
}

// sums of NV numbers over a team; `red` holds two sets of partial sums in turn, so one barrier a call is enough: a set is
// written again only after the barrier of the call in between
template <int NV>
__device__ __forceinline__ void team_sum(float (&v)[NV], int T, float *red, int &turn) {
  for (int o = (T < 64 ? T : 64) >> 1; o; o >>= 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] += __shfl_xor(v[i], o);
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
  } else if (a.w32) act8_load8<ACT8_F32>(p, c, a.C - c, a.vw != 0, v);
  else act8_load8<T>(p, c, a.C - c, a.vw != 0, v);
}

template <int T>
__device__ __forceinline__ float load_scale(const BnArgs &a) {
  if (!a.scale) return a.scale_host;
  return a.s32 ? *(const float *)a.scale : act8_get<T>(a.scale, 0);
}

template <int T>
__device__ __forceinline__ float rounded(float v) {
  if constexpr (T == ACT8_F32) return v;
  else if constexpr (T == ACT8_BF16) return act8_bf16_f32(act8_f32_bf16(v));
  else return (float)(_Float16)v;
}

// the values that 8 codes of a row stand for in the element type
template <int T>
__device__ __forceinline__ void load_codes(const uint8_t *codes, const uint8_t *exps, size_t row, int groups, int c, float *v) {
  const uint2 u = *(const uint2 *)(codes + (row * groups * ACT8_GROUP + c));
  const int e = (int)exps[row * groups + c / ACT8_GROUP] - 127;
  act8_decode4(u.x, e, v), act8_decode4(u.y, e, v + 4);
  if constexpr (T == ACT8_F16) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = v[k] != v[k] ? v[k] : rounded<T>(fminf(fmaxf(v[k], -65504.f), 65504.f));
  }
}

// mean and 1 / deviation of the row held by a team (values behind the width are 0); fixed two-step form: the deviation is taken around the
// mean, not from a difference of squares
template <bool LAYER, int NCH>
__device__ __forceinline__ void row_stats(const BnArgs &a, float (&v)[NCH][8], int tx, float *red, int &turn, float *mean, float *rstd) {
  float s[1] = {0.f};
  *mean = 0.f;
  if constexpr (LAYER) {
#pragma unroll
    for (int n = 0; n < NCH; ++n)
#pragma unroll
      for (int k = 0; k < 8; ++k) s[0] += v[n][k];
    team_sum<1>(s, a.T, red, turn);
    *mean = s[0] / (float)a.C;
    s[0] = 0.f;
  }
#pragma unroll
  for (int n = 0; n < NCH; ++n) {
    const int left = a.C - 8 * (tx + n * a.T);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float d = k < left ? v[n][k] - *mean : 0.f;
      s[0] = fmaf(d, d, s[0]);
    }
  }
  team_sum<1>(s, a.T, red, turn);
  *rstd = 1.f / sqrtf(s[0] / (float)a.C + a.eps);
}

template <int T, bool LAYER, int NCH, int BLOCK>
__global__ __launch_bounds__(BLOCK) void block_norm_fwd_kernel(BnArgs a) {
  __shared__ float red[64];
  const int tx = threadIdx.x & (a.T - 1), team = threadIdx.x / a.T, teams = BLOCK / a.T, groups8 = (a.C + 31) / 32;
  int turn = 0;
  const float scale = load_scale<T>(a);
  for (long long r0 = (long long)blockIdx.x * teams; r0 < a.rows; r0 += (long long)gridDim.x * teams) {
    const long long row = r0 + team;
    const bool live = row < a.rows;                 // (all teams of a workgroup take part in the sums)
    float y[NCH][8], u[NCH][8];
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int c = 8 * (tx + n * a.T), left = live ? a.C - c : 0;
      act8_load8<T>(a.x, (size_t)row * a.ldx + c, left, a.vx != 0, y[n]);
      if (a.f) act8_load8<T>(a.f, (size_t)row * a.ldf + c, left, a.vf != 0, u[n]);
    }
    if (a.f) {
      if (a.f_codes) {
#pragma unroll
        for (int n = 0; n < NCH; ++n) {
          const int c = 8 * (tx + n * a.T);
          int e;
          const uint2 w = act8_encode8(u[n], &e);
          if (live && c < groups8 * 32) {
            *(uint2 *)(a.f_codes + ((size_t)row * groups8 * 32 + c)) = w;
            if ((tx & 3) == 0) a.f_exps[(size_t)row * groups8 + c / 32] = (uint8_t)(e + 127);
          }
        }
      }
      float mean = 0.f, rstd = 1.f;
      if (a.post) {
        row_stats<LAYER, NCH>(a, u, tx, red, turn, &mean, &rstd);
        if (live && tx == 0 && a.f_rstd) {
          a.f_rstd[row] = rstd;
          if (LAYER) a.f_mean[row] = mean;
        }
      }
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        const int c = 8 * (tx + n * a.T);
        if (a.post) {
          float w[8], b[8];
          load_param<T>(a, a.post_w, c, w, 1.f);
          load_param<T>(a, a.post_b, c, b, 0.f);
#pragma unroll
          for (int k = 0; k < 8; ++k) u[n][k] = fmaf((u[n][k] - mean) * rstd, w[k], b[k]);
        }
        if (a.gate) {
          float g[8];
          act8_load8<T>(a.gate, (size_t)(row / a.each) * a.ldg + c, live ? a.C - c : 0, a.vg != 0, g);
#pragma unroll
          for (int k = 0; k < 8; ++k) u[n][k] *= act_of(a.act, g[k]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) y[n][k] = c + k < a.C ? fmaf(scale, u[n][k], y[n][k]) : 0.f;
        if (live && a.y) act8_store8<T>(a.y, (size_t)row * a.C + c, a.C - c, a.vo != 0, y[n]);
      }
    }
    if (a.y_codes) {
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        const int c = 8 * (tx + n * a.T);
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = rounded<T>(y[n][k]);
        int e;
        const uint2 w = act8_encode8(v, &e);
        if (live && c < groups8 * 32) {
          *(uint2 *)(a.y_codes + ((size_t)row * groups8 * 32 + c)) = w;
          if ((tx & 3) == 0) a.y_exps[(size_t)row * groups8 + c / 32] = (uint8_t)(e + 127);
        }
      }
    }
    if (a.h) {
      float mean, rstd;
      row_stats<LAYER, NCH>(a, y, tx, red, turn, &mean, &rstd);
      if (live && tx == 0 && a.y_rstd) {
        a.y_rstd[row] = rstd;
        if (LAYER) a.y_mean[row] = mean;
      }
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        const int c = 8 * (tx + n * a.T);
        float w[8], b[8];
        load_param<T>(a, a.pre_w, c, w, 1.f);
        load_param<T>(a, a.pre_b, c, b, 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = fmaf((y[n][k] - mean) * rstd, w[k], b[k]);
        if (live) act8_store8<T>(a.h, (size_t)row * a.C + c, a.C - c, a.vo != 0, w);
      }
    }
  }
}

// A team walks rows team, team + teams, ... of one group of rows (blockIdx.y) that share their gates, or, where there are many
// groups, whole groups one after another (by_unit); `each` rows have one row of gates.
template <int T, bool LAYER, int NCH, int BLOCK>
__global__ __launch_bounds__(BLOCK) void block_norm_bwd_kernel(BnArgs a) {
  __shared__ float red[64];
  __shared__ float sums[BLOCK <= 256 ? 256 * 8 : 1];
  const int tx = threadIdx.x & (a.T - 1), team = threadIdx.x / a.T, teams = BLOCK / a.T, groups8 = (a.C + 31) / 32;
  int turn = 0;
  const float scale = load_scale<T>(a);
  float acc[SETS][NCH][8], dscale = 0.f;
#pragma unroll
  for (int s = 0; s < SETS; ++s)
#pragma unroll
    for (int n = 0; n < NCH; ++n)
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[s][n][k] = 0.f;
  const long long stride = (long long)gridDim.x * teams, first = (long long)blockIdx.x * teams + team;
  const long long trips = a.by_unit ? (a.groups + stride - 1) / stride * a.each : (a.each + stride - 1) / stride;
  long long unit = first, in_unit = 0;
  for (long long i = 0; i < trips; ++i) {
    long long row;
    bool live;
    if (a.by_unit) {
      live = unit < a.groups;
      row = unit * a.each + in_unit;
    } else {
      const long long r = first + i * stride;
      live = r < a.each;
      row = (long long)blockIdx.y * a.each + r;
    }
    const long long gate_row = a.by_unit ? unit : blockIdx.y;
    float dy[NCH][8];
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int c = 8 * (tx + n * a.T);
      if (a.gy) act8_load8<T>(a.gy, (size_t)row * a.ldgy + c, live ? a.C - c : 0, a.vgy != 0, dy[n]);
      else
#pragma unroll
        for (int k = 0; k < 8; ++k) dy[n][k] = 0.f;
    }
    if (a.gh) {
      float hat[NCH][8], d[NCH][8], s[2] = {0.f, 0.f};
      const float rstd = live ? a.y_rstd[row] : 0.f, mean = LAYER && live ? a.y_mean[row] : 0.f;
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        const int c = 8 * (tx + n * a.T), left = live ? a.C - c : 0;
        float w[8];
        act8_load8<T>(a.gh, (size_t)row * a.ldgh + c, left, a.vgh != 0, d[n]);
        if (a.y_codes) {
          if (left > 0) load_codes<T>(a.y_codes, a.y_exps, (size_t)row, groups8, c, hat[n]);
          else
#pragma unroll
            for (int k = 0; k < 8; ++k) hat[n][k] = 0.f;
        } else act8_load8<T>(a.y_in, (size_t)row * a.ldx + c, left, a.vx != 0, hat[n]);
        load_param<T>(a, a.pre_w, c, w, 1.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          hat[n][k] = k < left ? (hat[n][k] - mean) * rstd : 0.f;
          acc[SET_PRE_W][n][k] = fmaf(d[n][k], hat[n][k], acc[SET_PRE_W][n][k]);
          if (LAYER) acc[SET_PRE_B][n][k] += d[n][k];
          d[n][k] = k < left ? d[n][k] * w[k] : 0.f;
          s[0] = fmaf(d[n][k], hat[n][k], s[0]);
          s[1] += d[n][k];
        }
      }
      if constexpr (LAYER) team_sum<2>(s, a.T, red, turn);
      else {
        float one[1] = {s[0]};
        team_sum<1>(one, a.T, red, turn);
        s[0] = one[0], s[1] = 0.f;
      }
      const float m0 = s[0] / (float)a.C, m1 = s[1] / (float)a.C;
#pragma unroll
      for (int n = 0; n < NCH; ++n)
#pragma unroll
        for (int k = 0; k < 8; ++k) dy[n][k] = fmaf(rstd, d[n][k] - m1 - hat[n][k] * m0, dy[n][k]);
    }
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int c = 8 * (tx + n * a.T);
      if (live && a.dx) act8_store8<T>(a.dx, (size_t)row * a.C + c, a.C - c, a.vo != 0, dy[n]);
    }
    if (a.f || a.f_codes) {
      float hat[NCH][8], s[2] = {0.f, 0.f};
      float rstd = 1.f, mean = 0.f;
      if (a.post) {
        rstd = live ? a.f_rstd[row] : 0.f;
        if (LAYER && live) mean = a.f_mean[row];
      }
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        const int c = 8 * (tx + n * a.T), left = live ? a.C - c : 0;
        float w[8], b[8], g[8];
        if (a.f_codes) {
          if (left > 0) load_codes<T>(a.f_codes, a.f_exps, (size_t)row, groups8, c, hat[n]);
          else
#pragma unroll
            for (int k = 0; k < 8; ++k) hat[n][k] = 0.f;
        } else act8_load8<T>(a.f, (size_t)row * a.ldf + c, left, a.vf != 0, hat[n]);
        if (a.post) {
          load_param<T>(a, a.post_w, c, w, 1.f);
          load_param<T>(a, a.post_b, c, b, 0.f);
        }
        if (a.gate) act8_load8<T>(a.gate, (size_t)gate_row * a.ldg + c, left, a.vg != 0, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float u = hat[n][k];
          if (a.post) {
            hat[n][k] = k < left ? (hat[n][k] - mean) * rstd : 0.f;
            u = fmaf(hat[n][k], w[k], b[k]);
          }
          const float up = k < left ? dy[n][k] : 0.f, gk = a.gate ? act_of(a.act, g[k]) : 1.f;
          dscale = fmaf(up * gk, k < left ? u : 0.f, dscale);
          float t = up * scale;
          if (a.gate) acc[SET_GATE][n][k] = fmaf(t, k < left ? u : 0.f, acc[SET_GATE][n][k]);
          t *= gk;
          if (a.post) {
            acc[SET_POST_W][n][k] = fmaf(t, hat[n][k], acc[SET_POST_W][n][k]);
            if (LAYER) acc[SET_POST_B][n][k] += k < left ? t : 0.f;
            t = k < left ? t * w[k] : 0.f;
            s[0] = fmaf(t, hat[n][k], s[0]);
            s[1] += t;
          }
          dy[n][k] = t;
        }
      }
      if (a.post) {
        if constexpr (LAYER) team_sum<2>(s, a.T, red, turn);
        else {
          float one[1] = {s[0]};
          team_sum<1>(one, a.T, red, turn);
          s[0] = one[0], s[1] = 0.f;
        }
        const float m0 = s[0] / (float)a.C, m1 = s[1] / (float)a.C;
#pragma unroll
        for (int n = 0; n < NCH; ++n)
#pragma unroll
          for (int k = 0; k < 8; ++k) dy[n][k] = rstd * (dy[n][k] - m1 - hat[n][k] * m0);
      }
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        const int c = 8 * (tx + n * a.T);
        if (live && a.df) act8_store8<T>(a.df, (size_t)row * a.C + c, a.C - c, a.vo != 0, dy[n]);
      }
    }
    if (a.by_unit && ++in_unit == a.each) {            // this group of rows is done: its gates' gradient is complete
      if (a.gate) {
#pragma unroll
        for (int n = 0; n < NCH; ++n) {
          const int c = 8 * (tx + n * a.T), left = live ? a.C - c : 0;
          float g[8];
          act8_load8<T>(a.gate, (size_t)unit * a.ldg + c, left, a.vg != 0, g);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            g[k] = acc[SET_GATE][n][k] * act_slope(a.act, act_of(a.act, g[k]));
            acc[SET_GATE][n][k] = 0.f;
          }
          if (live && a.dgate) act8_store8<T>(a.dgate, (size_t)unit * a.C + c, left, a.vo != 0, g);
        }
      }
      in_unit = 0, unit += stride;
    }
  }
  // this workgroup's sums
  const size_t block = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
  if (BLOCK <= 256 && teams > 1) {
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      if (s == SET_GATE && a.by_unit) continue;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 8; ++k) sums[threadIdx.x * 8 + k] = acc[s][0][k];
      __syncthreads();
      for (int c = threadIdx.x; c < a.C; c += BLOCK) {
        float v = 0.f;
        for (int t = 0; t < teams; ++t) v += sums[t * a.T * 8 + c];
        a.part[((size_t)s * a.n_blocks + block) * a.C + c] = v;
      }
    }
  } else {
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      if (s == SET_GATE && a.by_unit) continue;
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        const int c = 8 * (tx + n * a.T);
        for (int k = 0; k < 8; ++k)
          if (c + k < a.C) a.part[((size_t)s * a.n_blocks + block) * a.C + c + k] = acc[s][n][k];
      }
    }
  }
  float ds[1] = {dscale};
  __syncthreads();
  team_sum<1>(ds, BLOCK, red, turn);
  if (threadIdx.x == 0) a.part[(size_t)SETS * a.n_blocks * a.C + block] = ds[0];
}

struct SumArgs {
  const float *part;
  void *out[SETS], *dscale;
  const void *gate;
  long long ldg;
  int C, act, n_blocks, groups, w32, s32;
};

// sums over the workgroups, in order: 64 columns x 4 slices of the workgroups; blockIdx.y: set (gates: set + group)
template <int T>
__global__ __launch_bounds__(256) void block_norm_sum_kernel(SumArgs a) {
  __shared__ float sh[4][64];
  const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
  if (blockIdx.x * 64 >= (unsigned)a.C) {              // the workgroup behind the columns: the scale's gradient
    if (blockIdx.y || !a.dscale) return;
    float v = 0.f;
    for (int b = threadIdx.x; b < a.n_blocks; b += 256) v += a.part[(size_t)SETS * a.n_blocks * a.C + b];
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if (lane == 0) sh[0][slice] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
      v = (sh[0][0] + sh[0][1]) + (sh[0][2] + sh[0][3]);
      if (a.s32) *(float *)a.dscale = v;
      else act8_put<T>(a.dscale, 0, v);
    }
    return;
  }
  const int set = min((int)blockIdx.y, (int)SET_GATE), group = (int)blockIdx.y - set;
  if (!a.out[set]) return;
  const int c = blockIdx.x * 64 + lane;
  const int blocks = set == SET_GATE ? a.n_blocks / a.groups : a.n_blocks;
  const float *p = a.part + ((size_t)set * a.n_blocks + (size_t)group * blocks) * a.C + c;
  float v = 0.f;
  if (c < a.C)
    for (int b = slice; b < blocks; b += 4) v += p[(size_t)b * a.C];
  sh[slice][lane] = v;
  __syncthreads();
  if (slice || c >= a.C) return;
  v = (sh[0][lane] + sh[1][lane]) + (sh[2][lane] + sh[3][lane]);
  if (set == SET_GATE) {
    v *= act_slope(a.act, act_of(a.act, act8_get<T>(a.gate, (size_t)group * a.ldg + c)));
    act8_put<T>(a.out[set], (size_t)group * a.C + c, v);
  } else if (a.w32) ((float *)a.out[set])[c] = v;
  else act8_put<T>(a.out[set], c, v);
}

struct BnPlan {
  int T, nch, block;
};

bool bn_plan(int C, BnPlan *p) {
  const int chunks = dm_ceil_div(C, 8);
  int t = 8;
  while (t < chunks && t < 512) t <<= 1;
  if (chunks > 2 * t) t <<= 1;
  p->T = t;
  p->nch = dm_ceil_div(chunks, t);
  p->block = t <= 256 ? 256 : t;
  return p->nch <= 2;
}

// workgroups of the backward kernel: x for one group, y groups (by_unit: all groups in x)
struct BnGrid {
  int x, y, by_unit;
};

BnGrid bn_grid(const BnPlan &p, long long rows, long long groups) {
  const int teams = p.block / p.T;
  const int most = p.block >= 1024 ? 512 : p.block >= 512 ? 768 : 1024;
  BnGrid g;
  g.by_unit = groups > 64;
  const long long units = g.by_unit ? groups : rows / (groups > 0 ? groups : 1);
  g.y = g.by_unit || groups < 1 ? 1 : (int)groups;
  long long x = (units + teams - 1) / teams, cap = most / g.y > 0 ? most / g.y : 1;
  g.x = (int)(x < cap ? x : cap);
  return g;
}

template <int T, bool LAYER>
int launch_fwd(const BnArgs &a, const BnPlan &p, hipStream_t st) {
  const int teams = p.block / p.T;
  const long long blocks = (a.rows + teams - 1) / teams;
  const unsigned grid = (unsigned)(blocks < 16384 ? blocks : 16384);
  if (p.block == 256) block_norm_fwd_kernel<T, LAYER, 1, 256><<<grid, 256, 0, st>>>(a);
  else if (p.block == 512 && p.nch == 1) block_norm_fwd_kernel<T, LAYER, 1, 512><<<grid, 512, 0, st>>>(a);
  else if (p.block == 512) block_norm_fwd_kernel<T, LAYER, 2, 512><<<grid, 512, 0, st>>>(a);
  else block_norm_fwd_kernel<T, LAYER, 2, 1024><<<grid, 1024, 0, st>>>(a);
  DM_CHECK_LAUNCH();
  return DM_OK;
}

template <int T, bool LAYER>
int launch_bwd(const BnArgs &a, const BnPlan &p, const BnGrid &g, hipStream_t st) {
  const dim3 grid(g.x, g.y);
  if (p.block == 256) block_norm_bwd_kernel<T, LAYER, 1, 256><<<grid, 256, 0, st>>>(a);
  else if (p.block == 512 && p.nch == 1) block_norm_bwd_kernel<T, LAYER, 1, 512><<<grid, 512, 0, st>>>(a);
  else if (p.block == 512) block_norm_bwd_kernel<T, LAYER, 2, 512><<<grid, 512, 0, st>>>(a);
  else block_norm_bwd_kernel<T, LAYER, 2, 1024><<<grid, 1024, 0, st>>>(a);
  DM_CHECK_LAUNCH();
  return DM_OK;
}

int vec_of(const void *p, long long ld, int dtype) {
  return ((uintptr_t)p & 15) == 0 && ld % (dtype == ACT8_F32 ? 4 : 8) == 0;
}

// what forward and backward have in common; returns a DM_ERR_* code
int fill(BnArgs *a, const dm_block_norm *q, BnPlan *p) {
  if (!q || q->dtype < ACT8_F32 || q->dtype > ACT8_F16 || q->rows < 0 || q->width <= 0) return DM_ERR_INVALID_ARG;
  if (!bn_plan(q->width, p)) return DM_ERR_UNSUPPORTED;
  if (q->gate_act < ACT_NONE || q->gate_act > ACT_TANH || q->groups < 0 || (q->gate ? q->groups < 1 || q->rows % q->groups : q->groups != 0))
    return DM_ERR_INVALID_ARG;
  if (q->gate && q->ld_gate < q->width && q->groups > 1) return DM_ERR_INVALID_ARG;
  if (!(q->eps >= 0.f)) return DM_ERR_INVALID_ARG;
  const int dt = q->dtype;
  a->gate = q->gate, a->post_w = q->post_w, a->post_b = q->post_b, a->pre_w = q->pre_w, a->pre_b = q->pre_b, a->scale = q->scale;
  a->rows = q->rows, a->groups = q->groups, a->each = q->groups > 0 ? q->rows / q->groups : q->rows;
  a->ldg = q->ld_gate, a->eps = q->eps, a->scale_host = q->scale_host, a->C = q->width, a->T = p->T;
  a->act = q->gate_act, a->post = q->post, a->w32 = q->param_f32 || dt == ACT8_F32, a->s32 = q->scale_f32 || dt == ACT8_F32;
  a->vg = vec_of(q->gate, q->ld_gate, dt);
  a->vw = !(((uintptr_t)q->post_w | (uintptr_t)q->post_b | (uintptr_t)q->pre_w | (uintptr_t)q->pre_b) & 15);
  a->f_mean = q->f_mean, a->f_rstd = q->f_rstd, a->y_mean = q->y_mean, a->y_rstd = q->y_rstd;
  a->f_codes = q->f_codes, a->f_exps = q->f_exps, a->y_codes = q->y_codes, a->y_exps = q->y_exps;
  if ((!q->f_codes != !q->f_exps) || (!q->y_codes != !q->y_exps) || (((uintptr_t)q->f_codes | (uintptr_t)q->y_codes) & 7)) return DM_ERR_INVALID_ARG;
  return DM_OK;
}

}  // namespace

extern "C" int dm_block_norm_max_width(void) { return 2 * 1024 * 8; }

extern "C" int dm_block_norm_forward(const dm_block_norm *q, const void *x, long long ldx, const void *f, long long ldf, void *y, void *h,
                                     dm_stream_t stream) {
  BnArgs a = {};
  BnPlan p;
  const int rc = fill(&a, q, &p);
  if (rc != DM_OK) return rc;
  if (q->rows == 0) return DM_OK;
  if (!x || ldx < q->width || (f && (!y || ldf < q->width)) || (!f && (!h || y || q->gate)) || (q->f_codes && !f)) return DM_ERR_INVALID_ARG;
  const bool layer = q->layer != 0;
  if (layer && ((a.f_rstd && !a.f_mean) || (a.y_rstd && !a.y_mean))) return DM_ERR_INVALID_ARG;
  a.x = x, a.f = f, a.y = y, a.h = h, a.ldx = ldx, a.ldf = ldf;
  a.vx = vec_of(x, ldx, q->dtype), a.vf = vec_of(f, ldf, q->dtype);
  a.vo = !(((uintptr_t)y | (uintptr_t)h) & 15) && q->width % (q->dtype == ACT8_F32 ? 4 : 8) == 0;
  hipStream_t st = (hipStream_t)stream;
  if (q->dtype == ACT8_F32) return layer ? launch_fwd<ACT8_F32, true>(a, p, st) : launch_fwd<ACT8_F32, false>(a, p, st);
  if (q->dtype == ACT8_BF16) return layer ? launch_fwd<ACT8_BF16, true>(a, p, st) : launch_fwd<ACT8_BF16, false>(a, p, st);
  return layer ? launch_fwd<ACT8_F16, true>(a, p, st) : launch_fwd<ACT8_F16, false>(a, p, st);
}

extern "C" size_t dm_block_norm_workspace_bytes(long long rows, int width, long long groups) {
  BnPlan p;
  if (rows <= 0 || width <= 0 || groups < 0 || !bn_plan(width, &p)) return 0;
  const BnGrid g = bn_grid(p, rows, groups);
  return dm_align((size_t)g.x * g.y * ((size_t)SETS * width + 1) * sizeof(float));
}

extern "C" int dm_block_norm_backward(const dm_block_norm *q, const void *gy, long long ldgy, const void *gh, long long ldgh, const void *y,
                                      long long ldy, const void *f, long long ldf, void *dx, void *df, void *dgate, void *dpre_w, void *dpre_b,
                                      void *dpost_w, void *dpost_b, void *dscale, void *workspace, size_t workspace_bytes,
                                      dm_stream_t stream) {
  BnArgs a = {};
  BnPlan p;
  const int rc = fill(&a, q, &p);
  if (rc != DM_OK) return rc;
  if (q->rows == 0) return DM_ERR_INVALID_ARG;                     // (there is nothing to sum: the caller writes the zeros)
  const bool layer = q->layer != 0, has_f = f || q->f_codes;
  if ((gy && ldgy < q->width) || (gh && ldgh < q->width) || (!gy && !gh)) return DM_ERR_INVALID_ARG;
  if (gh && (!a.y_rstd || (layer && !a.y_mean) || !(y || q->y_codes) || (y && ldy < q->width))) return DM_ERR_INVALID_ARG;
  if (has_f && q->post && (!a.f_rstd || (layer && !a.f_mean))) return DM_ERR_INVALID_ARG;
  if ((f && ldf < q->width) || (!has_f && (df || dgate || dpost_w || dpost_b || dscale))) return DM_ERR_INVALID_ARG;
  if ((dgate && !q->gate) || ((dpost_w || dpost_b) && !q->post) || ((dpre_w || dpre_b) && !gh) || ((dpre_b || dpost_b) && !layer)) return DM_ERR_INVALID_ARG;
  if (!workspace || workspace_bytes < dm_block_norm_workspace_bytes(q->rows, q->width, q->groups)) return DM_ERR_WORKSPACE;
  const int dt = q->dtype;
  a.gy = gy, a.gh = gh, a.y_in = y, a.f = f, a.ldgy = ldgy, a.ldgh = ldgh, a.ldx = ldy, a.ldf = ldf;
  a.dx = dx, a.df = df, a.dgate = dgate, a.part = (float *)workspace;
  a.vgy = vec_of(gy, ldgy, dt), a.vgh = vec_of(gh, ldgh, dt), a.vx = vec_of(y, ldy, dt), a.vf = vec_of(f, ldf, dt);
  a.vo = !(((uintptr_t)dx | (uintptr_t)df | (uintptr_t)dgate) & 15) && q->width % (dt == ACT8_F32 ? 4 : 8) == 0;
  const BnGrid g = bn_grid(p, q->rows, q->groups);
  a.by_unit = g.by_unit, a.n_blocks = g.x * g.y;
  if (q->groups == 0) a.groups = 1;
  hipStream_t st = (hipStream_t)stream;
  int e;
  if (dt == ACT8_F32) e = layer ? launch_bwd<ACT8_F32, true>(a, p, g, st) : launch_bwd<ACT8_F32, false>(a, p, g, st);
  else if (dt == ACT8_BF16) e = layer ? launch_bwd<ACT8_BF16, true>(a, p, g, st) : launch_bwd<ACT8_BF16, false>(a, p, g, st);
  else e = layer ? launch_bwd<ACT8_F16, true>(a, p, g, st) : launch_bwd<ACT8_F16, false>(a, p, g, st);
  if (e != DM_OK) return e;
  SumArgs s = {};
  s.part = a.part, s.dscale = dscale, s.gate = q->gate, s.ldg = q->ld_gate, s.C = q->width, s.act = q->gate_act, s.n_blocks = a.n_blocks;
  s.groups = g.y, s.w32 = a.w32, s.s32 = a.s32;
  s.out[SET_PRE_W] = dpre_w, s.out[SET_PRE_B] = dpre_b, s.out[SET_POST_W] = dpost_w, s.out[SET_POST_B] = dpost_b;
  s.out[SET_GATE] = g.by_unit ? nullptr : dgate;
  if (!dpre_w && !dpre_b && !dpost_w && !dpost_b && !s.out[SET_GATE] && !dscale) return DM_OK;
  const dim3 grid(dm_ceil_div(q->width, 64) + 1, SET_GATE + g.y);
  if (dt == ACT8_F32) block_norm_sum_kernel<ACT8_F32><<<grid, 256, 0, st>>>(s);
  else if (dt == ACT8_BF16) block_norm_sum_kernel<ACT8_BF16><<<grid, 256, 0, st>>>(s);
  else block_norm_sum_kernel<ACT8_F16><<<grid, 256, 0, st>>>(s);
  DM_CHECK_LAUNCH();
  return DM_OK;
}
