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
#include "block_norm.h"

using namespace dm_bn;

namespace {

__device__ __forceinline__ void store_codes8(const float *v, uint8_t *codes, uint8_t *exps, size_t row, int groups, int c, bool live) {
  int e;
  const uint2 w = act8_encode8(v, &e);
  if (live && c < groups * ACT8_GROUP) {
    *(uint2 *)(codes + (row * groups * ACT8_GROUP + c)) = w;
    if ((threadIdx.x & 3) == 0) exps[row * groups + c / ACT8_GROUP] = (uint8_t)(e + 127);
  }
}

// mean and 1 / deviation of the row held by a team (values behind the width are 0); the deviation is taken around the mean, not from a
// difference of squares
template <bool LAYER, int NCH>
__device__ __forceinline__ void row_stats(const BnArgs &a, const float (&v)[NCH][8], int tx, float *red, int &turn, float *mean,
                                          float *rstd) {
  float s[1] = {0.f};
  *mean = 0.f;
  if constexpr (LAYER) {
#pragma unroll
    for (int n = 0; n < NCH; ++n)
#pragma unroll
      for (int k = 0; k < 8; ++k) s[0] += v[n][k];
    team_sum<1>(s, a.T, red, turn);
    *mean = s[0] * a.inv_c;
    s[0] = 0.f;
  }
#pragma unroll
  for (int n = 0; n < NCH; ++n) {
    const int left = a.C - 8 * (tx + n * a.T);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float d = LAYER ? (k < left ? v[n][k] - *mean : 0.f) : v[n][k];
      s[0] = fmaf(d, d, s[0]);
    }
  }
  team_sum<1>(s, a.T, red, turn);
  *rstd = rsqrt_of(fmaf(s[0], a.inv_c, a.eps));
}

// A workgroup's teams walk the rows with the grid's stride.  The next row's operands are under way while this one is computed.
// Bound by memory: 32 768 x 4 096 bf16 RMS 212 us = 5.0 TB/s, with a gate for each element 243 (5.5), and keeping codes 292 (5.5); LN 250; 16 384 x 640
// fp32 LN 42 (4.0), with the gates of a sample 49 (3.4: gates that rows share are loaded and activated for each row); 8 192 x 2 048 keeping codes 38 (4.4).
template <int T, bool LAYER, int NCH, int BLOCK, bool WAVES>
__global__ __launch_bounds__(BLOCK, NCH == 1 ? 4 : 2) void block_norm_fwd_kernel(BnArgs a) {
  __shared__ float red[64];
  const int tx = threadIdx.x & (a.T - 1), team = team_of<WAVES>(a.T), teams = BLOCK / a.T, groups8 = (a.C + 31) / 32;
  int turn = 0;
  const float scale = load_scale<T>(a);
  const bool has_f = a.f != nullptr, gate_each = a.gate && a.groups > 1;
  float post_w[NCH][8], post_b[LAYER ? NCH : 1][8], pre_w[NCH][8], pre_b[LAYER ? NCH : 1][8], g[NCH][8];
#pragma unroll
  for (int n = 0; n < NCH; ++n) {
    const int c = 8 * (tx + n * a.T);
    load_param<T>(a, a.post_w, c, post_w[n], 1.f), load_param<T>(a, a.pre_w, c, pre_w[n], 1.f);
    if constexpr (LAYER) load_param<T>(a, a.post_b, c, post_b[n], 0.f), load_param<T>(a, a.pre_b, c, pre_b[n], 0.f);
    if (a.gate && !gate_each) {
      act8_load8<T>(a.gate, c, a.C - c, g[n]);
#pragma unroll
      for (int k = 0; k < 8; ++k) g[n][k] = act_of(a.act, g[n][k]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) g[n][k] = 1.f;
    }
  }
  struct In {
    Act8Raw<T> x[NCH], f[NCH], g[NCH];
  } next;
  auto fetch = [&](uint32_t row) {
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int c = 8 * (tx + n * a.T), left = row < a.rows ? a.C - c : 0;
      next.x[n] = act8_load_raw<T>(a.x, (size_t)row * a.ldx + c, left);
      if (has_f) next.f[n] = act8_load_raw<T>(a.f, (size_t)row * a.ldf + c, left);
      if (gate_each) next.g[n] = act8_load_raw<T>(a.gate, (size_t)(a.each == 1 ? row : row / a.each) * a.ldg + c, left);
    }
  };
  const uint32_t stride = gridDim.x * teams;
  fetch(blockIdx.x * teams + team);
  for (uint32_t r0 = blockIdx.x * teams; r0 < a.rows; r0 += stride) {
    const uint32_t row = r0 + team;
    const bool live = row < a.rows;                 // (all teams of a workgroup take part in the sums)
    const In in = next;
    fetch(row + stride);
    float y[NCH][8];
#pragma unroll
    for (int n = 0; n < NCH; ++n) act8_unraw<T>(in.x[n], y[n]);
    if (has_f) {
      float u[NCH][8], mean = 0.f, rstd = 1.f;
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        act8_unraw<T>(in.f[n], u[n]);
        if (a.f_codes) store_codes8(u[n], a.f_codes, a.f_exps, row, groups8, 8 * (tx + n * a.T), live);
      }
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
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if constexpr (LAYER) u[n][k] = fmaf((u[n][k] - mean) * rstd, post_w[n][k], post_b[n][k]);
            else u[n][k] = u[n][k] * rstd * post_w[n][k];
          }
        }
        if (gate_each) {
          act8_unraw<T>(in.g[n], g[n]);
#pragma unroll
          for (int k = 0; k < 8; ++k) g[n][k] = act_of(a.act, g[n][k]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) y[n][k] = fmaf(scale, g[n][k] * u[n][k], y[n][k]);
        if (c + 8 > a.C) {                          // (gates and biases behind the width leave no trace)
#pragma unroll
          for (int k = 0; k < 8; ++k) y[n][k] = c + k < a.C ? y[n][k] : 0.f;
        }
        const Act8Raw<T> stored = act8_raw<T>(y[n]);
        if (live && a.y) act8_store_raw<T>(a.y, (size_t)row * a.C + c, a.C - c, stored);
        if (a.y_codes) {                            // of y as it is stored
          float v[8];
          act8_unraw<T>(stored, v);
          store_codes8(v, a.y_codes, a.y_exps, row, groups8, c, live);
        }
      }
    } else if (a.y_codes) {
#pragma unroll
      for (int n = 0; n < NCH; ++n) store_codes8(y[n], a.y_codes, a.y_exps, row, groups8, 8 * (tx + n * a.T), live);
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
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if constexpr (LAYER) y[n][k] = fmaf((y[n][k] - mean) * rstd, pre_w[n][k], pre_b[n][k]);
          else y[n][k] = y[n][k] * rstd * pre_w[n][k];
        }
        if (live) act8_store8<T>(a.h, (size_t)row * a.C + c, a.C - c, y[n]);
      }
    }
  }
}

struct SumArgs {
  const float *part;
  void *out[SETS], *dscale;
  const void *gate, *scale;
  long long ldg;
  float scale_host;
  int C, act, n_blocks, groups, w32, s32;
};

// Sums over the workgroups, in a fixed order: 32 columns x 32 slices of the workgroups, 8 loads of a thread under way at a time;
// blockIdx.y: set (gates: set + group).  Bound by the latency of the loads of a slice: few workgroups have little to read.
template <int T>
__global__ __launch_bounds__(1024) void block_norm_sum_kernel(SumArgs a) {
  __shared__ float sh[32][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const bool last = blockIdx.x * 32 >= (unsigned)a.C;    // the workgroup behind the columns: the scale's gradient
  const int set = min((int)blockIdx.y, (int)SET_GATE), group = (int)blockIdx.y - set;
  if (last ? blockIdx.y || !a.dscale : !a.out[set]) return;
  const int c = blockIdx.x * 32 + lane, blocks = set == SET_GATE ? a.n_blocks / a.groups : a.n_blocks;
  const float *p;
  size_t step;
  int b, n;
  if (last) p = a.part + (size_t)SETS * a.n_blocks * a.C, step = 1, b = threadIdx.x, n = 1024;
  else p = a.part + ((size_t)set * a.n_blocks + (size_t)group * blocks) * a.C + c, step = a.C, b = slice, n = 32;
  float v = 0.f;
  if (last || c < a.C) {
    for (; b + 7 * n < blocks; b += 8 * n) {
      float w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = p[(size_t)(b + k * n) * step];
#pragma unroll
      for (int k = 0; k < 8; ++k) v += w[k];
    }
    for (; b < blocks; b += n) v += p[(size_t)b * step];
  }
  sh[slice][lane] = v;
  __syncthreads();
  if (slice) return;
  v = 0.f;
#pragma unroll
  for (int k = 0; k < 32; ++k) v += sh[k][lane];
  if (last) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor(v, o);
    if (lane) return;
    if (a.s32) *(float *)a.dscale = v;
    else act8_put<T>(a.dscale, 0, v);
    return;
  }
  if (c >= a.C) return;
  if (set >= SET_POST_W) v *= !a.scale ? a.scale_host : a.s32 ? *(const float *)a.scale : act8_get<T>(a.scale, 0);
  if (set == SET_GATE) {
    v *= act_slope(a.act, act_of(a.act, act8_get<T>(a.gate, (size_t)group * a.ldg + c)));
    act8_put<T>(a.out[set], (size_t)group * a.C + c, v);
  } else if (a.w32) ((float *)a.out[set])[c] = v;
  else act8_put<T>(a.out[set], c, v);
}

template <int T, bool LAYER>
int launch_fwd(const BnArgs &a, const BnPlan &p, hipStream_t st) {
  const int teams = p.block / p.T;
  const uint32_t blocks = (a.rows + teams - 1) / teams, most = 1024;   // (as many as are resident at once, and parameters are read once)
  const unsigned grid = blocks < most ? blocks : most;
  if (p.T < 64) block_norm_fwd_kernel<T, LAYER, 1, 512, false><<<grid, 512, 0, st>>>(a);
  else if (p.block == 512 && p.nch == 1) block_norm_fwd_kernel<T, LAYER, 1, 512, true><<<grid, 512, 0, st>>>(a);
  else if (p.block == 512) block_norm_fwd_kernel<T, LAYER, 2, 512, true><<<grid, 512, 0, st>>>(a);
  else block_norm_fwd_kernel<T, LAYER, 2, 1024, true><<<grid, 1024, 0, st>>>(a);
  DM_CHECK_LAUNCH();
  return DM_OK;
}

// what forward and backward have in common; returns a DM_ERR_* code
int fill(BnArgs *a, const dm_block_norm *q, bool backward, BnPlan *p) {
  if (!q || q->dtype < ACT8_F32 || q->dtype > ACT8_F16 || q->rows < 0 || q->rows > 0x7ffffc00 || q->width <= 0) return DM_ERR_INVALID_ARG;
  if (!bn_plan(q->width, backward, p)) return DM_ERR_UNSUPPORTED;
  if (q->gate_act < ACT_NONE || q->gate_act > ACT_TANH || q->groups < 0 || (q->gate ? q->groups < 1 || q->rows % q->groups : q->groups != 0))
    return DM_ERR_INVALID_ARG;
  if (q->gate && q->ld_gate < q->width && q->groups > 1) return DM_ERR_INVALID_ARG;
  if (!(q->eps >= 0.f)) return DM_ERR_INVALID_ARG;
  const int dt = q->dtype;
  a->gate = q->gate, a->post_w = q->post_w, a->post_b = q->post_b, a->pre_w = q->pre_w, a->pre_b = q->pre_b, a->scale = q->scale;
  a->rows = (uint32_t)q->rows, a->groups = q->groups > 0 ? (uint32_t)q->groups : 1, a->each = a->rows / a->groups;
  a->ldg = q->ld_gate, a->inv_c = 1.f / (float)q->width, a->eps = q->eps, a->scale_host = q->scale_host, a->C = q->width, a->T = p->T;
  a->act = q->gate_act, a->post = q->post, a->w32 = q->param_f32 || dt == ACT8_F32, a->s32 = q->scale_f32 || dt == ACT8_F32;
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
  const int rc = fill(&a, q, false, &p);
  if (rc != DM_OK) return rc;
  if (q->rows == 0) return DM_OK;
  if (!x || ldx < q->width || (f && (!y || ldf < q->width)) || (!f && (!h || y || q->gate)) || (q->f_codes && !f)) return DM_ERR_INVALID_ARG;
  const bool layer = q->layer != 0;
  if (layer && ((a.f_rstd && !a.f_mean) || (a.y_rstd && !a.y_mean))) return DM_ERR_INVALID_ARG;
  a.x = x, a.f = f, a.y = y, a.h = h, a.ldx = ldx, a.ldf = ldf;
  hipStream_t st = (hipStream_t)stream;
  if (q->dtype == ACT8_F32) return layer ? launch_fwd<ACT8_F32, true>(a, p, st) : launch_fwd<ACT8_F32, false>(a, p, st);
  if (q->dtype == ACT8_BF16) return layer ? launch_fwd<ACT8_BF16, true>(a, p, st) : launch_fwd<ACT8_BF16, false>(a, p, st);
  return layer ? launch_fwd<ACT8_F16, true>(a, p, st) : launch_fwd<ACT8_F16, false>(a, p, st);
}

extern "C" size_t dm_block_norm_workspace_bytes(long long rows, int width, long long groups) {
  BnPlan p;
  if (rows <= 0 || width <= 0 || groups < 0 || !bn_plan(width, true, &p)) return 0;
  const BnGrid g = bn_grid(p, rows, groups);
  return dm_align((size_t)g.x * g.y * ((size_t)SETS * width + 1) * sizeof(float));
}

extern "C" int dm_block_norm_backward(const dm_block_norm *q, const void *gy, long long ldgy, const void *gh, long long ldgh, const void *y,
                                      long long ldy, const void *f, long long ldf, void *dx, void *df, void *dgate, void *dpre_w, void *dpre_b,
                                      void *dpost_w, void *dpost_b, void *dscale, void *workspace, size_t workspace_bytes,
                                      dm_stream_t stream) {
  BnArgs a = {};
  BnPlan p;
  const int rc = fill(&a, q, true, &p);
  if (rc != DM_OK) return rc;
  if (q->rows == 0) return DM_ERR_INVALID_ARG;                     // (there is nothing to sum: the caller writes the zeros)
  const bool layer = q->layer != 0, has_f = f || q->f_codes;
  if ((gy && ldgy < q->width) || (gh && ldgh < q->width) || (!gy && !gh)) return DM_ERR_INVALID_ARG;
  if ((q->f_codes || q->y_codes) && ((has_f && !q->f_codes) || (gh && !q->y_codes))) return DM_ERR_INVALID_ARG;
  if (gh && (!a.y_rstd || (layer && !a.y_mean) || !(y || q->y_codes) || (y && ldy < q->width))) return DM_ERR_INVALID_ARG;
  if (has_f && q->post && (!a.f_rstd || (layer && !a.f_mean))) return DM_ERR_INVALID_ARG;
  if ((f && ldf < q->width) || (!has_f && (df || dgate || dpost_w || dpost_b || dscale))) return DM_ERR_INVALID_ARG;
  if ((dgate && !q->gate) || ((dpost_w || dpost_b) && !q->post) || ((dpre_w || dpre_b) && !gh) || ((dpre_b || dpost_b) && !layer)) return DM_ERR_INVALID_ARG;
  if (!workspace || workspace_bytes < dm_block_norm_workspace_bytes(q->rows, q->width, q->groups)) return DM_ERR_WORKSPACE;
  const int dt = q->dtype;
  a.gy = gy, a.gh = gh, a.y_in = y, a.f = f, a.ldgy = ldgy, a.ldgh = ldgh, a.ldx = ldy, a.ldf = ldf;
  a.dx = dx, a.df = df, a.dgate = dgate, a.part = (float *)workspace;
  const BnGrid g = bn_grid(p, q->rows, q->groups);
  a.by_unit = g.by_unit, a.n_blocks = g.x * g.y;
  a.sets = (dpre_w ? 1 << SET_PRE_W : 0) | (dpre_b ? 1 << SET_PRE_B : 0) | (dpost_w ? 1 << SET_POST_W : 0) | (dpost_b ? 1 << SET_POST_B : 0) |
           (dgate && !g.by_unit ? 1 << SET_GATE : 0);
  hipStream_t st = (hipStream_t)stream;
  const int e = dm_block_norm_launch_backward(dt, layer, a, p, g, st);
  if (e != DM_OK) return e;
  SumArgs s = {};
  s.part = a.part, s.dscale = dscale, s.gate = q->gate, s.ldg = q->ld_gate, s.C = q->width, s.act = q->gate_act, s.n_blocks = a.n_blocks;
  s.groups = g.y, s.w32 = a.w32, s.s32 = a.s32, s.scale = q->scale, s.scale_host = q->scale_host;
  s.out[SET_PRE_W] = dpre_w, s.out[SET_PRE_B] = dpre_b, s.out[SET_POST_W] = dpost_w, s.out[SET_POST_B] = dpost_b;
  s.out[SET_GATE] = g.by_unit ? nullptr : dgate;
  if (!dpre_w && !dpre_b && !dpost_w && !dpost_b && !s.out[SET_GATE] && !dscale) return DM_OK;
  const dim3 grid(dm_ceil_div(q->width, 32) + 1, SET_GATE + g.y);
  if (dt == ACT8_F32) block_norm_sum_kernel<ACT8_F32><<<grid, 1024, 0, st>>>(s);
  else if (dt == ACT8_BF16) block_norm_sum_kernel<ACT8_BF16><<<grid, 1024, 0, st>>>(s);
  else block_norm_sum_kernel<ACT8_F16><<<grid, 1024, 0, st>>>(s);
  DM_CHECK_LAUNCH();
  return DM_OK;
}
