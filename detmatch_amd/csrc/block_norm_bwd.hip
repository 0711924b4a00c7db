// Backward pass of the norms around a residual block (formulas: block_norm.hip).
#include "block_norm.h"

using namespace dm_bn;

namespace {

// 8 elements of a row as they wait in registers: exact, or as codes and their exponent.  (A choice between the two at run time would make the
// compiler wait for the loads where they are issued, to move them into common registers.)
template <int T, bool KEEP8>
struct Waiting {
  Act8Raw<T> r;
  template <bool>
  __device__ __forceinline__ void load(const void *p, long long ld, const uint8_t *, const uint8_t *, uint32_t row, int, int c, int n) {
    r = act8_load_raw<T>(p, (size_t)row * ld + c, n);
  }
  __device__ __forceinline__ void take(float *v) const { act8_unraw<T>(r, v); }
};

template <int T>
struct Waiting<T, true> {
  uint2 u;
  uint32_t e;
  // Behind a row's end and for a team without a row: zeros.  CLAMP: behind a row's end other codes of the same row, without a branch.  (Gradients are 0 there; should
  // a code be a nan, that row's sums are nan already.  Another row's codes would not do: 0 * nan is nan.  So CLAMP is for teams that never lack a row.)
  template <bool CLAMP>
  __device__ __forceinline__ void load(const void *, long long, const uint8_t *codes, const uint8_t *exps, uint32_t row, int groups,
                                       int c, int n) {
    if (CLAMP) c = min(c, groups * ACT8_GROUP - 8);
    else u = make_uint2(0u, 0u), e = 127u;
    if (CLAMP || n > 0) {
      const size_t at = (size_t)row * groups;
      u = *(const uint2 *)(codes + (at * ACT8_GROUP + c));
      e = exps[at + c / ACT8_GROUP];
    }
  }
  __device__ __forceinline__ void take(float *v) const {
    act8_decode4(u.x, e, v), act8_decode4(u.y, e, v + 4);
    if constexpr (T == ACT8_F16) {                   // (the other types hold every code exactly)
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = v[k] != v[k] ? v[k] : (float)(_Float16)fminf(fmaxf(v[k], -65504.f), 65504.f);
    }
  }
};

// A row's number in a vector register: its statistics then come by vector loads.  As scalar loads they share a counter with LDS, and a team's sum
// would wait for memory.
__device__ __forceinline__ uint32_t in_vector(uint32_t v) {
  asm("" : "+v"(v));
  return v;
}

// Sums over the rows that a thread walks, 8 channels of one set, stay in registers; with 1 024 threads to a row there are too few of those, and the
// sums lie in LDS (16 384 x 8 192 bf16, exact RMS rows: 514 us against 620 with registers that spill, from codes 532 and 670; at 4 096 channels LDS costs 595 us against 343).
template <int BLOCK>
__device__ __forceinline__ float4 *sums_at(float4 *lds, int slot, int half) {
  return lds + (slot * 2 + half) * BLOCK + threadIdx.x;
}

template <int BLOCK>
__device__ __forceinline__ void sums_add(float4 *lds, int slot, const float (&v)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float4 *p = sums_at<BLOCK>(lds, slot, h);
    float4 w = *p;
    w.x += v[4 * h], w.y += v[4 * h + 1], w.z += v[4 * h + 2], w.w += v[4 * h + 3];
    *p = w;
  }
}

// A team walks rows team, team + teams, ... of one group of rows (blockIdx.y) that share their gates, or, where there are many
// groups, whole groups one after another (by_unit); `each` rows have one row of gates.
// Bound by memory, with 8 waves a compute unit (150 to 220 registers a thread: parameters, sums and two rows): 32 768 x 4 096 bf16 RMS 349 us = 4.6 TB/s
// exact, 324 (4.2) from codes, with a gate for each element 412 (5.2) and 409 (4.6); LN 362; 65 536 x 1 024 163 (4.9) and 170 (4.0).  Decoding and the
// products of fp32 rows are what keeps codes and LN from the rate of a copy; 128 registers, and twice the waves, spill: 752 us in place of 349.
// Above 4 096 channels 1 024 threads have 128 registers each, and rows come one at a time: 16 384 x 8 192 bf16 RMS 507 us = 3.2 TB/s exact, 528 (2.6) from codes, with
// a gate for each element 673 (2.8); LN 778 (2.1) and 789 (1.7).  Above 8 192 channels a thread has twice 8 channels and the sums spill: 8 192 x 16 384 RMS 1 619 us = 1.0
// TB/s, LN from codes 3 030 (0.45): right, but far from fast.
template <int T, bool LAYER, int NCH, int BLOCK, bool WAVES, bool KEEP8>
__global__ __launch_bounds__(BLOCK, 2) void block_norm_bwd_kernel(BnArgs a) {
  constexpr bool IN_LDS = BLOCK == 1024 && NCH == 1, AT_ONCE = KEEP8 && BLOCK == 512;
  __shared__ float team_sums[BLOCK == 512 ? BLOCK * 8 : 1];
  __shared__ float red[64];
  extern __shared__ __attribute__((aligned(16))) float4 bn_sums[];       // IN_LDS: [wanted set, SET_PRE_B apart][2][BLOCK]
  const int tx = threadIdx.x & (a.T - 1), team = team_of<WAVES>(a.T), teams = BLOCK / a.T, groups8 = (a.C + 31) / 32;
  int turn = 0;
  const float scale = load_scale<T>(a);
  const bool has_f = a.f || a.f_codes, has_h = a.gh != nullptr;
  // (SET_PRE_B, the first one of the layer norm's five, stays in registers: five sets of 1 024 threads are more than LDS holds)
  const int sets = a.sets, in_lds = sets & ~(1 << SET_PRE_B);
  auto slot = [&](int set) { return __builtin_popcount(in_lds & ((1 << set) - 1)); };
  float acc[IN_LDS ? 2 : SETS][NCH][8], dscale = 0.f;
  float (&gate_acc)[NCH][8] = acc[IN_LDS ? 1 : SET_GATE];        // (by_unit: of the group of rows under way)
  float post_w[NCH][8], post_b[LAYER ? NCH : 1][8], pre_w[NCH][8];
#pragma unroll
  for (int n = 0; n < NCH; ++n) {
    const int c = 8 * (tx + n * a.T);
    load_param<T>(a, a.post_w, c, post_w[n], 1.f), load_param<T>(a, a.pre_w, c, pre_w[n], 1.f);
    if constexpr (LAYER) load_param<T>(a, a.post_b, c, post_b[n], 0.f);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
#pragma unroll
      for (int s = 0; s < (IN_LDS ? 2 : SETS); ++s) acc[s][n][k] = 0.f;
    }
  }
  if constexpr (IN_LDS) {
    for (int i = 0; i < 2 * __builtin_popcount(in_lds); ++i) bn_sums[i * BLOCK + threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  auto add = [&](int set, const float (&v)[NCH][8]) {        // (a thread's own places: no barrier)
    if constexpr (IN_LDS) {
      if (LAYER && set == SET_PRE_B) {
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[0][0][k] += v[0][k];
      } else if ((sets >> set) & 1) sums_add<BLOCK>(bn_sums, slot(set), v[0]);
    } else {
#pragma unroll
      for (int n = 0; n < NCH; ++n)
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[set][n][k] += v[n][k];
    }
  };
  const uint32_t stride = gridDim.x * teams, first = blockIdx.x * teams + team;
  // Teams of a workgroup meet in the sums: all make as many trips as the first, the last ones perhaps without a row of their own.  Where codes are clamped a
  // workgroup is one team (1 024 threads), and walks its own rows alone (there are at most as many workgroups as rows or groups).
  const uint32_t ahead = KEEP8 && !AT_ONCE ? first : 0;
  const uint32_t trips = a.by_unit ? (a.groups - ahead + stride - 1) / stride * a.each : (a.each - ahead + stride - 1) / stride;
  // The next row's operands are under way while this one is computed: those of y's side from the row's begin on, those of f's side from where
  // this row's have been taken out of their registers.  Codes are so short that both sides can be under way from the row's begin on, AT_ONCE; teams do
  // without WAVES then, and loads without CLAMP (32 768 x 4 096 bf16 with a gate for each element 409 us; with late loads 449, with clamped ones 453;
  // exact rows 476, late and with WAVES 413).  With 1 024 threads and half the registers it is the other way round (16 384 x 8 192 with a gate for each element 969 and 688 us).
  uint32_t unit = a.by_unit ? first : blockIdx.y, in_unit = a.by_unit ? 0 : first;
  Act8Raw<T> raw_gh[NCH], raw_gy[NCH], raw_g[NCH];
  Waiting<T, KEEP8> raw_y[NCH], raw_f[NCH];
  float next_mean = 0.f, next_rstd = 0.f, next_f_mean = 0.f, next_f_rstd = 0.f;
  auto fetch_y = [&]() {
    const bool live = unit < a.groups && in_unit < a.each;
    const uint32_t row = unit * a.each + in_unit;
    next_mean = next_rstd = 0.f;
    if (live && has_h) {
      const uint32_t r = in_vector(row);
      next_rstd = a.y_rstd[r];
      if (LAYER) next_mean = a.y_mean[r];
    }
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int c = 8 * (tx + n * a.T), left = live ? a.C - c : 0;
      if (has_h) {
        raw_gh[n] = act8_load_raw<T>(a.gh, (size_t)row * a.ldgh + c, left);
        raw_y[n].template load<!AT_ONCE>(a.y_in, a.ldx, a.y_codes, a.y_exps, row, groups8, c, left);
      }
      if (a.gy) raw_gy[n] = act8_load_raw<T>(a.gy, (size_t)row * a.ldgy + c, left);
    }
  };
  auto fetch_f = [&]() {
    const bool live = unit < a.groups && in_unit < a.each;
    const uint32_t row = unit * a.each + in_unit;
    next_f_mean = next_f_rstd = 0.f;
    if (live && a.post) {
      const uint32_t r = in_vector(row);
      next_f_rstd = a.f_rstd[r];
      if (LAYER) next_f_mean = a.f_mean[r];
    }
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int c = 8 * (tx + n * a.T), left = live ? a.C - c : 0;
      raw_f[n].template load<!AT_ONCE>(a.f, a.ldf, a.f_codes, a.f_exps, row, groups8, c, left);
      if (a.gate) raw_g[n] = act8_load_raw<T>(a.gate, (size_t)unit * a.ldg + c, left);
    }
  };
  if (trips) {
    fetch_y();
    if (has_f) fetch_f();
  }
  for (uint32_t i = 0; i < trips; ++i) {
    const bool live = unit < a.groups && in_unit < a.each, last = a.by_unit && in_unit + 1 == a.each;     // last: the group's last row
    const uint32_t this_unit = unit;
    const size_t row = unit * a.each + in_unit;
    if (!a.by_unit) in_unit += stride;
    else if (++in_unit == a.each) in_unit = 0, unit += stride;
    float dy[NCH][8], hat[NCH][8], d[NCH][8];
    const float y_mean = next_mean, y_rstd = next_rstd;
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      if (a.gy) act8_unraw<T>(raw_gy[n], dy[n]);
      else
#pragma unroll
        for (int k = 0; k < 8; ++k) dy[n][k] = 0.f;
      if (has_h) {
        act8_unraw<T>(raw_gh[n], d[n]);
        raw_y[n].take(hat[n]);
      }
    }
    Waiting<T, KEEP8> now_f[NCH];                // (AT_ONCE)
    Act8Raw<T> now_g[NCH];
    float now_f_mean = next_f_mean, now_f_rstd = next_f_rstd;
    if (AT_ONCE && has_f) {
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        now_f[n] = raw_f[n];
        if (a.gate) now_g[n] = raw_g[n];
      }
    }
    if (i + 1 < trips) {
      fetch_y();
      if (AT_ONCE && has_f) fetch_f();
    }
    // (channels behind the width, and rows of a team without one: gradients are 0 there, and what multiplies them is finite)
    if (has_h) {
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int n = 0; n < NCH; ++n)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (LAYER) hat[n][k] -= y_mean;
          hat[n][k] *= y_rstd;
        }
      if (LAYER) add(SET_PRE_B, d);
      {
        float v[NCH][8];
#pragma unroll
        for (int n = 0; n < NCH; ++n)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (IN_LDS) v[n][k] = d[n][k] * hat[n][k];
            else acc[IN_LDS ? 0 : SET_PRE_W][n][k] = fmaf(d[n][k], hat[n][k], acc[IN_LDS ? 0 : SET_PRE_W][n][k]);
            d[n][k] *= pre_w[n][k];
            s[0] = fmaf(d[n][k], hat[n][k], s[0]);
            if (LAYER) s[1] += d[n][k];
          }
        if (IN_LDS) add(SET_PRE_W, v);
      }
      if constexpr (LAYER) team_sum<2>(s, a.T, red, turn);
      else {
        float one[1] = {s[0]};
        team_sum<1>(one, a.T, red, turn);
        s[0] = one[0];
      }
      const float m0 = s[0] * a.inv_c, m1 = s[1] * a.inv_c;
#pragma unroll
      for (int n = 0; n < NCH; ++n)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (LAYER) d[n][k] -= m1;
          dy[n][k] = fmaf(y_rstd, fmaf(-hat[n][k], m0, d[n][k]), dy[n][k]);
        }
    }
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int c = 8 * (tx + n * a.T);
      if (live && a.dx) act8_store8<T>(a.dx, row * a.C + c, a.C - c, dy[n]);
    }
    if (has_f) {
      float v[NCH][8], g[NCH][8], s[2] = {0.f, 0.f};
      const float f_mean = AT_ONCE ? now_f_mean : next_f_mean, f_rstd = AT_ONCE ? now_f_rstd : next_f_rstd;
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        if constexpr (AT_ONCE) now_f[n].take(hat[n]);
        else raw_f[n].take(hat[n]);
        if (a.gate) act8_unraw<T>(AT_ONCE ? now_g[n] : raw_g[n], g[n]);
      }
      if (!AT_ONCE && i + 1 < trips) fetch_f();
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        const int c = 8 * (tx + n * a.T);
        if (c + 8 > a.C) {
#pragma unroll
          for (int k = 0; k < 8; ++k) dy[n][k] = c + k < a.C ? dy[n][k] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {                        // v: the gradient times what the block put out, normalised
          float u = hat[n][k];
          if (a.post) {
            if (LAYER) hat[n][k] -= f_mean;
            hat[n][k] *= f_rstd;
            u = LAYER ? fmaf(hat[n][k], post_w[n][k], post_b[n][k]) : hat[n][k] * post_w[n][k];
          }
          v[n][k] = dy[n][k] * u;
        }
        if (a.gate) {
          if (a.by_unit) {
#pragma unroll
            for (int k = 0; k < 8; ++k) gate_acc[n][k] += v[n][k];
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) g[n][k] = act_of(a.act, g[n][k]);
          if (last) {                                     // this group of rows is done: its gates' gradient is complete
            float w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              w[k] = gate_acc[n][k] * scale * act_slope(a.act, g[n][k]);
              gate_acc[n][k] = 0.f;
            }
            if (live && a.dgate) act8_store8<T>(a.dgate, (size_t)this_unit * a.C + c, a.C - c, w);
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            dscale = fmaf(v[n][k], g[n][k], dscale);
            dy[n][k] *= g[n][k];
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) dscale += v[n][k];
        }
      }
      if (a.gate && !a.by_unit) add(SET_GATE, v);
      float r = scale;
      if (a.post) {
        if (LAYER) add(SET_POST_B, dy);
#pragma unroll
        for (int n = 0; n < NCH; ++n)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (IN_LDS) v[n][k] = dy[n][k] * hat[n][k];
            else acc[IN_LDS ? 0 : SET_POST_W][n][k] = fmaf(dy[n][k], hat[n][k], acc[IN_LDS ? 0 : SET_POST_W][n][k]);
            dy[n][k] *= post_w[n][k];
            s[0] = fmaf(dy[n][k], hat[n][k], s[0]);
            if (LAYER) s[1] += dy[n][k];
          }
        if (IN_LDS) add(SET_POST_W, v);
        if constexpr (LAYER) team_sum<2>(s, a.T, red, turn);
        else {
          float one[1] = {s[0]};
          team_sum<1>(one, a.T, red, turn);
          s[0] = one[0];
        }
        const float m0 = s[0] * a.inv_c, m1 = s[1] * a.inv_c;
        r *= f_rstd;
#pragma unroll
        for (int n = 0; n < NCH; ++n)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (LAYER) dy[n][k] -= m1;
            dy[n][k] = fmaf(-hat[n][k], m0, dy[n][k]);
          }
      }
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        const int c = 8 * (tx + n * a.T);
#pragma unroll
        for (int k = 0; k < 8; ++k) dy[n][k] *= r;
        if (live && a.df) act8_store8<T>(a.df, row * a.C + c, a.C - c, dy[n]);
      }
    }
  }
  // this workgroup's sums; the residual scale, the same for all, is multiplied on when they are added up
  const size_t block = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
  if constexpr (IN_LDS) {
    // (the set that is in registers last: it takes the place of the first)
    constexpr int order[SETS] = {SET_PRE_W, SET_POST_W, SET_POST_B, SET_GATE, SET_PRE_B};
#pragma unroll
    for (int i = 0; i < SETS; ++i) {
      const int s = order[i];
      if (!((sets >> s) & 1)) continue;
      if (s == SET_PRE_B) {
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *sums_at<BLOCK>(bn_sums, 0, h) = make_float4(acc[0][0][4 * h], acc[0][0][4 * h + 1], acc[0][0][4 * h + 2], acc[0][0][4 * h + 3]);
      }
      __syncthreads();
      // channel c of team t: float c % 4 of place [slot][c / 4 % 2][t * T + c / 8]
      const float *p = (const float *)(bn_sums + (size_t)(s == SET_PRE_B ? 0 : slot(s)) * 2 * BLOCK);
      for (int c = threadIdx.x; c < a.C; c += BLOCK) {
        const float *q = p + ((c >> 2) & 1) * BLOCK * 4 + (c >> 3) * 4 + (c & 3);
        float v = 0.f;
        for (int t = 0; t < teams; ++t) v += q[t * a.T * 4];
        a.part[((size_t)s * a.n_blocks + block) * a.C + c] = v;
      }
    }
  } else if (BLOCK == 512 && teams > 1) {
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      if (!((sets >> s) & 1)) continue;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 8; ++k) team_sums[threadIdx.x * 8 + k] = acc[s][0][k];
      __syncthreads();
      for (int c = threadIdx.x; c < a.C; c += BLOCK) {
        float v = 0.f;
        for (int t = 0; t < teams; ++t) v += team_sums[t * a.T * 8 + c];
        a.part[((size_t)s * a.n_blocks + block) * a.C + c] = v;
      }
    }
  } else {
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      if (!((sets >> s) & 1)) continue;
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        const int c = 8 * (tx + n * a.T);
        act8_store8<ACT8_F32>(a.part, ((size_t)s * a.n_blocks + block) * a.C + c, a.C - c, acc[s][n]);
      }
    }
  }
  float ds[1] = {dscale};
  __syncthreads();
  team_sum<1>(ds, BLOCK, red, turn);
  if (threadIdx.x == 0) a.part[(size_t)SETS * a.n_blocks * a.C + block] = ds[0];
}

template <int T, bool LAYER, int NCH, int BLOCK, bool WAVES>
int launch_bwd(const BnArgs &a, const BnGrid &g, hipStream_t st) {
  auto k = a.f_codes || a.y_codes ? block_norm_bwd_kernel<T, LAYER, NCH, BLOCK, WAVES && BLOCK != 512, true> : block_norm_bwd_kernel<T, LAYER, NCH, BLOCK, WAVES, false>;
  const int in_lds = a.sets & ~(1 << SET_PRE_B), slots = in_lds || !a.sets ? __builtin_popcount(in_lds) : 1;
  const int lds = BLOCK == 1024 && NCH == 1 ? slots * 2 * BLOCK * (int)sizeof(float4) : 0;
  if (lds > 65536 - 1024) DM_HIP(hipFuncSetAttribute((const void *)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  k<<<dim3(g.x, g.y), BLOCK, lds, st>>>(a);
  DM_CHECK_LAUNCH();
  return DM_OK;
}

template <int T, bool LAYER>
int launch_bwd(const BnArgs &a, const BnPlan &p, const BnGrid &g, hipStream_t st) {
  if (p.T < 64) return launch_bwd<T, LAYER, 1, 512, false>(a, g, st);
  if (p.block == 512) return launch_bwd<T, LAYER, 1, 512, true>(a, g, st);
  return p.nch == 1 ? launch_bwd<T, LAYER, 1, 1024, true>(a, g, st) : launch_bwd<T, LAYER, 2, 1024, true>(a, g, st);
}

}  // namespace

int dm_block_norm_launch_backward(int dtype, bool layer, const BnArgs &a, const BnPlan &p, const BnGrid &g, hipStream_t st) {
  if (dtype == ACT8_F32) return layer ? launch_bwd<ACT8_F32, true>(a, p, g, st) : launch_bwd<ACT8_F32, false>(a, p, g, st);
  if (dtype == ACT8_BF16) return layer ? launch_bwd<ACT8_BF16, true>(a, p, g, st) : launch_bwd<ACT8_BF16, false>(a, p, g, st);
  return layer ? launch_bwd<ACT8_F16, true>(a, p, g, st) : launch_bwd<ACT8_F16, false>(a, p, g, st);
}
