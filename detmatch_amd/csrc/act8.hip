// 8-bit copies of activations that wait for the backward pass (format: act8_codec.h), and what the backward pass of an FC
// layer reads besides them: the sign bits of a ReLU's output.
#include "act8_codec.h"

namespace {

constexpr int A8_BLOCK = 256;

// Rows of `width` elements -> codes (rows, 32 * groups) and exponents (rows, groups).  A thread holds 8 neighbouring
// elements, 4 threads a group; `tpr` threads (a power of two) walk one row, 256 / tpr rows to a workgroup.
// Bound by memory: element size in, 1 + 1/32 bytes out.  8 elements a thread make one 16-byte load (two in fp32), one 8-byte store and a
// maximum over 4 lanes without LDS.  4 096 x 12 544 bf16: 26 us, 6.0 TB/s (some of x is still in the last cache); with its way back 61 us, 5.1
// TB/s, the rate of a copy.  1 999 x 12 544 fp32: 22 us.
template <int T>
__global__ __launch_bounds__(A8_BLOCK) void act8_pack_kernel(const void *__restrict__ x, long long rows, int width, long long ld,
                                                             int groups, int tpr, uint8_t *__restrict__ codes,
                                                             uint8_t *__restrict__ exps) {
  const int tx = threadIdx.x & (tpr - 1), ty = threadIdx.x / tpr, rpb = A8_BLOCK / tpr;
  const int chunks = groups * 4;
  for (long long r = (long long)blockIdx.x * rpb + ty; r < rows; r += (long long)gridDim.x * rpb) {
    for (int c = tx; c < chunks; c += tpr) {             // (chunks and tpr are multiples of 4: a quad stays together)
      float v[8];
      const int n = width - 8 * c;
      act8_load8<T>(x, (size_t)r * ld + 8 * c, n, v);
      int e;
      const uint2 u = act8_encode8(v, &e);
      *(uint2 *)(codes + ((size_t)r * groups * ACT8_GROUP + 8 * c)) = u;
      if ((tx & 3) == 0) exps[(size_t)r * groups + (c >> 2)] = (uint8_t)(e + 127);
    }
  }
}

// The way back: a multiplication by a power of two, exact but for fp16's range.  Bound by memory; 4 096 x 12 544 bf16: 23 us.
template <int T>
__global__ __launch_bounds__(A8_BLOCK) void act8_unpack_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ exps,
                                                               long long rows, int width, int groups, int tpr,
                                                               void *__restrict__ out) {
  const int tx = threadIdx.x & (tpr - 1), ty = threadIdx.x / tpr, rpb = A8_BLOCK / tpr;
  const int chunks = (width + 7) / 8;
  const float most = act8_most<T>();
  for (long long r = (long long)blockIdx.x * rpb + ty; r < rows; r += (long long)gridDim.x * rpb) {
    for (int c = tx; c < chunks; c += tpr) {
      const uint2 u = *(const uint2 *)(codes + ((size_t)r * groups * ACT8_GROUP + 8 * c));
      const uint32_t e = exps[(size_t)r * groups + (c >> 2)];
      float v[8];
      act8_decode4(u.x, e, v);
      act8_decode4(u.y, e, v + 4);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = v[k] != v[k] ? v[k] : fminf(fmaxf(v[k], -most), most);
      act8_store8<T>(out, (size_t)r * width + 8 * c, width - 8 * c, v);
    }
  }
}

// threads that walk one row: the power of two above its chunks of 8 elements, a quad at least, a workgroup at most
int a8_threads_per_row(int chunks) {
  int t = 4;
  while (t < chunks && t < A8_BLOCK) t <<= 1;
  return t;
}

unsigned a8_grid(long long rows, int rpb) {
  const long long b = (rows + rpb - 1) / rpb;
  return (unsigned)(b < 65536 ? b : 65536);
}

}  // namespace

extern "C" int dm_act8_pack(const void *x, int dtype, long long rows, int width, long long ld, uint8_t *codes, uint8_t *exps,
                            dm_stream_t stream) {
  if (dtype < ACT8_F32 || dtype > ACT8_F16 || rows < 0 || width <= 0 || ld < width || width > (1 << 28)) return DM_ERR_INVALID_ARG;
  if (rows == 0) return DM_OK;
  if (!x || !codes || !exps || ((uintptr_t)codes & 7)) return DM_ERR_INVALID_ARG;
  const int groups = dm_ceil_div(width, ACT8_GROUP), tpr = a8_threads_per_row(groups * 4);
  const unsigned grid = a8_grid(rows, A8_BLOCK / tpr);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == ACT8_F32) act8_pack_kernel<ACT8_F32><<<grid, A8_BLOCK, 0, st>>>(x, rows, width, ld, groups, tpr, codes, exps);
  else if (dtype == ACT8_BF16) act8_pack_kernel<ACT8_BF16><<<grid, A8_BLOCK, 0, st>>>(x, rows, width, ld, groups, tpr, codes, exps);
  else act8_pack_kernel<ACT8_F16><<<grid, A8_BLOCK, 0, st>>>(x, rows, width, ld, groups, tpr, codes, exps);
  DM_CHECK_LAUNCH();
  return DM_OK;
}

extern "C" int dm_act8_unpack(const uint8_t *codes, const uint8_t *exps, long long rows, int width, void *out, int dtype,
                              dm_stream_t stream) {
  if (dtype < ACT8_F32 || dtype > ACT8_F16 || rows < 0 || width <= 0 || width > (1 << 28)) return DM_ERR_INVALID_ARG;
  if (rows == 0) return DM_OK;
  if (!out || !codes || !exps || ((uintptr_t)codes & 7)) return DM_ERR_INVALID_ARG;
  const int groups = dm_ceil_div(width, ACT8_GROUP), tpr = a8_threads_per_row(dm_ceil_div(width, 8));
  const unsigned grid = a8_grid(rows, A8_BLOCK / tpr);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == ACT8_F32) act8_unpack_kernel<ACT8_F32><<<grid, A8_BLOCK, 0, st>>>(codes, exps, rows, width, groups, tpr, out);
  else if (dtype == ACT8_BF16) act8_unpack_kernel<ACT8_BF16><<<grid, A8_BLOCK, 0, st>>>(codes, exps, rows, width, groups, tpr, out);
  else act8_unpack_kernel<ACT8_F16><<<grid, A8_BLOCK, 0, st>>>(codes, exps, rows, width, groups, tpr, out);
  DM_CHECK_LAUNCH();
  return DM_OK;
}
