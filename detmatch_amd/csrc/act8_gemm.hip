// Matrix products of an FC layer whose weight gradient reads the 8-bit copy of its input (act8_codec.h).
//   form 0   C[M][N] = A[M][K] . B[N][K]^T (+ bias, ReLU, sign bits)   forward            y  = x w^T + b
//   form 1   C[M][N] = A[M][K] . B[K][N]                               input gradient     gx = gy w
//   form 2   C[M][N] = A[K][M]^T . deq(B)[K][N] (+ row sums)           weight gradient    gw = gy^T x8, gb = sum of gy
// All on the 16-bit matrix instructions (v_mfma_f32_32x32x16, subnormal numbers included), accumulated in fp32.  deq(code) is exact in bf16, so form 2 loses
// nothing there.  fp32 operands are cut into three bf16 pieces (8 + 8 + 8 bits) while they are staged; a product of two such operands takes the 6 of the 9 piece
// products that matter in fp32, a product with codes takes 3.  The pieces are all of a finite value from 2^-109 on; below that, and of a code of an fp32 row, what
// lies under 2^-133, bf16's least number, is lost.
//
// A wave owns FM x FN blocks of 32 x 32; the matrix instruction gets its operands swapped (rows of its result = columns of C), so that a
// lane ends with 4 neighbouring elements of a row of C.  Few output tiles and a long contraction: the contraction is split over
// workgroups, partial sums go to a workspace and are added in split order by a second kernel (no atomics: the result is a
// function of the shapes and values alone).
#include <type_traits>

#include "act8_codec.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

struct A8Args {
  const void *A, *B, *bias;
  const uint8_t *exps;        // form 2: exponents of B's codes, groups per row = ldb / 32
  void *C;
  float *part;                // [splits][M][N] when splits > 1, and behind it [splits][M] row sums
  uint32_t *bits;             // sign bits of C, (M, ceil(N / 32)): see passes
  void *rowsum;               // form 2: sum over the contraction of A's columns (M)
  int M, N, K;
  long long lda, ldb;
  int relu, splits, steps_per_split, tiles_m, tiles_n, per_xcd, vec_c;
};

// ---- where a 16-byte piece of a staged tile lies in LDS ----------------------------------------------------------------
// contraction-contiguous tile [rows][BK]: a fragment read takes the same piece of 16 rows at once; the piece index is xored with bits
// of the row, so that those 16 reads fall on all 64 banks.
template <int BK>
__device__ __forceinline__ int kc_swizzle(int row) {
  return BK == 64 ? (row >> 1) & 7 : (row >> 2) & 3;
}
// contraction along the rows [BK][cols], 128-column (256-byte) lines or wider: a transposing read takes 64 bytes of 4 rows at once, a
// staging store the pieces 2 c + j of 2 rows
__device__ __forceinline__ int kr_swizzle(int k) { return ((k & 3) << 2) | (k & 1); }

// fragment of 32 rows x 16 of the contraction from a contraction-contiguous tile: lane -> row lane & 31, 8 elements from (lane >> 5) * 8
template <int BK>
__device__ __forceinline__ s16x8 frag_kc(const uint16_t *S, int row0, int kk, int lane) {
  const int row = row0 + (lane & 31), c = (kk * 2 + (lane >> 5)) ^ kc_swizzle<BK>(row);
  return *(const s16x8 *)(S + row * BK + c * 8);
}

// the same fragment from a tile whose rows run along the contraction: two transposing reads; lane i of a group of 16 reads 4 columns
// of row i / 4 and receives 4 rows of column i
template <int COLS>
__device__ __forceinline__ s16x8 frag_kr(const uint16_t *S, int col0, int kk, int lane) {
  const int i = lane & 15, col = col0 + ((lane >> 4) & 1) * 16 + (i & 3) * 4;
  const int k = kk * 16 + (lane >> 5) * 8 + (i >> 2);
  // (k and k + 4 have the same swizzle)
  const uint16_t *p = S + k * COLS + (((col >> 3) ^ kr_swizzle(k)) * 8 + (col & 7));
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + 4 * COLS));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <int T>
__device__ __forceinline__ f32x16 mfma16(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (T == ACT8_F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// 4 codes * 2^e -> 4 values of the 16-bit type (the exponent byte is the exponent field of the instruction's scale)
template <int T>
__device__ __forceinline__ uint2 deq4(uint32_t u, uint32_t eb) {
  const float scale = __uint_as_float(eb << 23);
  if constexpr (T == ACT8_F16) {
    if (eb >= 127 + 8) {                        // 256 * 2^8 is the one value that fp16 does not have: saturate
      float v[4];
      act8_decode4(u, eb, v);
      union { uint2 w; _Float16 h[4]; } r;
#pragma unroll
      for (int k = 0; k < 4; ++k) r.h[k] = (_Float16)(v[k] != v[k] ? v[k] : fminf(fmaxf(v[k], -65504.f), 65504.f));
      return r.w;
    }
    const f16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)u, scale, false);
    const f16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)u, scale, true);
    return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
  } else {
    const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)u, scale, false);
    const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)u, scale, true);
    return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
  }
}

// The ReLU's gradient passes where v, as it is stored, is not <= 0: half the smallest number of the type is rounded to 0 (a nan passes).
template <int T>
__device__ __forceinline__ bool passes(float v) {
  return !(v <= (T == ACT8_F32 ? 0.f : T == ACT8_BF16 ? 0x1p-134f : 0x1p-25f));
}

// three bf16 pieces of two fp32 values each: the leading 8 bits, the next 8, the last 8 (truncated, so that nothing overflows)
__device__ __forceinline__ void split3(float a, float b, uint32_t *p) {
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const uint32_t ua = __float_as_uint(a) & 0xffff0000u, ub = __float_as_uint(b) & 0xffff0000u;
    p[k] = (ua >> 16) | ub;
    a -= __uint_as_float(ua), b -= __uint_as_float(ub);
  }
}

// ---- tile staging ------------------------------------------------------------------------------------------------------
typedef __attribute__((address_space(3))) void *lptr_t;

// 16-bit operand, 16-byte pieces straight from memory into LDS, one BK after the other.  A wave's 64 pieces land side by side; the swizzle is
// in the offset that each lane reads at.  What lies beside the operand (rows of a contraction-contiguous tile, columns of the other kind)
// repeats its last part, and its results are not stored; the contraction behind its end is 0.  (Rows are readable, and 0 along the
// contraction, up to the next multiple of 8 elements: the entry's contract.)  A whole step is exactly H loads.
// Buffer loads: a tile's base is uniform, a lane's offset in it (< 2^31 bytes, checked by the entry) the same in every step.  (The global form of
// these loads makes the compiler wait for all LDS reads under way before each matrix instruction.)
constexpr int BUFFER_WORD3 = 0x00027000;         // untyped 32-bit data

template <bool ALONG_K, int SIDE, int BK, int THREADS>
struct Stager {
  static constexpr int H = SIDE * BK / 8 / THREADS;
  const uint16_t *base;
  long long step;                // elements from one step's tile to the next
  uint32_t at[H];                // bytes from the base
  int k[H];                      // where piece h lies along the contraction, from the step's begin on

  __device__ __forceinline__ void start(const uint16_t *P, long long ld, int side0, int side, int k0, int tid) {
    base = P + (ALONG_K ? k0 * ld + side0 : side0 * ld + k0);
    step = ALONG_K ? BK * ld : BK;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int i = tid + THREADS * h;
      if (!ALONG_K) {
        const int row = i / (BK / 8);
        k[h] = 8 * ((i % (BK / 8)) ^ kc_swizzle<BK>(row));
        at[h] = 2 * ((uint32_t)min(row, side - 1 - side0) * (uint32_t)ld + k[h]);
      } else {
        k[h] = i / (SIDE / 8);
        const int c = (i % (SIDE / 8)) ^ kr_swizzle(k[h]);
        at[h] = 2 * ((uint32_t)k[h] * (uint32_t)ld + min(8 * c, ((side - side0 + 7) & ~7) - 8));
      }
    }
  }

  // left: what is left of the contraction at this step's begin
  __device__ __forceinline__ void issue(uint16_t *S, int wave, int left) {
#ifdef __HIP_DEVICE_COMPILE__                       // (the host pass has no type for a buffer descriptor)
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, 0x7fffffff, BUFFER_WORD3);
    base += step;
    if (left >= BK) {
#pragma unroll
      for (int h = 0; h < H; ++h)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lptr_t)(S + (size_t)(wave * 64 + THREADS * h) * 8), 16, at[h], 0, 0, 0);
    } else {
#pragma unroll
      for (int h = 0; h < H; ++h) {
        uint16_t *d = S + (size_t)(wave * 64 + THREADS * h) * 8;
        if (k[h] < left) __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lptr_t)d, 16, at[h], 0, 0, 0);
        else *(uint4 *)(d + 8 * (threadIdx.x & 63)) = make_uint4(0, 0, 0, 0);
      }
    }
#endif
  }
};

// The same through registers, for rows at any address: 8 elements a thread, any alignment, nothing read behind a row's end.
template <int T, bool ALONG_K, int SIDE, int BK, int THREADS>
struct RowRegs {
  static constexpr int H = SIDE * BK / 8 / THREADS;
  Act8Raw<T> r[H];

  __device__ __forceinline__ void fetch(const uint16_t *P, long long ld, int side0, int side, int k0, int k_hi, int tid) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int i = tid + THREADS * h;
      if (!ALONG_K) {
        const int row = side0 + i / (BK / 8), k = k0 + 8 * (i % (BK / 8));
        r[h] = act8_load_raw<T>(P, (size_t)((long long)row * ld + k), row < side ? k_hi - k : 0);
      } else {
        const int k = k0 + i / (SIDE / 8), c = side0 + 8 * (i % (SIDE / 8));
        r[h] = act8_load_raw<T>(P, (size_t)((long long)k * ld + c), k < k_hi ? side - c : 0);
      }
    }
  }

  __device__ __forceinline__ void put(uint16_t *S, int tid) const {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int i = tid + THREADS * h, row = ALONG_K ? i / (SIDE / 8) : i / (BK / 8);
      const int c = ALONG_K ? (i % (SIDE / 8)) ^ kr_swizzle(row) : (i % (BK / 8)) ^ kc_swizzle<BK>(row);
      *(act8_u32x4 *)(S + row * (ALONG_K ? SIDE : BK) + c * 8) = r[h].w[0];
    }
  }
};

// 8-bit operand: 16 codes of a row at a time through registers
template <int COLS, int BK, int THREADS>
struct CodeRegs {
  static constexpr int H = COLS * BK / 16 / THREADS;
  uint4 u[H];
  uint32_t e[H];
};

template <int COLS, int BK, int THREADS>
__device__ __forceinline__ void fetch_codes(CodeRegs<COLS, BK, THREADS> &t, const uint8_t *P, const uint8_t *E, long long ld, int n0,
                                            int k0, int k_hi, int tid) {
#pragma unroll
  for (int h = 0; h < CodeRegs<COLS, BK, THREADS>::H; ++h) {
    const int i = tid + THREADS * h, k = k0 + i / (COLS / 16), c = n0 + 16 * (i % (COLS / 16));
    t.u[h] = make_uint4(0, 0, 0, 0), t.e[h] = 127;
    if (k < k_hi && c < ld) {
      t.u[h] = *(const uint4 *)(P + (long long)k * ld + c);
      t.e[h] = E[(long long)k * (ld / 32) + c / 32];
    }
  }
}

template <int T, int COLS, int BK, int THREADS>
__device__ __forceinline__ void store_codes(const CodeRegs<COLS, BK, THREADS> &t, uint16_t *S, int tid) {
#pragma unroll
  for (int h = 0; h < CodeRegs<COLS, BK, THREADS>::H; ++h) {
    const int i = tid + THREADS * h, r = i / (COLS / 16), c = 2 * (i % (COLS / 16)), z = kr_swizzle(r);
    const uint2 a = deq4<T>(t.u[h].x, t.e[h]), b = deq4<T>(t.u[h].y, t.e[h]), d = deq4<T>(t.u[h].z, t.e[h]), f = deq4<T>(t.u[h].w, t.e[h]);
    *(uint4 *)(S + r * COLS + ((c ^ z) * 8)) = make_uint4(a.x, a.y, b.x, b.y);
    *(uint4 *)(S + r * COLS + (((c + 1) ^ z) * 8)) = make_uint4(d.x, d.y, f.x, f.y);
  }
}

// fp32 operand: 8 elements at a time through registers, three planes in LDS
template <int ROWS, int BK, int THREADS>
struct F32Regs {
  static constexpr int H = ROWS * BK / 8 / THREADS;
  float v[H][8];
};

template <bool ALONG_K, int ROWS, int BK, int THREADS>
__device__ __forceinline__ void fetch_f32(F32Regs<ROWS, BK, THREADS> &t, const float *P, long long ld, int row0, int rows, int k0, int k_hi,
                                          int tid) {
#pragma unroll
  for (int h = 0; h < F32Regs<ROWS, BK, THREADS>::H; ++h) {
    const int i = tid + THREADS * h;
    int n;                                    // elements of this piece that exist
    long long at;
    if (!ALONG_K) {
      const int row = row0 + i / (BK / 8), k = k0 + 8 * (i % (BK / 8));
      n = row < rows ? k_hi - k : 0;
      at = (long long)row * ld + k;
    } else {
      const int k = k0 + i / (ROWS / 8), row = row0 + 8 * (i % (ROWS / 8));
      n = k < k_hi ? rows - row : 0;
      at = (long long)k * ld + row;
    }
    act8_load8<ACT8_F32>(P, (size_t)at, n, t.v[h]);
  }
}

template <bool ALONG_K, int ROWS, int BK, int THREADS>
__device__ __forceinline__ void store_f32(const F32Regs<ROWS, BK, THREADS> &t, uint16_t *S, int tid) {
#pragma unroll
  for (int h = 0; h < F32Regs<ROWS, BK, THREADS>::H; ++h) {
    const int i = tid + THREADS * h;
    int at;
    if (!ALONG_K) {
      const int r = i / (BK / 8);
      at = r * BK + ((i % (BK / 8)) ^ kc_swizzle<BK>(r)) * 8;
    } else {
      const int r = i / (ROWS / 8);
      at = r * ROWS + ((i % (ROWS / 8)) ^ kr_swizzle(r)) * 8;
    }
    uint32_t p[4][3];
#pragma unroll
    for (int k = 0; k < 4; ++k) split3(t.v[h][2 * k], t.v[h][2 * k + 1], p[k]);
#pragma unroll
    for (int q = 0; q < 3; ++q) *(uint4 *)(S + q * ROWS * BK + at) = make_uint4(p[0][q], p[1][q], p[2][q], p[3][q]);
  }
}

// ---- tile order and epilogue -------------------------------------------------------------------------------------------
struct Tile {
  int m, n, split;
};

// workgroup ids go round-robin over the 8 XCDs (each with its own L2): an XCD gets consecutive logical tiles, and those go
// down 8 tile rows at a time, so that the tiles in flight on one XCD share rows of A and columns of B
__device__ __forceinline__ bool tile_of(const A8Args &a, Tile *t) {
  const int logical = (int)(blockIdx.x % 8) * a.per_xcd + (int)(blockIdx.x / 8), tiles = a.tiles_m * a.tiles_n;
  if (logical >= tiles * a.splits) return false;
  t->split = logical / tiles;
  const int i = logical - t->split * tiles, band = i / (8 * a.tiles_n), m_lo = band * 8, high = min(8, a.tiles_m - m_lo);
  const int j = i - band * 8 * a.tiles_n;
  t->m = m_lo + j % high, t->n = j / high;
  return true;
}

// 4 neighbouring elements of row m from n on
template <int T>
__device__ __forceinline__ void put4(const A8Args &a, int m, int n, const float *v) {
  const size_t at = (size_t)m * a.N + n;
  if (a.vec_c && n + 3 < a.N) {
    if constexpr (T == ACT8_F32) *(float4 *)((float *)a.C + at) = make_float4(v[0], v[1], v[2], v[3]);
    else {
      union { uint2 w; uint16_t h[4]; } u;
#pragma unroll
      for (int k = 0; k < 4; ++k) act8_put<T>(u.h, k, v[k]);
      *(uint2 *)((uint16_t *)a.C + at) = u.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (n + k < a.N) act8_put<T>(a.C, at + k, v[k]);
  }
}

// 32 rows x 64 columns of a wave's results, from row m0 and column n0 on.  They go through LDS, 32 x 68 floats of the wave's own, so that
// 8 lanes write 64 neighbouring elements of a row: straight from the accumulators an instruction would write 16 bytes in each of 32 rows
// (4 096 x 4 096 bf16 results of a product over 64: 46 us, this way 14).
constexpr int EPI_PITCH = 68, EPI_FLOATS = 32 * EPI_PITCH;

template <int T>
__device__ __forceinline__ void store_rows(const A8Args &a, const Tile &t, const f32x16 &left, const f32x16 &right, float *S, const float *bias,
                                           int m0, int n0, int lane) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float *d = S + (lane & 31) * EPI_PITCH + 8 * q + 4 * (lane >> 5);
    *(float4 *)d = make_float4(left[4 * q], left[4 * q + 1], left[4 * q + 2], left[4 * q + 3]);
    *(float4 *)(d + 32) = make_float4(right[4 * q], right[4 * q + 1], right[4 * q + 2], right[4 * q + 3]);
  }
  __builtin_amdgcn_wave_barrier();
  const int n = n0 + 8 * (lane & 7);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int m = m0 + 8 * r + (lane >> 3);
    const float *p = S + (8 * r + (lane >> 3)) * EPI_PITCH + 8 * (lane & 7);
    const float4 lo = *(const float4 *)p, hi = *(const float4 *)(p + 4);
    float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    const int left_n = m < a.M ? a.N - n : 0;
    if (a.splits > 1) {
      act8_store8<ACT8_F32>(a.part, ((size_t)t.split * a.M + m) * a.N + n, left_n, v);
      continue;
    }
    uint32_t word = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] += bias[k];
      if (passes<T>(v[k])) word |= 1u << k;
      if (a.relu) v[k] = v[k] < 0.f ? 0.f : v[k];            // (a nan stays one)
    }
    act8_store8<T>(a.C, (size_t)m * a.N + n, left_n, v);
    if (a.bits) {
      word <<= 8 * (lane & 3);
      word |= __shfl_xor(word, 1), word |= __shfl_xor(word, 2);
      if ((lane & 3) == 0 && left_n > 0) a.bits[(size_t)m * ((a.N + 31) / 32) + n / 32] = word;
    }
  }
  __builtin_amdgcn_wave_barrier();
}

// the bias of the 8 columns that a lane writes
template <int T>
__device__ __forceinline__ void load_bias(const A8Args &a, int n0, int lane, float *v) {
  const int n = n0 + 8 * (lane & 7);
  if (a.bias && a.splits == 1) act8_load8<T>(a.bias, n, a.N - n, v);
  else
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.f;
}

// ---- the 16-bit product --------------------------------------------------------------------------------------------------
// STAGES tiles of BK in LDS.  Fragments are read one group of 16 of the contraction ahead of the matrix instructions, also across the border of
// two steps: before a step's last group is multiplied, the wave waits for its own loads of the next step (all but those issued after
// them) and for its last fragments, and meets the others at the barrier.  Behind it the next tile is complete, and nobody reads this step's
// any more: the loads of step s + STAGES go there.
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (15 << 8) | (7 << 4));       // vmcnt(N)
}

// (Builtins and not inline assembly: the compiler then knows that no scalar load is pending either, and waits for the fragments that it
// needs instead of for all that are under way.)
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));                                 // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <int T>
__device__ __forceinline__ float add8(s16x8 v, float acc) {          // acc + the sum of 8 values
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (T == ACT8_F16) {
      const f16x2 x = {__builtin_bit_cast(f16x8, v)[2 * k], __builtin_bit_cast(f16x8, v)[2 * k + 1]}, one = {(_Float16)1.f, (_Float16)1.f};
      acc = __builtin_amdgcn_fdot2(x, one, acc, false);
    } else {
      const __bf16 b1 = (__bf16)1.f;
      const bf16x2 x = {__builtin_bit_cast(bf16x8, v)[2 * k], __builtin_bit_cast(bf16x8, v)[2 * k + 1]}, one = {b1, b1};
      acc = __builtin_amdgcn_fdot2_f32_bf16(x, one, acc, false);
    }
  }
  return acc;
}

// row sums (form 2): lane -> column m0 + (lane & 31) of A, half of the contraction each
template <int T>
__device__ __forceinline__ void store_sum(const A8Args &a, const Tile &t, float v, int m0, int lane) {
  v += __shfl_xor(v, 32);
  const int m = m0 + lane;
  if (lane >= 32 || m >= a.M) return;
  if (a.splits > 1) a.part[(size_t)a.splits * a.M * a.N + (size_t)t.split * a.M + m] = v;
  else act8_put<T>(a.rowsum, m, v);
}

// REGS: operands at any address, through registers.  WK groups of WM x WN waves share a tile: each multiplies its part of every step's
// contraction, and they add up at the end.
// Large products are bound by the matrix instructions and the clock that they leave (8 192^3 bf16, forms 0 / 1 / 2: 1 211 / 1 170 / 1 004 TFLOP/s, the
// library's plain product 1 357 to 1 550; 16 384 x 4 096 x 4 096: 464 / 509 / 558 us = 1 184 / 1 080 / 985).  Form 2 pays for its transposed reads and for
// the codes' way through registers.  Small ones are bound by the loads' latency over a few steps: 777 x 1 001 x 515 fp16 13 / 14 / 17 us.
template <int T, int FORM, int WM, int WN, int FM, int FN, int BK, int STAGES, int WK, bool REGS>
__global__ __launch_bounds__(64 * WM * WN * WK, 2) void a8_gemm16_kernel(A8Args a) {
  constexpr int BM = WM * FM * 32, BN = WN * FN * 32, THREADS = 64 * WM * WN * WK, STAGE = (BM + BN) * BK;
  extern __shared__ __attribute__((aligned(16))) uint16_t a8_lds[];      // [STAGES][A tile, B tile]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wk = wave / (WM * WN),
            wm = wave % (WM * WN) / WN, wn = wave % WN;
  Tile t;
  if (!tile_of(a, &t)) return;
  const int m0 = t.m * BM, n0 = t.n * BN;
  const int s_lo = t.split * a.steps_per_split, s_hi = min((a.K + BK - 1) / BK, s_lo + a.steps_per_split);
  f32x16 acc[FM][FN];
  float sum[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    sum[i] = 0.f;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  }
  typedef Stager<FORM == 2, BM, BK, THREADS> SA;
  typedef Stager<FORM == 1, BN, BK, THREADS> SB;
  SA sa;
  SB sb;
  RowRegs<T, FORM == 2, BM, BK, THREADS> ra;
  RowRegs<T, FORM == 1, BN, BK, THREADS> rb;
  CodeRegs<BN, BK, THREADS> codes;
  constexpr int LOADS = REGS ? 0 : SA::H + (FORM == 2 ? 0 : SB::H);
  if constexpr (!REGS) {
    sa.start((const uint16_t *)a.A, a.lda, m0, a.M, s_lo * BK, tid);
    if constexpr (FORM != 2) sb.start((const uint16_t *)a.B, a.ldb, n0, a.N, s_lo * BK, tid);
  }

  // what goes through registers: fetched one step before put stores it
  auto fetch = [&](int s) {
    if constexpr (REGS) {
      ra.fetch((const uint16_t *)a.A, a.lda, m0, a.M, s * BK, a.K, tid);
      if constexpr (FORM != 2) rb.fetch((const uint16_t *)a.B, a.ldb, n0, a.N, s * BK, a.K, tid);
    }
    if constexpr (FORM == 2) fetch_codes<BN, BK, THREADS>(codes, (const uint8_t *)a.B, a.exps, a.ldb, n0, s * BK, a.K, tid);
  };
  auto issue = [&](int s, int buf) {
    if constexpr (!REGS) {
      sa.issue(a8_lds + buf * STAGE, wave, a.K - s * BK);
      if constexpr (FORM != 2) sb.issue(a8_lds + buf * STAGE + BM * BK, wave, a.K - s * BK);
    }
  };
  auto put = [&](int buf) {
    if constexpr (REGS) {
      ra.put(a8_lds + buf * STAGE, tid);
      if constexpr (FORM != 2) rb.put(a8_lds + buf * STAGE + BM * BK, tid);
    }
    if constexpr (FORM == 2) store_codes<T, BN, BK, THREADS>(codes, a8_lds + buf * STAGE + BM * BK, tid);
  };

  const int steps = s_hi - s_lo;
#pragma unroll
  for (int i = 0; i < STAGES; ++i) {
    if (i < steps) {
      fetch(s_lo + i);
      issue(s_lo + i, i);
      if (i < STAGES - 1) put(i);                    // (the last ones wait in registers)
    }
  }
  constexpr int KK = BK / 16 / WK;                         // groups of 16 that a wave multiplies of a step
  static_assert(KK % 2 == 0, "a fragment set's index is a constant in the unrolled loops");
  s16x8 fa[2][FM], fb[2][FN];
  auto read = [&](int buf, int kk) {                       // kk == KK: the first of the tile in buf
    const int set = kk % 2;
    kk = wk * KK + kk % KK;
    const uint16_t *As = a8_lds + buf * STAGE, *Bs = As + BM * BK;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      if constexpr (FORM == 2) fa[set][i] = frag_kr<BM>(As, (wm * FM + i) * 32, kk, lane);
      else fa[set][i] = frag_kc<BK>(As, (wm * FM + i) * 32, kk, lane);
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      if constexpr (FORM == 0) fb[set][j] = frag_kc<BK>(Bs, (wn * FN + j) * 32, kk, lane);
      else fb[set][j] = frag_kr<BN>(Bs, (wn * FN + j) * 32, kk, lane);
    }
  };
  if (steps > 0) {
    if (steps > STAGES) wait_loads<LOADS * (STAGES - 1)>();    // (the very last step may be less than LOADS)
    else wait_loads<0>();
    meet();
    read(0, 0);
  }
  auto loop = [&](auto with_sums) {                        // (one branch outside of the loop: a branch inside keeps instructions from mixing)
    auto multiply = [&](int kk) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma16<T>(fb[kk % 2][j], fa[kk % 2][i], acc[i][j]);
      if constexpr (decltype(with_sums)::value) {
#pragma unroll
        for (int i = 0; i < FM; ++i) sum[i] = add8<T>(fa[kk % 2][i], sum[i]);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    int buf = 0, s = 0;
    // steps with STAGES more behind them, without a branch
    for (; s + STAGES < steps; ++s) {
      const int now = buf, before = now == 0 ? STAGES - 1 : now - 1;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if (kk == KK - 1) {             // the last fragments of this tile are under way: the border
          buf = buf + 1 == STAGES ? 0 : buf + 1;
          put(before);            // what arrived during this step belongs to step s + STAGES - 1, in the buffer of the step before this one
          wait_loads<LOADS * (STAGES - 2)>();
          meet();
        }
        read(buf, kk + 1);
        if (kk == KK - 1) {
          fetch(s_lo + s + STAGES);
          issue(s_lo + s + STAGES, now);
        }
        multiply(kk);
      }
    }
    for (; s < steps; ++s) {
      const int before = buf == 0 ? STAGES - 1 : buf - 1;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if (kk == KK - 1 && s + 1 < steps) {
          buf = buf + 1 == STAGES ? 0 : buf + 1;
          if (s + STAGES == steps) put(before);
          wait_loads<0>();              // (fewer loads behind the next step's than in the middle: wait for all)
          meet();
        }
        if (kk < KK - 1 || s + 1 < steps) read(buf, kk + 1);
        multiply(kk);
      }
    }
  };
  const bool sums = FORM == 2 && a.rowsum && t.n == 0 && wn == 0;
  if constexpr (FORM == 2) {
    if (sums) loop(std::true_type{});
    else loop(std::false_type{});
  } else loop(std::false_type{});
  static_assert(FN == 2, "store_rows takes two blocks side by side");
  __syncthreads();                                         // the tiles have been read: their place is free
  float *S = (float *)a8_lds;
  if constexpr (WK == 2) {
    // Each group stores half of the rows: it gives the other half's sums away, [wave of the group][FM / 2][FN][16][lane].
    static_assert(FM % 2 == 0 && WK * WM * WN * (FM / 2) * (FN * 16 + 1) * 64 * 4 <= STAGES * STAGE * 2, "");
    constexpr int EACH = (FM / 2) * (FN * 16 + 1) * 64;
    float *give = S + wave * EACH + lane, *take = S + (wave ^ (WM * WN)) * EACH + lane;
#pragma unroll
    for (int i = 0; i < FM / 2; ++i) {
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) give[((i * FN + j) * 16 + r) * 64] = wk ? acc[i][j][r] : acc[FM / 2 + i][j][r];
      give[((FM / 2) * FN * 16 + i) * 64] = wk ? sum[i] : sum[FM / 2 + i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FM / 2; ++i) {
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float v = take[((i * FN + j) * 16 + r) * 64];
          acc[i][j][r] = wk ? v + acc[FM / 2 + i][j][r] : acc[i][j][r] + v;      // (group 0 + group 1)
        }
      const float v = take[((FM / 2) * FN * 16 + i) * 64];
      sum[i] = wk ? v + sum[FM / 2 + i] : sum[i] + v;
    }
    __syncthreads();
  }
  float bias[8];
  load_bias<T>(a, n0 + wn * 64, lane, bias);
#pragma unroll
  for (int i = 0; i < FM / WK; ++i) {
    const int m = m0 + (wm * FM + wk * (FM / WK) + i) * 32;
    store_rows<T>(a, t, acc[i][0], acc[i][1], S + wave * EPI_FLOATS, bias, m, n0 + wn * 64, lane);
    if (FORM == 2 && sums) store_sum<T>(a, t, sum[i], m, lane);
  }
}

// ---- the fp32 product ----------------------------------------------------------------------------------------------------
// 128 x 128 tile, 4 waves of 64 x 64, 32 of the contraction at a time; the next step's operands are in registers while this
// one's planes are multiplied.  Bound by matrix instructions and the cutting beside them: 1 999 x 12 544 -> 1 024, forms 0 / 1 / 2: 274 / 309 / 206 us,
// 1 124 / 997 / 747 TFLOP/s of bf16 products = 187 / 166 / 249 of fp32 ones (the library's fp32 product: 152); 256 x 27 648 -> 256: 33 / 30 / 20 us.
template <int FORM>
__global__ __launch_bounds__(256, 3) void a8_gemm32_kernel(A8Args a) {
  constexpr int BM = 128, BN = 128, BK = 32, THREADS = 256, FM = 2, FN = 2, PB = FORM == 2 ? 1 : 3;
  extern __shared__ __attribute__((aligned(16))) uint16_t a8_lds[];
  uint16_t *As = a8_lds, *Bs = a8_lds + 3 * BM * BK;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  Tile t;
  if (!tile_of(a, &t)) return;
  const int m0 = t.m * BM, n0 = t.n * BN;
  const int s_lo = t.split * a.steps_per_split, s_hi = min((a.K + BK - 1) / BK, s_lo + a.steps_per_split);
  const bool sums = FORM == 2 && a.rowsum && t.n == 0 && wn == 0;
  f32x16 acc[FM][FN];
  float sum[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    sum[i] = 0.f;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  }
  F32Regs<BM, BK, THREADS> ra;
  F32Regs<BN, BK, THREADS> rb;
  CodeRegs<BN, BK, THREADS> codes;

  auto fetch = [&](int s) {
    fetch_f32<FORM == 2, BM, BK, THREADS>(ra, (const float *)a.A, a.lda, m0, a.M, s * BK, a.K, tid);
    if constexpr (FORM == 2) fetch_codes<BN, BK, THREADS>(codes, (const uint8_t *)a.B, a.exps, a.ldb, n0, s * BK, a.K, tid);
    else fetch_f32<FORM == 1, BN, BK, THREADS>(rb, (const float *)a.B, a.ldb, n0, a.N, s * BK, a.K, tid);
  };

  if (s_lo < s_hi) fetch(s_lo);
  for (int s = s_lo; s < s_hi; ++s) {
    __syncthreads();                                      // the previous step's fragments have been read
    store_f32<FORM == 2, BM, BK, THREADS>(ra, As, tid);
    if constexpr (FORM == 2) store_codes<ACT8_BF16, BN, BK, THREADS>(codes, Bs, tid);
    else store_f32<FORM == 1, BN, BK, THREADS>(rb, Bs, tid);
    __syncthreads();
    if (s + 1 < s_hi) fetch(s + 1);
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) {
      s16x8 fa[3][FM], fb[PB][FN];
#pragma unroll
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          if constexpr (FORM == 2) fa[q][i] = frag_kr<BM>(As + q * BM * BK, (wm * FM + i) * 32, kk, lane);
          else fa[q][i] = frag_kc<BK>(As + q * BM * BK, (wm * FM + i) * 32, kk, lane);
        }
#pragma unroll
      for (int q = 0; q < PB; ++q)
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          if constexpr (FORM >= 1) fb[q][j] = frag_kr<BN>(Bs + q * BN * BK, (wn * FN + j) * 32, kk, lane);
          else fb[q][j] = frag_kc<BK>(Bs + q * BN * BK, (wn * FN + j) * 32, kk, lane);
        }
      // smallest products first
#pragma unroll
      for (int o = 2; o >= 0; --o)
#pragma unroll
        for (int q = 0; q < PB; ++q) {
          if (o - q < 0) continue;
#pragma unroll
          for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = mfma16<ACT8_BF16>(fb[q][j], fa[o - q][i], acc[i][j]);
        }
      if constexpr (FORM == 2) {
        if (sums) {
#pragma unroll
          for (int q = 2; q >= 0; --q)
#pragma unroll
            for (int i = 0; i < FM; ++i) sum[i] = add8<ACT8_BF16>(fa[q][i], sum[i]);
        }
      }
    }
  }
  __syncthreads();                                         // the tiles have been read: their place is free
  float bias[8];
  load_bias<ACT8_F32>(a, n0 + wn * 64, lane, bias);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    store_rows<ACT8_F32>(a, t, acc[i][0], acc[i][1], (float *)a8_lds + wave * EPI_FLOATS, bias, m0 + (wm * FM + i) * 32, n0 + wn * 64, lane);
    if (FORM == 2 && sums) store_sum<ACT8_F32>(a, t, sum[i], m0 + (wm * FM + i) * 32, lane);
  }
}

// ---- partial sums, in a fixed order ---------------------------------------------------------------------------------------
// A thread has 4 neighbouring columns and every SLICES-th part, 4 loads under way at a time; the slices are added in LDS.  Many parts of few
// results are bound by the latency of that chain: 64 parts of 256 x 256 took 19 us one after the other.  The last workgroups take the
// row sums.
template <int T, int SLICES>
__global__ __launch_bounds__(256) void a8_reduce_kernel(A8Args a, int col4, unsigned main_blocks) {
  constexpr int THREADS = 256 / SLICES;
  __shared__ float4 sh[SLICES > 1 ? 256 : 1];
  if (blockIdx.x >= main_blocks) {
    const long long m = (long long)(blockIdx.x - main_blocks) * 256 + threadIdx.x;
    if (m >= a.M) return;
    const float *p = a.part + (size_t)a.splits * a.M * a.N + m;
    float v = 0.f;
    for (int s = 0; s < a.splits; ++s) v += p[(size_t)s * a.M];
    act8_put<T>(a.rowsum, m, v);
    return;
  }
  const int tx = threadIdx.x % THREADS, slice = threadIdx.x / THREADS;
  const long long i = (long long)blockIdx.x * THREADS + tx;
  const int m = (int)(i / col4), n = 4 * (int)(i % col4);     // col4: a multiple of 8 (a word of sign bits is 8 threads)
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (m < a.M && n < a.N) {
    const size_t step = (size_t)a.M * a.N * SLICES;
    const float *p = a.part + ((size_t)slice * a.M + m) * a.N + n;
    const bool whole = a.N % 4 == 0;
    int s = slice;
    if (whole) {
      for (; s + 3 * SLICES < a.splits; s += 4 * SLICES, p += 4 * step) {
        const float4 w0 = *(const float4 *)p, w1 = *(const float4 *)(p + step), w2 = *(const float4 *)(p + 2 * step), w3 = *(const float4 *)(p + 3 * step);
        v[0] += (w0.x + w1.x) + (w2.x + w3.x), v[1] += (w0.y + w1.y) + (w2.y + w3.y);
        v[2] += (w0.z + w1.z) + (w2.z + w3.z), v[3] += (w0.w + w1.w) + (w2.w + w3.w);
      }
    }
    for (; s < a.splits; s += SLICES, p += step) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n + k < a.N) v[k] += p[k];
    }
  }
  if constexpr (SLICES > 1) {
    sh[threadIdx.x] = make_float4(v[0], v[1], v[2], v[3]);
    __syncthreads();
    if (slice) return;
#pragma unroll
    for (int k = 1; k < SLICES; ++k) {
      const float4 w = sh[k * THREADS + tx];
      v[0] += w.x, v[1] += w.y, v[2] += w.z, v[3] += w.w;
    }
  }
  if (m >= a.M) return;
  uint32_t word = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (a.bias && n + k < a.N) v[k] += act8_get<T>(a.bias, n + k);
    if (passes<T>(v[k])) word |= 1u << ((n & 31) + k);
    if (a.relu) v[k] = v[k] < 0.f ? 0.f : v[k];
  }
  put4<T>(a, m, n, v);
  if (a.bits) {
    word |= __shfl_xor(word, 1), word |= __shfl_xor(word, 2), word |= __shfl_xor(word, 4);
    if ((n & 31) == 0 && n < a.N) a.bits[(size_t)m * ((a.N + 31) / 32) + n / 32] = word;
  }
}

// ---- a gradient behind a ReLU / rows moved to a 16-byte pitch --------------------------------------------------------------
// out (rows, ldo) = bits ? (bit set ? x : 0) : x, 0 behind the width; a thread has 8 elements.  Bound by memory: 4 096 x 4 096 bf16 13 us, 5.2 TB/s.
// (Taking the mask inside the products instead would put the gradient through registers there: the direct path to LDS is worth more.)
template <int T>
__global__ __launch_bounds__(256) void a8_mask_kernel(const void *__restrict__ x, long long rows, int width, long long ld,
                                                      const uint32_t *__restrict__ bits, void *__restrict__ out, int ldo) {
  const int chunks = ldo / 8;
  const long long total = rows * chunks;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long r = i / chunks;
    const int c = 8 * (int)(i % chunks);
    float v[8];
    act8_load8<T>(x, (size_t)r * ld + c, width - c, v);
    if (bits && c < width) {
      const uint32_t w = bits[r * ((width + 31) / 32) + c / 32] >> (c & 31);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = (w >> k) & 1 ? v[k] : 0.f;
    }
    act8_store8<T>(out, (size_t)r * ldo + c, 8, v);
  }
}

// Large tiles where there are this many of them: 256 x 256 for forms 0 and 1 (rows of 128 bytes a step: 32 of the contraction read half of each
// 128-byte line at a time, 776 against 863 TFLOP/s at 16 384 x 4 096 x 4 096), 256 x 128 with two workgroups to a compute unit for form 2
// (1 047 TFLOP/s there; the 256 x 256 tile spills: 535).
constexpr int A8_BIG_TILES = 200;

template <int WM_, int WN_, int FM_, int FN_, int BK_, int STAGES_, int WK_>
struct Shape {
  static constexpr int WM = WM_, WN = WN_, FM = FM_, FN = FN_, BK = BK_, STAGES = STAGES_, WK = WK_, BM = WM * FM * 32, BN = WN * FN * 32,
                       THREADS = 64 * WM * WN * WK, TILES = STAGES * (BM + BN) * BK * 2, ROWS = WK * WM * WN * EPI_FLOATS * 4,
                       LDS = TILES > ROWS ? TILES : ROWS;
};
// Fewer results: 128 x 128, 8 waves in two groups that share the contraction (4 096 x 1 024 results of a product over 4 096, us of forms 0 / 1 / 2: 4
// waves and two stages 50 / 66 / 74, 8 waves of 32 x 64 and four stages 41 / 60 / 69, this 41 / 55 / 63).
typedef Shape<2, 2, 2, 2, 64, 4, 2> Small;
typedef Shape<2, 4, 4, 2, 64, 2, 1> BigForward;
typedef Shape<2, 2, 4, 2, 32, 3, 1> BigWeight;

constexpr long long A8_MAX_PITCH = (1ll << 31) / 512 - 8;
// sizes are 32-bit numbers in the kernels, which add a tile's width to them
constexpr int A8_MAX_SIZE = 0x7fffffff - 1023;

struct Plan {
  int big, bm, bn, bk, tiles_m, tiles_n, splits, steps_per_split;
};

Plan a8_plan(int form, int dtype, bool regs, int M, int N, int K) {
  Plan p;
  p.bm = p.bn = 128;
  p.bk = dtype == ACT8_F32 ? 32 : Small::BK;
  p.big = 0;
  if (dtype != ACT8_F32 && !regs) {
    const int bm = form == 2 ? BigWeight::BM : BigForward::BM, bn = form == 2 ? BigWeight::BN : BigForward::BN;
    if ((long long)dm_ceil_div(M, bm) * dm_ceil_div(N, bn) >= A8_BIG_TILES)
      p.big = 1, p.bm = bm, p.bn = bn, p.bk = form == 2 ? BigWeight::BK : BigForward::BK;
  }
  p.tiles_m = dm_ceil_div(M, p.bm), p.tiles_n = dm_ceil_div(N, p.bn);
  const long long tiles = (long long)p.tiles_m * p.tiles_n;
  const int steps = dm_ceil_div(K, p.bk);
  const int fill = dtype == ACT8_F32 ? 512 : 256;                       // workgroups that are resident at once, about
  long long want = p.big || tiles >= 256 ? 1 : (fill + tiles - 1) / tiles;
  // A split has 256 of the contraction at least, and a short contraction is not worth the second kernel (1 024^3 bf16: 13.5 us, split 20; 256 x 2 000
  // x 256 bf16: 20, split 13; through registers, a step's loads are not hidden as well: 777 x 1 001 x 515 fp16 25, split 18, fp32 78 and 31).
  const long long most = K < (dtype == ACT8_F32 || regs ? 512 : 1536) ? 1 : (long long)steps * p.bk / 256;
  if (want > most) want = most;
  if (want > 64) want = 64;
  if (want < 1) want = 1;
  p.steps_per_split = dm_ceil_div(steps, want);
  p.splits = dm_ceil_div(steps, p.steps_per_split);                     // no empty split
  return p;
}

template <int T, int FORM, typename S, bool REGS = false>
int launch16(const A8Args &a, unsigned grid, hipStream_t st) {
  auto k = a8_gemm16_kernel<T, FORM, S::WM, S::WN, S::FM, S::FN, S::BK, S::STAGES, S::WK, REGS>;
  if (S::LDS > 65536) DM_HIP(hipFuncSetAttribute((const void *)k, hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS));
  k<<<grid, S::THREADS, S::LDS, st>>>(a);
  DM_CHECK_LAUNCH();
  return DM_OK;
}

template <int T>
int launch16(int form, bool regs, const A8Args &a, const Plan &p, unsigned grid, hipStream_t st) {
  if (regs)
    return form == 0 ? launch16<T, 0, Small, true>(a, grid, st) : form == 1 ? launch16<T, 1, Small, true>(a, grid, st) : launch16<T, 2, Small, true>(a, grid, st);
  if (form == 0) return p.big ? launch16<T, 0, BigForward>(a, grid, st) : launch16<T, 0, Small>(a, grid, st);
  if (form == 1) return p.big ? launch16<T, 1, BigForward>(a, grid, st) : launch16<T, 1, Small>(a, grid, st);
  return p.big ? launch16<T, 2, BigWeight>(a, grid, st) : launch16<T, 2, Small>(a, grid, st);
}

template <int FORM>
int launch32(const A8Args &a, unsigned grid, hipStream_t st) {
  constexpr size_t tiles = (size_t)(3 * 128 * 32 + (FORM == 2 ? 1 : 3) * 128 * 32) * 2, rows = (size_t)4 * EPI_FLOATS * sizeof(float);
  a8_gemm32_kernel<FORM><<<grid, 256, tiles > rows ? tiles : rows, st>>>(a);
  DM_CHECK_LAUNCH();
  return DM_OK;
}

template <int T>
int reduce(const A8Args &a, hipStream_t st) {
  const int col4 = dm_ceil_div(a.N, 32) * 8, threads = a.splits >= 8 ? 64 : 256;
  const long long main_blocks = ((long long)a.M * col4 + threads - 1) / threads, more = a.rowsum ? (a.M + 255) / 256 : 0;
  if (threads == 64) a8_reduce_kernel<T, 4><<<(unsigned)(main_blocks + more), 256, 0, st>>>(a, col4, (unsigned)main_blocks);
  else a8_reduce_kernel<T, 1><<<(unsigned)(main_blocks + more), 256, 0, st>>>(a, col4, (unsigned)main_blocks);
  DM_CHECK_LAUNCH();
  return DM_OK;
}

}  // namespace

// rows that 16-byte loads straight into LDS fit: every address a multiple of 16, a tile's 256 rows less than 2^31 bytes; `whole`: no row ends inside
// of a 16-byte piece, or (padded) what is behind its end may be read
static bool a8_direct(const void *p, long long ld, int whole, int padded) {
  return ld % 8 == 0 && ld <= A8_MAX_PITCH && ((uintptr_t)p & 15) == 0 && (padded || whole % 8 == 0);
}

static bool a8_regs(int form, int dtype, const void *A, long long lda, const void *B, long long ldb, int padded, int M, int N, int K) {
  if (dtype == ACT8_F32) return false;
  return !a8_direct(A, lda, form == 2 ? M : K, padded & 1) || (form != 2 && !a8_direct(B, ldb, form == 0 ? K : N, padded & 2));
}

extern "C" size_t dm_act8_gemm_workspace_bytes(int form, int dtype, const void *A, long long lda, const void *B, long long ldb, int padded, int M,
                                               int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || M > A8_MAX_SIZE || N > A8_MAX_SIZE || K > A8_MAX_SIZE) return 0;
  const Plan p = a8_plan(form, dtype, a8_regs(form, dtype, A, lda, B, ldb, padded, M, N, K), M, N, K);
  return p.splits > 1 ? dm_align(((size_t)p.splits * M * N + (form == 2 ? (size_t)p.splits * M : 0)) * sizeof(float)) : 0;
}

extern "C" int dm_act8_gemm(int form, int dtype, const void *A, long long lda, const void *B, long long ldb, int padded, const uint8_t *exps,
                            const void *bias, int relu, int M, int N, int K, void *C, uint32_t *sign_bits, void *rowsum,
                            void *workspace, size_t workspace_bytes, dm_stream_t stream) {
  hipStream_t st = (hipStream_t)stream;
  if (form < 0 || form > 2 || dtype < ACT8_F32 || dtype > ACT8_F16 || M <= 0 || N <= 0 || K <= 0 || !A || !B || !C)
    return DM_ERR_INVALID_ARG;
  if (M > A8_MAX_SIZE || N > A8_MAX_SIZE || K > A8_MAX_SIZE) return DM_ERR_INVALID_ARG;
  if ((form == 2) != (exps != nullptr) || (form != 2 && rowsum) || (form == 2 && (bias || relu || sign_bits))) return DM_ERR_INVALID_ARG;
  if (lda < (form == 2 ? M : K) || ldb < (form == 0 ? K : N)) return DM_ERR_INVALID_ARG;
  if (form == 2 && (ldb % 32 || ((uintptr_t)B & 15))) return DM_ERR_INVALID_ARG;
  const bool regs = a8_regs(form, dtype, A, lda, B, ldb, padded, M, N, K);
  const Plan p = a8_plan(form, dtype, regs, M, N, K);
  A8Args a = {};
  a.A = A, a.B = B, a.bias = bias, a.exps = exps, a.C = C, a.bits = sign_bits, a.rowsum = rowsum;
  a.M = M, a.N = N, a.K = K, a.lda = lda, a.ldb = ldb, a.relu = relu;
  a.splits = p.splits, a.steps_per_split = p.steps_per_split, a.tiles_m = p.tiles_m, a.tiles_n = p.tiles_n;
  a.vec_c = N % 4 == 0 && ((uintptr_t)C & 15) == 0;
  if (p.splits > 1) {
    if (!workspace || workspace_bytes < dm_act8_gemm_workspace_bytes(form, dtype, A, lda, B, ldb, padded, M, N, K)) return DM_ERR_WORKSPACE;
    a.part = (float *)workspace;
  }
  const long long total = (long long)p.tiles_m * p.tiles_n * p.splits;
  if (total > 0x3fffffff || (long long)M * (dm_ceil_div(N, 32) * 8) / 64 > 0x7ffffff0) return DM_ERR_INVALID_ARG;
  a.per_xcd = (int)((total + 7) / 8);
  const unsigned grid = (unsigned)a.per_xcd * 8;
  int rc;
  if (dtype == ACT8_F32) rc = form == 0 ? launch32<0>(a, grid, st) : form == 1 ? launch32<1>(a, grid, st) : launch32<2>(a, grid, st);
  else rc = dtype == ACT8_BF16 ? launch16<ACT8_BF16>(form, regs, a, p, grid, st) : launch16<ACT8_F16>(form, regs, a, p, grid, st);
  if (rc != DM_OK || p.splits == 1) return rc;
  return dtype == ACT8_F32 ? reduce<ACT8_F32>(a, st) : dtype == ACT8_BF16 ? reduce<ACT8_BF16>(a, st) : reduce<ACT8_F16>(a, st);
}

extern "C" int dm_act8_mask_rows(const void *x, int dtype, long long rows, int width, long long ld, const uint32_t *sign_bits, void *out,
                                 int ldo, dm_stream_t stream) {
  if (dtype < ACT8_F32 || dtype > ACT8_F16 || rows < 0 || width <= 0 || ld < width || ldo < width || ldo % 8 || ldo > A8_MAX_SIZE) return DM_ERR_INVALID_ARG;
  if (rows == 0) return DM_OK;
  if (!x || !out || ((uintptr_t)out & 15)) return DM_ERR_INVALID_ARG;
  const long long blocks = (rows * (ldo / 8) + 255) / 256;
  const unsigned grid = (unsigned)(blocks < 65536 ? blocks : 65536);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == ACT8_F32) a8_mask_kernel<ACT8_F32><<<grid, 256, 0, st>>>(x, rows, width, ld, sign_bits, out, ldo);
  else if (dtype == ACT8_BF16) a8_mask_kernel<ACT8_BF16><<<grid, 256, 0, st>>>(x, rows, width, ld, sign_bits, out, ldo);
  else a8_mask_kernel<ACT8_F16><<<grid, 256, 0, st>>>(x, rows, width, ld, sign_bits, out, ldo);
  DM_CHECK_LAUNCH();
  return DM_OK;
}
