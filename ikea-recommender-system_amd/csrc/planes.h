// Matrices in LDS as bf16 planes, for v_mfma_f32_16x16x32_bf16 (csrc/delta.hip).
//
// An fp32 value is kept as N bf16 planes x = x0 + x1 (+ x2), largest first; bf16 inputs are one plane, exactly.  A matrix
// of R x C values (C a multiple of 32) stores its rows with 8 values of padding and, inside each block of 32
// columns, in the order in which two 16x16 accumulator tiles hold 32 rows: column 16·hi + 4·kg + i at place
// 8·kg + 4·hi + i.  So one 16-byte read gives a lane its 8 values of a 32-deep contraction, in the same order
// in which a pair of accumulators (rows 4·kg + i of either tile) gives them, and accumulators feed the next
// product without leaving their registers.  With the contraction along the rows instead, ds_read_b64_tr_b16 transposes
// on the way: 16 lanes fetch 4 rows x 16 columns and lane j receives column j.
#pragma once
#include "common.h"

typedef short pl_s4 __attribute__((ext_vector_type(4)));
typedef short pl_s8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ int pl_place(int c) {
  return (c & ~31) | ((c & 12) << 1) | ((c & 16) >> 2) | (c & 3);
}

template <int R, int C, int N>
struct PlaneMat {
  static constexpr int LD = C + 8, PLANE = R * LD, BYTES = N * PLANE * 2;
  __bf16* p;
  // contraction along the columns: rows r0 + (lane & 15), columns 32·kb ..
  __device__ __forceinline__ void row(bf16x8* f, int r0, int kb) const {
    const int l = threadIdx.x & 63;
    const __bf16* a = p + (r0 + (l & 15)) * LD + 32 * kb + 8 * (l >> 4);
#pragma unroll
    for (int q = 0; q < N; ++q) f[q] = *reinterpret_cast<const bf16x8*>(a + q * PLANE);
  }
  // contraction along the rows 32·kb ..: columns c0 + (lane & 15), c0 a multiple of 16
  __device__ __forceinline__ void col(bf16x8* f, int kb, int c0) const {
    const int l = threadIdx.x & 63, j = l & 15;
    __bf16* a = p + (32 * kb + 4 * (l >> 4) + (j >> 2)) * LD + (c0 & ~31) + 8 * (j & 3) + ((c0 >> 2) & 4);
#pragma unroll
    for (int q = 0; q < N; ++q) {
      pl_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pl_s4*)(a + q * PLANE));
      pl_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) pl_s4*)(a + q * PLANE + 16 * LD));
      const pl_s8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      f[q] = __builtin_bit_cast(bf16x8, v);
    }
  }
  // 8 consecutive columns c .. c + 7 (c a multiple of 8)
  __device__ __forceinline__ void put8(int r, int c, const bf16x8* v) const {
    __bf16* a = p + r * LD + pl_place(c);
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const pl_s8 s = __builtin_bit_cast(pl_s8, v[q]);
      *reinterpret_cast<pl_s4*>(a + q * PLANE) = (pl_s4){s[0], s[1], s[2], s[3]};
      *reinterpret_cast<pl_s4*>(a + q * PLANE + 8) = (pl_s4){s[4], s[5], s[6], s[7]};
    }
  }
};

// 8 fp32 values -> N planes, round to nearest even each
template <int N>
__device__ __forceinline__ void pl_split(const f4& lo, const f4& hi, bf16x8* p) {
  if constexpr (N == 3) {
    split3x8_pair(lo, hi, p[0], p[1], p[2]);
  } else {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    typedef float fl2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float xa = i < 2 ? lo[2 * i] : hi[2 * i - 4], xb = i < 2 ? lo[2 * i + 1] : hi[2 * i - 3];
      const bf2 b0 = __builtin_convertvector((fl2){xa, xb}, bf2);
      p[0][2 * i] = b0.x;
      p[0][2 * i + 1] = b0.y;
      if constexpr (N == 2) {
        const uint32_t u0 = __builtin_bit_cast(uint32_t, b0);
        const bf2 b1 = __builtin_convertvector(
            (fl2){xa - __uint_as_float(u0 << 16), xb - __uint_as_float(u0 & 0xFFFF0000u)}, bf2);
        p[1][2 * i] = b1.x;
        p[1][2 * i + 1] = b1.y;
      }
    }
  }
}

// c += a·b over the plane products with p + q below the larger plane count, smallest first
template <int NA, int NB>
__device__ __forceinline__ f4 pl_mm(const bf16x8* a, const bf16x8* b, f4 c) {
  constexpr int T = NA > NB ? NA : NB;
#pragma unroll
  for (int s = T - 1; s >= 0; --s)
#pragma unroll
    for (int p = s; p >= 0; --p)
      if (p < NA && s - p < NB) c = mfma16bf(a[p], b[s - p], c);
  return c;
}
