// Item scores from a 4-bit item table: y[m, n] = Σ_k x[m, k]·s[n, k/G]·(c[n, k] − 8) + bias[n],
// c four-bit codes (two a byte, the even k in the low half), s one bf16 scale per G = 32 / 64 / 128 codes of an item.
//
// Bound: the table's bytes (N·K/2 codes and 2·N·K/G scales, each read once) and, for many rows, the M·N fp32 scores
// written.  The products run on v_mfma_f32_16x16x32_bf16 with x as the A operand (its 16 rows are sessions) and 16 items
// as B, so that a lane belongs to one item: its scale multiplies the lane's four accumulators once per group, in
// fp32.  A code enters the MFMA exactly, as the bf16 value 16 + c (its bits are 0x4180 | c << 3: one shift and one
// and-or for two codes); the offset 24 goes into the accumulator's start, −24·Σ x of the group, itself an MFMA
// against a constant.  (128 + c would save a shift, but then the sums carry 30 times the result's size and lose five
// bits.)  fp32 x is split into three bf16 planes, whose products are exact; the first plane's sums, eight-bit values times
// small integers, are as good as exact, and the other planes', 2^-8 as large, run beside them and join at a group's
// end: in one chain their low bits would be rounded at the size of 24·Σ x (1.3e-6 of the result instead of 1e-7).
//
// Infinities would meet their own negative in that offset, and values from 2^96 on could leave fp32 before the scale brings
// them back: such rows of x are marked when x is split, and behind the last job the table is read once more and their
// scores made as plain fp32 sums of x·w, w = s·(c − 8) an exact value.
//
// A lane's share of an item's group is G/4 consecutive codes; reading those straight from HBM makes 16 rows' short
// pieces per instruction (64 lanes, 8 cache lines of which 4 B to 16 B are used), so a wave first copies the 16·U
// items of a job, contiguous in memory, to LDS with 16-byte buffer -> LDS loads and reads them from there.  One buffer a
// wave; the next job's copy starts when the last code has been read, before this job's scores are stored.  A second
// buffer a wave halves the waves that fit and measured 36 us against 30 on 1M x 128.
//
// Measured: 1M x 128 for one fp32 session, G = 32: 25 to 28 us, 76 MB, 2.7 to 3 TB/s with the launch (the vector instructions
// take 18 of them: 44 a step of 16 items x 32 codes, of which 8 expand the codes; the three planes are three MFMAs and three
// operand reads, each for one row of 16); 5M x 256 for 16 bf16 sessions, G = 64: 248 us, 0.68 GB read and 0.32 GB
// written, 4.0 TB/s, 78 % of a large copy's rate: the scores of 16 rows end anywhere in a cache line.  10K x 64: 3 to
// 4 us of kernel, less than a launch costs.  64 rows of 1M x 128: 110 us.
#include "common.h"

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

#define Q4_WAVES 4
#define Q4_K_MAX 1024
#define Q4_GRID 2048   // 5M x 256: 250 us; 1024 305, 1280 257, 4096 259 (before x was loaded under one guard: now 248)

// two bf16 values (16 + c) of the codes at bits 4j .. and 16 + 4j .. of w
template <int J>
__device__ __forceinline__ uint32_t q4_pair(uint32_t w) {
  const uint32_t v = J == 0 ? w << 3 : w >> (4 * J - 3);
  return (v & 0x00780078u) | 0x41804180u;
}
// eight codes -> MFMA operand; its k order is (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ bf16x8 q4_codes(uint32_t w) {
  const u32x4 v = {q4_pair<0>(w), q4_pair<1>(w), q4_pair<2>(w), q4_pair<3>(w)};
  return __builtin_bit_cast(bf16x8, v);
}
__device__ __forceinline__ int q4_order(int e) { return (e >> 1) + 4 * (e & 1); }

#define Q4_LARGE 0x1p96f   // rows of x with larger values, infinities or NaN are summed plainly

__device__ __forceinline__ float q4_x(const float* x, int64_t i) { return x[i]; }
__device__ __forceinline__ float q4_x(const __bf16* x, int64_t i) { return (float)x[i]; }

// LDS: x fragments [K / 32][NP][64 lanes] of 16 B, then per wave `cbytes` of codes and `sbytes` of scales (both
// multiples of 1 KB) of the 16·U items that it has in hand.  A granule (16 B of codes) l of a job lies at
// l ^ (l >> shift & 7): 2^shift granules or fewer make a row, so 16 rows' granules of one group spread over the banks
// (a row of 128 B would put them all on eight).  Four waves a SIMD keep the accumulators in vector registers.
template <typename XT, int NP, int G, int U>
__global__ __launch_bounds__(64 * Q4_WAVES, 4) void k_q4_scores(const XT* __restrict__ x, int64_t ldx,
                                                             const uint8_t* __restrict__ codes,
                                                             const uint16_t* __restrict__ scales,
                                                             const float* __restrict__ bias, int M, int64_t N, int K,
                                                             int cbytes, int sbytes, int shift,
                                                             float* __restrict__ y, int64_t ldy) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  constexpr int SG = G / 32;   // MFMA steps of a group; a lane's codes of a group: 4·SG bytes
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15,
            kg = lane >> 4;
  const int steps = K / 32, groups = K / G;
  const int m0 = blockIdx.y * 16;
  bf16x8* xf = reinterpret_cast<bf16x8*>(lds);
  uint8_t* cl = lds + (size_t)steps * NP * 1024 + (size_t)wave * (cbytes + sbytes);
  const uint8_t* sl = cl + cbytes;
  // behind them a word a wave, bit m: row m0 + m is marked
  uint32_t* marks = reinterpret_cast<uint32_t*>(lds + (size_t)steps * NP * 1024 + (size_t)Q4_WAVES * (cbytes + sbytes));

  constexpr int per = 16 * U;
  const int64_t jobs = (N + per - 1) / per, stride = (int64_t)gridDim.x * Q4_WAVES;
  int64_t job = (int64_t)blockIdx.x * Q4_WAVES + wave;
  auto slot = [&](int l) { return l ^ ((l >> shift) & 7); };   // its own inverse: shift >= 3
  // 16-byte loads of a job's codes and scales; behind the table's end the buffer's bound makes them zero
  auto fetch = [&](int64_t j) {
    const int64_t i0 = j * per;
    const int64_t cleft = (N - i0) * (K / 2), sleft = (N - i0) * groups * 2;
    const auto rc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(codes) + i0 * (K / 2), 0,
                                                      (int)min(cleft, (int64_t)cbytes), 0x00020000);
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(scales)) + i0 * groups * 2, 0,
        (int)min((sleft + 3) & ~(int64_t)3, (int64_t)sbytes), 0x00020000);
    for (int o = 0; o < cbytes; o += 1024) rg_blds16(rc, cl + o, 16 * slot((o >> 4) + lane), 0);
    for (int o = 0; o < sbytes; o += 1024) rg_blds16(rs, cl + cbytes + o, o + 16 * lane, 0);
  };
  if (job < jobs) fetch(job);

  uint32_t marked = 0;
  for (int f = threadIdx.x; f < steps * 64; f += 64 * Q4_WAVES) {   // (a wave's lanes together)
    const int s = f >> 6, l = f & 63, m = m0 + (l & 15);
    const int k0 = (s / SG) * G + (G / 4) * (l >> 4) + 8 * (s % SG);
    f4 v[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    uint32_t top = 0;   // of the values' bits without their signs: infinities and NaN are above the finite ones
    if (m < M) {
      const XT* at = x + (int64_t)m * ldx + k0;
      XT r[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = at[q4_order(e)];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e >> 2][e & 3] = (float)r[e];
        top = max(top, __float_as_uint(v[e >> 2][e & 3]) & 0x7fffffff);
      }
    }
    const uint64_t on = __ballot(top >= __float_as_uint(Q4_LARGE));
    marked |= (uint32_t)(on | on >> 16 | on >> 32 | on >> 48) & 0xffff;
    bf16x8 p[3];
    split3x8(v[0], v[1], p[0], p[1], p[2]);
#pragma unroll
    for (int q = 0; q < NP; ++q) xf[(s * NP + q) * 64 + l] = p[q];
  }
  if (lane == 0) marks[wave] = marked;
  __syncthreads();

  const bf16x8 minus24 = {(__bf16)-24.f, (__bf16)-24.f, (__bf16)-24.f, (__bf16)-24.f,
                          (__bf16)-24.f, (__bf16)-24.f, (__bf16)-24.f, (__bf16)-24.f};
  for (; job < jobs; job += stride) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    f4 acc[U];
    float b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t item = job * per + 16 * u + n;
      acc[u] = (f4){0.f, 0.f, 0.f, 0.f};
      b[u] = bias != nullptr && item < N ? bias[item] : 0.f;
    }
    for (int g = 0; g < groups; ++g) {
      bf16x8 a[SG][NP];
      f4 start[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int s = 0; s < SG; ++s)
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          a[s][q] = xf[((g * SG + s) * NP + q) * 64 + lane];
          start[q > 0] = mfma16bf(a[s][q], minus24, start[q > 0]);
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = 16 * u + n;
        const int off = row * (K / 2) + g * (G / 2) + kg * (G / 8);
        const uint32_t* c = reinterpret_cast<const uint32_t*>(cl + 16 * slot(off >> 4) + (off & 15));
        f4 d = start[0], rest = start[1];
#pragma unroll
        for (int s = 0; s < SG; ++s) {
          const bf16x8 w = q4_codes(c[s]);
          d = mfma16bf(a[s][0], w, d);
#pragma unroll
          for (int q = NP - 1; q >= 1; --q) rest = mfma16bf(a[s][q], w, rest);
        }
        if constexpr (NP > 1) d += rest;
        const float sc = __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(sl)[row * groups + g] << 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[u][i] = __builtin_fmaf(sc, d[i], acc[u][i]);
      }
    }
    // every LDS read of this job has returned before the next job's loads land there; they go before the stores,
    // since the wait for them at the loop's head is one for everything in flight
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (job + stride < jobs) fetch(job + stride);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t item = job * per + 16 * u + n;
      if (item < N) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int m = m0 + 4 * kg + i;
          if (m < M) y[(int64_t)m * ldy + item] = acc[u][i] + b[u];
        }
      }
    }
  }

  static_assert(Q4_WAVES == 4, "");
  marked = __builtin_amdgcn_readfirstlane((marks[0] | marks[1]) | (marks[2] | marks[3]));
  if (marked == 0) return;
  for (job = (int64_t)blockIdx.x * Q4_WAVES + wave; job < jobs; job += stride) {
    fetch(job);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    for (uint32_t left = marked; left != 0; left &= left - 1) {
      const int m = m0 + __builtin_ctz(left);
#pragma unroll 1
      for (int u = 0; u < U; ++u) {   // a lane has the quarter kg of each group
        const int row = 16 * u + n;
        float sum = 0.f;
        for (int g = 0; g < groups; ++g) {
          const int off = row * (K / 2) + g * (G / 2) + kg * (G / 8);
          const uint8_t* c = cl + 16 * slot(off >> 4) + (off & 15);
          const float sc = __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(sl)[row * groups + g] << 16);
          for (int k = 0; k < G / 8; ++k) {
            const int64_t at = (int64_t)m * ldx + g * G + kg * (G / 4) + 2 * k;
            sum = __builtin_fmaf(sc * (float)((c[k] & 15) - 8), q4_x(x, at), sum);
            sum = __builtin_fmaf(sc * (float)((c[k] >> 4) - 8), q4_x(x, at + 1), sum);
          }
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        const int64_t item = job * per + row;
        if (kg == (m - m0) >> 2 && item < N)   // the lane that stored it before
          y[(int64_t)m * ldy + item] = sum + (bias != nullptr ? bias[item] : 0.f);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// codes and scales of a row-major table: s = bf16(max |w| / 7) of each group, c = clamp(round(w / s) + 8, 0, 15) with
// the rounded scale, ties to even; an all-zero group has s = 0 and c = 8.  One lane per 8 codes, a group's lanes join
// by shuffles.
template <typename WT>
__global__ __launch_bounds__(256) void k_q4_pack(const WT* __restrict__ W, int64_t ldw, int64_t N, int K, int G,
                                                 uint8_t* __restrict__ codes, uint16_t* __restrict__ scales) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;   // eighth of the table
  const int64_t per = K / 8, total = N * per;
  const int64_t row = i < total ? i / per : N - 1;
  const int k0 = i < total ? (int)(i % per) * 8 : 0;
  float v[8], top = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = q4_x(W, row * ldw + k0 + e);
    top = fmaxf(top, fabsf(v[e]));
  }
  for (int o = 1; o < G / 8; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
  const __bf16 sb = (__bf16)(top / 7.f);
  const float s = (float)sb, inv = s > 0.f ? s : 1.f;
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) w |= (uint32_t)(int)fminf(fmaxf(rintf(v[e] / inv) + 8.f, 0.f), 15.f) << (4 * e);
  if (i < total) {
    *reinterpret_cast<uint32_t*>(codes + row * (K / 2) + k0 / 2) = w;
    if (k0 % G == 0) scales[row * (K / G) + k0 / G] = __builtin_bit_cast(uint16_t, sb);
  }
}

static bool q4_shape(int64_t N, int K, int G) {
  return N > 0 && (G == 32 || G == 64 || G == 128) && K > 0 && K % G == 0 && K <= Q4_K_MAX && N <= ((int64_t)1 << 40);
}

extern "C" int rg_q4_pack(const void* W, int wtype, int64_t ldw, int64_t N, int K, int G, uint8_t* codes,
                          uint16_t* scales, hipStream_t stream) {
  if (!q4_shape(N, K, G)) return RG_ERR_SHAPE;
  if (W == nullptr || codes == nullptr || scales == nullptr || ldw < K || (wtype != 0 && wtype != 1)) return RG_ERR_ARG;
  if ((uintptr_t)codes & 15) return RG_ERR_ARG;
  const int64_t blocks = (N * (K / 8) + 255) / 256;
  if (blocks > 0x7fffffff) return RG_ERR_SHAPE;
  if (wtype == 0)
    k_q4_pack<float><<<(int)blocks, 256, 0, stream>>>((const float*)W, ldw, N, K, G, codes, scales);
  else
    k_q4_pack<__bf16><<<(int)blocks, 256, 0, stream>>>((const __bf16*)W, ldw, N, K, G, codes, scales);
  RG_LAUNCH_CHECK();
  return RG_OK;
}

template <typename XT, int NP, int G, int U>
static int q4_launch(const void* x, int64_t ldx, const uint8_t* codes, const uint16_t* scales, const float* bias, int M,
                     int64_t N, int K, float* y, int64_t ldy, hipStream_t stream) {
  const int cbytes = (U * 8 * K + 1023) & ~1023, sbytes = (U * 32 * (K / G) + 1023) & ~1023;
  const size_t shared = (size_t)(K / 32) * NP * 1024 + (size_t)Q4_WAVES * (cbytes + sbytes + 4);
  int shift = 3;   // rows of 2^shift granules or fewer
  while ((K >> 5) >> (shift + 1)) ++shift;
  auto kern = k_q4_scores<XT, NP, G, U>;
  if (shared > 64 * 1024 &&
      hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shared) != hipSuccess)
    return RG_ERR_LAUNCH;
  const int64_t jobs = (N + 16 * U - 1) / (16 * U);
  const int64_t wgs = (jobs + Q4_WAVES - 1) / Q4_WAVES;
  const int gx = (int)(wgs < Q4_GRID ? wgs : Q4_GRID);
  hipLaunchKernelGGL(kern, dim3(gx, (M + 15) / 16), dim3(64 * Q4_WAVES), shared, stream, (const XT*)x, ldx, codes, scales,
                     bias, M, N, K, cbytes, sbytes, shift, y, ldy);
  RG_LAUNCH_CHECK();
  return RG_OK;
}

// Four units a wave read x's operands once for 64 items (5M x 256: 250 us against 276 with two); one where four would
// hold over 8 KB of codes, or where the items are so few that CUs would stand idle (10K x 64: 39 workgroups of four
// units, 157 of one).
template <typename XT, int NP, int G>
static int q4_units(const void* x, int64_t ldx, const uint8_t* codes, const uint16_t* scales, const float* bias, int M,
                    int64_t N, int K, float* y, int64_t ldy, hipStream_t stream) {
  return K <= 256 && N > 64 * Q4_WAVES * 256
             ? q4_launch<XT, NP, G, 4>(x, ldx, codes, scales, bias, M, N, K, y, ldy, stream)
             : q4_launch<XT, NP, G, 1>(x, ldx, codes, scales, bias, M, N, K, y, ldy, stream);
}

extern "C" int rg_q4_scores(const void* x, int xtype, int64_t ldx, const uint8_t* codes, const uint16_t* scales,
                            const float* bias, int M, int64_t N, int K, int G, float* y, int64_t ldy,
                            hipStream_t stream) {
  if (!q4_shape(N, K, G)) return RG_ERR_SHAPE;
  if (M <= 0 || M > 65535 * 16) return RG_ERR_SHAPE;
  if (x == nullptr || codes == nullptr || scales == nullptr || y == nullptr || ldx < K || ldy < N) return RG_ERR_ARG;
  if (((uintptr_t)codes & 15) || ((uintptr_t)scales & 15)) return RG_ERR_ARG;
#define Q4_GO(XT, NP)                                                                                       \
  return G == 32   ? q4_units<XT, NP, 32>(x, ldx, codes, scales, bias, M, N, K, y, ldy, stream)            \
         : G == 64 ? q4_units<XT, NP, 64>(x, ldx, codes, scales, bias, M, N, K, y, ldy, stream)            \
                   : q4_units<XT, NP, 128>(x, ldx, codes, scales, bias, M, N, K, y, ldy, stream)
  if (xtype == 0) Q4_GO(float, 3);
  if (xtype == 1) Q4_GO(__bf16, 1);
#undef Q4_GO
  return RG_ERR_ARG;
}
