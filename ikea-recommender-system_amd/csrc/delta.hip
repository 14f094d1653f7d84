// Gated delta rule: a linear-attention recurrence beside the GRU (csrc/gru.hip), per value head with a Dk x Dv state
//     S_t = a_t S_{t-1} + b_t k_t (v_t − a_t S_{t-1}ᵀ k_t)ᵀ,   o_t = scale · S_tᵀ q_t,   a_t = exp(g_t)
//
// Chunks of 32 positions.  With G_i the running sum of g inside a chunk, D_ij = exp(G_i − G_j), S the state before it:
//     A_ij = b_i D_ij k_i·k_j (j < i),  P_ij = scale · D_ij q_i·k_j (j <= i),  T = (1 + A)^-1   (unit lower triangular)
//     X = diag(b)(V − diag(e^G) K S),   U = T X,   O = scale · diag(e^G) Q S + P U
//     S' = e^{G_end} S + Kᵀ diag(D_end) U
// Backwards, with dS the gradient of S':
//     dU = Pᵀ dO + diag(D_end) K dS,   dX = Tᵀ dU,   dV = diag(b) dX
//     dS_prev = e^{G_end} dS + Qᵀ diag(scale · e^G) dO − Kᵀ diag(b e^G) dX
// and, per chunk and independent of the others, dP = dO Uᵀ, dA = −dX Uᵀ and the rest (k_delta_grads).
//
// One wave owns 16·CT value columns of one (row, value head) and their part of the state, in accumulators; it makes the
// chunk's P and T itself and never waits for another wave.  What bounds these kernels is latency inside a chunk (about 20
// products and a triangular solve of 16 steps), not bandwidth or MFMAs; T needs no state, so its part of that is not
// in the chain from chunk to chunk, but every wave makes it for itself, in every pass.  Sessions are
// short, so the answer is many independent waves with little LDS, and each step small.  Forwards, 8192 sessions x
// heads of up to 50 positions of width 64, bf16: 104 us.  (Workgroups of four waves with 64-position chunks, K, Q, P and T
// shared through LDS and a barrier between steps, two to a CU: 320 us.  Three waves a SIMD spill: 602 us a
// training step against 350.  A second copy of the code with half the tiles, for chunks of 16 positions or fewer,
// spills 19 registers: 120 us.)  A long row is cut into segments whose waves run side by side (below).
//
// The state, G and every sum are fp32 or wider (G in fp64: differences of long sums enter an exponential).  Products run
// on bf16 MFMA with fp32 operands split into three planes (planes.h); bf16 inputs are one exact plane.  Two planes
// would halve the products, but leave the fp32 outputs (state, dg, dbeta) at 2^-18 instead of fp32's own rounding; they do
// for o where it is rounded to bf16 (2^-8) in the end.
// Positions at or behind a sequence's length are read as k = v = q = 0, b = 0, g = 0, which leaves the state as it is;
// nothing is read there.
//
// Accumulator tiles feed the next product from their registers: a tile of rows i and columns n packs (with the next 16
// rows) into an operand with n as its free index and i contracted, whichever side it stands on.  So P and T are made in
// the orientation in which they are used and never pass through LDS; T's blocks come from forward substitution in
// registers, by columns or by rows as the use wants.
#include "planes.h"

#define DL_C 32
#define DL_NP 3
#define DL_G_MIN (-1000.0)   // exp of anything below is 0 in fp32; keeps −inf (a full reset) out of differences

struct DeltaArgs {
  const void *q, *k, *v, *d_o;
  const float *g, *beta, *state0, *dstate;
  const int64_t* lens;
  int64_t qs[3], ks[3], vs[3], gs[3], bs[3], dos[3];   // strides of (B, T, H), in elements
  int B, T, Hk, Hv, Dk, Dv;
  float scale;
  void *o, *dq, *dk, *dv;                   // contiguous
  float *state, *dstate0, *dg, *dbeta;
  float *U, *dX;                            // (B, Hv, T, Dv)
  float *S0, *dS;                           // (B, Hv, chunks - 1, Dk, Dv): states before chunk c + 1, gradients after chunk c
  // segments of `per` chunks; nseg = 1: none.  trans (B, Hv, nseg, dl_trans_floats): what a segment does to the state it
  // starts with; local (B, Hv, nseg, Dk, Dv): the state (or its gradient) it leaves when it starts from zero, then, joined,
  // the one it really starts from
  int nseg, per;
  float *trans, *local;
};

typedef uint32_t dl_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t dl_u2 __attribute__((ext_vector_type(2)));

// Memory through buffer resources.  A lane's part of an offset is one register, the rest (row, tile) is uniform and goes
// into the scalar offset; rows behind the last one lie behind the resource's end and a lane whose column does not exist
// has an offset behind any end: such loads give 0 and such stores do nothing, without a branch or a mask per access.
// (All elements of a vector load have to be used: narrowed to its last elements, this compiler reads the first.)
typedef __amdgpu_buffer_rsrc_t DlBuf;
// rows of `cols` elements, `st` apart (st >= cols, or one row)
__device__ __forceinline__ DlBuf dl_buf(const void* p, int rows, int64_t st, int cols, int size) {
  const int64_t bytes = rows > 0 ? ((rows - 1) * st + cols) * size : 0;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ int dl_lane(bool on, int bytes) { return on ? bytes : (int)0x80000000; }

template <typename IO>
struct DlIO;
template <>
struct DlIO<float> {
  static constexpr int N = 3, SIZE = 4;
  static __device__ __forceinline__ float load1(DlBuf b, int v, int s) {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(b, v, s, 0));
  }
  static __device__ __forceinline__ f4 load4(DlBuf b, int v, int s) {
    return __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(b, v, s, 0));
  }
  static __device__ __forceinline__ void load44(DlBuf b, int v, int s, int v2, int s2, bf16x8* f) {
    pl_split<3>(load4(b, v, s), load4(b, v2, s2), f);
  }
  struct Raw8 {
    f4 a, b;
  };
  static __device__ __forceinline__ Raw8 load8(DlBuf b, int v, int s) { return {load4(b, v, s), load4(b, v + 16, s)}; }
  static __device__ __forceinline__ void planes(const Raw8& x, bf16x8* f) { pl_split<3>(x.a, x.b, f); }
  static __device__ __forceinline__ float dot(const Raw8& x, const f4& p, const f4& q, float s) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s = __builtin_fmaf(x.a[i], p[i], __builtin_fmaf(x.b[i], q[i], s));
    return s;
  }
  static __device__ __forceinline__ void store1(DlBuf b, int v, int s, float x) {
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, x), b, v, s, 0);
  }
  // the scalar offset stays constant here: a 16-byte store with one in a register may read its data after the next
  // instruction has overwritten it (the compiler only waits where the offset is a constant)
  static __device__ __forceinline__ void store4(DlBuf b, int v, int s, f4 x) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(dl_u4, x), b, v + s, 0, 0);
  }
};
template <>
struct DlIO<__bf16> {
  static constexpr int N = 1, SIZE = 2;
  static __device__ __forceinline__ float load1(DlBuf b, int v, int s) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_raw_buffer_load_b16(b, v, s, 0) << 16);
  }
  static __device__ __forceinline__ void load44(DlBuf b, int v, int s, int v2, int s2, bf16x8* f) {
    const dl_u2 x = __builtin_amdgcn_raw_buffer_load_b64(b, v, s, 0), y = __builtin_amdgcn_raw_buffer_load_b64(b, v2, s2, 0);
    f[0] = __builtin_bit_cast(bf16x8, (dl_u4){x[0], x[1], y[0], y[1]});
  }
  typedef bf16x8 Raw8;
  static __device__ __forceinline__ Raw8 load8(DlBuf b, int v, int s) {
    return __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(b, v, s, 0));
  }
  static __device__ __forceinline__ void planes(const Raw8& x, bf16x8* f) { f[0] = x; }
  static __device__ __forceinline__ float dot(const Raw8& x, const f4& p, const f4& q, float s) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s = __builtin_fmaf((float)x[i], p[i], __builtin_fmaf((float)x[4 + i], q[i], s));
    return s;
  }
  static __device__ __forceinline__ void store1(DlBuf b, int v, int s, float x) {
    __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (__bf16)x), b, v, s, 0);
  }
  static __device__ __forceinline__ void store4(DlBuf b, int v, int s, f4 x) {
    typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(dl_u2, __builtin_convertvector(x, bf4)), b, v, s, 0);
  }
};

__device__ __forceinline__ int dl_len(const DeltaArgs& a, int b) {
  if (a.lens == nullptr) return a.T;
  const int64_t n = a.lens[b];
  return n < 0 ? 0 : n > a.T ? a.T : (int)n;
}

// 32 rows of a (.., D) operand (zeros behind the buffer's rows and behind column D): from memory, then into planes
template <typename IO, int DP, int THREADS>
struct DlTile {
  static constexpr int N = DlIO<IO>::N, W = DP / 8, ALL = DL_C * W, PER = ALL / THREADS > 0 ? ALL / THREADS : 1;
  typename DlIO<IO>::Raw8 x[PER];
  __device__ __forceinline__ void load(DlBuf buf, int64_t st, int D, int tid) {
    const int r = tid / W, c = tid % W * 8, v = dl_lane(c < D && tid < ALL, (int)(r * st + c) * DlIO<IO>::SIZE);
    const int step = (int)(THREADS / W * st) * DlIO<IO>::SIZE;
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = DlIO<IO>::load8(buf, v, i * step);
  }
  __device__ __forceinline__ void put(const PlaneMat<DL_C, DP, N>& m, int tid) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      bf16x8 f[N];
      DlIO<IO>::planes(x[i], f);
      if (ALL >= THREADS || tid < ALL) m.put8(tid / W + i * (THREADS / W), tid % W * 8, f);
    }
  }
};
// operand straight from memory: rows `row` + n, columns c0 + 4·kg .. and 16 further on
template <typename IO>
__device__ __forceinline__ void dl_operand(bf16x8* f, DlBuf buf, int row, int64_t st, int c0, int D) {
  const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4, v = (int)(n * st + 4 * kg) * DlIO<IO>::SIZE;
  const int s = (int)(row * st + c0) * DlIO<IO>::SIZE;
  DlIO<IO>::load44(buf, dl_lane(c0 + 4 * kg < D, v), s, dl_lane(c0 + 16 + 4 * kg < D, v), s + 16 * DlIO<IO>::SIZE, f);
}

// per-position scalars of a chunk
struct DlGates {
  double G[DL_C];        // running sum of g · log2 e
  float gam[DL_C];       // 2^G_i
  float rest[DL_C];      // 2^(G_end − G_i)
  float beta[DL_C];
};
__device__ __forceinline__ float dl_exp2(double x) { return __builtin_amdgcn_exp2f((float)x); }
// one wave: g and beta of a chunk's positions from memory, then their sums and exponentials
__device__ __forceinline__ void dl_gates_load(float* x, const DeltaArgs& a, int b, int h, int t0, int len) {
  const int i = threadIdx.x & 31;
  const DlBuf gbuf = dl_buf(a.g + b * a.gs[0] + t0 * a.gs[1] + h * a.gs[2], 32, a.gs[1], 1, 4),
              bbuf = dl_buf(a.beta + b * a.bs[0] + t0 * a.bs[1] + h * a.bs[2], 32, a.bs[1], 1, 4);
  x[0] = DlIO<float>::load1(gbuf, dl_lane(t0 + i < len, (int)(i * a.gs[1]) * 4), 0);
  x[1] = DlIO<float>::load1(bbuf, dl_lane(t0 + i < len, (int)(i * a.bs[1]) * 4), 0);
}
__device__ __forceinline__ void dl_gates(DlGates& s, const float* x) {
  const int i = threadIdx.x & 31;
  double g = (x[0] < DL_G_MIN ? DL_G_MIN : (double)x[0]) * 1.4426950408889634;   // NaN stays
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double up = __shfl_up(g, o, 32);
    if (i >= o) g += up;
  }
  const double end = __shfl(g, 31, 32);
  if ((threadIdx.x & 63) < 32) {
    s.G[i] = g;
    s.gam[i] = dl_exp2(g);
    s.rest[i] = dl_exp2(end - g);
    s.beta[i] = x[1];
  }
}

#define DL_ZERO ((f4){0.f, 0.f, 0.f, 0.f})

// LDS between the lanes of one wave: its LDS instructions run in order, so only the compiler has to keep it
__device__ __forceinline__ void dl_fence() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

// Forward substitution: column n of (1 + A)^-1, A strictly lower, 16 x 16 in LDS (rows of 20 floats, read by many lanes at
// once).  The next row is read while this one's sum runs; left to itself the compiler reads all of A first (120 registers).
__device__ __forceinline__ void dl_solve(const float* A, int n, float* t) {
  f4 row[4], next[4];
  t[0] = n == 0 ? 1.f : 0.f;
  next[0] = *reinterpret_cast<const f4*>(A + 20);
#pragma unroll
  for (int i = 1; i < 16; ++i) {
#pragma unroll
    for (int q = 0; q < 4; ++q) row[q] = next[q];
    if (i < 15) {
#pragma unroll
      for (int q = 0; q < (i + 4) / 4; ++q) next[q] = *reinterpret_cast<const f4*>(A + (i + 1) * 20 + 4 * q);
    }
    float x = i == n ? 1.f : 0.f;
#pragma unroll
    for (int j = 0; j < i; ++j) x = __builtin_fmaf(-row[j >> 2][j & 3], t[j], x);
    t[i] = x;
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }
}

// LDS of one wave: K (and Q) in planes, the gates, the diagonal blocks of A, then of T
template <int DP, int NI, bool Q>
struct DlLds {
  static constexpr int KQ = PlaneMat<DL_C, DP, NI>::BYTES;
  static constexpr int BYTES = (Q ? 2 : 1) * KQ + (int)sizeof(DlGates) + 2 * 16 * 20 * 4;
};

// T of a chunk as operands: FWD: T (free index i), two per 32 rows; else its transpose (free index j).
//   FWD  t[0] = {T00, 0}, t[1] = {T10, T11}      else  t[0] = {T00ᵀ, T10ᵀ}, t[1] = {0, T11ᵀ}
// Rows behind the length are zero in K, so A is zero and T the identity there.
template <int DP, int NI, bool FWD>
__device__ __forceinline__ void dl_inverse(const PlaneMat<DL_C, DP, NI>& K, const DlGates& s, float* Ad,
                                           bf16x8 (*t)[DL_NP]) {
  const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;
  f4 d0 = DL_ZERO, d1 = DL_ZERO, off = DL_ZERO;   // off: rows j of block 0, columns i of block 1
#pragma unroll
  for (int x = 0; x < DP / 32; ++x) {
    bf16x8 k0[NI], k1[NI];
    K.row(k0, 0, x);
    K.row(k1, 16, x);
    d0 = pl_mm<NI, NI>(k0, k0, d0);
    d1 = pl_mm<NI, NI>(k1, k1, d1);
    off = pl_mm<NI, NI>(k0, k1, off);
  }
  const double gn0 = s.G[n], gn1 = s.G[16 + n];
  const float bn1 = s.beta[16 + n];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = 4 * kg + r;
    const double g0 = s.G[i], g1 = s.G[16 + i];
    Ad[i * 20 + n] = n < i ? s.beta[i] * dl_exp2(g0 - gn0) * d0[r] : 0.f;
    Ad[320 + i * 20 + n] = n < i ? s.beta[16 + i] * dl_exp2(g1 - gn1) * d1[r] : 0.f;
    off[r] *= bn1 * dl_exp2(gn1 - g0);
  }
  dl_fence();
  {   // lanes of kg 0, 1 solve block 0, the others block 1; T goes where A was, each lane half a column
    float x[16];
    dl_solve(Ad + 320 * (kg >> 1), n, x);
    dl_fence();
    float* to = Ad + 320 * (kg >> 1) + n;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float lo = x[i], hi = x[8 + i];
      to[(i + 8 * (kg & 1)) * 20] = kg & 1 ? hi : lo;
    }
  }
  dl_fence();
  f4 c0, r1;
#pragma unroll
  for (int r = 0; r < 4; ++r) c0[r] = Ad[(4 * kg + r) * 20 + n];   // column n of T00
  r1 = *reinterpret_cast<const f4*>(Ad + 320 + n * 20 + 4 * kg);   // row n of T11
  // T10 = −T11 (A10 T00)
  bf16x8 fa[DL_NP], fb[DL_NP];
  pl_split<DL_NP>(off, DL_ZERO, fa);
  pl_split<DL_NP>(c0, DL_ZERO, fb);
  const f4 m = pl_mm<DL_NP, DL_NP>(fa, fb, DL_ZERO);   // rows i of block 1, columns j of block 0
  pl_split<DL_NP>(m, DL_ZERO, fa);
  pl_split<DL_NP>(r1, DL_ZERO, fb);
  if (FWD) {
    const f4 low = -pl_mm<DL_NP, DL_NP>(fa, fb, DL_ZERO), r0 = *reinterpret_cast<const f4*>(Ad + n * 20 + 4 * kg);
    pl_split<DL_NP>(r0, DL_ZERO, t[0]);
    pl_split<DL_NP>(low, r1, t[1]);
  } else {
    const f4 low = -pl_mm<DL_NP, DL_NP>(fb, fa, DL_ZERO);
    f4 c1;
#pragma unroll
    for (int r = 0; r < 4; ++r) c1[r] = Ad[320 + (4 * kg + r) * 20 + n];
    pl_split<DL_NP>(c0, low, t[0]);
    pl_split<DL_NP>(DL_ZERO, c1, t[1]);
  }
}

template <typename IO>
__device__ __forceinline__ void dl_zero4(IO* p) {
  typedef IO IO4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<IO4*>(p) = (IO4)(IO)0.f;
}

// the state of one wave: rows d = 16·u + 4·kg + r, columns col0 + 16·ct + n of a (Dk, cols) fp32 matrix
template <int CT, int UT>
__device__ __forceinline__ void dl_state_load(f4 (*S)[UT], const float* src, int Dk, int cols, int col0) {
  const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;
  const DlBuf buf = dl_buf(src, src != nullptr ? Dk : 0, cols, cols, 4);
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int col = col0 + 16 * ct + n, v = dl_lane(col < cols, (4 * kg * cols + col) * 4);
#pragma unroll
    for (int u = 0; u < UT; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[ct][u][r] = DlIO<float>::load1(buf, v, (16 * u + r) * cols * 4);
  }
}
template <int CT, int UT>
__device__ __forceinline__ void dl_state_store(const f4 (*S)[UT], float* dst, int Dk, int cols, int col0) {
  const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;
  const DlBuf buf = dl_buf(dst, Dk, cols, cols, 4);
  int row[CT], at = 0;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int col = col0 + 16 * ct + n;
    row[ct] = dl_lane(col < cols, (4 * kg * cols + col) * 4);
  }
#pragma unroll
  for (int u = 0; u < UT; ++u)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      asm volatile("" : "+s"(at));   // one running offset; the compiler would keep all of them and spill
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) DlIO<float>::store1(buf, row[ct], at, S[ct][u][r]);
      at += (r < 3 ? 1 : 13) * cols * 4;
    }
}

// A transition is kept as its 16 x 16 tiles in the order in which the join's operands want them, so that a wave reads 1 KB
// in one piece (from rows, half a cache line a lane: 2.2 us a segment of width 128 against 1.55): lane (kg, n), value r of
// tile (w, t) is row 16·w + n, column 16·t + 4·kg + r, then, for the backward pass, row 16·t + 4·kg + r, column 16·w + n.
__host__ __device__ __forceinline__ int64_t dl_trans_floats(int Dk) {
  const int N = (Dk + 15) / 16;
  return 2 * 256 * (int64_t)N * N;
}
template <int CT, int UT>
__device__ __forceinline__ void dl_trans_store(const f4 (*S)[UT], float* dst, int Dk, int col0, bool back) {
  const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4, N = (Dk + 15) / 16;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = col0 / 16 + ct;
    if (c >= N) break;
#pragma unroll
    for (int u = 0; u < UT; ++u) {
      if (u >= N) break;
      float* p = dst + (u * N + c) * 256 + (16 * (n >> 2) + 4 * kg) * 4 + (n & 3);
#pragma unroll
      for (int r = 0; r < 4; ++r) p[4 * r] = S[ct][u][r];
      if (back) *reinterpret_cast<f4*>(dst + N * N * 256 + (c * N + u) * 256 + lane * 4) = S[ct][u];
    }
  }
}

// ---------------------------------------------------------------- forward ----
// TRANS: only the states a segment leaves, from zero (columns of the value) or from the identity with v = 0 (the columns
// behind them: the segment's transition)
template <typename IO, int DP, int CT, bool TRANS>
__global__ __launch_bounds__(64, 2) void k_delta_fwd(DeltaArgs a) {
  constexpr int NI = DlIO<IO>::N, KT = DP / 32, NP = DL_NP, NO = NI == 1 ? 2 : 3;
  using L = DlLds<DP, NI, false>;
  __shared__ __attribute__((aligned(16))) uint8_t lds[L::BYTES];
  const PlaneMat<DL_C, DP, NI> K{(__bf16*)lds};
  DlGates& s = *(DlGates*)(lds + L::KQ);
  float* Ad = (float*)(lds + L::KQ + sizeof(DlGates));

  const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;
  const int seg = blockIdx.x / (a.B * a.Hv), bhi = blockIdx.x % (a.B * a.Hv);
  const int b = bhi / a.Hv, h = bhi % a.Hv, hk = h / (a.Hv / a.Hk);
  const int len = dl_len(a, b), nC = (a.T + DL_C - 1) / DL_C;
  const int vblocks = (a.Dv + 16 * CT - 1) / (16 * CT);
  const bool unit = TRANS && (int)blockIdx.y >= vblocks;      // columns of the transition
  const int col0 = (unit ? blockIdx.y - vblocks : blockIdx.y) * 16 * CT, cols = unit ? a.Dk : a.Dv;
  const IO* q = (const IO*)a.q + b * a.qs[0] + hk * a.qs[2];
  const IO* k = (const IO*)a.k + b * a.ks[0] + hk * a.ks[2];
  const IO* v = (const IO*)a.v + b * a.vs[0] + h * a.vs[2];
  const int64_t bh = bhi, os = (int64_t)a.Hv * a.Dv, size = (int64_t)a.Dk * a.Dv;
  IO* o = (IO*)a.o + ((int64_t)b * a.T * a.Hv + h) * a.Dv;   // row stride Hv * Dv

  const float* init = TRANS ? nullptr : seg > 0 ? a.local + (bh * a.nseg + seg) * size : a.state0 ? a.state0 + bh * size : nullptr;
  bool zero = init == nullptr && !unit;   // the state is still zero
  f4 S[CT][2 * KT];
  dl_state_load<CT, 2 * KT>(S, init, a.Dk, a.Dv, col0);
  if (unit) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int u = 0; u < 2 * KT; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[ct][u][r] = 16 * u + 4 * kg + r == col0 + 16 * ct + n ? 1.f : 0.f;
  }

  const int tfrom = seg * a.per * DL_C, tend = a.nseg == 1 ? len : min(len, tfrom + a.per * DL_C);
  for (int t0 = tfrom; t0 < tend; t0 += DL_C) {
    const int left = len - t0;   // positions from here on
    const int rows = min(left, DL_C);
    const DlBuf vbuf = dl_buf(v + t0 * a.vs[1], unit ? 0 : rows, a.vs[1], a.Dv, DlIO<IO>::SIZE);
    auto values = [&](int ct, float* x) __attribute__((always_inline)) {
      const int col = col0 + 16 * ct + n, at = dl_lane(col < cols, (int)(4 * kg * a.vs[1] + col) * DlIO<IO>::SIZE);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] = DlIO<IO>::load1(vbuf, at, (int)((16 * (i >> 2) + (i & 3)) * a.vs[1]) * DlIO<IO>::SIZE);
    };
    DlTile<IO, DP, 64> kt;
    kt.load(dl_buf(k + t0 * a.ks[1], rows, a.ks[1], a.Dk, DlIO<IO>::SIZE), a.ks[1], a.Dk, lane);
    float gates[2];
    dl_gates_load(gates, a, b, h, t0, len);
    float vv[8], vnext[8];
    values(0, vnext);
    bf16x8 qf[2][KT][NI];
    if constexpr (!TRANS) {
      const DlBuf qbuf = dl_buf(q + t0 * a.qs[1], rows, a.qs[1], a.Dk, DlIO<IO>::SIZE);
#pragma unroll
      for (int it = 0; it < 2; ++it)
#pragma unroll
        for (int t = 0; t < KT; ++t) dl_operand<IO>(qf[it][t], qbuf, 16 * it, a.qs[1], 32 * t, a.Dk);
      if (a.S0 != nullptr && t0 > 0)
        dl_state_store<CT, 2 * KT>(S, a.S0 + (bh * (nC - 1) + t0 / DL_C - 1) * size, a.Dk, a.Dv, col0);
    }
    dl_fence();
    kt.put(K, lane);
    dl_gates(s, gates);
    dl_fence();
    bf16x8 T[2][NP], P[2][NO];
    dl_inverse<DP, NI, true>(K, s, Ad, T);
    if constexpr (!TRANS) {
      f4 p00 = DL_ZERO, p01 = DL_ZERO, p11 = DL_ZERO;   // rows j, columns i
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        bf16x8 k0[NI], k1[NI];
        K.row(k0, 0, t);
        K.row(k1, 16, t);
        p00 = pl_mm<NI, NI>(k0, qf[0][t], p00);
        p01 = pl_mm<NI, NI>(k0, qf[1][t], p01);
        p11 = pl_mm<NI, NI>(k1, qf[1][t], p11);
      }
      const double g0 = s.G[n], g1 = s.G[16 + n];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 4 * kg + r;
        const double h0 = s.G[j], h1 = s.G[16 + j];
        p00[r] = j <= n ? a.scale * dl_exp2(g0 - h0) * p00[r] : 0.f;
        p01[r] *= a.scale * dl_exp2(g1 - h0);
        p11[r] = j <= n ? a.scale * dl_exp2(g1 - h1) * p11[r] : 0.f;
      }
      pl_split<NO>(p00, DL_ZERO, P[0]);
      pl_split<NO>(p01, p11, P[1]);
    }
    const float last = s.gam[DL_C - 1];
    const DlBuf obuf = dl_buf(o + t0 * os, min(a.T - t0, DL_C), os, a.Dv, DlIO<IO>::SIZE),
                ubuf = dl_buf(a.U + (bh * a.T + t0) * a.Dv, a.U != nullptr ? rows : 0, a.Dv, a.Dv, 4);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
      for (int i = 0; i < 8; ++i) vv[i] = vnext[i];
      if (ct + 1 < CT) values(ct + 1, vnext);
      f4 x[2] = {DL_ZERO, DL_ZERO}, oo[2] = {DL_ZERO, DL_ZERO};   // oo: rows v, columns i
      if (!zero) {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          bf16x8 sb[NP], f[NI];
          pl_split<NP>(S[ct][2 * t], S[ct][2 * t + 1], sb);
          K.row(f, 0, t);
          x[0] = pl_mm<NI, NP>(f, sb, x[0]);
          K.row(f, 16, t);
          x[1] = pl_mm<NI, NP>(f, sb, x[1]);
          if constexpr (!TRANS) {
            oo[0] = pl_mm<NO, NI>(sb, qf[0][t], oo[0]);
            oo[1] = pl_mm<NO, NI>(sb, qf[1][t], oo[1]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f4 be = *reinterpret_cast<const f4*>(s.beta + 16 * j + 4 * kg), gam = *reinterpret_cast<const f4*>(s.gam + 16 * j + 4 * kg);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[j][r] = be[r] * (vv[4 * j + r] - gam[r] * x[j][r]);
      }
      bf16x8 xb[NP];
      pl_split<NP>(x[0], x[1], xb);
      f4 u[2];
      u[0] = pl_mm<NP, NP>(T[0], xb, DL_ZERO);
      u[1] = pl_mm<NP, NP>(T[1], xb, DL_ZERO);
      if constexpr (!TRANS) {
        bf16x8 ub[NO];
        pl_split<NO>(u[0], u[1], ub);
        const int row = col0 + 16 * ct + 4 * kg, at = dl_lane(row < a.Dv, (int)(n * os + row) * DlIO<IO>::SIZE);
#pragma unroll
        for (int it = 0; it < 2; ++it) {
          oo[it] *= a.scale * s.gam[16 * it + n];
          oo[it] = pl_mm<NO, NO>(ub, P[it], oo[it]);
          DlIO<IO>::store4(obuf, at, (int)(16 * it * os) * DlIO<IO>::SIZE, oo[it]);
        }
        if (a.U != nullptr) {
          const int col = col0 + 16 * ct + n, up = dl_lane(col < cols, (4 * kg * a.Dv + col) * 4);
          int to = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            asm volatile("" : "+s"(to));
            DlIO<float>::store1(ubuf, up, to, u[i >> 2][i & 3]);
            to += (i == 3 ? 13 : 1) * a.Dv * 4;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) u[j] *= *reinterpret_cast<const f4*>(s.rest + 16 * j + 4 * kg);
      pl_split<NP>(u[0], u[1], xb);
#pragma unroll
      for (int t = 0; t < 2 * KT; ++t) {
        bf16x8 f[NI];
        K.col(f, 0, 16 * t);
        S[ct][t] = pl_mm<NI, NP>(f, xb, S[ct][t] * last);
      }
    }
    zero = false;
  }
  if constexpr (TRANS) {
    if (unit)
      dl_trans_store<CT, 2 * KT>(S, a.trans + (bh * a.nseg + seg) * dl_trans_floats(a.Dk), a.Dk, col0, a.U != nullptr);
    else
      dl_state_store<CT, 2 * KT>(S, a.local + (bh * a.nseg + seg) * size, a.Dk, cols, col0);
  } else {
    // outputs behind the length, in this segment's part
    const int tto = seg == a.nseg - 1 ? a.T : min(a.T, tfrom + a.per * DL_C);
    const int tdone = max(tfrom, (len + DL_C - 1) / DL_C * DL_C);
    for (int t = tdone + n; t < tto; t += 16)
      for (int c = col0 + 4 * kg; c < min(a.Dv, col0 + 16 * CT); c += 16) dl_zero4(o + t * os + c);
    if (seg == a.nseg - 1) dl_state_store<CT, 2 * KT>(S, a.state + bh * size, a.Dk, a.Dv, col0);
  }
}

// ------------------------------------------------------- backward, the scan ----
// The same split, chunks last to first; leaves dX, dV, the gradients after each chunk but the last, and dstate0.  LOCAL: only
// the gradient that a segment leaves when it starts from zero.
template <typename IO, int DP, int CT, bool LOCAL>
__global__ __launch_bounds__(64, 2) void k_delta_scan(DeltaArgs a) {
  constexpr int NI = DlIO<IO>::N, KT = DP / 32, NP = DL_NP;
  using L = DlLds<DP, NI, true>;
  __shared__ __attribute__((aligned(16))) uint8_t lds[L::BYTES];
  const PlaneMat<DL_C, DP, NI> K{(__bf16*)lds}, Q{(__bf16*)(lds + L::KQ)};
  DlGates& s = *(DlGates*)(lds + 2 * L::KQ);
  float* Ad = (float*)(lds + 2 * L::KQ + sizeof(DlGates));

  const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;
  const int seg = blockIdx.x / (a.B * a.Hv), bhi = blockIdx.x % (a.B * a.Hv);
  const int b = bhi / a.Hv, h = bhi % a.Hv, hk = h / (a.Hv / a.Hk);
  const int len = dl_len(a, b), nC = (a.T + DL_C - 1) / DL_C, col0 = blockIdx.y * 16 * CT;
  const IO* q = (const IO*)a.q + b * a.qs[0] + hk * a.qs[2];
  const IO* k = (const IO*)a.k + b * a.ks[0] + hk * a.ks[2];
  const IO* d_o = (const IO*)a.d_o + b * a.dos[0] + h * a.dos[2];
  const int64_t bh = bhi, os = (int64_t)a.Hv * a.Dv, size = (int64_t)a.Dk * a.Dv;
  IO* dv = (IO*)a.dv + ((int64_t)b * a.T * a.Hv + h) * a.Dv;

  const float* init = LOCAL                ? nullptr
                      : seg < a.nseg - 1 ? a.local + (bh * a.nseg + seg) * size
                      : a.dstate         ? a.dstate + bh * size
                                         : nullptr;
  bool zero = init == nullptr;
  f4 S[CT][2 * KT];
  dl_state_load<CT, 2 * KT>(S, init, a.Dk, a.Dv, col0);

  const int nc = (len + DL_C - 1) / DL_C, cfrom = seg * a.per, cend = a.nseg == 1 ? nc : min(nc, cfrom + a.per);
  for (int c = cend - 1; c >= cfrom; --c) {
    const int t0 = c * DL_C, left = len - t0;
    const int rows = min(left, DL_C);
    const DlBuf gbuf = dl_buf(d_o + t0 * a.dos[1], rows, a.dos[1], a.Dv, DlIO<IO>::SIZE);
    DlTile<IO, DP, 64> kt, qt;
    kt.load(dl_buf(k + t0 * a.ks[1], rows, a.ks[1], a.Dk, DlIO<IO>::SIZE), a.ks[1], a.Dk, lane);
    qt.load(dl_buf(q + t0 * a.qs[1], rows, a.qs[1], a.Dk, DlIO<IO>::SIZE), a.qs[1], a.Dk, lane);
    float gates[2];
    dl_gates_load(gates, a, b, h, t0, len);
    f4 go[CT][2];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int col = col0 + 16 * ct + n, at = dl_lane(col < a.Dv, (int)(4 * kg * a.dos[1] + col) * DlIO<IO>::SIZE);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        go[ct][i >> 2][i & 3] = DlIO<IO>::load1(gbuf, at, (int)((16 * (i >> 2) + (i & 3)) * a.dos[1]) * DlIO<IO>::SIZE);
    }
    // before the segment's first chunk nobody asks for the state's gradient but dstate0 (8192 sessions x heads
    // of up to 50 positions: 86 us against 96)
    const bool on = LOCAL || c > cfrom || (seg == 0 && a.dstate0 != nullptr);
    if (!LOCAL && c < nc - 1) dl_state_store<CT, 2 * KT>(S, a.dS + (bh * (nC - 1) + c) * size, a.Dk, a.Dv, col0);
    dl_fence();
    kt.put(K, lane);
    qt.put(Q, lane);
    dl_gates(s, gates);
    dl_fence();
    bf16x8 T[2][NP], P[2][NP];
    dl_inverse<DP, NI, false>(K, s, Ad, T);
    {
      f4 p00 = DL_ZERO, p10 = DL_ZERO, p11 = DL_ZERO;   // rows i, columns j
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        bf16x8 k0[NI], k1[NI], f[NI];
        K.row(k0, 0, t);
        K.row(k1, 16, t);
        Q.row(f, 0, t);
        p00 = pl_mm<NI, NI>(f, k0, p00);
        Q.row(f, 16, t);
        p10 = pl_mm<NI, NI>(f, k0, p10);
        p11 = pl_mm<NI, NI>(f, k1, p11);
      }
      const double g0 = s.G[n], g1 = s.G[16 + n];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 4 * kg + r;
        const double h0 = s.G[i], h1 = s.G[16 + i];
        p00[r] = n <= i ? a.scale * dl_exp2(h0 - g0) * p00[r] : 0.f;
        p10[r] *= a.scale * dl_exp2(h1 - g0);
        p11[r] = n <= i ? a.scale * dl_exp2(h1 - g1) * p11[r] : 0.f;
      }
      pl_split<NP>(p00, p10, P[0]);
      pl_split<NP>(DL_ZERO, p11, P[1]);
    }
    const float last = s.gam[DL_C - 1];
    const DlBuf dvbuf = dl_buf(dv + t0 * os, min(a.T - t0, DL_C), os, a.Dv, DlIO<IO>::SIZE),
                xbuf = dl_buf(a.dX + (bh * a.T + t0) * a.Dv, rows, a.Dv, a.Dv, 4);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      f4 du[2] = {DL_ZERO, DL_ZERO};
      if (!zero) {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          bf16x8 sb[NP], f[NI];
          pl_split<NP>(S[ct][2 * t], S[ct][2 * t + 1], sb);
          K.row(f, 0, t);
          du[0] = pl_mm<NI, NP>(f, sb, du[0]);
          K.row(f, 16, t);
          du[1] = pl_mm<NI, NP>(f, sb, du[1]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) du[j] *= *reinterpret_cast<const f4*>(s.rest + 16 * j + 4 * kg);
      }
      bf16x8 gb[NI], xb[NP];
      pl_split<NI>(go[ct][0], go[ct][1], gb);
      du[0] = pl_mm<NP, NI>(P[0], gb, du[0]);
      du[1] = pl_mm<NP, NI>(P[1], gb, du[1]);
      pl_split<NP>(du[0], du[1], xb);
      f4 dx[2];
      dx[0] = pl_mm<NP, NP>(T[0], xb, DL_ZERO);
      dx[1] = pl_mm<NP, NP>(T[1], xb, DL_ZERO);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f4 be = *reinterpret_cast<const f4*>(s.beta + 16 * j + 4 * kg), gam = *reinterpret_cast<const f4*>(s.gam + 16 * j + 4 * kg);
        if constexpr (!LOCAL) {
          const int col = col0 + 16 * ct + n, at = dl_lane(col < a.Dv, (int)(4 * kg * os + col) * DlIO<IO>::SIZE),
                    up = dl_lane(col < a.Dv, (4 * kg * a.Dv + col) * 4);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            DlIO<IO>::store1(dvbuf, at, (int)((16 * j + r) * os) * DlIO<IO>::SIZE, be[r] * dx[j][r]);
            DlIO<float>::store1(xbuf, up, (16 * j + r) * a.Dv * 4, dx[j][r]);
          }
        }
        go[ct][j] *= a.scale * gam;
        dx[j] *= -be * gam;
      }
      if (!on) continue;
      bf16x8 hb[NP];
      pl_split<NP>(go[ct][0], go[ct][1], hb);
      pl_split<NP>(dx[0], dx[1], xb);
#pragma unroll
      for (int t = 0; t < 2 * KT; ++t) {
        bf16x8 f[NI];
        Q.col(f, 0, 16 * t);
        S[ct][t] = pl_mm<NI, NP>(f, hb, S[ct][t] * last);
        K.col(f, 0, 16 * t);
        S[ct][t] = pl_mm<NI, NP>(f, xb, S[ct][t]);
      }
    }
    zero = false;
  }
  if (!LOCAL) {
    const int tto = seg == a.nseg - 1 ? a.T : min(a.T, (cfrom + a.per) * DL_C);
    for (int t = max(cfrom, nc) * DL_C + kg; t < tto; t += 4)
      for (int c = col0 + n; c < min(a.Dv, col0 + 16 * CT); c += 16) dv[t * os + c] = (IO)0.f;
  }
  float* dst = LOCAL ? a.local + (bh * a.nseg + seg) * size : seg == 0 && a.dstate0 ? a.dstate0 + bh * size : nullptr;
  if (dst != nullptr) dl_state_store<CT, 2 * KT>(S, dst, a.Dk, a.Dv, col0);
}

// ------------------------------------------------------- segments ----
// The state a segment starts from: S_{s+1} = trans_s S_s + local_s, put in local's place; backwards the gradient it starts
// from: dS_{s-1} = trans_sᵀ dS_s + local_s.  One workgroup per (row, head, 16 value columns), a wave per 16 rows of the
// state: its rows of trans straight from memory (the next segments' while this one's products run), the state from LDS, in
// two buffers, so that a segment costs one barrier.  On fp32 MFMA, whose four steps take a lane's four values of an
// accumulator as they are.  What bounds it is a CU's way to the 64 KB of trans of each segment (width 128): neither the
// products (fp32, or bf16 planes split here) nor loading one or three segments ahead move it.  (8 heads, 32 segments: 49 us.)
template <int DP, bool BACK>
__global__ __launch_bounds__(4 * DP) void k_delta_join(DeltaArgs a) {
  constexpr int NT = DP / 16, AHEAD = 3;
  __shared__ f4 lds[2][NT][64];
  const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), d0 = 16 * wave, col = blockIdx.y * 16 + n, N = (a.Dk + 15) / 16;
  const int64_t bh = blockIdx.x, size = (int64_t)a.Dk * a.Dv;
  const float* first = BACK ? a.dstate : a.state0;
  const int at = dl_lane(col < a.Dv, ((d0 + 4 * kg) * a.Dv + col) * 4);
  auto state = [&](const float* p) { return dl_buf(p, p != nullptr ? a.Dk : 0, a.Dv, a.Dv, 4); };
  f4 S;
#pragma unroll
  for (int r = 0; r < 4; ++r) S[r] = DlIO<float>::load1(state(first != nullptr ? first + bh * size : nullptr), at, r * a.Dv * 4);

  struct Part {
    f4 w[NT], loc;   // this wave's rows of trans (BACK: of its transpose), and of local
  } part[AHEAD];
  auto fetch = [&](Part& x, int i) __attribute__((always_inline)) {
    const int seg = BACK ? a.nseg - 1 - i : i;
    const DlBuf tb = dl_buf(a.trans + (bh * a.nseg + seg) * dl_trans_floats(a.Dk) + (BACK ? N * N * 256 : 0), 1, 0, N * N * 256, 4);
#pragma unroll
    for (int t = 0; t < NT; ++t)
      x.w[t] = DlIO<float>::load4(tb, dl_lane(wave < N && t < N, lane * 16), (wave * N + t) * 1024);
    const DlBuf lb = state(a.local + (bh * a.nseg + seg) * size);
#pragma unroll
    for (int r = 0; r < 4; ++r) x.loc[r] = DlIO<float>::load1(lb, at, r * a.Dv * 4);
  };
  const int last = a.nseg - 1;   // (what the last segment leaves is not asked for)
  auto put = [&](int i) __attribute__((always_inline)) {
    const DlBuf lb = state(a.local + (bh * a.nseg + (BACK ? last - i : i)) * size);
#pragma unroll
    for (int r = 0; r < 4; ++r) DlIO<float>::store1(lb, at, r * a.Dv * 4, S[r]);
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    fetch(part[k], min(k, last));
    __builtin_amdgcn_sched_barrier(0);   // in this order, so that the first wait leaves the others in flight
  }
  int i = 0;
  while (true) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k, ++i) {
      if (i >= last) {
        put(i);
        return;
      }
      f4 sum[4] = {part[k].loc, DL_ZERO, DL_ZERO, DL_ZERO};
      put(i);
      lds[i & 1][wave][lane] = S;
      __syncthreads();
      f4 x[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) x[t] = lds[i & 1][t][lane];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[r] = mfma16(part[k].w[t][r], x[t][r], sum[r]);
      __builtin_amdgcn_sched_barrier(0);
      // without a branch, so that the waits for the segments before count only what they have to
      fetch(part[k], min(i + AHEAD, last));
      __builtin_amdgcn_sched_barrier(0);
      S = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
  }
}

// -------------------------------------- backward, the rest of a chunk's gradients ----
// One workgroup of four waves per (row, key head, chunk), independent of the others; the value heads of a key head one
// after the other, their dq and dk summed in registers (no atomics: the same result every time).  The contractions over the
// value columns,
//     dP = dO Uᵀ,  dA = −dX Uᵀ,  E1 = dO Sᵀ,  E2 = dX Sᵀ,  E3 = U dS'ᵀ,
// go 32 columns at a time: dX, U and dO are split into planes once, in LDS, and shared, while each wave loads and
// splits its own key tiles of S and dS' (rows of contiguous values are what an operand's lanes want) and multiplies them
// with both tiles of positions; of the four tiles of dP and dA each wave has one.  Then
//     dQ = scale e^G E1 + M1 K,  dK = M1ᵀ Q + (M2 + M2ᵀ) K − b e^G E2 + D_end E3,  M1 = scale D dP,  M2 = b D dA
// with M1 and M2 passed through LDS, in dX's and U's place, and the scalars' gradients from their row and column sums, by
// one wave while the others load the next value head.  Every product is made with the position i as its column, so a
// lane's scalars are one position's and its four results lie side by side.
// What bounds it is vector instructions, most of them splitting operands into planes, and the chain of loads, products and sums.  (Two
// waves, one per tile of positions, each splitting all of S, dS', dX and U for itself: 270 us against 157 on 4 x 8
// heads x 4096 positions of width 128, 181 against 165 on 8192 sessions x heads of up to 50 positions of width 64.  Waves a
// SIMD: with three, fp32 spills 23 registers at width 64, 91 us against 75 on 2048 sessions x heads; bf16 does not, 165 us against
// 219 with two.  At width 128 fp32 spills 37 with two: 547 us for the whole backward pass of 2048 sessions x heads, bf16 158.
// Rows of one chunk, which have no states, in a kernel of their own with four waves a SIMD: 56 + 118 us against 165.)
template <int DP, int NI>
struct DlGradLds {
  static constexpr int KQ = PlaneMat<DL_C, DP, NI>::BYTES, X = PlaneMat<DL_C, 32, DL_NP>::BYTES,
                       G = PlaneMat<DL_C, 32, NI>::BYTES;
  static constexpr int THREADS = 256, WAVES = 4;
  static constexpr int SUMS = 2 * 32 + 3 * WAVES * 32 + 5 * 32 + WAVES;   // floats, once per parity of the value head
  static constexpr int BYTES = 2 * KQ + 2 * X + G + (int)sizeof(DlGates) + 2 * SUMS * 4;
};

// sum over the 16 lanes of a group, by rotations of a row of lanes
__device__ __forceinline__ float dl_sum16(float x) {
  x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, true));
  x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x124, 0xf, 0xf, true));
  x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x122, 0xf, 0xf, true));
  x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x121, 0xf, 0xf, true));
  return x;
}
// sum over the four groups
__device__ __forceinline__ float dl_sum4(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// four neighbouring columns c .. c + 3 (c a multiple of 4) of a matrix in planes
template <int R, int C, int N>
__device__ __forceinline__ f4 dl_get4(const PlaneMat<R, C, N>& m, int r, int c) {
  const __bf16* p = m.p + r * PlaneMat<R, C, N>::LD + pl_place(c);
  f4 x = DL_ZERO;
#pragma unroll
  for (int q = N - 1; q >= 0; --q) {
    const dl_u2 u = *reinterpret_cast<const dl_u2*>(p + q * PlaneMat<R, C, N>::PLANE);
    x += (f4){__uint_as_float(u[0] << 16), __uint_as_float(u[0] & 0xffff0000u), __uint_as_float(u[1] << 16),
              __uint_as_float(u[1] & 0xffff0000u)};
  }
  return x;
}
template <int R, int C, int N>
__device__ __forceinline__ void dl_put4(const PlaneMat<R, C, N>& m, int r, int c, const f4& x) {
  bf16x8 f[N];
  pl_split<N>(x, DL_ZERO, f);
  __bf16* p = m.p + r * PlaneMat<R, C, N>::LD + pl_place(c);
#pragma unroll
  for (int q = 0; q < N; ++q) {
    const pl_s8 v = __builtin_bit_cast(pl_s8, f[q]);
    *reinterpret_cast<pl_s4*>(p + q * PlaneMat<R, C, N>::PLANE) = (pl_s4){v[0], v[1], v[2], v[3]};
  }
}

// 8 values of an operand as fp32, and their products' sum with another's
struct DlRow {
  f4 a, b;
  __device__ __forceinline__ void load(DlBuf buf, int row, int64_t st, int c0, int D) {
    const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4, v = (int)(n * st + 4 * kg) * 4;
    a = DlIO<float>::load4(buf, dl_lane(c0 + 4 * kg < D, v), (int)(row * st + c0) * 4);
    b = DlIO<float>::load4(buf, dl_lane(c0 + 16 + 4 * kg < D, v), (int)(row * st + c0 + 16) * 4);
  }
  __device__ __forceinline__ void planes(bf16x8* f) const { pl_split<DL_NP>(a, b, f); }
  __device__ __forceinline__ float dot(const f4& x, const f4& y, float s) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) s = __builtin_fmaf(a[i], x[i], __builtin_fmaf(b[i], y[i], s));
    return s;
  }
};

template <typename IO, int DP>
__global__ __launch_bounds__(256, DP > 64 || DlIO<IO>::N > 1 ? 2 : 3) void k_delta_grads(DeltaArgs a) {
  using L = DlGradLds<DP, DlIO<IO>::N>;
  constexpr int NI = DlIO<IO>::N, NP = DL_NP, THREADS = L::THREADS, WAVES = L::WAVES, SIZE = DlIO<IO>::SIZE;
  constexpr int KT = DP / 16 / WAVES;   // key tiles of a wave
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const PlaneMat<DL_C, DP, NI> K{(__bf16*)lds}, Q{(__bf16*)(lds + L::KQ)};
  // 32 columns of dX, U and dO; then dX's and U's place is M1's and M2's
  const PlaneMat<DL_C, 32, NP> X{(__bf16*)(lds + 2 * L::KQ)}, Y{(__bf16*)(lds + 2 * L::KQ + L::X)}, M1 = X, M2 = Y;
  const PlaneMat<DL_C, 32, NI> G{(__bf16*)(lds + 2 * L::KQ + 2 * L::X)};
  DlGates& s = *(DlGates*)(lds + 2 * L::KQ + 2 * L::X + L::G);
  float* sums = (float*)(lds + 2 * L::KQ + 2 * L::X + L::G + sizeof(DlGates));

  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int it = wave & 1, jt = wave < 2 ? it : 1 - it;   // this wave's tile of dP and dA: positions i, j
  const int group = a.Hv / a.Hk, b = blockIdx.x / a.Hk, hk = blockIdx.x % a.Hk, c = blockIdx.y, t0 = c * DL_C;
  const int len = dl_len(a, b), nC = (a.T + DL_C - 1) / DL_C, nc = (len + DL_C - 1) / DL_C;
  const int64_t ks = (int64_t)a.Hk * a.Dk;
  const int d0 = wave * 16 * KT;   // this wave's key columns
  const int outrows = min(a.T - t0, DL_C);
  const DlBuf dqbuf = dl_buf((IO*)a.dq + (((int64_t)b * a.T + t0) * a.Hk + hk) * a.Dk, outrows, ks, a.Dk, SIZE),
              dkbuf = dl_buf((IO*)a.dk + (((int64_t)b * a.T + t0) * a.Hk + hk) * a.Dk, outrows, ks, a.Dk, SIZE);
  f4 gq[KT][2], gk[KT][2];   // rows: key columns, columns: positions
#pragma unroll
  for (int u = 0; u < KT; ++u) gq[u][0] = gq[u][1] = gk[u][0] = gk[u][1] = DL_ZERO;
  auto store = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < KT; ++u)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int at = dl_lane(d0 + 16 * u + 4 * kg < a.Dk, (int)((16 * p + n) * ks + 4 * kg) * SIZE);
        DlIO<IO>::store4(dqbuf, at, (d0 + 16 * u) * SIZE, gq[u][p]);
        DlIO<IO>::store4(dkbuf, at, (d0 + 16 * u) * SIZE, gk[u][p]);
      }
  };
  if (c >= nc) {   // behind the row's length
    store();
    if (tid < outrows)
      for (int h = hk * group; h < (hk + 1) * group; ++h) {
        const int64_t at = ((int64_t)b * a.T + t0 + tid) * a.Hv + h;
        a.dg[at] = 0.f;
        a.dbeta[at] = 0.f;
      }
    return;
  }
  const int left = min(len - t0, DL_C);

  // 8 columns of a row: two waves take dX and V, the others U and dO
  const int pr = (tid & 127) >> 2, pc = (tid & 3) * 8;
  typename DlIO<float>::Raw8 rx;   // dX or U
  typename DlIO<IO>::Raw8 rv;      // V or dO
  auto fetch = [&](int h, int c0) __attribute__((always_inline)) {
    const int64_t row = ((int64_t)b * a.Hv + h) * a.T + t0;
    const bool on = c0 + pc < a.Dv;
    const int v = dl_lane(on, (pr * a.Dv + pc) * 4);
    const bool x = wave < 2;
    const IO* p = x ? (const IO*)a.v + b * a.vs[0] + h * a.vs[2] + t0 * a.vs[1]
                    : (const IO*)a.d_o + b * a.dos[0] + h * a.dos[2] + t0 * a.dos[1];
    const int64_t st = x ? a.vs[1] : a.dos[1];
    rx = DlIO<float>::load8(dl_buf((x ? a.dX : a.U) + row * a.Dv, left, a.Dv, a.Dv, 4), v, c0 * 4);
    rv = DlIO<IO>::load8(dl_buf(p, left, st, a.Dv, SIZE), dl_lane(on, (int)(pr * st + pc) * SIZE), c0 * SIZE);
  };
  float gates[2];
  if (wave == 0) dl_gates_load(gates, a, b, hk * group, t0, len);
  fetch(hk * group, 0);
  DlTile<IO, DP, THREADS> kt, qt;
  kt.load(dl_buf((const IO*)a.k + b * a.ks[0] + hk * a.ks[2] + t0 * a.ks[1], left, a.ks[1], a.Dk, SIZE), a.ks[1], a.Dk, tid);
  qt.load(dl_buf((const IO*)a.q + b * a.qs[0] + hk * a.qs[2] + t0 * a.qs[1], left, a.qs[1], a.Dk, SIZE), a.qs[1], a.Dk, tid);

  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    float* colsum = sums + (h & 1) * L::SUMS;    // [2 tiles of i][32]
    float* part = colsum + 2 * 32;               // [3][waves][32]: q·E1, k·E2, k·E3
    float* rows = part + 3 * WAVES * 32;         // [5][32]: row sums of M, of the terms of dbeta (two tiles of j each), dX·V
    float* dots = rows + 5 * 32;                 // [waves]: sums of S·dS'
    const int64_t bh = (int64_t)b * a.Hv + h, size = (int64_t)a.Dk * a.Dv;
    const float* S0 = c > 0 ? a.S0 + (bh * (nC - 1) + c - 1) * size : a.state0 ? a.state0 + bh * size : nullptr;
    // (after the last chunk of the row's length: the gradient handed in)
    const float* dS = c < nc - 1 ? a.dS + (bh * (nC - 1) + c) * size : a.dstate ? a.dstate + bh * size : nullptr;
    const DlBuf sbuf = dl_buf(S0, S0 != nullptr ? a.Dk : 0, a.Dv, a.Dv, 4),
                ebuf = dl_buf(dS, dS != nullptr ? a.Dk : 0, a.Dv, a.Dv, 4);
    const bool states = S0 != nullptr || dS != nullptr;
    DlRow rs[KT], re[KT];   // (a state that is not there has no rows: nothing is read)
    auto rows_of = [&](int c0) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < KT; ++u) {
        rs[u].load(sbuf, d0 + 16 * u, a.Dv, c0, a.Dv);
        re[u].load(ebuf, d0 + 16 * u, a.Dv, c0, a.Dv);
      }
    };
    if (states) rows_of(0);

    // dP, dA and the states' part
    f4 dp = DL_ZERO, da = DL_ZERO;
    f4 e1[KT][2], e2[KT][2], e3[KT][2];
#pragma unroll
    for (int u = 0; u < KT; ++u)
#pragma unroll
      for (int p = 0; p < 2; ++p) e1[u][p] = e2[u][p] = e3[u][p] = DL_ZERO;
    float dot = 0.f, both = 0.f;
    for (int c0 = 0; c0 < a.Dv; c0 += 32) {
      {
        bf16x8 f[NP];
        DlIO<float>::planes(rx, f);
        (wave < 2 ? X : Y).put8(pr, pc, f);
        if (wave < 2) {
          dot = DlIO<IO>::dot(rv, rx.a, rx.b, dot);
        } else {
          DlIO<IO>::planes(rv, f);
          G.put8(pr, pc, f);
        }
      }
      if (c0 == 0) {
        if (wave == 0) dl_gates(s, gates);
        if (h == hk * group) {
          kt.put(K, tid);
          qt.put(Q, tid);
        }
      }
      __syncthreads();
      if (c0 + 32 < a.Dv) fetch(h, c0 + 32);
      if (jt <= it) {
        bf16x8 go[NI], gx[NP], y[NP];
        G.row(go, 16 * it, 0);
        X.row(gx, 16 * it, 0);
        Y.row(y, 16 * jt, 0);
        dp = pl_mm<NP, NI>(y, go, dp);
        da = pl_mm<NP, NP>(y, gx, da);
      }
      if (states) {
#pragma unroll
        for (int u = 0; u < KT; ++u) {
          bf16x8 y[NP], f[NP];
          both = rs[u].dot(re[u].a, re[u].b, both);
          if (S0 != nullptr) {
            rs[u].planes(y);
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              bf16x8 go[NI];
              G.row(go, 16 * p, 0);
              X.row(f, 16 * p, 0);
              e1[u][p] = pl_mm<NP, NI>(y, go, e1[u][p]);
              e2[u][p] = pl_mm<NP, NP>(y, f, e2[u][p]);
            }
          }
          if (dS != nullptr) {
            re[u].planes(y);
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              Y.row(f, 16 * p, 0);
              e3[u][p] = pl_mm<NP, NP>(y, f, e3[u][p]);
            }
          }
        }
        if (c0 + 32 < a.Dv) rows_of(c0 + 32);
      }
      __syncthreads();
    }
    if (wave < 2) {
      dot += __shfl_xor(dot, 1);
      dot += __shfl_xor(dot, 2);
      if ((tid & 3) == 0) rows[4 * 32 + pr] = dot;
    }
    {
      const int i = 16 * it + n;   // this lane's position
      f4 kk = DL_ZERO, qk = DL_ZERO, m1 = DL_ZERO, m2 = DL_ZERO, cs = DL_ZERO;
      float rm = 0.f, rb = 0.f;
      if (jt <= it) {
        const float be = s.beta[i];
        const double gi = s.G[i];
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) {
          bf16x8 ki[NI], qi[NI], kj[NI];
          K.row(ki, 16 * it, t);
          Q.row(qi, 16 * it, t);
          K.row(kj, 16 * jt, t);
          kk = pl_mm<NI, NI>(kj, ki, kk);
          qk = pl_mm<NI, NI>(kj, qi, qk);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = 16 * jt + 4 * kg + r;
          const float d = j <= i ? dl_exp2(gi - s.G[j]) : 0.f;
          const float w = j < i ? -d * da[r] : 0.f;
          m1[r] = j <= i ? a.scale * d * dp[r] : 0.f;
          m2[r] = be * w;
          cs[r] = m1[r] * qk[r] + m2[r] * kk[r];
          rm += cs[r];
          rb += w * kk[r];
          cs[r] = dl_sum16(cs[r]);
        }
        rm = dl_sum4(rm);
        rb = dl_sum4(rb);
      }
      dl_put4(M1, i, 16 * jt + 4 * kg, m1);
      dl_put4(M2, i, 16 * jt + 4 * kg, m2);
      if (n == 0) *reinterpret_cast<f4*>(colsum + it * 32 + 16 * jt + 4 * kg) = cs;
      if (kg == 0) {
        rows[(wave >> 1) * 32 + i] = rm;
        rows[(2 + (wave >> 1)) * 32 + i] = rb;
      }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      float r1 = 0.f, r2 = 0.f, r3 = 0.f;
      if (states) {
        const float gam = s.gam[16 * p + n], be = s.beta[16 * p + n], rest = s.rest[16 * p + n];
#pragma unroll
        for (int u = 0; u < KT; ++u) {
          const f4 kx = dl_get4(K, 16 * p + n, d0 + 16 * u + 4 * kg), qx = dl_get4(Q, 16 * p + n, d0 + 16 * u + 4 * kg);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            r1 = __builtin_fmaf(qx[r], e1[u][p][r], r1);
            r2 = __builtin_fmaf(kx[r], e2[u][p][r], r2);
            r3 = __builtin_fmaf(kx[r], e3[u][p][r], r3);
          }
          gq[u][p] += (a.scale * gam) * e1[u][p];
          gk[u][p] += rest * e3[u][p] - (be * gam) * e2[u][p];
        }
        r1 = dl_sum4(r1);
        r2 = dl_sum4(r2);
        r3 = dl_sum4(r3);
      }
      if (kg == 0) {
        part[wave * 32 + 16 * p + n] = r1;
        part[(WAVES + wave) * 32 + 16 * p + n] = r2;
        part[(2 * WAVES + wave) * 32 + 16 * p + n] = r3;
      }
    }
    if (states) both = dl_sum4(dl_sum16(both));
    if (lane == 0) dots[wave] = both;
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      bf16x8 m1[NP], m1t[NP], m2[NP], m2t[NP];
      M1.row(m1, 16 * p, 0);
      M2.row(m2, 16 * p, 0);
      M1.col(m1t, 0, 16 * p);
      M2.col(m2t, 0, 16 * p);
#pragma unroll
      for (int u = 0; u < KT; ++u) {
        bf16x8 f[NI];
        K.col(f, 0, d0 + 16 * u);
        gq[u][p] = pl_mm<NI, NP>(f, m1, gq[u][p]);
        gk[u][p] = pl_mm<NI, NP>(f, m2, gk[u][p]);
        gk[u][p] = pl_mm<NI, NP>(f, m2t, gk[u][p]);
        Q.col(f, 0, d0 + 16 * u);
        gk[u][p] = pl_mm<NI, NP>(f, m1t, gk[u][p]);
      }
    }
    const bool more = h + 1 < (hk + 1) * group;
    if (more) {
      fetch(h + 1, 0);
      __syncthreads();   // M is read: the next value head's dX and U take its place
    }
    if (wave == 0) {
      const int j = lane & 31;
      const float gj = s.gam[j];
      float qe = 0.f, ke = 0.f, kd = 0.f;
      double sd = 0.0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        qe += part[w * 32 + j];
        ke += part[(WAVES + w) * 32 + j];
        kd += part[(2 * WAVES + w) * 32 + j];
        sd += dots[w];
      }
      const double leave = (double)s.rest[j] * kd;
      double at = (double)rows[j] + rows[32 + j] + (double)a.scale * gj * qe - (double)s.beta[j] * gj * ke - leave;
      at -= (double)colsum[j] + (double)colsum[32 + j];
      double all = leave;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        all += __shfl_xor(all, o, 32);
        const double down = __shfl_down(at, o, 32);
        if (j + o < 32) at += down;
      }
      at += all + (double)s.gam[DL_C - 1] * sd;
      const int64_t out = ((int64_t)b * a.T + t0 + j) * a.Hv + h;
      if (lane < 32 && j < outrows) {
        a.dg[out] = j < left ? (float)at : 0.f;
        a.dbeta[out] = j < left ? rows[128 + j] - gj * ke + (rows[64 + j] + rows[96 + j]) : 0.f;
      }
      if (more) dl_gates_load(gates, a, b, h + 1, t0, len);
    }
  }
#pragma unroll
  for (int p = 0; p < 2; ++p)
    if (16 * p + n >= left)
#pragma unroll
      for (int u = 0; u < KT; ++u) gq[u][p] = gk[u][p] = DL_ZERO;
  store();
}

// ------------------------------------------------------------- one token ----
// A workgroup owns 32 value columns of one (row, value head) state: read once, kept in registers, written once.  Sᵀk and
// Sᵀq come out of the same pass, since o = scale (a Sᵀq + (k·q) u) with u = b (v − a Sᵀk).
template <typename IO>
__global__ __launch_bounds__(256) void k_delta_step(DeltaArgs a, int64_t sb) {
  __shared__ float part[4][2][32], uo[2][32];
  const int tid = threadIdx.x, wave = tid >> 6, c4 = (tid & 7) * 4, rg = tid >> 3;   // 32 groups of rows
  const int b = blockIdx.x / a.Hv, h = blockIdx.x % a.Hv, hk = h / (a.Hv / a.Hk), col = blockIdx.y * 32 + c4;
  const bool mine = col < a.Dv;
  float* S = a.state + b * sb + (int64_t)h * a.Dk * a.Dv + col;
  const IO* q = (const IO*)a.q + b * a.qs[0] + hk * a.qs[2];
  const IO* k = (const IO*)a.k + b * a.ks[0] + hk * a.ks[2];
  f4 x[4];
  float kx[4], qx[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = rg + 32 * i;
    const bool on = d < a.Dk;
    x[i] = on && mine ? *reinterpret_cast<const f4*>(S + (int64_t)d * a.Dv) : (f4){0.f, 0.f, 0.f, 0.f};
    kx[i] = on ? (float)k[d] : 0.f;
    qx[i] = on ? (float)q[d] : 0.f;
  }
  const float gam = expf(a.g[b * a.gs[0] + h * a.gs[2]]), be = a.beta[b * a.bs[0] + h * a.bs[2]];
  f4 sk = {0.f, 0.f, 0.f, 0.f}, sq = sk;
  float kq = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // a decay of 0 leaves nothing of the old state, infinities included
    x[i] = gam == 0.f ? (f4){0.f, 0.f, 0.f, 0.f} : x[i] * gam;
    sk += x[i] * kx[i];
    sq += x[i] * qx[i];
    kq = __builtin_fmaf(kx[i], qx[i], kq);
  }
#pragma unroll
  for (int o = 8; o < 64; o <<= 1) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sk[e] += __shfl_xor(sk[e], o);
      sq[e] += __shfl_xor(sq[e], o);
    }
    kq += __shfl_xor(kq, o);
  }
  if ((tid & 63) < 8) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      part[wave][0][c4 + e] = sk[e];
      part[wave][1][c4 + e] = sq[e];
    }
    if ((tid & 63) == 0) uo[0][wave] = kq;
  }
  __syncthreads();
  kq = (uo[0][0] + uo[0][1]) + (uo[0][2] + uo[0][3]);
  f4 u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float k0 = (part[0][0][c4 + e] + part[1][0][c4 + e]) + (part[2][0][c4 + e] + part[3][0][c4 + e]);
    const float vv = mine ? (float)((const IO*)a.v)[b * a.vs[0] + h * a.vs[2] + col + e] : 0.f;
    u[e] = be * (vv - k0);
  }
  if (!mine) return;
  if (rg == 0) {
    IO* o = (IO*)a.o + ((int64_t)b * a.Hv + h) * a.Dv + col;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float q0 = (part[0][1][c4 + e] + part[1][1][c4 + e]) + (part[2][1][c4 + e] + part[3][1][c4 + e]);
      o[e] = (IO)(a.scale * __builtin_fmaf(kq, u[e], q0));
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = rg + 32 * i;
    if (d < a.Dk) {
      f4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(kx[i], u[e], x[i][e]);
      *reinterpret_cast<f4*>(S + (int64_t)d * a.Dv) = y;
    }
  }
}

// ------------------------------------------------------------------ host ----
static int delta_check(const DeltaArgs& a, int type) {
  if (type != 0 && type != 1) return RG_ERR_ARG;
  if (a.B <= 0 || a.T <= 0 || a.Hk <= 0 || a.Hv <= 0 || a.Hv % a.Hk) return RG_ERR_SHAPE;
  if (a.Dk <= 0 || a.Dk > 128 || a.Dk % 8 || a.Dv <= 0 || a.Dv > 128 || a.Dv % 8) return RG_ERR_SHAPE;
  if ((int64_t)a.B * a.Hv >= (1 << 24) || (a.T + DL_C - 1) / DL_C > 65535) return RG_ERR_SHAPE;
  if (a.q == nullptr || a.k == nullptr || a.v == nullptr || a.g == nullptr || a.beta == nullptr) return RG_ERR_ARG;
  return RG_OK;
}
// positions at least a row apart, a chunk's 32 of them within a buffer's 2 GB
static bool delta_apart(const int64_t* s, int T, int width) { return T == 1 || (s[1] >= width && s[1] < (1 << 23)); }
// so lie the contiguous outputs' positions, all heads of one next to another
static bool delta_wide(int Hk, int Hv, int Dk, int Dv) { return (int64_t)Hk * Dk >= (1 << 23) || (int64_t)Hv * Dv >= (1 << 23); }
// rows at multiples of 16 bytes
static bool delta_aligned(const void* p, const int64_t* s, int type) {
  const int64_t e = type == 0 ? 4 : 2;
  return ((uintptr_t)p & 15) == 0 && s[0] * e % 16 == 0 && s[1] * e % 16 == 0 && s[2] * e % 16 == 0;
}

// column tiles a wave owns: as many as its registers hold (the chunk's P and T are made once for all of them), fewer
// where that would leave CUs without work
static int delta_ct(int64_t heads, int Dk, int Dv, int type) {
  int ct = (Dk <= 64 ? 4 : 2) / (type == 0 ? 2 : 1);
  while (ct > 1 && (16 * (ct / 2) >= Dv || heads * ((Dv + 16 * ct - 1) / (16 * ct)) < 1024)) ct /= 2;
  return ct;
}

// Segments.  A chunk takes a wave of 1, 2, 4 column tiles about 4.5, 7.5, 12 us with a SIMD of its own (1024 of them), 1.75
// times that beside another (2048 at once); with segments there are two passes, the first over the transition's
// columns too but without outputs, each a segment long, and a join of 1 to 1.5 us a segment.  Measured at width 128,
// 4 x 8 heads x 4096 positions, forward and backward: 8 segments 819 us, 16 749, 32 808, 64 960; 8 heads x 8191
// positions, forward: 8 segments 269 us, 16 188, 32 192, 37 (a wave too many for the SIMDs in either pass) 225, 64 241
// (before the joins and the gradients' kernel were made faster: then 16 612, 20 589, 24 651, 32 674, and 16 180, 20 190, 32 176).
struct DeltaCut {
  int nseg, per;
};
static DeltaCut delta_cut(int B, int T, int Hv, int Dk, int Dv) {
  const int nC = (T + DL_C - 1) / DL_C;
  const int64_t heads = (int64_t)B * Hv;
  auto chunk = [&](int nseg, int cols) {
    const int ct = delta_ct(heads * nseg, Dk, Dv, 1);
    const int64_t waves = heads * nseg * ((cols + 16 * ct - 1) / (16 * ct));
    return (ct == 1 ? 4.5 : ct == 2 ? 7.5 : 12.0) * (waves > 1024 ? 1.75 : 1.0) * (double)((waves + 2047) / 2048);
  };
  DeltaCut best = {1, nC};
  double cost = nC * chunk(1, Dv);
  for (int want = 2; want <= 64 && want <= nC; ++want) {
    const int per = (nC + want - 1) / want, nseg = (nC + per - 1) / per;
    const double t = per * (chunk(nseg, Dv) + 0.7 * chunk(nseg, Dv + Dk)) + 1.06 * nseg + 15.0;
    if (t < cost) cost = t, best = {nseg, per};
  }
  return best;
}

template <typename K>
static int delta_go(K kern, dim3 grid, int threads, int shared, const DeltaArgs& a, hipStream_t st) {
  if (shared > 64 * 1024 &&
      hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, shared) != hipSuccess)
    return RG_ERR_LAUNCH;
  hipLaunchKernelGGL(kern, grid, dim3(threads), shared, st, a);
  RG_LAUNCH_CHECK();
  return RG_OK;
}

template <typename IO, int DP, int CT>
static int delta_fwd_ct(const DeltaArgs& a, hipStream_t st) {
  const int heads = a.B * a.Hv, vb = (a.Dv + 16 * CT - 1) / (16 * CT), kb = (a.Dk + 16 * CT - 1) / (16 * CT);
  if (a.nseg > 1) {
    int rc = delta_go(k_delta_fwd<IO, DP, CT, true>, dim3(heads * a.nseg, vb + kb), 64, 0, a, st);
    if (rc != RG_OK) return rc;
    rc = delta_go(k_delta_join<DP, false>, dim3(heads, (a.Dv + 15) / 16), 4 * DP, 0, a, st);
    if (rc != RG_OK) return rc;
  }
  return delta_go(k_delta_fwd<IO, DP, CT, false>, dim3(heads * a.nseg, vb), 64, 0, a, st);
}
template <typename IO, int DP, int CT>
static int delta_scan_ct(const DeltaArgs& a, hipStream_t st) {
  const int heads = a.B * a.Hv, vb = (a.Dv + 16 * CT - 1) / (16 * CT);
  if (a.nseg > 1) {
    int rc = delta_go(k_delta_scan<IO, DP, CT, true>, dim3(heads * a.nseg, vb), 64, 0, a, st);
    if (rc != RG_OK) return rc;
    rc = delta_go(k_delta_join<DP, true>, dim3(heads, (a.Dv + 15) / 16), 4 * DP, 0, a, st);
    if (rc != RG_OK) return rc;
  }
  return delta_go(k_delta_scan<IO, DP, CT, false>, dim3(heads * a.nseg, vb), 64, 0, a, st);
}
template <typename IO, int DP>
static int delta_fwd_t(const DeltaArgs& a, hipStream_t st) {
  const int ct = delta_ct((int64_t)a.B * a.Hv * a.nseg, a.Dk, a.Dv, DlIO<IO>::N == 3 ? 0 : 1);
  if constexpr (DP <= 64 && DlIO<IO>::N == 1)
    if (ct == 4) return delta_fwd_ct<IO, DP, 4>(a, st);
  if constexpr (DP <= 64 || DlIO<IO>::N == 1)
    if (ct >= 2) return delta_fwd_ct<IO, DP, 2>(a, st);
  return delta_fwd_ct<IO, DP, 1>(a, st);
}
template <typename IO, int DP>
static int delta_bwd_t(const DeltaArgs& a, hipStream_t st) {
  const int ct = delta_ct((int64_t)a.B * a.Hv * a.nseg, a.Dk, a.Dv, DlIO<IO>::N == 3 ? 0 : 1);
  int rc = RG_OK;
  bool done = false;
  if constexpr (DP <= 64 && DlIO<IO>::N == 1)
    if (ct == 4) rc = delta_scan_ct<IO, DP, 4>(a, st), done = true;
  if constexpr (DP <= 64 || DlIO<IO>::N == 1)
    if (!done && ct >= 2) rc = delta_scan_ct<IO, DP, 2>(a, st), done = true;
  if (!done) rc = delta_scan_ct<IO, DP, 1>(a, st);
  if (rc != RG_OK) return rc;
  constexpr int GP = DP > 64 ? 128 : 64;   // (two key tiles at least: four waves have one or two each)
  using L = DlGradLds<GP, DlIO<IO>::N>;
  return delta_go(k_delta_grads<IO, GP>, dim3(a.B * a.Hk, (a.T + DL_C - 1) / DL_C), L::THREADS, L::BYTES, a, st);
}
#define DL_DISPATCH(F)                                                                             \
  (type == 0 ? (a.Dk <= 32 ? F<float, 32>(a, st) : a.Dk <= 64 ? F<float, 64>(a, st) : F<float, 128>(a, st)) \
             : (a.Dk <= 32 ? F<__bf16, 32>(a, st) : a.Dk <= 64 ? F<__bf16, 64>(a, st) : F<__bf16, 128>(a, st)))

// (one position: its stride means nothing, but the rows behind it have to lie behind the buffer's end)
static void delta_strides(DeltaArgs& a, const int64_t* strides, int T) {
  int64_t s[18];
  for (int i = 0; i < 18; ++i) s[i] = T == 1 && i % 3 == 1 ? 128 : strides[i];
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = s[i];
    a.ks[i] = s[3 + i];
    a.vs[i] = s[6 + i];
    a.gs[i] = s[9 + i];
    a.bs[i] = s[12 + i];
    a.dos[i] = s[15 + i];
  }
}
static void delta_segments(DeltaArgs& a, float* trans, float* local) {
  const DeltaCut c = delta_cut(a.B, a.T, a.Hv, a.Dk, a.Dv);
  a.nseg = c.nseg, a.per = c.per, a.trans = trans, a.local = local;
}

extern "C" int64_t rg_delta_chunk_floats(int B, int T, int Hv, int Dk, int Dv) {
  return T > 0 ? (int64_t)B * Hv * ((T + DL_C - 1) / DL_C - 1) * Dk * Dv : 0;
}
extern "C" int rg_delta_segments(int B, int T, int Hv, int Dk, int Dv) {
  return B > 0 && T > 0 ? delta_cut(B, T, Hv, Dk, Dv).nseg : 1;
}

extern "C" int64_t rg_delta_trans_floats(int B, int T, int Hv, int Dk, int Dv) {
  const int n = rg_delta_segments(B, T, Hv, Dk, Dv);
  return n > 1 ? (int64_t)B * Hv * n * dl_trans_floats(Dk) : 0;
}

extern "C" int rg_delta_fwd(const void* q, const void* k, const void* v, const float* g, const float* beta,
                            const int64_t* strides, const int64_t* lens, const float* state0, int type, int B, int T,
                            int Hk, int Hv, int Dk, int Dv, float scale, void* o, float* state, float* U, float* S0,
                            float* trans, float* local, hipStream_t st) {
  DeltaArgs a = {};
  if (strides == nullptr) return RG_ERR_ARG;
  delta_strides(a, strides, T);
  a.q = q, a.k = k, a.v = v, a.g = g, a.beta = beta, a.lens = lens, a.state0 = state0;
  a.B = B, a.T = T, a.Hk = Hk, a.Hv = Hv, a.Dk = Dk, a.Dv = Dv, a.scale = scale, a.o = o, a.state = state, a.U = U;
  a.S0 = U != nullptr && T > DL_C ? S0 : nullptr;
  const int rc = delta_check(a, type);
  if (rc != RG_OK) return rc;
  if (delta_wide(Hk, Hv, Dk, Dv)) return RG_ERR_SHAPE;
  if (!delta_apart(a.qs, T, Dk) || !delta_apart(a.ks, T, Dk) || !delta_apart(a.vs, T, Dv) || !delta_apart(a.gs, T, 1) ||
      !delta_apart(a.bs, T, 1))
    return RG_ERR_ARG;
  delta_segments(a, trans, local);
  if (o == nullptr || state == nullptr || (U != nullptr && T > DL_C && S0 == nullptr) || (a.nseg > 1 && (trans == nullptr || local == nullptr)))
    return RG_ERR_ARG;
  if (!delta_aligned(q, a.qs, type) || !delta_aligned(k, a.ks, type) || (((uintptr_t)o | (uintptr_t)trans | (uintptr_t)local) & 15))
    return RG_ERR_ARG;
  return DL_DISPATCH(delta_fwd_t);
}

extern "C" int rg_delta_bwd(const void* q, const void* k, const void* v, const float* g, const float* beta,
                            const void* d_o, const int64_t* strides, const int64_t* lens, const float* state0,
                            const float* dstate, const float* U, const float* S0, const float* trans, int type, int B, int T,
                            int Hk, int Hv, int Dk, int Dv, float scale, float* dX, float* dS, float* local, void* dq,
                            void* dk, void* dv, float* dg, float* dbeta, float* dstate0, hipStream_t st) {
  DeltaArgs a = {};
  if (strides == nullptr) return RG_ERR_ARG;
  delta_strides(a, strides, T);
  a.q = q, a.k = k, a.v = v, a.g = g, a.beta = beta, a.d_o = d_o, a.lens = lens, a.state0 = state0, a.dstate = dstate;
  a.B = B, a.T = T, a.Hk = Hk, a.Hv = Hv, a.Dk = Dk, a.Dv = Dv, a.scale = scale;
  a.U = const_cast<float*>(U), a.S0 = const_cast<float*>(S0), a.dX = dX, a.dS = dS;
  a.dq = dq, a.dk = dk, a.dv = dv, a.dg = dg, a.dbeta = dbeta, a.dstate0 = dstate0;
  const int rc = delta_check(a, type);
  if (rc != RG_OK) return rc;
  if (delta_wide(Hk, Hv, Dk, Dv)) return RG_ERR_SHAPE;
  if (!delta_apart(a.qs, T, Dk) || !delta_apart(a.ks, T, Dk) || !delta_apart(a.vs, T, Dv) || !delta_apart(a.gs, T, 1) ||
      !delta_apart(a.bs, T, 1))
    return RG_ERR_ARG;
  delta_segments(a, const_cast<float*>(trans), local);
  if (!delta_apart(a.dos, T, Dv)) return RG_ERR_ARG;
  if (d_o == nullptr || U == nullptr || dX == nullptr || dq == nullptr || dk == nullptr || dv == nullptr ||
      dg == nullptr || dbeta == nullptr || (T > DL_C && (S0 == nullptr || dS == nullptr)) ||
      (a.nseg > 1 && (trans == nullptr || local == nullptr)))
    return RG_ERR_ARG;
  if (!delta_aligned(q, a.qs, type) || !delta_aligned(k, a.ks, type) || !delta_aligned(v, a.vs, type) ||
      !delta_aligned(d_o, a.dos, type) || (((uintptr_t)dq | (uintptr_t)dk) & 15) ||
      (((uintptr_t)state0 | (uintptr_t)dstate | (uintptr_t)U | (uintptr_t)S0 | (uintptr_t)dX | (uintptr_t)dS |
        (uintptr_t)trans | (uintptr_t)local) & 15))
    return RG_ERR_ARG;
  return DL_DISPATCH(delta_bwd_t);
}

extern "C" int rg_delta_step(const void* q, const void* k, const void* v, const float* g, const float* beta,
                             const int64_t* strides, int type, int B, int Hk, int Hv, int Dk, int Dv, float scale,
                             float* state, int64_t state_stride, void* o, hipStream_t st) {
  DeltaArgs a = {};
  if (strides == nullptr) return RG_ERR_ARG;
  delta_strides(a, strides, 1);
  a.q = q, a.k = k, a.v = v, a.g = g, a.beta = beta, a.state = state, a.o = o;
  a.B = B, a.T = 1, a.Hk = Hk, a.Hv = Hv, a.Dk = Dk, a.Dv = Dv, a.scale = scale;
  const int rc = delta_check(a, type);
  if (rc != RG_OK) return rc;
  if (state == nullptr || o == nullptr || ((uintptr_t)state & 15) || state_stride % 4) return RG_ERR_ARG;
  if (B > 1 && state_stride < (int64_t)Hv * Dk * Dv) return RG_ERR_ARG;
  const dim3 grid(B * Hv, (Dv + 31) / 32);
  if (type == 0)
    hipLaunchKernelGGL(k_delta_step<float>, grid, dim3(256), 0, st, a, state_stride);
  else
    hipLaunchKernelGGL(k_delta_step<__bf16>, grid, dim3(256), 0, st, a, state_stride);
  RG_LAUNCH_CHECK();
  return RG_OK;
}
