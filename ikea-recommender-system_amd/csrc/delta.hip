// Gated delta rule: a linear-attention recurrence beside the GRU (csrc/gru.hip), per value head with a Dk x Dv state
//     S_t = a_t S_{t-1} + b_t k_t (v_t − a_t S_{t-1}ᵀ k_t)ᵀ,   o_t = scale · S_tᵀ q_t,   a_t = exp(g_t)
//
// Chunks of 64 positions.  With G_i the running sum of g inside a chunk, D_ij = exp(G_i − G_j), S the state before it:
//     A_ij = b_i D_ij k_i·k_j (j < i),  P_ij = scale · D_ij q_i·k_j (j <= i),  T = (1 + A)^-1   (unit lower triangular)
//     X = diag(b)(V − diag(e^G) K S),   U = T X,   O = scale · diag(e^G) Q S + P U
//     S' = e^{G_end} S + Kᵀ diag(D_end) U
// Backwards, with dS the gradient of S':
//     dU = Pᵀ dO + diag(D_end) K dS,   dX = Tᵀ dU,   dV = diag(b) dX
//     dS_prev = e^{G_end} dS + Qᵀ diag(scale · e^G) dO − Kᵀ diag(b e^G) dX
// and, per chunk and independent of the others, dP = dO Uᵀ, dA = −dX Uᵀ and the rest (k_delta_grads).
//
// The state, G and every sum are fp32 or wider (G in fp64: differences of long sums enter an exponential).  Products run
// on bf16 MFMA with fp32 operands split into planes (planes.h): three planes (six products) for fp32 inputs; bf16
// inputs are one exact plane.  Positions at or behind a sequence's length are read as k = v = q = 0, b = 0, g = 0,
// which leaves the state as it is; nothing is read there.
#include "planes.h"

#define DL_C 64
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
};

template <typename IO>
struct DlIO;
template <>
struct DlIO<float> {
  static constexpr int N = 3;
  static __device__ __forceinline__ void load8(const float* p, bf16x8* f) {
    pl_split<3>(*reinterpret_cast<const f4*>(p), *reinterpret_cast<const f4*>(p + 4), f);
  }
};
template <>
struct DlIO<__bf16> {
  static constexpr int N = 1;
  static __device__ __forceinline__ void load8(const __bf16* p, bf16x8* f) {
    f[0] = *reinterpret_cast<const bf16x8*>(p);
  }
};

__device__ __forceinline__ int dl_len(const DeltaArgs& a, int b) {
  if (a.lens == nullptr) return a.T;
  const int64_t n = a.lens[b];
  return n < 0 ? 0 : n > a.T ? a.T : (int)n;
}

// rows t0 .. t0 + 63 of a (T, D) operand into planes; zeros behind `len` and behind column D
template <typename IO, int DP>
__device__ __forceinline__ void dl_load(const PlaneMat<DL_C, DP, DlIO<IO>::N>& m, const IO* base, int64_t st, int t0,
                                        int len, int D, int tid, int nthreads) {
  constexpr int N = DlIO<IO>::N;
  for (int e = tid; e < DL_C * (DP / 8); e += nthreads) {
    const int r = e / (DP / 8), c = (e % (DP / 8)) * 8;
    bf16x8 f[N] = {};
    if (t0 + r < len && c < D) DlIO<IO>::load8(base + (int64_t)(t0 + r) * st + c, f);
    m.put8(r, c, f);
  }
}

// per-position scalars of a chunk
struct DlGates {
  double G[DL_C];        // running sum of g
  float gam[DL_C];       // exp(G_i)
  float rest[DL_C];      // exp(G_end − G_i)
  float beta[DL_C];
};
// one wave
__device__ __forceinline__ void dl_gates(DlGates& s, const DeltaArgs& a, int b, int h, int t0, int len) {
  const int i = threadIdx.x & 63, t = t0 + i;
  double g = 0.0;
  float be = 0.f;
  if (t < len) {
    g = a.g[b * a.gs[0] + t * a.gs[1] + h * a.gs[2]];
    g = g < DL_G_MIN ? DL_G_MIN : g;   // NaN stays
    be = a.beta[b * a.bs[0] + t * a.bs[1] + h * a.bs[2]];
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double up = __shfl_up(g, o);
    if (i >= o) g += up;
  }
  const double end = __shfl(g, 63);
  s.G[i] = g;
  s.gam[i] = expf((float)g);
  s.rest[i] = expf((float)(end - g));
  s.beta[i] = be;
}

// T and P of a chunk in planes, from K and Q in planes and the gates.  P's place holds A first: its off-diagonal blocks
// in planes, its diagonal 16 x 16 blocks in fp32 in the quadrant of rows 0 .. 31 and columns 32 .. 63, which no product
// reads.  The other upper tiles must be zero before and stay so.  All waves call it; ends with every wave's writes visible.
template <int NP>
__device__ __forceinline__ float* dl_diag(const PlaneMat<DL_C, 64, NP>& P, int r) {   // row r of 64: 16 floats
  using M = PlaneMat<DL_C, 64, NP>;
  return reinterpret_cast<float*>(P.p + (r >> 5) * M::PLANE + (r & 31) * M::LD + 32);
}
template <int DP, int NI, int NP>
__device__ __forceinline__ void dl_prep(const PlaneMat<DL_C, DP, NI>& K, const PlaneMat<DL_C, DP, NI>& Q,
                                        const PlaneMat<DL_C, 64, NP>& P, const PlaneMat<DL_C, 64, NP>& T,
                                        const DlGates& s, float scale, int nt, int wave, int nw) {
  static_assert(NP >= 2, "the diagonal blocks need two planes' room");
  const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;
  auto lower = [&](const PlaneMat<DL_C, DP, NI>& X, auto use) {   // the lower tiles of X Kᵀ times D
    for (int job = wave; job < 10; job += nw) {
      const int it = job < 1 ? 0 : job < 3 ? 1 : job < 6 ? 2 : 3, jt = job - it * (it + 1) / 2;
      if (it >= nt) break;
      f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < DP / 32; ++t) {
        bf16x8 xi[NI], kj[NI];
        X.row(xi, 16 * it, t);
        K.row(kj, 16 * jt, t);
        x = pl_mm<NI, NI>(xi, kj, x);
      }
      const int j = 16 * jt + n;
      const double gj = s.G[j];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * it + 4 * kg + r;
        use(i, j, it == jt, expf((float)(s.G[i] - gj)) * x[r]);
      }
    }
  };
  lower(K, [&](int i, int j, bool diag, float x) {
    x = j < i ? s.beta[i] * x : 0.f;
    if (diag)
      dl_diag(P, i)[j & 15] = x;
    else
      P.put(i, j, x);
  });
  __syncthreads();
  // T of the diagonal blocks: lane (kg, n) solves column n of block kg forwards
  if (wave == 0 && kg < nt) {
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const f4* row = reinterpret_cast<const f4*>(dl_diag(P, 16 * kg + i));
      float x = i == n ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) x = __builtin_fmaf(-row[j >> 2][j & 3], t[j], x);
      t[i] = x;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) T.put(16 * kg + i, 16 * kg + n, t[i]);
  }
  __syncthreads();
  // T_10 = −T_11 (A_10 T_00) inside each 32 x 32 diagonal block; the operands' other halves are zeroed
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  if (nt > 1) {
    for (int p = wave; 2 * p + 1 < nt; p += nw) {
      bf16x8 x[NP], y[NP];
      P.row(x, 16 * (2 * p + 1), p);
      T.col(y, p, 32 * p);
#pragma unroll
      for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int e = 4; e < 8; ++e) y[q][e] = (__bf16)0.f, x[q][e] = (__bf16)0.f;
      const f4 m1 = pl_mm<NP, NP>(x, y, zero);
      T.row(x, 16 * (2 * p + 1), p);
#pragma unroll
      for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[q][e] = (__bf16)0.f;
      pl_split<NP>(zero, m1, y);
      const f4 m2 = pl_mm<NP, NP>(x, y, zero);
#pragma unroll
      for (int r = 0; r < 4; ++r) T.put(32 * p + 16 + 4 * kg + r, 32 * p + n, -m2[r]);
    }
    __syncthreads();
  }
  if (nt > 2) {   // and of the 64 x 64 block
    for (int jt = wave; jt < 2; jt += nw) {
      bf16x8 x[NP], y[NP];
      T.col(y, 0, 16 * jt);
      f4 m[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        P.row(x, 32 + 16 * r, 0);
        m[r] = pl_mm<NP, NP>(x, y, zero);
      }
      if (nt < 4) m[1] = zero;
      pl_split<NP>(m[0], m[1], y);
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (2 + r < nt) {
          T.row(x, 32 + 16 * r, 1);
          const f4 m2 = pl_mm<NP, NP>(x, y, zero);
#pragma unroll
          for (int i = 0; i < 4; ++i) T.put(32 + 16 * r + 4 * kg + i, 16 * jt + n, -m2[i]);
        }
    }
    __syncthreads();
  }
  lower(Q, [&](int i, int j, bool diag, float x) { P.put(i, j, j <= i ? scale * x : 0.f); });
  __syncthreads();
}

template <int DP, int NI, int NP>
struct DlLds {
  static constexpr int KQ = PlaneMat<DL_C, DP, NI>::BYTES, M = PlaneMat<DL_C, 64, NP>::BYTES;
  static constexpr int BYTES = 2 * KQ + 2 * M + (int)sizeof(DlGates);
  static_assert(BYTES <= 160 * 1024, "LDS of a CU");
};

// clear the planes of P and T: their upper triangles (and the parts behind a short sequence) stay zero
__device__ __forceinline__ void dl_clear(void* p, int bytes) {
  for (int i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16)
    *reinterpret_cast<f4*>(reinterpret_cast<uint8_t*>(p) + i) = (f4){0.f, 0.f, 0.f, 0.f};
}

// ---------------------------------------------------------------- forward ----
// One workgroup per (batch row, value head, group of value columns); a wave owns 16 value columns and their part of
// the state, which stays in its accumulators from the first chunk to the last.  The chunk's K, Q, P, T are shared.
template <typename IO, int DP, int NP>
__global__ __launch_bounds__(512) void k_delta_fwd(DeltaArgs a) {
  constexpr int NI = DlIO<IO>::N, KT = DP / 32;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  using L = DlLds<DP, NI, NP>;
  const PlaneMat<DL_C, DP, NI> K{(__bf16*)lds}, Q{(__bf16*)(lds + L::KQ)};
  const PlaneMat<DL_C, 64, NP> P{(__bf16*)(lds + 2 * L::KQ)}, T{(__bf16*)(lds + 2 * L::KQ + L::M)};
  DlGates& s = *(DlGates*)(lds + 2 * L::KQ + 2 * L::M);

  const int tid = threadIdx.x, nth = blockDim.x, lane = tid & 63, n = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = nth >> 6;
  const int b = blockIdx.x / a.Hv, h = blockIdx.x % a.Hv, hk = h / (a.Hv / a.Hk);
  const int len = dl_len(a, b), col = (blockIdx.y * nw + wave) * 16 + n;
  const bool mine = col < a.Dv;
  const int nC = (a.T + DL_C - 1) / DL_C;
  const IO* q = (const IO*)a.q + b * a.qs[0] + hk * a.qs[2];
  const IO* k = (const IO*)a.k + b * a.ks[0] + hk * a.ks[2];
  const IO* v = (const IO*)a.v + b * a.vs[0] + h * a.vs[2] + col;
  const int64_t bh = (int64_t)b * a.Hv + h;
  IO* o = (IO*)a.o + ((int64_t)b * a.T * a.Hv + h) * a.Dv + col;   // row stride Hv * Dv
  const int64_t os = (int64_t)a.Hv * a.Dv;

  f4 S[2 * KT];
#pragma unroll
  for (int u = 0; u < 2 * KT; ++u)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * u + 4 * kg + r;
      S[u][r] = a.state0 != nullptr && mine && d < a.Dk ? a.state0[(bh * a.Dk + d) * a.Dv + col] : 0.f;
    }
  dl_clear(P.p, 2 * L::M);

  for (int t0 = 0; t0 < len; t0 += DL_C) {
    const int nt = min((len - t0 + 15) / 16, 4);
    if (a.S0 != nullptr && t0 > 0 && mine) {
      float* dst = a.S0 + ((bh * (nC - 1) + t0 / DL_C - 1) * a.Dk) * a.Dv + col;
#pragma unroll
      for (int u = 0; u < 2 * KT; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * u + 4 * kg + r < a.Dk) dst[(int64_t)(16 * u + 4 * kg + r) * a.Dv] = S[u][r];
    }
    float vv[4][4];
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = t0 + 16 * it + 4 * kg + r;
        vv[it][r] = mine && t < len ? (float)v[t * a.vs[1]] : 0.f;
      }
    __syncthreads();   // the last chunk's reads are done
    dl_load<IO, DP>(K, k, a.ks[1], t0, len, a.Dk, tid, nth);
    dl_load<IO, DP>(Q, q, a.qs[1], t0, len, a.Dk, tid, nth);
    if (wave == 0) dl_gates(s, a, b, h, t0, len);
    __syncthreads();
    dl_prep<DP, NI, NP>(K, Q, P, T, s, a.scale, nt, wave, nw);

    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    f4 x[4] = {zero, zero, zero, zero}, oo[4] = {zero, zero, zero, zero};
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      bf16x8 sb[NP];
      pl_split<NP>(S[2 * t], S[2 * t + 1], sb);
#pragma unroll
      for (int it = 0; it < 4; ++it)
        if (it < nt) {
          bf16x8 f[NI];
          K.row(f, 16 * it, t);
          x[it] = pl_mm<NI, NP>(f, sb, x[it]);
          Q.row(f, 16 * it, t);
          oo[it] = pl_mm<NI, NP>(f, sb, oo[it]);
        }
    }
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * it + 4 * kg + r;
        const float gam = s.gam[i];
        x[it][r] = s.beta[i] * (vv[it][r] - gam * x[it][r]);
        oo[it][r] *= a.scale * gam;
      }
    bf16x8 xb[2][NP];
    pl_split<NP>(x[0], x[1], xb[0]);
    pl_split<NP>(x[2], x[3], xb[1]);
    f4 u[4] = {zero, zero, zero, zero};
#pragma unroll
    for (int it = 0; it < 4; ++it)
      if (it < nt) {
#pragma unroll
        for (int kb = 0; kb <= it / 2; ++kb) {
          bf16x8 f[NP];
          T.row(f, 16 * it, kb);
          u[it] = pl_mm<NP, NP>(f, xb[kb], u[it]);
        }
      }
    pl_split<NP>(u[0], u[1], xb[0]);
    pl_split<NP>(u[2], u[3], xb[1]);
#pragma unroll
    for (int it = 0; it < 4; ++it)
      if (it < nt) {
#pragma unroll
        for (int kb = 0; kb <= it / 2; ++kb) {
          bf16x8 f[NP];
          P.row(f, 16 * it, kb);
          oo[it] = pl_mm<NP, NP>(f, xb[kb], oo[it]);
        }
      }
    if (mine) {
#pragma unroll
      for (int it = 0; it < 4; ++it)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int t = t0 + 16 * it + 4 * kg + r;
          if (t < a.T) o[t * os] = (IO)oo[it][r];
          if (a.U != nullptr && t < len) a.U[(bh * a.T + t) * a.Dv + col] = u[it][r];
        }
    }
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
      for (int r = 0; r < 4; ++r) u[it][r] *= s.rest[16 * it + 4 * kg + r];
    pl_split<NP>(u[0], u[1], xb[0]);
    pl_split<NP>(u[2], u[3], xb[1]);
    const float last = s.gam[DL_C - 1];
#pragma unroll
    for (int t = 0; t < 2 * KT; ++t) {
      S[t] *= last;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
        if (2 * kb < nt) {
          bf16x8 f[NI];
          K.col(f, kb, 16 * t);
          S[t] = pl_mm<NI, NP>(f, xb[kb], S[t]);
        }
    }
  }
  if (mine) {
    for (int t = (len + DL_C - 1) / DL_C * DL_C + kg; t < a.T; t += 4) o[t * os] = (IO)0.f;
#pragma unroll
    for (int u = 0; u < 2 * KT; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 16 * u + 4 * kg + r;
        if (d < a.Dk) a.state[(bh * a.Dk + d) * a.Dv + col] = S[u][r];
      }
  }
}

// ------------------------------------------------------- backward, the scan ----
// The same split, chunks last to first; leaves dX, dV, the gradients after each chunk but the last, and dstate0.
template <typename IO, int DP, int NP>
__global__ __launch_bounds__(512) void k_delta_scan(DeltaArgs a) {
  constexpr int NI = DlIO<IO>::N, KT = DP / 32;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  using L = DlLds<DP, NI, NP>;
  const PlaneMat<DL_C, DP, NI> K{(__bf16*)lds}, Q{(__bf16*)(lds + L::KQ)};
  const PlaneMat<DL_C, 64, NP> P{(__bf16*)(lds + 2 * L::KQ)}, T{(__bf16*)(lds + 2 * L::KQ + L::M)};
  DlGates& s = *(DlGates*)(lds + 2 * L::KQ + 2 * L::M);

  const int tid = threadIdx.x, nth = blockDim.x, lane = tid & 63, n = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = nth >> 6;
  const int b = blockIdx.x / a.Hv, h = blockIdx.x % a.Hv, hk = h / (a.Hv / a.Hk);
  const int len = dl_len(a, b), col = (blockIdx.y * nw + wave) * 16 + n;
  const bool mine = col < a.Dv;
  const int nC = (a.T + DL_C - 1) / DL_C;
  const IO* q = (const IO*)a.q + b * a.qs[0] + hk * a.qs[2];
  const IO* k = (const IO*)a.k + b * a.ks[0] + hk * a.ks[2];
  const IO* d_o = (const IO*)a.d_o + b * a.dos[0] + h * a.dos[2] + col;
  const int64_t bh = (int64_t)b * a.Hv + h;
  IO* dv = (IO*)a.dv + ((int64_t)b * a.T * a.Hv + h) * a.Dv + col;
  const int64_t os = (int64_t)a.Hv * a.Dv;

  f4 S[2 * KT];
#pragma unroll
  for (int u = 0; u < 2 * KT; ++u)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * u + 4 * kg + r;
      S[u][r] = a.dstate != nullptr && mine && d < a.Dk ? a.dstate[(bh * a.Dk + d) * a.Dv + col] : 0.f;
    }
  dl_clear(P.p, 2 * L::M);

  const int nc = (len + DL_C - 1) / DL_C;
  for (int c = nc - 1; c >= 0; --c) {
    const int t0 = c * DL_C, nt = min((len - t0 + 15) / 16, 4);
    if (c < nc - 1 && mine) {
      float* dst = a.dS + ((bh * (nC - 1) + c) * a.Dk) * a.Dv + col;
#pragma unroll
      for (int u = 0; u < 2 * KT; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * u + 4 * kg + r < a.Dk) dst[(int64_t)(16 * u + 4 * kg + r) * a.Dv] = S[u][r];
    }
    f4 go[4];
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = t0 + 16 * it + 4 * kg + r;
        go[it][r] = mine && t < len ? (float)d_o[t * a.dos[1]] : 0.f;
      }
    __syncthreads();
    dl_load<IO, DP>(K, k, a.ks[1], t0, len, a.Dk, tid, nth);
    dl_load<IO, DP>(Q, q, a.qs[1], t0, len, a.Dk, tid, nth);
    if (wave == 0) dl_gates(s, a, b, h, t0, len);
    // parts that a shorter last chunk left untouched hold no older chunk's values: it comes first
    __syncthreads();
    dl_prep<DP, NI, NP>(K, Q, P, T, s, a.scale, nt, wave, nw);

    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    f4 du[4] = {zero, zero, zero, zero};
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      bf16x8 sb[NP];
      pl_split<NP>(S[2 * t], S[2 * t + 1], sb);
#pragma unroll
      for (int it = 0; it < 4; ++it)
        if (it < nt) {
          bf16x8 f[NI];
          K.row(f, 16 * it, t);
          du[it] = pl_mm<NI, NP>(f, sb, du[it]);
        }
    }
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
      for (int r = 0; r < 4; ++r) du[it][r] *= s.rest[16 * it + 4 * kg + r];
    {
      bf16x8 gb[2][NI];
      pl_split<NI>(go[0], go[1], gb[0]);
      pl_split<NI>(go[2], go[3], gb[1]);
#pragma unroll
      for (int it = 0; it < 4; ++it)
        if (it < nt) {
#pragma unroll
          for (int kb = it / 2; kb < 2; ++kb)
            if (2 * kb < nt) {
              bf16x8 f[NP];
              P.col(f, kb, 16 * it);
              du[it] = pl_mm<NP, NI>(f, gb[kb], du[it]);
            }
        }
    }
    bf16x8 xb[2][NP];
    pl_split<NP>(du[0], du[1], xb[0]);
    pl_split<NP>(du[2], du[3], xb[1]);
    f4 dx[4] = {zero, zero, zero, zero};
#pragma unroll
    for (int it = 0; it < 4; ++it)
      if (it < nt) {
#pragma unroll
        for (int kb = it / 2; kb < 2; ++kb)
          if (2 * kb < nt) {
            bf16x8 f[NP];
            T.col(f, kb, 16 * it);
            dx[it] = pl_mm<NP, NP>(f, xb[kb], dx[it]);
          }
      }
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * it + 4 * kg + r, t = t0 + i;
        if (mine) {
          if (t < a.T) dv[t * os] = (IO)(s.beta[i] * dx[it][r]);
          if (t < len) a.dX[(bh * a.T + t) * a.Dv + col] = dx[it][r];
        }
        const float gam = s.gam[i];
        go[it][r] *= a.scale * gam;
        dx[it][r] *= -s.beta[i] * gam;
      }
    const float last = s.gam[DL_C - 1];
    bf16x8 gb[2][NP];
    pl_split<NP>(go[0], go[1], gb[0]);
    pl_split<NP>(go[2], go[3], gb[1]);
    pl_split<NP>(dx[0], dx[1], xb[0]);
    pl_split<NP>(dx[2], dx[3], xb[1]);
#pragma unroll
    for (int t = 0; t < 2 * KT; ++t) {
      S[t] *= last;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
        if (2 * kb < nt) {
          bf16x8 f[NI];
          Q.col(f, kb, 16 * t);
          S[t] = pl_mm<NI, NP>(f, gb[kb], S[t]);
          K.col(f, kb, 16 * t);
          S[t] = pl_mm<NI, NP>(f, xb[kb], S[t]);
        }
    }
  }
  if (mine) {
    for (int t = nc * DL_C + kg; t < a.T; t += 4) dv[t * os] = (IO)0.f;
    if (a.dstate0 != nullptr) {
#pragma unroll
      for (int u = 0; u < 2 * KT; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int d = 16 * u + 4 * kg + r;
          if (d < a.Dk) a.dstate0[(bh * a.Dk + d) * a.Dv + col] = S[u][r];
        }
    }
  }
}

// -------------------------------------- backward, the rest of a chunk's gradients ----
// One workgroup of four waves per (batch row, key head, chunk), independent of the others; the value heads of a key head
// one after the other, their dq and dk summed in registers (no atomics: the same result every time).  Wave w owns the
// chunk's rows 16w .. 16w + 15.  First the contractions over the value columns, staged in blocks of 32,
//     dP = dO Uᵀ,  dA = −dX Uᵀ,  E1 = dO Sᵀ,  E2 = dX Sᵀ,  E3 = U dS'ᵀ,
// then K and Q take the staging area's place for  dQ = scale e^G E1 + M1 K,  dK = M1ᵀ Q + (M2 + M2ᵀ) K − b e^G E2 +
// D_end E3  with M1 = scale D dP, M2 = b D dA, and for the scalars' gradients.
template <int DP, int NI, int NP>
struct DlGradLds {
  static constexpr int KQ = PlaneMat<DL_C, DP, NI>::BYTES, M = PlaneMat<DL_C, 64, NP>::BYTES;
  static constexpr int GO = PlaneMat<DL_C, 32, NI>::BYTES, X = PlaneMat<DL_C, 32, NP>::BYTES,
                       ST = PlaneMat<DP, 32, NP>::BYTES;
  static constexpr int ONE = GO + 2 * X + 2 * ST, TWO = 2 * KQ + 2 * M;
  static constexpr int AREA = ONE > TWO ? ONE : TWO;
  static constexpr int SUMS = (4 * 64 + 6 * 64) * 4;
  static constexpr int BYTES = AREA + (int)sizeof(DlGates) + SUMS;
  static_assert(BYTES <= 160 * 1024, "LDS of a CU");
};

// rows r < rows of a (.., Dv) fp32 matrix, columns c0 .. c0 + 31, into planes; zeros elsewhere.  With `with`: also the
// sum of products with that matrix.
template <int R, int NP>
__device__ __forceinline__ float dl_stage(const PlaneMat<R, 32, NP>& m, const float* src, int rows, int c0, int Dv,
                                          const float* with) {
  float sum = 0.f;
  for (int e = threadIdx.x; e < R * 4; e += blockDim.x) {
    const int r = e >> 2, c = (e & 3) * 8;
    bf16x8 f[NP] = {};
    if (r < rows && c0 + c < Dv) {
      const float* s = src + (int64_t)r * Dv + c0 + c;
      const f4 lo = *reinterpret_cast<const f4*>(s), hi = *reinterpret_cast<const f4*>(s + 4);
      pl_split<NP>(lo, hi, f);
      if (with != nullptr) {
        const float* w = with + (int64_t)r * Dv + c0 + c;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = __builtin_fmaf(lo[i], w[i], __builtin_fmaf(hi[i], w[4 + i], sum));
      }
    }
    m.put8(r, c, f);
  }
  return sum;
}

__device__ __forceinline__ float dl_sum16(float x) {   // over the 16 lanes of a group
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) x += __shfl_xor(x, o);
  return x;
}

template <int R, int C, int N>
__device__ __forceinline__ float dl_get(const PlaneMat<R, C, N>& m, int r, int c) {
  const __bf16* p = m.p + r * PlaneMat<R, C, N>::LD + pl_place(c);
  float x = 0.f;
#pragma unroll
  for (int q = N - 1; q >= 0; --q) x += (float)p[q * PlaneMat<R, C, N>::PLANE];
  return x;
}

template <typename IO, int DP, int NP>
__global__ __launch_bounds__(256) void k_delta_grads(DeltaArgs a) {
  constexpr int NI = DlIO<IO>::N, UT = DP / 16;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  using L = DlGradLds<DP, NI, NP>;
  const PlaneMat<DL_C, 32, NI> GO{(__bf16*)lds};
  const PlaneMat<DL_C, 32, NP> DX{(__bf16*)(lds + L::GO)}, UU{(__bf16*)(lds + L::GO + L::X)};
  const PlaneMat<DP, 32, NP> SS{(__bf16*)(lds + L::GO + 2 * L::X)}, DS{(__bf16*)(lds + L::GO + 2 * L::X + L::ST)};
  const PlaneMat<DL_C, DP, NI> K{(__bf16*)lds}, Q{(__bf16*)(lds + L::KQ)};
  const PlaneMat<DL_C, 64, NP> M1{(__bf16*)(lds + 2 * L::KQ)}, M2{(__bf16*)(lds + 2 * L::KQ + L::M)};
  DlGates& s = *(DlGates*)(lds + L::AREA);
  float* colsum = (float*)(lds + L::AREA + sizeof(DlGates));   // [4 waves][64]
  float* rows = colsum + 4 * 64;                               // [6][64]

  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = a.Hv / a.Hk, b = blockIdx.x / a.Hk, hk = blockIdx.x % a.Hk, c = blockIdx.y, t0 = c * DL_C;
  const int len = dl_len(a, b), nC = (a.T + DL_C - 1) / DL_C, nc = (len + DL_C - 1) / DL_C;
  IO* dq = (IO*)a.dq + ((int64_t)b * a.T * a.Hk + hk) * a.Dk;
  IO* dk = (IO*)a.dk + ((int64_t)b * a.T * a.Hk + hk) * a.Dk;
  const int64_t ks = (int64_t)a.Hk * a.Dk;

  if (c >= nc) {
    const int end = min(a.T, t0 + DL_C);
    for (int e = tid; e < (end - t0) * a.Dk; e += 256) {
      dq[(t0 + e / a.Dk) * ks + e % a.Dk] = (IO)0.f;
      dk[(t0 + e / a.Dk) * ks + e % a.Dk] = (IO)0.f;
    }
    for (int e = tid; e < (end - t0) * group; e += 256) {
      const int64_t at = ((int64_t)b * a.T + t0 + e / group) * a.Hv + hk * group + e % group;
      a.dg[at] = 0.f;
      a.dbeta[at] = 0.f;
    }
    return;
  }

  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  f4 gq[UT], gk[UT];
#pragma unroll
  for (int u = 0; u < UT; ++u) gq[u] = gk[u] = zero;

  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    const int64_t bh = (int64_t)b * a.Hv + h, state = (int64_t)a.Dk * a.Dv;
    const float* S0 = c > 0 ? a.S0 + (bh * (nC - 1) + c - 1) * state : a.state0 ? a.state0 + bh * state : nullptr;
    const float* dS = c < nc - 1 ? a.dS + (bh * (nC - 1) + c) * state : a.dstate ? a.dstate + bh * state : nullptr;
    const float* U = a.U + (bh * a.T + t0) * a.Dv;
    const float* dX = a.dX + (bh * a.T + t0) * a.Dv;
    const IO* d_o = (const IO*)a.d_o + b * a.dos[0] + h * a.dos[2];
    const IO* v = (const IO*)a.v + b * a.vs[0] + h * a.vs[2];
    const int left = min(len - t0, DL_C);

    f4 dp[4] = {zero, zero, zero, zero}, da[4] = {zero, zero, zero, zero}, e1[UT], e2[UT], e3[UT];
#pragma unroll
    for (int u = 0; u < UT; ++u) e1[u] = e2[u] = e3[u] = zero;
    float both = 0.f;
    for (int c0 = 0; c0 < a.Dv; c0 += 32) {
      __syncthreads();
      for (int e = tid; e < DL_C * 4; e += 256) {
        const int r = e >> 2, cc = (e & 3) * 8;
        bf16x8 f[NI] = {};
        if (r < left && c0 + cc < a.Dv) DlIO<IO>::load8(d_o + (int64_t)(t0 + r) * a.dos[1] + c0 + cc, f);
        GO.put8(r, cc, f);
      }
      dl_stage<DL_C, NP>(DX, dX, left, c0, a.Dv, nullptr);
      dl_stage<DL_C, NP>(UU, U, left, c0, a.Dv, nullptr);
      if (S0 != nullptr) both += dl_stage<DP, NP>(SS, S0, a.Dk, c0, a.Dv, dS);
      if (dS != nullptr) dl_stage<DP, NP>(DS, dS, a.Dk, c0, a.Dv, nullptr);
      __syncthreads();
      bf16x8 go[NI], gx[NP], y[NP];
      GO.row(go, 16 * wave, 0);
      DX.row(gx, 16 * wave, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j <= wave) {
          UU.row(y, 16 * j, 0);
          dp[j] = pl_mm<NI, NP>(go, y, dp[j]);
          da[j] = pl_mm<NP, NP>(gx, y, da[j]);
        }
      if (S0 != nullptr) {
#pragma unroll
        for (int u = 0; u < UT; ++u) {
          SS.row(y, 16 * u, 0);
          e1[u] = pl_mm<NI, NP>(go, y, e1[u]);
          e2[u] = pl_mm<NP, NP>(gx, y, e2[u]);
        }
      }
      if (dS != nullptr) {
        UU.row(gx, 16 * wave, 0);
#pragma unroll
        for (int u = 0; u < UT; ++u) {
          DS.row(y, 16 * u, 0);
          e3[u] = pl_mm<NP, NP>(gx, y, e3[u]);
        }
      }
    }
    // dX · V of each row: four lanes a row
    {
      const int r = tid >> 2;
      float x = 0.f;
      if (r < left)
        for (int cc = (tid & 3) * 4; cc < a.Dv; cc += 16)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            x = __builtin_fmaf(dX[(int64_t)r * a.Dv + cc + i], (float)v[(int64_t)(t0 + r) * a.vs[1] + cc + i], x);
      x += __shfl_xor(x, 1);
      x += __shfl_xor(x, 2);
      if ((tid & 3) == 0) rows[5 * 64 + r] = x;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) both += __shfl_xor(both, o);
    }
    __syncthreads();   // the staged blocks are read: K and Q take their place
    dl_load<IO, DP>(K, (const IO*)a.k + b * a.ks[0] + hk * a.ks[2], a.ks[1], t0, len, a.Dk, tid, 256);
    dl_load<IO, DP>(Q, (const IO*)a.q + b * a.qs[0] + hk * a.qs[2], a.qs[1], t0, len, a.Dk, tid, 256);
    if (wave == 0) dl_gates(s, a, b, h, t0, len);
    __syncthreads();
    float rm[4] = {0.f, 0.f, 0.f, 0.f}, rb[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f4 kk = zero, qk = zero;
      if (j <= wave) {
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) {
          bf16x8 ki[NI], qi[NI], kj[NI];
          K.row(ki, 16 * wave, t);
          Q.row(qi, 16 * wave, t);
          K.row(kj, 16 * j, t);
          kk = pl_mm<NI, NI>(ki, kj, kk);
          qk = pl_mm<NI, NI>(qi, kj, qk);
        }
      }
      const int jj = 16 * j + n;
      float cs = 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * wave + 4 * kg + r;
        float m1 = 0.f, m2 = 0.f;
        if (jj <= i) {
          const float d = expf((float)(s.G[i] - s.G[jj]));
          m1 = a.scale * d * dp[j][r];
          float m = m1 * qk[r];
          if (jj < i) {
            const float w = -d * da[j][r];
            m2 = s.beta[i] * w;
            m += m2 * kk[r];
            rb[r] += w * kk[r];
          }
          rm[r] += m;
          cs += m;
        }
        M1.put(i, jj, m1);
        M2.put(i, jj, m2);
      }
      cs += __shfl_xor(cs, 16);
      cs += __shfl_xor(cs, 32);
      if (kg == 0) colsum[wave * 64 + jj] = cs;
    }
    float r1[4] = {0.f, 0.f, 0.f, 0.f}, r2[4] = {0.f, 0.f, 0.f, 0.f}, r3[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < UT; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * wave + 4 * kg + r;
        const float gam = s.gam[i], kx = dl_get(K, i, 16 * u + n), qx = dl_get(Q, i, 16 * u + n);
        r1[r] = __builtin_fmaf(qx, e1[u][r], r1[r]);
        r2[r] = __builtin_fmaf(kx, e2[u][r], r2[r]);
        r3[r] = __builtin_fmaf(kx, e3[u][r], r3[r]);
        gq[u][r] += a.scale * gam * e1[u][r];
        gk[u][r] += s.rest[i] * e3[u][r] - s.beta[i] * gam * e2[u][r];
      }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * wave + 4 * kg + r;
      const float x0 = dl_sum16(rm[r]), x1 = dl_sum16(rb[r]), x2 = dl_sum16(r1[r]), x3 = dl_sum16(r2[r]),
                  x4 = dl_sum16(r3[r]);
      if (n == 0) {
        rows[i] = x0;
        rows[64 + i] = x1;
        rows[2 * 64 + i] = x2;
        rows[3 * 64 + i] = x3;
        rows[4 * 64 + i] = x4;
      }
    }
    // one sum of S · dS' per wave in the gates' place of G, which is not read any more behind the barrier
    __syncthreads();
    if (lane == 0) s.G[wave] = both;
    __syncthreads();
    if (wave == 0) {
      const int i = lane;
      const float gam = s.gam[i], be = s.beta[i];
      const double leave = (double)s.rest[i] * rows[4 * 64 + i];
      double at = (double)rows[i] + (double)a.scale * gam * rows[2 * 64 + i] - (double)be * gam * rows[3 * 64 + i] - leave;
#pragma unroll
      for (int w = 0; w < 4; ++w) at -= (double)colsum[w * 64 + i];
      double all = leave;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        all += __shfl_xor(all, o);
        const double down = __shfl_down(at, o);
        if (i + o < 64) at += down;
      }
      at += all + (double)s.gam[DL_C - 1] * (s.G[0] + s.G[1] + s.G[2] + s.G[3]);
      const int64_t out = ((int64_t)b * a.T + t0 + i) * a.Hv + h;
      if (t0 + i < a.T) {
        a.dg[out] = t0 + i < len ? (float)at : 0.f;
        a.dbeta[out] = t0 + i < len ? rows[5 * 64 + i] - gam * rows[3 * 64 + i] + rows[64 + i] : 0.f;
      }
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      bf16x8 m1[NP], m1t[NP], m2[NP], m2t[NP];
      M1.row(m1, 16 * wave, kb);
      M2.row(m2, 16 * wave, kb);
      M1.col(m1t, kb, 16 * wave);
      M2.col(m2t, kb, 16 * wave);
#pragma unroll
      for (int u = 0; u < UT; ++u) {
        bf16x8 f[NI];
        K.col(f, kb, 16 * u);
        if (kb <= wave / 2) {
          gq[u] = pl_mm<NP, NI>(m1, f, gq[u]);
          gk[u] = pl_mm<NP, NI>(m2, f, gk[u]);
        }
        if (kb >= wave / 2) {
          gk[u] = pl_mm<NP, NI>(m2t, f, gk[u]);
          Q.col(f, kb, 16 * u);
          gk[u] = pl_mm<NP, NI>(m1t, f, gk[u]);
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < UT; ++u)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = t0 + 16 * wave + 4 * kg + r, d = 16 * u + n;
      if (t < a.T && d < a.Dk) {
        dq[t * ks + d] = (IO)(t < len ? gq[u][r] : 0.f);
        dk[t * ks + d] = (IO)(t < len ? gk[u][r] : 0.f);
      }
    }
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
  if ((int64_t)a.B * a.Hv > 0x7fffffff || (a.T + DL_C - 1) / DL_C > 65535) return RG_ERR_SHAPE;
  if (a.q == nullptr || a.k == nullptr || a.v == nullptr || a.g == nullptr || a.beta == nullptr) return RG_ERR_ARG;
  return RG_OK;
}
static bool delta_aligned(const void* p, const int64_t* s, int type) {   // 16-byte rows
  const int64_t e = type == 0 ? 4 : 2;
  return ((uintptr_t)p & 15) == 0 && s[0] * e % 16 == 0 && s[1] * e % 16 == 0 && s[2] * e % 16 == 0;
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

// waves of a workgroup: all value columns together (K, Q, P and T of a chunk are then made once), fewer where that would
// leave most of the 256 CUs without work
static int delta_waves(const DeltaArgs& a) {
  int w = (a.Dv + 15) / 16;
  while (w > 2 && (int64_t)a.B * a.Hv * ((a.Dv + 16 * w - 1) / (16 * w)) < 128) w = (w + 1) / 2;
  return w;
}

// three planes of fp32 operands also for bf16 inputs: two would halve their products, but leave the fp32 outputs
// (state, dg, dbeta) at 2^-18 instead of fp32's own rounding
#define DL_NP 3

template <typename IO, int DP>
static int delta_fwd_t(const DeltaArgs& a, hipStream_t st) {
  const int w = delta_waves(a);
  return delta_go(k_delta_fwd<IO, DP, DL_NP>, dim3(a.B * a.Hv, (a.Dv + 16 * w - 1) / (16 * w)), 64 * w,
                  DlLds<DP, DlIO<IO>::N, DL_NP>::BYTES, a, st);
}
template <typename IO, int DP>
static int delta_bwd_t(const DeltaArgs& a, hipStream_t st) {
  const int w = delta_waves(a);
  const int rc = delta_go(k_delta_scan<IO, DP, DL_NP>, dim3(a.B * a.Hv, (a.Dv + 16 * w - 1) / (16 * w)), 64 * w,
                          DlLds<DP, DlIO<IO>::N, DL_NP>::BYTES, a, st);
  if (rc != RG_OK) return rc;
  return delta_go(k_delta_grads<IO, DP, DL_NP>, dim3(a.B * a.Hk, (a.T + DL_C - 1) / DL_C), 256,
                  DlGradLds<DP, DlIO<IO>::N, DL_NP>::BYTES, a, st);
}
#define DL_DISPATCH(F)                                                                             \
  (type == 0 ? (a.Dk <= 32 ? F<float, 32>(a, st) : a.Dk <= 64 ? F<float, 64>(a, st) : F<float, 128>(a, st)) \
             : (a.Dk <= 32 ? F<__bf16, 32>(a, st) : a.Dk <= 64 ? F<__bf16, 64>(a, st) : F<__bf16, 128>(a, st)))

static void delta_strides(DeltaArgs& a, const int64_t* s) {
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = s[i];
    a.ks[i] = s[3 + i];
    a.vs[i] = s[6 + i];
    a.gs[i] = s[9 + i];
    a.bs[i] = s[12 + i];
    a.dos[i] = s[15 + i];
  }
}

extern "C" int64_t rg_delta_chunk_floats(int B, int T, int Hv, int Dk, int Dv) {
  return T > 0 ? (int64_t)B * Hv * ((T + DL_C - 1) / DL_C - 1) * Dk * Dv : 0;
}

extern "C" int rg_delta_fwd(const void* q, const void* k, const void* v, const float* g, const float* beta,
                            const int64_t* strides, const int64_t* lens, const float* state0, int type, int B, int T,
                            int Hk, int Hv, int Dk, int Dv, float scale, void* o, float* state, float* U, float* S0,
                            hipStream_t st) {
  DeltaArgs a = {};
  if (strides == nullptr) return RG_ERR_ARG;
  delta_strides(a, strides);
  a.q = q, a.k = k, a.v = v, a.g = g, a.beta = beta, a.lens = lens, a.state0 = state0;
  a.B = B, a.T = T, a.Hk = Hk, a.Hv = Hv, a.Dk = Dk, a.Dv = Dv, a.scale = scale, a.o = o, a.state = state, a.U = U;
  a.S0 = T > DL_C ? S0 : nullptr;
  const int rc = delta_check(a, type);
  if (rc != RG_OK) return rc;
  if (o == nullptr || state == nullptr || (U != nullptr && T > DL_C && S0 == nullptr)) return RG_ERR_ARG;
  if (!delta_aligned(q, a.qs, type) || !delta_aligned(k, a.ks, type)) return RG_ERR_ARG;
  return DL_DISPATCH(delta_fwd_t);
}

extern "C" int rg_delta_bwd(const void* q, const void* k, const void* v, const float* g, const float* beta,
                            const void* d_o, const int64_t* strides, const int64_t* lens, const float* state0,
                            const float* dstate, const float* U, const float* S0, int type, int B, int T, int Hk,
                            int Hv, int Dk, int Dv, float scale, float* dX, float* dS, void* dq, void* dk, void* dv,
                            float* dg, float* dbeta, float* dstate0, hipStream_t st) {
  DeltaArgs a = {};
  if (strides == nullptr) return RG_ERR_ARG;
  delta_strides(a, strides);
  a.q = q, a.k = k, a.v = v, a.g = g, a.beta = beta, a.d_o = d_o, a.lens = lens, a.state0 = state0, a.dstate = dstate;
  a.B = B, a.T = T, a.Hk = Hk, a.Hv = Hv, a.Dk = Dk, a.Dv = Dv, a.scale = scale;
  a.U = const_cast<float*>(U), a.S0 = const_cast<float*>(S0), a.dX = dX, a.dS = dS;
  a.dq = dq, a.dk = dk, a.dv = dv, a.dg = dg, a.dbeta = dbeta, a.dstate0 = dstate0;
  const int rc = delta_check(a, type);
  if (rc != RG_OK) return rc;
  if (d_o == nullptr || U == nullptr || dX == nullptr || dq == nullptr || dk == nullptr || dv == nullptr ||
      dg == nullptr || dbeta == nullptr || (T > DL_C && (S0 == nullptr || dS == nullptr)))
    return RG_ERR_ARG;
  if (!delta_aligned(q, a.qs, type) || !delta_aligned(k, a.ks, type) || !delta_aligned(d_o, a.dos, type) ||
      (((uintptr_t)state0 | (uintptr_t)dstate | (uintptr_t)U | (uintptr_t)S0 | (uintptr_t)dX | (uintptr_t)dS) & 15))
    return RG_ERR_ARG;
  return DL_DISPATCH(delta_bwd_t);
}

extern "C" int rg_delta_step(const void* q, const void* k, const void* v, const float* g, const float* beta,
                             const int64_t* strides, int type, int B, int Hk, int Hv, int Dk, int Dv, float scale,
                             float* state, int64_t state_stride, void* o, hipStream_t st) {
  DeltaArgs a = {};
  if (strides == nullptr) return RG_ERR_ARG;
  delta_strides(a, strides);
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
