// Linear cross entropy over a large item vocabulary on half-precision activations, without keeping the logits: beside the
// fp32 training heads (csrc/head.hip, csrc/head_flash.hip), for any number of rows, ignored rows and widths.
//     z = h Wᵀ + b,   loss_r = lse(z_r) − z_{r, t_r},   dz = g (softmax(z) − onehot),   dh = dz W,  dW = dzᵀ h,  db = Σ_r dz
//
// Two passes of the same shape; each recomputes z tile by tile and feeds it on from registers (8 N V D flops; 6 with the
// N x V logits kept).  A workgroup holds a block of one matrix ("X") in registers and streams the other ("Y") through
// LDS in chunks of 64 rows:
//     S = Y_c Xᵀ (MFMA),   P = f(S) rounded to the inputs' type,   Oᵀ += Y_cᵀ P (MFMA)
//   forward   X = rows of h, Y = W: f = 2^(z − m) with a reference m of the row, 0 at the row's target; O = Σ_v 2^(z − m) W_v
//             and the sum of P per row and split of the vocabulary.  k_ce_join takes the target's logit in fp32 and has the
//             odds q against it, loss = log(1 + q), and dh = (Σ_{v ≠ t} p_v W_v) − (1 − p_t) W_t with 1 − p_t = q / (1 + q):
//             where a row is predicted well both are small, and neither is a difference of large rounded values (with
//             the target inside P, dh is off by up to 0.36 % of |W_t|: 7 % of itself at p_t = 0.98, nine times at 0.9998).
//   backward  X = items of W, Y = rows of h: f = g_r e^(z − lse_r), and −g_r (1 − p_t) at the row's target; O = dW, and
//             Σ_r P = db from the unrounded P.  A target's share is most of a target item's gradient; rounded to the type it
//             moved that by as much as the output's own rounding again (0.2 beside 1.0, clicks beside purchases: every
//             click's share by 1e-3 the same way).  So what the rounding leaves off follows behind the last chunk, for the
//             N rows of a whole pass alone: a wave remembers in which chunks it met targets of its items, lists those
//             rows, and takes 32 of them for one more product; a popular item's rows are shared among the workgroup's waves.
//             Less than 2^-16 of a share stays off (1/32 of fp16's half step): with the weights of a mean, scaled to 2^13,
//             2^13 (1 - p_t) is so near 2^13 for most rows of a large vocabulary.
// The accumulator of S (16 rows of Y x 16 of X per tile; lane (kg, n) holds rows 4·kg + i of column n) is already the B
// operand of the second product, whose A operand is Y_c read from LDS with ds_read_b64_tr_b16.  The biases are
// S's start value and cost no instruction an element; backwards −lse and log2 |g| enter with the exponent's scaling (as a
// start value of size 20 they would cost S its low bits: db was off by 1.5e-6 instead of 1e-7).  That matters because
// the exponentials, not the MFMAs, take the longer at small D: an element costs a scaling, an exponential (four
// issue slots), a sum and half a conversion, so there is no running maximum either: forwards the reference only
// moves when a lane's eight powers sum to more than LIM, which needs one comparison per eight elements.  A wave that
// has met only masked items, or logits beyond CE_FAR, looks for the largest one each time and takes it off first.  Per 32
// rows of Y a wave reads 2·32·D values from LDS for 4·16·NX·32·D MFMA flops.
//
// Measured, whole step: 4096 rows x 1M items x 128 bf16 3.47 to 3.53 ms, 1190 to 1210 TFLOP/s of these 8 N V D (88 to 90 % of
// what a large library product reaches, with the exponentials beside it); 7867 of 13111 rows x 78341 items x 256 fp16 1.17
// to 1.19 ms, 1060 to 1080 TFLOP/s, and 1.25 ms where the rows' weights differ: half of these targets are among 256 items, whose
// shares one workgroup adds (row by row, by one wave each: 4.4 ms); 64 x 10001 x 32 32 to 36 us, of which the launches and the
// waits between its five kernels (3 to 8 us each) are most.
//
// Rows with a negative target are left out from the start: k_ce_rows lists the others in order, and the passes run on a
// packed copy of h (padded to 64 / 128 / 256 columns), so an ignored position costs nothing.
// P is rounded to bf16 / fp16 for the second product (half a step of the type, once, as its other operand is held); sums
// of P, lse, O and the gradients are fp32, and each output is rounded once.  Backwards g is scaled so that the largest
// |g| is 2^13, and back in fp32: it keeps fp16's small probabilities out of its subnormals; forwards P <= 2^15 does.
#include "common.h"

typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t ce_u2 __attribute__((ext_vector_type(2)));
typedef short ce_s4 __attribute__((ext_vector_type(4)));
typedef short ce_s8 __attribute__((ext_vector_type(8)));

#define CE_CH 64           // rows of Y per chunk
#define CE_PAD 512         // packed rows are allocated in multiples of this
#define CE_L2E 1.4426950408889634f
#define CE_LN2 0.6931471805599453f
#define CE_LOW (-2.0e38f)  // the running reference before any logit
#define CE_REST 0x1p-16f   // what is left off a target's share and is less than this of it stays off
#define CE_FAR 32768.f     // references beyond it: exponents from differences of logits

template <typename T>
struct CeT;
template <>
struct CeT<__bf16> {
  typedef bf16x8 V;
  static constexpr float OFF = 0.f, LIM = 0x1p40f;
  static __device__ __forceinline__ f4 mm(V a, V b, f4 c) { return mfma16bf(a, b, c); }
};
template <>
struct CeT<_Float16> {
  typedef h16x8 V;
  static constexpr float OFF = 7.f, LIM = 0x1p15f;
  static __device__ __forceinline__ f4 mm(V a, V b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// Powers are 2^(z log2 e + base) with a base per reference, one fused operation an element.  The base is rounded to half a
// unit of its last place, which moves all powers of the reference alike and drops out as long as everything that meets
// them uses the same base; but beyond CE_FAR that half unit grows (64 at a logit of 1e9) until the powers leave fp32's range
// on either side, and there they are 2^((z - m) log2 e), whose difference is exact where it matters.
template <typename T>
__device__ __forceinline__ float ce_base(float m) {
  return __builtin_fmaf(-m, CE_L2E, CeT<T>::OFF);
}
__device__ __forceinline__ bool ce_near(float m) { return fabsf(m) <= CE_FAR; }
// what sums taken with the reference m count beside sums with the reference top >= m
template <typename T>
__device__ __forceinline__ float ce_weight(float m, float top) {
  return __builtin_amdgcn_exp2f(ce_near(m) && ce_near(top) ? ce_base<T>(top) - ce_base<T>(m) : (m - top) * CE_L2E);
}

struct CeArgs {
  const void *X, *Y;
  int64_t ldx, ldy;        // row strides in elements
  const int* tc;           // forward: targets of the packed rows
  int nx, ny;              // rows (host bounds)
  int D;                   // columns of W's rows (h's packed copy has DP, zeros behind D)
  const int* count;        // packed rows
  const float* bias;       // (V) or null
  const float* recs;       // backward: [chunk][4][64], see k_ce_dh
  int nsplit, nblock, block0;   // blocks of X: nblock of them, from block0 on
  float *pm, *pl, *pO;     // forward: [split][row], [split][row][DP]; backward: pO slabs [split][items from block0 on][D], pl likewise
  void* dW;
  float* db;
  const float* scale;      // backward: what g's scaling left out
};

// 16-byte chunk c of row r sits at place c ^ swz(r): 16 rows' reads of one column spread over all banks
template <int DP>
__device__ __forceinline__ int ce_swz(int r) {
  return DP == 64 ? (r >> 1) & 7 : r & 15;
}

// FWD: forward pass (else backward); GRAD: with the second product; BIAS: backward with biases
template <typename T, int DP, int NX, int NW, bool FWD, bool GRAD, bool BIAS>
__global__ __launch_bounds__(64 * NW, DP == 64 ? 4 : 2) void k_ce_pass(CeArgs a) {
  typedef typename CeT<T>::V V;
  constexpr int KS = DP / 32, RB = DP * 2, FB = GRAD ? DP / 16 : 1;
  constexpr int LOADS = CE_CH * RB / (NW * 1024);
  // the swizzled addresses of a tile's reads, remade for each: kept over the loop they would cost a tile's registers
  constexpr bool REMAKE = DP == 256 && NX > 1;
  static_assert(LOADS >= 1, "a chunk is at least one load a wave");
  __shared__ __attribute__((aligned(16))) uint8_t y0[CE_CH * RB], y1[CE_CH * RB];
  __shared__ __attribute__((aligned(16))) float r0[4 * CE_CH], r1[4 * CE_CH];
  __shared__ int target[FWD ? 16 * NX * NW : 1];
  __shared__ float xbias[BIAS ? 16 * NX * NW : 1];   // (registers are short at 256 columns)
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, kg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // neighbouring blocks of one split run on one XCD (workgroups go round the 8 XCDs) and share its L2
  int split, block;
  if (a.nsplit % 8 == 0) {
    const int k = blockIdx.x >> 3;
    split = (blockIdx.x & 7) + 8 * (k / a.nblock);
    block = k % a.nblock;
  } else {
    split = blockIdx.x / a.nblock;
    block = blockIdx.x % a.nblock;
  }
  block += a.block0;
  const int rows = *a.count;
  const int nx = FWD ? rows : a.nx, ny = FWD ? a.ny : rows;
  const int x0 = block * 16 * NX * NW + wave * 16 * NX;
  if (FWD && block * 16 * NX * NW >= nx) return;
  const int nch = (ny + CE_CH - 1) / CE_CH;
  const int c0 = (int)((int64_t)nch * split / a.nsplit), c1 = (int)((int64_t)nch * (split + 1) / a.nsplit);

  const T* Y = (const T*)a.Y;
  const int ycols = FWD ? a.D : DP;
  auto issue = [&](int c, uint8_t* y, float* r) __attribute__((always_inline)) {
    const int64_t at = (int64_t)c * CE_CH;
    const int64_t left = ny - at;   // rows
    const int64_t bytes = left <= 0 ? 0 : ((left < CE_CH ? left : CE_CH) - 1) * a.ldy * 2 + ycols * 2;
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(Y) + at * a.ldy, 0, (int)bytes, 0x00020000);
    // a load's rows are the first one's and ROWS more each, with the same swizzle: one register for all
    constexpr int ROWS = NW * 1024 / RB;
    static_assert(ROWS % 16 == 0, "");
    const int e = wave * 64 + lane, row = e / (RB / 16), col = (e % (RB / 16) ^ ce_swz<DP>(row)) * 8;
    const int off = col < ycols ? (int)(row * a.ldy + col) * 2 : 0x7ffffff0;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) rg_blds16(rs, y + (i * NW + wave) * 1024, off, i * ROWS * (int)a.ldy * 2);
    if (wave == 0) {
      if constexpr (FWD) {   // 64 biases
        const int nb = a.bias != nullptr ? (int)(left < CE_CH ? left : CE_CH) * 4 : 0;
        const auto rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.bias) + (a.bias ? at : 0), 0,
                                                          nb < 0 ? 0 : nb, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (__attribute__((address_space(3))) void*)r, 4, lane * 4, 0, 0, 0);
      } else {
        const auto rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.recs) + at * 4, 0,
                                                          left > 0 ? 4 * CE_CH * 4 : 0, 0x00020000);
        rg_blds16(rb, r, 16 * lane, 0);
      }
    }
  };
  if (c0 < c1) issue(c0, y0, r0);

  V xf[NX][KS];
  float ref[NX], sum[NX];
  bool away = true;   // a reference of this wave lies beyond CE_FAR
  uint64_t met = 0;   // backward: a bit for each 2^fold chunks with targets among this wave's items
  int fold = 2;
  while (c1 - c0 > 64 << fold) ++fold;
  const T* X = (const T*)a.X;
  const int xcols = FWD ? DP : a.D;
#pragma unroll
  for (int t = 0; t < NX; ++t) {
    const int64_t x = x0 + 16 * t + n;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int col = 32 * s + 8 * kg;
      xf[t][s] = x < nx && col < xcols ? *reinterpret_cast<const V*>(X + x * a.ldx + col) : (V)(T)0.f;
    }
    ref[t] = CE_LOW;
    sum[t] = 0.f;
    if (BIAS && kg == 0) xbias[wave * 16 * NX + 16 * t + n] = x < nx ? a.bias[x] : 0.f;
    if (FWD && kg == 0) target[wave * 16 * NX + 16 * t + n] = x < nx ? a.tc[x] : -1;
  }
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  f4 O[FB][NX];
#pragma unroll
  for (int f = 0; f < FB; ++f)
#pragma unroll
    for (int t = 0; t < NX; ++t) O[f][t] = zero;

  auto work = [&](int c, uint8_t* y, const float* r) __attribute__((always_inline)) {
    // a target of this wave's rows among the chunk's items, or backwards one of the chunk's rows among this wave's items;
    // a negative g among the chunk's rows, and one whose logits lie beyond CE_FAR
    bool mine = false, sign = false, far = false;
    if constexpr (FWD) {
#pragma unroll
      for (int t = 0; t < NX; ++t) mine |= (unsigned)(target[wave * 16 * NX + 16 * t + n] - c * CE_CH) < CE_CH;
      mine = __any(mine);
    } else {
      const int t = __float_as_int(r[2 * CE_CH + lane]) - x0;
      mine = __any(t >= 0 && t < 16 * NX);
      if (mine) met |= 1ull << ((c - c0) >> fold);
      sign = __any(!__builtin_signbitf(r[CE_CH + lane]));
      far = __any(r[3 * CE_CH + lane] != 0.f);
    }
    const bool tail = FWD && c * CE_CH + CE_CH > ny;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      V P[NX];
      int nn = n;
      if constexpr (REMAKE) asm volatile("" : "+v"(nn));
      f4 S[2][NX];
      const int at = 32 * h + 4 * kg;   // this lane's rows: at .. at + 3 and 16 further on
#pragma unroll
      for (int t = 0; t < NX; ++t) {
        const float xb = BIAS ? xbias[wave * 16 * NX + 16 * t + nn] : 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          S[j][t] = FWD ? *reinterpret_cast<const f4*>(r + at + 16 * j) : BIAS ? (f4){xb, xb, xb, xb} : zero;
      }
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint8_t* p = y + (32 * h + nn) * RB + (((4 * s + kg) ^ ce_swz<DP>(nn)) << 4);
        const V f0 = *reinterpret_cast<const V*>(p), f1 = *reinterpret_cast<const V*>(p + 16 * RB);
#pragma unroll
        for (int t = 0; t < NX; ++t) S[0][t] = CeT<T>::mm(f0, xf[t][s], S[0][t]);
#pragma unroll
        for (int t = 0; t < NX; ++t) S[1][t] = CeT<T>::mm(f1, xf[t][s], S[1][t]);
      }
      if constexpr (FWD) {
        float base[NX];
#pragma unroll
        for (int t = 0; t < NX; ++t) base[t] = ce_base<T>(ref[t]);
        // the reference moves up to the logits in hand, what was summed follows, and the powers are made from differences
        auto move = [&]() __attribute__((always_inline)) {
          bool up = false, beyond = false;
          float now[NX];
#pragma unroll
          for (int t = 0; t < NX; ++t) {
            float m = fmaxf(fmaxf(fmaxf(S[0][t][0], S[0][t][1]), fmaxf(S[0][t][2], S[0][t][3])),
                            fmaxf(fmaxf(S[1][t][0], S[1][t][1]), fmaxf(S[1][t][2], S[1][t][3])));
            m = fmaxf(m, __shfl_xor(m, 16));
            m = fmaxf(m, __shfl_xor(m, 32));
            now[t] = fmaxf(ref[t], m);
            up |= now[t] != ref[t];
            beyond |= !ce_near(now[t]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i) S[j][t][i] -= now[t];
            base[t] = CeT<T>::OFF;
          }
          if (__any(up)) {
#pragma unroll
            for (int t = 0; t < NX; ++t) {
              const float fac = ce_weight<T>(ref[t], now[t]);
              ref[t] = now[t];
              sum[t] *= fac;
#pragma unroll
              for (int f = 0; f < FB; ++f) O[f][t] *= fac;
            }
          }
          away = __any(beyond);
        };
        bool fresh = false;
        if (tail || mine || away) {
          if (tail) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (c * CE_CH + at + 16 * (i >> 2) + (i & 3) >= ny)
#pragma unroll
                for (int t = 0; t < NX; ++t) S[i >> 2][t][i & 3] = -__builtin_inff();
          }
          if (mine) {
#pragma unroll
            for (int t = 0; t < NX; ++t) {
              const int place = target[wave * 16 * NX + 16 * t + n] - c * CE_CH - at;
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (place == 16 * (i >> 2) + (i & 3)) S[i >> 2][t][i & 3] = -__builtin_inff();
            }
          }
          if (away) {
            move();
            fresh = true;
          }
        }
        float p[NX][8], add[NX];
        auto powers = [&]() __attribute__((always_inline)) {
          bool up = false;
#pragma unroll
          for (int t = 0; t < NX; ++t) {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i >> 2][t][i & 3], CE_L2E, base[t]));
            add[t] = ((p[t][0] + p[t][1]) + (p[t][2] + p[t][3])) + ((p[t][4] + p[t][5]) + (p[t][6] + p[t][7]));
            up |= !(add[t] <= CeT<T>::LIM);
          }
          return up;
        };
        if (__any(powers()) && !fresh) {   // rare: no power is above 2^OFF afterwards
          move();
          powers();
        }
#pragma unroll
        for (int t = 0; t < NX; ++t) {
          sum[t] += add[t];
#pragma unroll
          for (int i = 0; i < 8; ++i) P[t][i] = (T)p[t][i];
        }
      } else {
        f4 e[2];   // log2(|g| / Σ exp) of this lane's rows
#pragma unroll
        for (int j = 0; j < 2; ++j) e[j] = *reinterpret_cast<const f4*>(r + at + 16 * j);
        if (far) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int t = 0; t < NX; ++t) S[j][t] -= *reinterpret_cast<const f4*>(r + 3 * CE_CH + at + 16 * j);
        }
        float p[NX][8];
#pragma unroll
        for (int t = 0; t < NX; ++t)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            p[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i >> 2][t][i & 3], CE_L2E, e[i >> 2][i & 3]));
        if (mine || sign) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float share = r[CE_CH + at + 16 * (i >> 2) + (i & 3)];
            const int tg = __float_as_int(r[2 * CE_CH + at + 16 * (i >> 2) + (i & 3)]);
#pragma unroll
            for (int t = 0; t < NX; ++t) {
              if (!__builtin_signbitf(share)) p[t][i] = -p[t][i];
              if (tg == x0 + 16 * t + n) p[t][i] = share;
            }
          }
        }
#pragma unroll
        for (int t = 0; t < NX; ++t) {
          if constexpr (BIAS)
            sum[t] += ((p[t][0] + p[t][1]) + (p[t][2] + p[t][3])) + ((p[t][4] + p[t][5]) + (p[t][6] + p[t][7]));
#pragma unroll
          for (int i = 0; i < 8; ++i) P[t][i] = (T)p[t][i];
        }
      }
      if constexpr (GRAD) {
        const int row = 32 * h + 4 * kg + (nn >> 2);
#pragma unroll
        for (int f = 0; f < FB; ++f) {
          const int ch = 2 * f + ((nn >> 1) & 1);
          uint8_t* p0 = y + row * RB + ((ch ^ ce_swz<DP>(row)) << 4) + 8 * (nn & 1);
          uint8_t* p1 = p0 + 16 * RB;   // 16 rows on, the same swizzle
          const ce_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ce_s4*)p0);
          const ce_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ce_s4*)p1);
          const ce_s8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
          for (int t = 0; t < NX; ++t) O[f][t] = CeT<T>::mm(__builtin_bit_cast(V, v), P[t], O[f][t]);
        }
      }
    }
  };
  __syncthreads();
  for (int c = c0; c < c1; c += 2) {
    if (c + 1 < c1) issue(c + 1, y1, r1);
    __builtin_amdgcn_sched_barrier(0);
    work(c, y0, r0);
    __syncthreads();
    if (c + 1 < c1) {
      if (c + 2 < c1) issue(c + 2, y0, r0);
      __builtin_amdgcn_sched_barrier(0);
      work(c + 1, y1, r1);
      __syncthreads();
    }
  }

  if constexpr (!FWD) {   // what rounding left off the targets' shares
    // each wave's rows with targets among its items, as item << 24 | row: as many as there is room for, the others are in
    // the chunks from `resume` on.  Four chunks are looked through at once, four rows a lane.
    constexpr int LIST = DP == 64 ? 640 : 1024;   // (two workgroups a CU at 64 columns, one at more)
    static_assert(16 * NX <= 256, "");
    __shared__ uint32_t list[NW][LIST];
    __shared__ float left_off[NW][LIST];
    __shared__ int have_of[NW], resume_of[NW];
    auto next = [&](int c) {   // the first of the chunks c, c + 4, .. that may have some, or one behind the last
      const int group = (c - c0) >> fold;
      const uint64_t rest = c < c1 ? met >> group : 0;
      return rest == 0 ? c1 : rest & 1 ? c : c0 + ((group + __builtin_ctzll(rest)) << fold);
    };
    int n = threadIdx.x & 15, kg = (threadIdx.x & 63) >> 4;
    asm volatile("" : "+v"(n), "+v"(kg));   // what is derived from them is not kept over the loop above
    const int lane = 16 * kg + n;
    int have = 0, resume = next(c0);
    auto fill = [&]() __attribute__((always_inline)) {
      have = 0;
      for (bool room = true; resume < c1 && room;) {
        constexpr int AHEAD = DP == 64 ? 2 : 4;
        int c[AHEAD];
        f4 share[AHEAD], target[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          c[i] = i == 0 ? resume : next(c[i - 1] + 4);
          const float* rec = a.recs + (int64_t)min(c[i] + kg, c1 - 1) * 4 * CE_CH + 4 * n;
          share[i] = *reinterpret_cast<const f4*>(rec + CE_CH);
          target[i] = *reinterpret_cast<const f4*>(rec + 2 * CE_CH);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          uint64_t mask[4];
          int more = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = __float_as_int(target[i][e]) - x0;
            const float all = share[i][e];
            share[i][e] = all - (float)(T)all;
            mask[e] = __ballot(c[i] + kg < c1 && at >= 0 && at < 16 * NX && fabsf(share[i][e]) > CE_REST * fabsf(all));
            more += __popcll(mask[e]);
          }
          room = room && have + more <= LIST;
          if (!room) continue;
          if (more > 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int place = have + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask[e] >> 32),
                                                                      __builtin_amdgcn_mbcnt_lo((uint32_t)mask[e], 0));
              if (mask[e] >> lane & 1) {
                list[wave][place] = (uint32_t)(__float_as_int(target[i][e]) - x0) << 24 |
                                    (uint32_t)((c[i] + kg) * CE_CH + 4 * n + e);
                left_off[wave][place] = share[i][e];
              }
              have += __popcll(mask[e]);
            }
          }
          resume = next(c[i] + 4);
        }
      }
      if (lane == 0) {
        have_of[wave] = have;
        resume_of[wave] = resume;
      }
    };
    auto entries = [&](uint32_t* e, int w, int first, int count) __attribute__((always_inline)) {   // 32 of wave w's list
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = first + 8 * kg + j;
        e[j] = list[w][at < count ? at : 0];
      }
    };
    auto shares = [&](V* P, const uint32_t* e, int w, int first, int count) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = first + 8 * kg + j;
        const T rest = (T)(at < count ? left_off[w][at] : 0.f);
#pragma unroll
        for (int t = 0; t < NX; ++t) P[t][j] = e[j] >> 24 == 16 * t + n ? rest : (T)0.f;
      }
    };
    auto columns = [&](uint32_t* v, const uint32_t* e, int f) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = reinterpret_cast<const uint16_t*>(Y)[(int64_t)(e[j] & 0xffffff) * DP + 16 * f + n];
    };
    auto pack = [](const uint32_t* v) __attribute__((always_inline)) {
      typedef uint32_t u4 __attribute__((ext_vector_type(4)));
      const u4 w = {v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16};
      return __builtin_bit_cast(V, w);
    };
    fill();
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) all += have_of[w];
    // a long list that is a good part of the workgroup's is shared: each wave takes 64 of the columns and some of the rows.  A
    // lane loads four neighbouring columns, so column 4·i + q of them is row i of the wave's tile q.
    uint32_t together = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w)
      together |= resume_of[w] < c1 || (have_of[w] > 64 && have_of[w] > all / 4) ? 1u << w : 0;
    together = __builtin_amdgcn_readfirstlane(together);
    for (; together != 0; together &= together - 1) {
      const int w = __builtin_ctz(together);
      constexpr int SPLIT = NW * 64 / DP, AT_ONCE = DP == 64 ? 1 : 2;
      const int group = wave / SPLIT, split = wave % SPLIT;
      f4 part[4][NX];
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int t = 0; t < NX; ++t) part[q][t] = zero;
      while (true) {
        const int count = __builtin_amdgcn_readfirstlane(have_of[w]);
        const bool last = __builtin_amdgcn_readfirstlane(resume_of[w]) >= c1;
        for (int k = split * 32 * AT_ONCE; k < count; k += SPLIT * 32 * AT_ONCE) {
          uint32_t e[AT_ONCE][8];
          ce_u2 v[AT_ONCE][8];
#pragma unroll
          for (int i = 0; i < AT_ONCE; ++i) entries(e[i], w, k + 32 * i, count);
#pragma unroll
          for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j)
              v[i][j] = *reinterpret_cast<const ce_u2*>(Y + (int64_t)(e[i][j] & 0xffffff) * DP + 64 * group + 4 * n);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < AT_ONCE; ++i) {
            V P[NX];
            shares(P, e[i], w, k + 32 * i, count);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t x[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) x[j] = q & 1 ? v[i][j][q >> 1] >> 16 : v[i][j][q >> 1] & 0xffff;
#pragma unroll
              for (int t = 0; t < NX; ++t) part[q][t] = CeT<T>::mm(pack(x), P[t], part[q][t]);
            }
          }
        }
        if (last) break;
        __syncthreads();
        if (wave == w) fill();
        __syncthreads();
      }
      // joined where a chunk was, one split after the other: [column][tile][item], 4 bytes
      static_assert(sizeof(y0) >= DP * NX * 16 * 4, "");
      float* parts = reinterpret_cast<float*>(y0);
#pragma unroll
      for (int x = 0; x < SPLIT; ++x) {
        if (split == x) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int t = 0; t < NX; ++t)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float* p = parts + ((64 * group + 4 * (4 * kg + i) + q) * NX + t) * 16 + n;
                *p = x == 0 ? part[q][t][i] : *p + part[q][t][i];
              }
        }
        __syncthreads();
      }
      if (wave == w) {
        have = 0;
#pragma unroll
        for (int f = 0; f < FB; ++f)
#pragma unroll
          for (int t = 0; t < NX; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) O[f][t][i] += parts[((16 * f + 4 * kg + i) * NX + t) * 16 + n];
      }
      __syncthreads();
    }
    for (int k = 0; k < have; k += 32) {
      uint32_t e[8];
      V P[NX];
      entries(e, wave, k, have);
      shares(P, e, wave, k, have);
      constexpr int BATCH = FB < 8 ? FB : 8;   // tiles of columns whose loads are in flight at once
#pragma unroll
      for (int f0 = 0; f0 < FB; f0 += BATCH) {
        uint32_t v[BATCH][8];
#pragma unroll
        for (int f = 0; f < BATCH; ++f) columns(v[f], e, f0 + f);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int f = 0; f < BATCH; ++f)
#pragma unroll
          for (int t = 0; t < NX; ++t) O[f0 + f][t] = CeT<T>::mm(pack(v[f]), P[t], O[f0 + f][t]);
      }
    }
  }

#pragma unroll
  for (int t = 0; t < NX; ++t) {
    sum[t] += __shfl_xor(sum[t], 16);
    sum[t] += __shfl_xor(sum[t], 32);
    const int64_t x = x0 + 16 * t + n;
    if (x >= nx) continue;
    if constexpr (FWD) {
      const int64_t at = (int64_t)split * a.nx + x;
      if (kg == 0) {
        a.pm[at] = ref[t];
        a.pl[at] = sum[t];
      }
      if constexpr (GRAD) {
#pragma unroll
        for (int f = 0; f < FB; ++f) *reinterpret_cast<f4*>(a.pO + at * DP + 16 * f + 4 * kg) = O[f][t];
      }
    } else {
      const float back = *a.scale;
      if (a.nsplit > 1) {
        const int64_t first = (int64_t)a.block0 * 16 * NX * NW, at = split * (a.nx - first) + x - first;
        if (a.db != nullptr && kg == 0) a.pl[at] = sum[t] * back;
#pragma unroll
        for (int f = 0; f < FB; ++f)
          if (16 * f + 4 * kg < a.D) *reinterpret_cast<f4*>(a.pO + at * a.D + 16 * f + 4 * kg) = O[f][t] * back;
      } else {
        if (a.db != nullptr && kg == 0) a.db[x] = sum[t] * back;
        typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int f = 0; f < FB; ++f)
          if (16 * f + 4 * kg < a.D)
            *reinterpret_cast<T4*>((T*)a.dW + x * a.D + 16 * f + 4 * kg) =
                __builtin_convertvector(O[f][t] * back, T4);
      }
    }
  }
}

// Rows with a target >= 0, in order: tc (their targets, −1 for one that is no item), rows (their places), inv (the way
// back, −1: ignored), count; the losses of ignored rows.  A workgroup lists 1024 rows; with more than one the groups'
// counts come first and the packed copy of h (zeros behind column D and behind the last row) after.  Up to 1024 rows
// each workgroup lists them all and packs its share: two launches less.
__global__ __launch_bounds__(1024) void k_ce_count(const int64_t* __restrict__ tgt, int64_t st, int N, int* __restrict__ counts) {
  __shared__ int part[16];
  const int r = blockIdx.x * 1024 + threadIdx.x;
  const uint64_t on = __ballot(r < N && tgt[r < N ? r * st : 0] >= 0);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = __popcll(on);
  __syncthreads();
  if (threadIdx.x == 0) {
    int k = 0;
    for (int w = 0; w < 16; ++w) k += part[w];
    counts[blockIdx.x] = k;
  }
}
__device__ __forceinline__ void ce_pack8(const uint16_t* h, int64_t ldh, int D, int DP, int c, int r, int col, uint16_t* hp) {
  ce_s8 v = {0, 0, 0, 0, 0, 0, 0, 0};
  if (r >= 0 && col < D) v = *reinterpret_cast<const ce_s8*>(h + r * ldh + col);
  *reinterpret_cast<ce_s8*>(hp + (int64_t)c * DP + col) = v;
}
template <bool PACK>
__global__ __launch_bounds__(1024) void k_ce_rows(const int64_t* __restrict__ tgt, int64_t st, int N, int npad, int V,
                                                  const int* __restrict__ counts, int* __restrict__ count,
                                                  int* __restrict__ rows, int* __restrict__ tc, int* __restrict__ inv,
                                                  float* __restrict__ loss, const uint16_t* __restrict__ h, int64_t ldh,
                                                  int D, int DP, uint16_t* __restrict__ hp) {
  __shared__ int part[16], before[16], list[PACK ? 1024 : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = (PACK ? 0 : blockIdx.x * 1024) + tid;
  const int64_t t = tgt[r < N ? r * st : 0];
  const bool on = r < N && t >= 0;
  const uint64_t mask = __ballot(on);
  int base = 0;
  if constexpr (PACK)
    list[tid] = -1;
  else
    for (int i = tid; i < (int)blockIdx.x; i += 1024) base += counts[i];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) base += __shfl_xor(base, o);
  if (lane == 0) {
    part[wave] = __popcll(mask);
    before[wave] = base;
  }
  __syncthreads();
  int at = 0, all = 0;
  for (int w = 0; w < 16; ++w) {
    at += before[w];
    all += before[w] + part[w];
    if (w < wave) at += part[w];
  }
  at += __popcll(mask & ((1ull << lane) - 1));
  if (PACK && on) list[at] = r;
  if (!PACK || blockIdx.x == 0) {
    if (on) {
      rows[at] = r;
      tc[at] = t < V ? (int)t : -1;
      inv[r] = at;
    } else if (r < N) {
      inv[r] = -1;
      loss[r] = 0.f;
    }
  }
  if (blockIdx.x == (PACK ? 0 : gridDim.x - 1)) {
    if (tid == 0) *count = all;
    for (int c = all + tid; c < npad; c += 1024) rows[c] = -1;
  }
  if constexpr (PACK) {
    __syncthreads();
    const int e = blockIdx.x * 1024 + tid, c = e / (DP / 8);
    if (c < npad) ce_pack8(h, ldh, D, DP, c, list[c], e % (DP / 8) * 8, hp);
  }
}
__global__ __launch_bounds__(256) void k_ce_pack(const uint16_t* __restrict__ h, int64_t ldh, int D, int DP, int npad,
                                                 const int* __restrict__ rows, uint16_t* __restrict__ hp) {
  const int e = blockIdx.x * 256 + threadIdx.x, c = e / (DP / 8);
  if (c < npad) ce_pack8(h, ldh, D, DP, c, rows[c], e % (DP / 8) * 8, hp);
}

// One wave per packed row: the splits' sums (without the target) and the target's logit joined.  With the odds q against the
// target, as x = log2 q: loss = log(1 + q), and (GRAD) dh for g = 1 in fp32, with the target's share 1 − p_t = q / (1 + q).  For
// the backward pass the row's log-sum-exp: `lse` in base 2, or, where it lies beyond CE_FAR, `top` the largest logit and
// `lse` what is added to it.
template <typename T, bool GRAD>
__global__ __launch_bounds__(256) void k_ce_join(const float* __restrict__ pm, const float* __restrict__ pl,
                                                 const float* __restrict__ pO, int nsplit, int N, int D, int DP,
                                                 const T* __restrict__ hp, const T* __restrict__ W, int64_t ldw,
                                                 const float* __restrict__ bias, const int* __restrict__ count,
                                                 const int* __restrict__ rows, const int* __restrict__ tc,
                                                 float* __restrict__ loss, float* __restrict__ lse,
                                                 float* __restrict__ top, float* __restrict__ against,
                                                 float* __restrict__ dh) {
  const int lane = threadIdx.x & 63, c = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (c >= *count) return;
  float m = CE_LOW;
  for (int s = lane; s < nsplit; s += 64) m = fmaxf(m, pm[(int64_t)s * N + c]);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
  float l = 0.f;
  for (int s = lane; s < nsplit; s += 64)
    l += pl[(int64_t)s * N + c] * ce_weight<T>(pm[(int64_t)s * N + c], m);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o);
  const int t = tc[c];
  const T* w = W + (int64_t)(t < 0 ? 0 : t) * ldw;
  float z = 0.f;
  for (int f = lane; f < D; f += 64) z = __builtin_fmaf((float)hp[(int64_t)c * DP + f], (float)w[f], z);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) z += __shfl_xor(z, o);
  if (bias != nullptr && t >= 0) z += bias[t];
  // a target that is no item: NaN in the loss and, through lse, in the gradients; so does an infinite logit of the target
  if (t < 0 || z == __builtin_inff()) z = __builtin_nanf("");
  const bool near = ce_near(m);
  const float rest = __log2f(l) - (near ? ce_base<T>(m) : CeT<T>::OFF);   // of the others, to the base of m
  const float x = near ? __builtin_fmaf(-z, CE_L2E, rest) : __builtin_fmaf(m - z, CE_L2E, rest);
  const float e = __builtin_amdgcn_exp2f(-fabsf(x)), share = (x >= 0.f ? 1.f : e) / (1.f + e);
  if (lane == 0) {
    const bool own = !(x >= 0.f);   // the target's logit is the larger part of the sum
    const float big = own ? z : m;
    loss[rows[c]] = __builtin_fmaf(own ? 0.f : x, CE_LN2, log1pf(e));
    lse[c] = (own ? ce_near(z) ? z * CE_L2E : 0.f : rest) + __log2f(1.f + e);
    top[c] = ce_near(big) ? 0.f : big;
    against[c] = share;
  }
  if constexpr (GRAD) {
    // DP / 4 lanes per split, several splits at once
    const float one = l != 0.f ? share / l : 0.f;
    const int per = DP / 4, f = lane % per * 4;
    f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = lane / per; s < nsplit; s += 64 / per)
      o += *reinterpret_cast<const f4*>(pO + ((int64_t)s * N + c) * DP + f) * ce_weight<T>(pm[(int64_t)s * N + c], m);
    for (int x = per; x < 64; x <<= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], x);
    if (lane < per && f < D) {
      f4 d;
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = t < 0 ? __builtin_nanf("") : __builtin_fmaf(o[i], one, -share * (float)w[f + i]);
      *reinterpret_cast<f4*>(dh + (int64_t)c * D + f) = d;
    }
  }
}

// the largest |g| of 1024 rows that are not ignored
__global__ __launch_bounds__(1024) void k_ce_largest(const float* __restrict__ g, int64_t sg, const int* __restrict__ inv,
                                                     int N, float* __restrict__ largest) {
  __shared__ float part[16];
  const int r = blockIdx.x * 1024 + threadIdx.x;
  float m = r < N && inv[r] >= 0 ? fabsf(g[r * sg]) : 0.f;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 0; w < 16; ++w) m = fmaxf(m, part[w]);
    largest[blockIdx.x] = m;
  }
}

// dh = g times what the forward left, zeros for ignored rows; the backward pass's records of the packed rows (four
// values: log2 |g| − lse in base 2; the target's −g (1 − p_t), whose sign bit is clear where g is negative; the target as
// int bits; and what is taken off the logits first, not 0 only beyond CE_FAR), and the factor that the scaled g leave
// out.  largest: of every 1024 rows, or null, and each wave looks at the rows itself.
template <typename T>
__global__ __launch_bounds__(256) void k_ce_dh(const float* __restrict__ g, int64_t sg, const int* __restrict__ inv,
                                               const int* __restrict__ count, const int* __restrict__ tc,
                                               const float* __restrict__ lse, const float* __restrict__ far,
                                               const float* __restrict__ against, const float* __restrict__ dh0, int N,
                                               int npad, int D, const float* __restrict__ largest, T* __restrict__ dh,
                                               float* __restrict__ recs, float* __restrict__ scale) {
  const int lane = threadIdx.x & 63, r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= npad) return;
  float top = 0.f;
  if (largest != nullptr)
    for (int i = lane; i < (N + 1023) / 1024; i += 64) top = fmaxf(top, largest[i]);
  else
    for (int i = lane; i < N; i += 64) top = fmaxf(top, inv[i] >= 0 ? fabsf(g[i * sg]) : 0.f);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
  top = top < __builtin_inff() ? fmaxf(top, 0x1p-100f) : 1.f;
  if (r == 0 && lane == 0) *scale = top * 0x1p-13f;
  if (lane == 0 && r >= *count) {   // behind the last packed row
    float* rec = recs + (int64_t)(r / CE_CH) * 4 * CE_CH + r % CE_CH;
    rec[0] = -__builtin_inff();
    rec[CE_CH] = -0.f;
    rec[2 * CE_CH] = __int_as_float(-1);
    rec[3 * CE_CH] = 0.f;
  }
  if (r >= N) return;
  const int c = inv[r];
  const float gr = c >= 0 ? g[r * sg] : 0.f;
  for (int f = lane * 4; f < D; f += 256) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const f4 v = c >= 0 ? *reinterpret_cast<const f4*>(dh0 + (int64_t)c * D + f) * gr : (f4){0.f, 0.f, 0.f, 0.f};
    *reinterpret_cast<T4*>(dh + (int64_t)r * D + f) = __builtin_convertvector(v, T4);
  }
  if (lane == 0 && c >= 0) {
    float* rec = recs + (int64_t)(c / CE_CH) * 4 * CE_CH + c % CE_CH;
    const float w = gr / top * 0x1p13f;
    rec[0] = __log2f(fabsf(w)) - lse[c];
    rec[CE_CH] = -w * against[c];
    rec[2 * CE_CH] = __int_as_float(tc[c]);
    rec[3 * CE_CH] = far[c];
  }
}

// backward slabs added up in a fixed order
template <typename T>
__global__ __launch_bounds__(256) void k_ce_slabs(const float* __restrict__ pO, const float* __restrict__ pl,
                                                  int nsplit, int V, int D, T* __restrict__ dW, float* __restrict__ db) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  const int64_t n = (int64_t)V * D / 4, step = (int64_t)gridDim.x * 256;
  const f4* p = reinterpret_cast<const f4*>(pO);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += step) {
    f4 x = p[i];
    for (int s = 1; s < nsplit; ++s) x += p[s * n + i];
    reinterpret_cast<T4*>(dW)[i] = __builtin_convertvector(x, T4);
  }
  if (db != nullptr)
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < V; i += step) {
      float x = pl[i];
      for (int s = 1; s < nsplit; ++s) x += pl[(int64_t)s * V + i];
      db[i] = x;
    }
}

// ------------------------------------------------------------------ host ----
static int ce_dp(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
static int64_t ce_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
// a workgroup holds CE_NW · CE_NX · 16 = 256 rows of X: eight waves, two on a SIMD, so that one's exponentials run beside
// the other's MFMAs, and two tiles a wave.  Measured (4096 x 1M x 128 bf16 / 7867 rows x 78K x 256 fp16, whole
// step, as the passes were then): two tiles 3.52 / 1.31 ms, three (128 columns; registers full) 4.36 ms, one 4.17 / 1.41 ms,
// four waves with two to six tiles each 5.2 ms and more (nothing beside the exponentials).  Exponentials woven between the
// MFMAs of the tiles before and after by hand (three buffers, sched_group_barrier): 116 to 800 registers spilled, 14.9 / 9.5 ms.
#define CE_NX 2
#define CE_NW 8

// splits of the streamed axis: fewest rounds of 256 workgroups times a split's chunks (and two chunks' worth of start
// and end), a chunk of 64 rows taking a CU about `chunk` us; every split's partial results are written and read
static int ce_splits(int64_t nblock, int64_t nch, double chunk, double bytes, int64_t most) {
  if (most > nch) most = nch;
  int best = 1;
  double cost = 1e30;
  for (int64_t s = 1; s <= most && s <= 512; ++s) {
    if (s > 8 && s % 8) continue;
    const double c = (double)((nblock * s + 255) / 256) * ((nch + s - 1) / s + 2) * chunk + (s > 1 ? s * bytes / 4e6 : 0.0);
    if (c < cost * 0.999) cost = c, best = (int)s;
  }
  return best;
}

struct CePlan {
  int DP, xw, npad, fblocks, fsplits;
  int bwhole, brest, bsplits;   // backward: blocks done whole (rounds of 256 workgroups), and the rest in splits
  int64_t items;                // of the rest
};
static CePlan ce_plan(int N, int V, int D) {
  CePlan p;
  p.DP = ce_dp(D);
  p.xw = 16 * CE_NW * CE_NX;
  p.npad = (int)ce_up(N, CE_PAD);
  p.fblocks = (N + p.xw - 1) / p.xw;
  // partial results: at most 2^28 values
  const double chunk = p.xw * (p.DP / 64) * 0.006;
  p.fsplits = ce_splits(p.fblocks, (V + CE_CH - 1) / CE_CH, chunk, 8.0 * N * p.DP,
                        ((int64_t)1 << 28) / ((int64_t)p.npad * p.DP) + 1);
  // backwards full rounds of 256 blocks go whole, the last, partial one is split over the rows to fill the CUs
  const int blocks = (V + p.xw - 1) / p.xw;
  p.bwhole = blocks / 256 * 256;
  p.brest = blocks - p.bwhole;
  p.items = V - (int64_t)p.bwhole * p.xw;
  p.bsplits = p.brest == 0 ? 1 : ce_splits(p.brest, (N + CE_CH - 1) / CE_CH, chunk, 8.0 * p.items * D,
                                           ((int64_t)1 << 28) / (p.items * D) + 1);
  return p;
}

static int ce_check(int64_t N, int64_t V, int D, int type) {
  if (type != 1 && type != 2) return RG_ERR_ARG;
  if (N <= 0 || N > (1 << 24) || V <= 0 || V > 0x7ffffff0 - 4096 || D <= 0 || D % 8 || D > 256) return RG_ERR_SHAPE;
  return RG_OK;
}

// forward scratch (floats): pm, pl, pO; backward: scale, recs, pO slabs and pl slabs (before them the largest |g|s)
extern "C" int64_t rg_linear_ce_work_floats(int N, int V, int D, int pass) {
  if (ce_check(N, V, D, 1) != RG_OK) return 0;
  const CePlan p = ce_plan(N, V, D);
  if (pass == 0) return 2 * (int64_t)p.fsplits * N + 64;
  if (pass == 1) return 2 * (int64_t)p.fsplits * N + 64 + (int64_t)p.fsplits * N * p.DP;
  const int64_t slabs = p.bsplits > 1 ? p.bsplits * p.items * (D + 1) + 64 : 0, groups = (N + 1023) / 1024;
  return 64 + 4 * (int64_t)p.npad + (slabs > groups ? slabs : groups);
}
// what the backward pass needs of the forward (bytes): packed h, lists, lse (two values), 1 − p_t, dh for g = 1
extern "C" int64_t rg_linear_ce_saved_bytes(int N, int V, int D) {
  if (ce_check(N, V, D, 1) != RG_OK) return 0;
  const int64_t npad = ce_up(N, CE_PAD);
  return 256 + npad * (ce_dp(D) * 2 + 6 * 4) + (int64_t)N * D * 4;
}
struct CeSaved {
  void* hp;
  int *count, *rows, *tc, *inv;
  float *lse, *top, *against, *dh0;
};
static CeSaved ce_saved(void* base, int N, int D) {
  const int64_t npad = ce_up(N, CE_PAD);
  CeSaved s;
  uint8_t* p = (uint8_t*)base;
  s.count = (int*)p;
  p += 256;
  s.hp = p;
  p += npad * ce_dp(D) * 2;
  s.rows = (int*)p;
  s.tc = s.rows + npad;
  s.inv = s.tc + npad;
  s.lse = (float*)(s.inv + npad);
  s.top = s.lse + npad;
  s.against = s.top + npad;
  s.dh0 = s.against + npad;
  return s;
}

template <typename T, int DP, bool FWD, bool GRAD, bool BIAS>
static int ce_pass(const CeArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((k_ce_pass<T, DP, CE_NX, CE_NW, FWD, GRAD, BIAS>), dim3(a.nblock * a.nsplit),
                     dim3(64 * CE_NW), 0, st, a);
  RG_LAUNCH_CHECK();
  return RG_OK;
}
template <typename T, bool FWD, bool GRAD, bool BIAS>
static int ce_pass(int DP, const CeArgs& a, hipStream_t st) {
  return DP == 64    ? ce_pass<T, 64, FWD, GRAD, BIAS>(a, st)
         : DP == 128 ? ce_pass<T, 128, FWD, GRAD, BIAS>(a, st)
                     : ce_pass<T, 256, FWD, GRAD, BIAS>(a, st);
}

template <typename T>
static int ce_fwd(const void* h, int64_t ldh, const void* W, int64_t ldw, const float* bias, const int64_t* tgt,
                  int64_t st_t, int N, int V, int D, bool grad, float* work, void* saved, float* loss, hipStream_t st) {
  const CePlan p = ce_plan(N, V, D);
  const CeSaved s = ce_saved(saved, N, D);
  const int groups = (N + 1023) / 1024;
  int* counts = (int*)s.lse;   // not written before the join
  const int pieces = p.npad * (p.DP / 8);
  auto list = [&](auto kern, int grid) {
    hipLaunchKernelGGL(kern, dim3(grid), dim3(1024), 0, st, tgt, st_t, N, p.npad, V, counts, s.count, s.rows, s.tc, s.inv,
                       loss, (const uint16_t*)h, ldh, D, p.DP, (uint16_t*)s.hp);
  };
  if (groups == 1) {
    list(k_ce_rows<true>, (pieces + 1023) / 1024);
  } else {
    hipLaunchKernelGGL(k_ce_count, dim3(groups), dim3(1024), 0, st, tgt, st_t, N, counts);
    list(k_ce_rows<false>, groups);
    hipLaunchKernelGGL(k_ce_pack, dim3((pieces + 255) / 256), dim3(256), 0, st, (const uint16_t*)h, ldh, D, p.DP, p.npad,
                       s.rows, (uint16_t*)s.hp);
  }
  RG_LAUNCH_CHECK();
  CeArgs a = {};
  a.X = s.hp, a.ldx = p.DP, a.nx = N, a.Y = W, a.ldy = ldw, a.ny = V, a.D = D, a.count = s.count, a.bias = bias, a.tc = s.tc;
  a.nsplit = p.fsplits, a.nblock = p.fblocks;
  a.pm = work, a.pl = work + (int64_t)p.fsplits * N;
  a.pO = work + ce_up(2 * (int64_t)p.fsplits * N, 64);
  const int rc = grad ? ce_pass<T, true, true, false>(p.DP, a, st) : ce_pass<T, true, false, false>(p.DP, a, st);
  if (rc != RG_OK) return rc;
  auto join = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((N + 3) / 4), dim3(256), 0, st, a.pm, a.pl, a.pO, p.fsplits, N, D, p.DP,
                       (const T*)s.hp, (const T*)W, ldw, bias, s.count, s.rows, s.tc, loss, s.lse, s.top, s.against, s.dh0);
  };
  if (grad)
    join(k_ce_join<T, true>);
  else
    join(k_ce_join<T, false>);
  RG_LAUNCH_CHECK();
  return RG_OK;
}

template <typename T>
static int ce_bwd(const void* W, int64_t ldw, const float* bias, const float* g, int64_t sg, int N, int V, int D,
                  const void* saved, float* work, void* dh, void* dW, float* db, hipStream_t st) {
  const CePlan p = ce_plan(N, V, D);
  const CeSaved s = ce_saved(const_cast<void*>(saved), N, D);
  const int groups = (N + 1023) / 1024;
  float *scale = work, *recs = work + 64, *largest = groups > 1 ? recs + 4 * (int64_t)p.npad : nullptr;
  if (groups > 1) hipLaunchKernelGGL(k_ce_largest, dim3(groups), dim3(1024), 0, st, g, sg, s.inv, N, largest);
  hipLaunchKernelGGL(k_ce_dh<T>, dim3((p.npad + 3) / 4), dim3(256), 0, st, g, sg, s.inv, s.count, s.tc, s.lse, s.top, s.against, s.dh0, N,
                     p.npad, D, largest, (T*)dh, recs, scale);
  RG_LAUNCH_CHECK();
  CeArgs a = {};
  a.X = W, a.ldx = ldw, a.nx = V, a.Y = s.hp, a.ldy = p.DP, a.ny = N, a.D = D, a.count = s.count, a.bias = bias;
  a.recs = recs, a.dW = dW, a.db = db, a.scale = scale;
  auto pass = [&]() {
    return bias != nullptr ? ce_pass<T, false, true, true>(p.DP, a, st) : ce_pass<T, false, true, false>(p.DP, a, st);
  };
  if (p.bwhole > 0) {
    a.nsplit = 1, a.nblock = p.bwhole, a.block0 = 0;
    const int rc = pass();
    if (rc != RG_OK) return rc;
  }
  if (p.brest > 0) {
    a.nsplit = p.bsplits, a.nblock = p.brest, a.block0 = p.bwhole;
    a.pO = recs + 4 * (int64_t)p.npad, a.pl = a.pO + ce_up(p.bsplits * p.items * D, 64);
    const int rc = pass();
    if (rc != RG_OK) return rc;
  }
  if (p.bsplits > 1) {
    const int64_t first = V - p.items, blocks = (p.items * D / 4 + 255) / 256;
    hipLaunchKernelGGL(k_ce_slabs<T>, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, a.pO, a.pl,
                       p.bsplits, (int)p.items, D, (T*)dW + first * D, db != nullptr ? db + first : nullptr);
    RG_LAUNCH_CHECK();
  }
  return RG_OK;
}

// 16-byte rows; a chunk's 64 rows have to stay within a buffer's 2 GB
static bool ce_rows_ok(const void* p, int64_t ld, int D) {
  return p != nullptr && ((uintptr_t)p & 15) == 0 && ld >= D && ld % 8 == 0 && ld < ((int64_t)1 << 23);
}

extern "C" int rg_linear_ce_fwd(const void* h, int64_t ldh, const void* W, int64_t ldw, const float* bias,
                                const int64_t* target, int64_t target_stride, int type, int N, int V, int D, int grad,
                                float* work, void* saved, float* loss, hipStream_t stream) {
  const int rc = ce_check(N, V, D, type);
  if (rc != RG_OK) return rc;
  if (!ce_rows_ok(h, ldh, D) || !ce_rows_ok(W, ldw, D) || target == nullptr || work == nullptr || saved == nullptr ||
      loss == nullptr || (((uintptr_t)work | (uintptr_t)saved) & 15))
    return RG_ERR_ARG;
  return type == 1 ? ce_fwd<__bf16>(h, ldh, W, ldw, bias, target, target_stride, N, V, D, grad != 0, work, saved, loss, stream)
                   : ce_fwd<_Float16>(h, ldh, W, ldw, bias, target, target_stride, N, V, D, grad != 0, work, saved, loss, stream);
}

extern "C" int rg_linear_ce_bwd(const void* W, int64_t ldw, const float* bias, const float* dloss, int64_t dloss_stride,
                                int type, int N, int V, int D, const void* saved, float* work, void* dh, void* dW,
                                float* db, hipStream_t stream) {
  const int rc = ce_check(N, V, D, type);
  if (rc != RG_OK) return rc;
  if (!ce_rows_ok(W, ldw, D) || dloss == nullptr || saved == nullptr || work == nullptr || dh == nullptr ||
      dW == nullptr || (((uintptr_t)work | (uintptr_t)saved | (uintptr_t)dh | (uintptr_t)dW) & 15) ||
      (db != nullptr && bias == nullptr))
    return RG_ERR_ARG;
  return type == 1 ? ce_bwd<__bf16>(W, ldw, bias, dloss, dloss_stride, N, V, D, saved, work, dh, dW, db, stream)
                   : ce_bwd<_Float16>(W, ldw, bias, dloss, dloss_stride, N, V, D, saved, work, dh, dW, db, stream);
}
