// ---- activations of a few tokens times weights of 4 bits ----
//   Y[m][n] = sum over groups of scale[n][group] * sum over the group's k of X[m][k] * (code[n][k] - zero[n][group])
// X [M][K] in 16 bits; codes two to a byte, [N][K / 2], the even k in the low four bits; a scale, and if Q4_ZERO a zero (a byte), for each
// Q4_GROUP codes of a row, else zero = 8.
//
// The weights are read once and bound the launch, so they are spent as little on as they can be: the bits of a code are shifted into
// the mantissa of 1.0, which gives 1 + code / 16 exactly in either 16-bit type, eight codes in eight instructions.  The matrix
// product takes these and begins a group at -(1 + zero / 16) times the group's sum of X, which the wavefronts take on X's way into LDS;
// 16 scale times what comes out is the group's part of the result: codes, zeros and X enter unrounded, sums are fp32, the scale is applied in
// fp32.
// X is the left operand, so the result's lanes hold one column n and four rows: a group's scale is one number per lane.
//
// A dword of codes gives the pairs (0, 4) (1, 5) (2, 6) (3, 7) of its eight, and X is put into that order on its way into LDS.
//
// A wavefront has 16 Q4_NT columns and takes 256 k a step: 128 bytes of a row, whole lines.  Neighbouring lanes load neighbouring bytes
// and the tile goes through LDS rows that belong to the wavefront alone, where lane l finds column l % 16 (read where a lane needs them,
// four neighbouring lanes touch four lines).  Q4_WN wavefronts beside one another share the rows of X, Q4_WK groups of them split k and add
// their sums through LDS, and Q4_SPLIT workgroups split it again, whose fp32 results gemm_q4_join adds in order.
// Where a group has 128 codes or more, product j of a step's half takes k = 32 g + 8 j .. + 7 for quarter g of the wavefront, 16 bytes
// of codes as they come; smaller groups need products of 32 neighbouring k, so the quarters exchange dwords (four permlane swaps).
// Measured: 1 row, N = K = 4096, bf16, groups of 128: 3.8 to 4.4 us by the process (2 TB/s; reading as many bytes alone takes 3.0); 16 rows, N 11008, K 4096, half
// precision with zeros: 8.6 us (2.8 TB/s; reading alone 5.1); 61 rows, N 4096, K 11008, groups of 64: 17.9 us with the join's 3.  One row is
// bound by the launch and one trip to memory.  At 61 rows vector instructions are under way half of the time (codes to numbers, sums to results), LDS
// accesses, of X by every wavefront's columns anew, 57 %, matrix products 20 %, each step's one after the other.  The sums of X taken by the
// matrix product itself, with ones in the weights' place, cost this case 1.5 us.
// Parameters: Q4_NAME, Q4_N, Q4_K, Q4_GROUP, Q4_F16, Q4_ZERO, Q4_ST (type of the scales), Q4_YT (of the result), Q4_MB, Q4_MR (rows of X in
// LDS, up to 16 Q4_MB), Q4_NT, Q4_WN, Q4_WK, Q4_SPLIT, Q4_WIDE, Q4_JOIN (this is gemm_q4_join).
typedef _Float16 q4_f16x8 __attribute__((ext_vector_type(8)));
#if Q4_F16
typedef _Float16 q4_x;
#define Q4_MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(q4_f16x8, a), __builtin_bit_cast(q4_f16x8, b), c, 0, 0, 0)
#define Q4_ONE 0x3c003c00u
#define Q4_MASK 0x03c003c0u
#define Q4_DOT(a, c) __builtin_amdgcn_fdot2(__builtin_bit_cast(kcg_f16x2, a), __builtin_bit_cast(kcg_f16x2, Q4_ONE), c, false)
#define Q4_SHIFT(w, p) ((p) == 0 ? (w) << 6 : (p) == 1 ? (w) << 2 : (p) == 2 ? (w) >> 2 : (w) >> 6)
#else
typedef __bf16 q4_x;
#define Q4_MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(kcg_bf16x8, a), __builtin_bit_cast(kcg_bf16x8, b), c, 0, 0, 0)
#define Q4_ONE 0x3f803f80u
#define Q4_MASK 0x00780078u
#define Q4_DOT(a, c) __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(kcg_bf16x2, a), __builtin_bit_cast(kcg_bf16x2, Q4_ONE), c, false)
#define Q4_SHIFT(w, p) ((p) == 0 ? (w) << 3 : (p) == 1 ? (w) >> 1 : (p) == 2 ? (w) >> 5 : (w) >> 9)
#endif
#define Q4_STEPS ((Q4_K + 255) / 256)
#define Q4_PARTS (Q4_WK * Q4_SPLIT)
#define Q4_SHARE ((Q4_STEPS + Q4_PARTS - 1) / Q4_PARTS)       // steps of a wavefront
#define Q4_EXACT (Q4_K % 256 == 0 && Q4_STEPS == Q4_SHARE * Q4_PARTS)
#define Q4_GROUPS (Q4_K / Q4_GROUP)
#if Q4_WIDE            // offsets that 32 bits do not hold
typedef long long q4_offset;
#else
typedef unsigned q4_offset;
#endif
#define Q4_PER (Q4_GROUP >= 128 ? 1 : 128 / Q4_GROUP)         // groups of half a step
#define Q4_J (4 / Q4_PER)                                     // products of a group of half a step
#define Q4_COLS (16 * Q4_NT)
// A read of 16 bytes serves sixteen lanes at a time: rows 0 to 3 and 12 to 15 of one quarter and 4 to 11 of the next.  They meet all banks
// where rows are an odd number of 16 bytes apart and an odd quarter lies a multiple of 256 bytes behind the even one before it, in X within a
// row, in W in a plane of its own.  Lanes bring the chunks in an order whose writes meet few banks twice.
#define Q4_XPITCH 528                                         // bytes of a row of X in LDS
#define Q4_WPITCH 80                                          // and of one in a plane of W
#define Q4_WPLANE (Q4_COLS * Q4_WPITCH)
#define Q4_XPLACE(g, h, j) (((g) & 1) * 16 + ((g) >> 1) * 8 + (h) * 4 + (j))
#define Q4_XC ((Q4_MR * 32 + 64 * Q4_WN - 1) / (64 * Q4_WN))  // chunks of X that a lane brings
#define Q4_SC ((Q4_COLS * 2 * Q4_PER + 63) / 64)              // scales that a lane brings

#if Q4_JOIN
extern "C" __global__ __launch_bounds__(256)
void Q4_NAME(const float* __restrict__ part, long long M, Q4_YT* __restrict__ Y) {
  const long long total = M * Q4_N, at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= total) return;
  float sum = part[at];
#pragma unroll
  for (int i = 1; i < Q4_SPLIT; ++i) sum += part[i * total + at];
  Y[at] = (Q4_YT)sum;
}
#else
struct Q4Step {
  kcg_u32x4 w[2 * Q4_NT], x[Q4_XC];
  Q4_ST s[Q4_SC];
  unsigned char z[Q4_SC];
};

extern "C" __global__ __launch_bounds__(64 * Q4_WN * Q4_WK, 1)
void Q4_NAME(const q4_x* __restrict__ X, const unsigned char* __restrict__ W, const Q4_ST* __restrict__ scale, const unsigned char* __restrict__ zero,
             long long M_,
#if Q4_SPLIT > 1
             float* __restrict__ part
#else
             Q4_YT* __restrict__ Y
#endif
) {
  struct Tiles {
    __attribute__((aligned(16))) unsigned char x[Q4_WK][Q4_WN > 1 ? 2 : 1][Q4_MR * Q4_XPITCH], w[Q4_WK * Q4_WN][2 * Q4_WPLANE];
    kcg_f32x2 s[Q4_WK * Q4_WN][2 * Q4_PER][Q4_COLS];
    __attribute__((aligned(16))) float u[Q4_WK][Q4_WN > 1 ? 2 : 1][2 * Q4_PER][16 * Q4_MB];        // sums of X of a group
  };
  union Shared {
    Tiles t;
    kcg_f32x4 red[Q4_WK][Q4_WN * Q4_MB * Q4_NT][64];
  };
  __shared__ Shared sh;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % Q4_WN, wk = wave / Q4_WN, lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int M = (int)M_, n0 = (blockIdx.x * Q4_WN + wn) * Q4_COLS, m0 = blockIdx.y * (16 * Q4_MB);
  kcg_f32x4 acc[Q4_MB][Q4_NT];
#pragma unroll
  for (int a = 0; a < Q4_MB; ++a)
#pragma unroll
    for (int b = 0; b < Q4_NT; ++b) acc[a][b] = kcg_f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // mask and one in a scalar and a vector register: one v_and_or_b32 a pair, of which an instruction takes no more than one constant
  unsigned mask = Q4_MASK, one = Q4_ONE;
  asm("" : "+s"(mask));
  asm("" : "+v"(one));

  const int share = blockIdx.z * Q4_WK + wk, first = share * Q4_SHARE, kend = (first + Q4_SHARE) * 256 < Q4_K ? (first + Q4_SHARE) * 256 : Q4_K;
  // Rows and columns behind the last are read as the last, and their results are not stored; k behind the last is read as the first and
  // takes part with zeros of X.  (All loads are unconditional: one behind a branch would be waited for there.)  Addresses are a uniform
  // base, which goes on with the steps, and an offset of the lane's.
  q4_offset wo[2 * Q4_NT], xo[Q4_XC], so[Q4_SC];
  const int wc = lane % 4 * 2 + lane % 8 / 4;        // chunk of a row of W: lanes 0 to 3 the even ones, which go into one plane
#pragma unroll
  for (int b = 0; b < 2 * Q4_NT; ++b) {
    const int n = n0 + b * 8 + lane / 8;
    wo[b] = (q4_offset)(n < Q4_N ? n : Q4_N - 1) * (Q4_K / 2) + wc * 16;
  }
  int xk[Q4_XC], xat[Q4_XC];
#pragma unroll
  for (int c = 0; c < Q4_XC; ++c) {
    const int u = (c * Q4_WN + wn) * 64 + lane, row = u / 32, m = m0 + row;
    const int q = u % 16 / 4, j = u % 4;       // quarter and product that this lane's chunk of 8 k is for
    xk[c] = u % 32 / 16 * 128 + (Q4_PER == 1 ? q * 4 + j : j * 4 + q) * 8;
    xo[c] = (q4_offset)((m < M ? m : M - 1) - m0) * Q4_K + xk[c];
    xat[c] = row < Q4_MR ? row * Q4_XPITCH + Q4_XPLACE(q, u % 32 / 16, j) * 16 : -1;
  }
  int se[Q4_SC], sat[Q4_SC];
#pragma unroll
  for (int c = 0; c < Q4_SC; ++c) {
    const int u = c * 64 + lane, col = u / (2 * Q4_PER), n = n0 + col;
    se[c] = u % (2 * Q4_PER);
    so[c] = (q4_offset)(n < Q4_N ? n : Q4_N - 1) * Q4_GROUPS;
    sat[c] = col < Q4_COLS ? se[c] * Q4_COLS + col : -1;
  }
  auto load = [&](int n, Q4Step& s) {
    int k0 = (first + n) * 256;
    k0 = k0 < Q4_K ? k0 : 0;             // (the last wavefront's may lie behind the last k)
    // the first group of the step and the second half's; smaller groups follow one another
    const int g0 = k0 / Q4_GROUP, g1 = Q4_PER > 1 || k0 + 128 < Q4_K ? (k0 + 128) / Q4_GROUP : g0;
#pragma unroll
    for (int c = 0; c < Q4_SC; ++c) {
      int at = Q4_PER > 1 ? g0 + se[c] : se[c] ? g1 : g0;
      if (Q4_PER > 1 && Q4_K % 256) at = at < Q4_GROUPS ? at : 0;
      s.s[c] = scale[so[c] + at];
      if (Q4_ZERO) s.z[c] = zero[so[c] + at];
    }
    const unsigned char* wk0 = W + k0 / 2;
#pragma unroll
    for (int b = 0; b < 2 * Q4_NT; ++b) s.w[b] = *(const kcg_u32x4*)(wk0 + (Q4_K % 256 == 0 || k0 + wc * 32 < Q4_K ? wo[b] : wo[b] - wc * 16));
    const q4_x* xk0 = X + (long long)m0 * Q4_K + k0;
#pragma unroll
    for (int c = 0; c < Q4_XC; ++c) s.x[c] = *(const kcg_u32x4*)(xk0 + (Q4_K % 256 == 0 || k0 + xk[c] < Q4_K ? xo[c] : xo[c] - xk[c]));
  };
  auto stage = [&](int n, Q4Step& s, unsigned char* xs, float* us) {
    const int k0 = (first + n) * 256;
#pragma unroll
    for (int c = 0; c < Q4_XC; ++c) {
      const kcg_u32x4 v = Q4_EXACT || k0 + xk[c] < kend ? s.x[c] : kcg_u32x4{0, 0, 0, 0};
      const kcg_u32x4 o = {__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
                           __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
      if (Q4_MR * 32 % (64 * Q4_WN) == 0 || xat[c] >= 0) *(kcg_u32x4*)(xs + xat[c]) = o;
      // the sum over the lanes that have a group of the row (16, 8 or 4), times -1.5 where that is 1 + zero / 16 for all columns
      const unsigned v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3];      // (bit_cast of a vector's element takes the first)
      float sum = Q4_DOT(v0, Q4_DOT(v1, Q4_DOT(v2, Q4_DOT(v3, 0.0f))));
#define Q4_ADD(control) sum += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, sum), control, 0xf, 0xf, true))
      if (Q4_PER < 4) Q4_ADD(0xb1);            // quad_perm: 1 0 3 2
      if (Q4_PER < 2) Q4_ADD(0x4e);            // quad_perm: 2 3 0 1
      Q4_ADD(0x124);                           // row_ror 4, 8: over the quarters
      Q4_ADD(0x128);
#undef Q4_ADD
      if (lane % 16 / 4 == 0 && lane % (4 / Q4_PER) == 0 && xat[c] >= 0)
        us[(lane % 32 / 16 * Q4_PER + lane % 4 / (4 / Q4_PER)) * (16 * Q4_MB) + xat[c] / Q4_XPITCH] = Q4_ZERO ? sum : -1.5f * sum;
    }
#pragma unroll
    for (int b = 0; b < 2 * Q4_NT; ++b) *(kcg_u32x4*)(sh.t.w[wave] + lane % 8 / 4 * Q4_WPLANE + (b * 8 + lane / 8) * Q4_WPITCH + lane % 4 * 16) = s.w[b];
#pragma unroll
    for (int c = 0; c < Q4_SC; ++c)
      if (Q4_COLS * 2 * Q4_PER % 64 == 0 || sat[c] >= 0)
        (&sh.t.s[wave][0][0])[sat[c]] = kcg_f32x2{(float)s.s[c], Q4_ZERO ? -1.0f - (float)s.z[c] * 0.0625f : 0.0f};
  };
  auto multiply = [&](const unsigned char* xs, const float* us) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      kcg_u32x4 w4[Q4_NT];
#pragma unroll
      for (int b = 0; b < Q4_NT; ++b) {
        w4[b] = *(const kcg_u32x4*)(sh.t.w[wave] + g % 2 * Q4_WPLANE + (b * 16 + i) * Q4_WPITCH + (h * 2 + g / 2) * 16);
#if Q4_PER > 1
        // dword j of quarter g becomes dword g of quarter j
        auto x02 = __builtin_amdgcn_permlane32_swap(w4[b][0], w4[b][2], false, false);
        auto x13 = __builtin_amdgcn_permlane32_swap(w4[b][1], w4[b][3], false, false);
        auto x01 = __builtin_amdgcn_permlane16_swap(x02[0], x13[0], false, false);
        auto x23 = __builtin_amdgcn_permlane16_swap(x02[1], x13[1], false, false);
        w4[b] = kcg_u32x4{x01[0], x01[1], x23[0], x23[1]};
#endif
      }
#pragma unroll
      for (int p = 0; p < Q4_PER; ++p) {
        kcg_f32x4 t[Q4_MB][Q4_NT];
        float by[Q4_NT];
#pragma unroll
        for (int b = 0; b < Q4_NT; ++b) {
          const kcg_f32x2 s = sh.t.s[wave][h * Q4_PER + p][b * 16 + i];
          by[b] = s[0];
#pragma unroll
          for (int a = 0; a < Q4_MB; ++a) {
            t[a][b] = *(const kcg_f32x4*)(us + (h * Q4_PER + p) * (16 * Q4_MB) + a * 16 + g * 4);
            if (Q4_ZERO) t[a][b] *= s[1];
          }
        }
#pragma unroll
        for (int j = p * Q4_J; j < (p + 1) * Q4_J; ++j) {
          kcg_u32x4 x[Q4_MB];
#pragma unroll
          for (int a = 0; a < Q4_MB; ++a) {
            const int row = a * 16 + i < Q4_MR ? a * 16 + i : Q4_MR - 1;
            x[a] = *(const kcg_u32x4*)(xs + row * Q4_XPITCH + Q4_XPLACE(g, h, j) * 16);
          }
#pragma unroll
          for (int b = 0; b < Q4_NT; ++b) {
            const unsigned w = w4[b][j];
            const kcg_u32x4 f = {Q4_SHIFT(w, 0) & mask | one, Q4_SHIFT(w, 1) & mask | one, Q4_SHIFT(w, 2) & mask | one, Q4_SHIFT(w, 3) & mask | one};
#pragma unroll
            for (int a = 0; a < Q4_MB; ++a) t[a][b] = Q4_MFMA(x[a], f, t[a][b]);
          }
        }
#pragma unroll
        for (int b = 0; b < Q4_NT; ++b)
#pragma unroll
          for (int a = 0; a < Q4_MB; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[a][b][r] = __builtin_fmaf(by[b], t[a][b][r], acc[a][b][r]);
      }
    }
  };

  // Every wavefront makes Q4_SHARE steps; one that has fewer multiplies zeros in those behind its last.  A step is under way in registers
  // while the one before it is multiplied (two or three were no faster in any form).
  Q4Step next;
  load(0, next);
  auto step = [&](int n, bool more) __attribute__((always_inline)) {
    const int buffer = Q4_WN > 1 ? n & 1 : 0;
    __builtin_amdgcn_sched_barrier(0);
    stage(n, next, sh.t.x[wk][buffer], &sh.t.u[wk][buffer][0][0]);
    if (more) load(n + 1, next);
    // the rows of X are there, and those of the step before last have been read (a wavefront's own LDS accesses are carried out in order)
    if (Q4_WN > 1) __syncthreads(); else __builtin_amdgcn_wave_barrier();
    multiply(sh.t.x[wk][buffer], &sh.t.u[wk][buffer][0][0]);
  };
#pragma unroll 1
  for (int n = 0; n < Q4_SHARE - 1; ++n) step(n, true);
  step(Q4_SHARE - 1, false);
  __syncthreads();
#pragma unroll
  for (int a = 0; a < Q4_MB; ++a)
#pragma unroll
    for (int b = 0; b < Q4_NT; ++b) sh.red[wk][(wn * Q4_MB + a) * Q4_NT + b][lane] = acc[a][b];
  __syncthreads();
  for (int u = wave; u < Q4_WN * Q4_MB * Q4_NT; u += Q4_WN * Q4_WK) {
    kcg_f32x4 sum = sh.red[0][u][lane];
#pragma unroll
    for (int w = 1; w < Q4_WK; ++w) sum += sh.red[w][u][lane];
    const int n = (blockIdx.x * Q4_WN + u / (Q4_MB * Q4_NT)) * Q4_COLS + (u % Q4_NT) * 16 + i;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = m0 + (u / Q4_NT % Q4_MB) * 16 + g * 4 + r;
      if (n < Q4_N && m < M) {
#if Q4_SPLIT > 1
        part[((long long)blockIdx.z * M + m) * Q4_N + n] = 16.0f * sum[r];
#else
        Y[(long long)m * Q4_N + n] = (Q4_YT)(16.0f * sum[r]);
#endif
      }
    }
  }
}
#endif
