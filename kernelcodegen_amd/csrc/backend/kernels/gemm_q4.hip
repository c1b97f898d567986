// ---- activations of a few tokens times weights of 4 bits ----
//   Y[m][n] = sum over groups of scale[n][group] * sum over the group's k of X[m][k] * (code[n][k] - zero[n][group])
// X [M][K] in 16 bits; codes two to a byte, [N][K / 2], the even k in the low four bits; a scale, and if Q4_ZERO a zero (a byte), for each
// Q4_GROUP codes of a row, else zero = 8.
//
// The weights are read once and bound the launch, so they are spent as little on as they can be: the bits of a code are shifted into
// the mantissa of 1.0, which gives 1 + code / 16 exactly in either 16-bit type, eight codes in eight instructions.  The matrix
// product takes these, and a second one with ones in the weights' place sums X; from a group's two fp32 sums t and u
//   16 scale (t - (1 + zero / 16) u)
// is the group's part of the result: codes, zeros and X enter unrounded, sums are fp32, the scale is applied in fp32.
// X is the left operand, so the result's lanes hold one column n and four rows: a group's scale is one number per lane.
//
// A dword of codes gives the pairs (0, 4) (1, 5) (2, 6) (3, 7) of its eight, and X is put into that order.  Where a group is 128 or more, a
// lane of quarter g takes k = 32 g + 8 j .. + 7 of a step of 128 for product j, 16 bytes of codes as they come; smaller groups
// need products of 32 neighbouring k, so the quarters exchange dwords first (four permlane swaps).
//
// A workgroup has 16 Q4_NT columns of up to 16 Q4_MB rows; its wavefronts split k (and the grid's z axis, if Q4_SPLIT) and add through LDS.
// Parameters: Q4_NAME, Q4_N, Q4_K, Q4_GROUP, Q4_F16, Q4_ZERO, Q4_ST (type of the scales), Q4_YT (of the result), Q4_MB, Q4_NT, Q4_WAVES.
typedef _Float16 q4_f16x8 __attribute__((ext_vector_type(8)));
#if Q4_F16
typedef _Float16 q4_x;
#define Q4_MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(q4_f16x8, a), __builtin_bit_cast(q4_f16x8, b), c, 0, 0, 0)
#define Q4_ONE 0x3c003c00u
#define Q4_MASK 0x03c003c0u
#define Q4_PAIR(w, p) (((p) == 0 ? (w) << 6 : (p) == 1 ? (w) << 2 : (p) == 2 ? (w) >> 2 : (w) >> 6) & Q4_MASK | Q4_ONE)
#else
typedef __bf16 q4_x;
#define Q4_MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(kcg_bf16x8, a), __builtin_bit_cast(kcg_bf16x8, b), c, 0, 0, 0)
#define Q4_ONE 0x3f803f80u
#define Q4_MASK 0x00780078u
#define Q4_PAIR(w, p) (((p) == 0 ? (w) << 3 : (p) == 1 ? (w) >> 1 : (p) == 2 ? (w) >> 5 : (w) >> 9) & Q4_MASK | Q4_ONE)
#endif
#define Q4_STEPS ((Q4_K + 127) / 128)
#define Q4_GROUPS (Q4_K / Q4_GROUP)
#define Q4_PER (Q4_GROUP >= 128 ? 1 : 128 / Q4_GROUP)         // groups of a step
#define Q4_J (4 / Q4_PER)                                     // products of a group of a step

struct Q4Step {
  kcg_u32x4 w[Q4_NT], x[Q4_MB][4];
  float s[Q4_NT][Q4_PER], z[Q4_NT][Q4_PER];
};

extern "C" __global__ __launch_bounds__(64 * Q4_WAVES)
void Q4_NAME(const q4_x* __restrict__ X, const unsigned char* __restrict__ W, const Q4_ST* __restrict__ scale, const unsigned char* __restrict__ zero,
             long long M_, Q4_YT* __restrict__ Y) {
  __shared__ kcg_f32x4 red[Q4_WAVES][Q4_MB * Q4_NT][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int M = (int)M_, n0 = blockIdx.x * (16 * Q4_NT), m0 = blockIdx.y * (16 * Q4_MB);
  kcg_f32x4 acc[Q4_MB][Q4_NT];
#pragma unroll
  for (int a = 0; a < Q4_MB; ++a)
#pragma unroll
    for (int b = 0; b < Q4_NT; ++b) acc[a][b] = kcg_f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // rows and columns behind the last are read as the last; their results are not stored
  const unsigned char* wp[Q4_NT];
  int col[Q4_NT];
#pragma unroll
  for (int b = 0; b < Q4_NT; ++b) {
    const int n = n0 + b * 16 + i;
    col[b] = n < Q4_N ? n : Q4_N - 1;
    wp[b] = W + (long long)col[b] * (Q4_K / 2);
  }
  const q4_x* xp[Q4_MB];
#pragma unroll
  for (int a = 0; a < Q4_MB; ++a) {
    const int m = m0 + a * 16 + i;
    xp[a] = X + (long long)(m < M ? m : M - 1) * Q4_K;
  }

  auto load = [&](int step, Q4Step& s) {
    const int k0 = step * 128;
    const int kw = k0 + g * 32;
#pragma unroll
    for (int b = 0; b < Q4_NT; ++b) {
      s.w[b] = *(const kcg_u32x4*)(wp[b] + (Q4_K % 128 == 0 || kw < Q4_K ? kw : 0) / 2);
#pragma unroll
      for (int p = 0; p < Q4_PER; ++p) {
        int at = (k0 + p * 128 / Q4_PER) / Q4_GROUP;
        if (Q4_K % 128 != 0 && at >= Q4_GROUPS) at = Q4_GROUPS - 1;
        s.s[b][p] = (float)scale[(long long)col[b] * Q4_GROUPS + at];
        s.z[b][p] = Q4_ZERO ? 1.0f + (float)zero[(long long)col[b] * Q4_GROUPS + at] * 0.0625f : 1.5f;
      }
    }
#pragma unroll
    for (int a = 0; a < Q4_MB; ++a)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = Q4_PER == 1 ? kw + j * 8 : k0 + j * 32 + g * 8;
        if (Q4_K % 128 == 0 || k < Q4_K)
          s.x[a][j] = *(const kcg_u32x4*)(xp[a] + k);
        else
          s.x[a][j] = kcg_u32x4{0, 0, 0, 0};          // takes the codes read in place of those behind the row out of all sums
      }
  };

  auto compute = [&](Q4Step& s) {
    const kcg_f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
    const kcg_u32x4 ones = {Q4_ONE, Q4_ONE, Q4_ONE, Q4_ONE};
#pragma unroll
    for (int a = 0; a < Q4_MB; ++a)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const kcg_u32x4 v = s.x[a][j];
        s.x[a][j] = kcg_u32x4{__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
                              __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
      }
#if Q4_PER > 1
    // dword j of quarter g becomes dword g of quarter j
#pragma unroll
    for (int b = 0; b < Q4_NT; ++b) {
      auto x02 = __builtin_amdgcn_permlane32_swap(s.w[b][0], s.w[b][2], false, false);
      auto x13 = __builtin_amdgcn_permlane32_swap(s.w[b][1], s.w[b][3], false, false);
      auto x01 = __builtin_amdgcn_permlane16_swap(x02[0], x13[0], false, false);
      auto x23 = __builtin_amdgcn_permlane16_swap(x02[1], x13[1], false, false);
      s.w[b] = kcg_u32x4{x01[0], x01[1], x23[0], x23[1]};
    }
#endif
#pragma unroll
    for (int p = 0; p < Q4_PER; ++p) {
      kcg_f32x4 u[Q4_MB], t[Q4_MB][Q4_NT];
#pragma unroll
      for (int a = 0; a < Q4_MB; ++a) {
        u[a] = none;
#pragma unroll
        for (int b = 0; b < Q4_NT; ++b) t[a][b] = none;
      }
#pragma unroll
      for (int j = p * Q4_J; j < (p + 1) * Q4_J; ++j) {
#pragma unroll
        for (int a = 0; a < Q4_MB; ++a) u[a] = Q4_MFMA(s.x[a][j], ones, u[a]);
#pragma unroll
        for (int b = 0; b < Q4_NT; ++b) {
          const unsigned w = s.w[b][j];
          const kcg_u32x4 f = {Q4_PAIR(w, 0), Q4_PAIR(w, 1), Q4_PAIR(w, 2), Q4_PAIR(w, 3)};
#pragma unroll
          for (int a = 0; a < Q4_MB; ++a) t[a][b] = Q4_MFMA(s.x[a][j], f, t[a][b]);
        }
      }
#pragma unroll
      for (int a = 0; a < Q4_MB; ++a)
#pragma unroll
        for (int b = 0; b < Q4_NT; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            acc[a][b][r] = __builtin_fmaf(s.s[b][p], __builtin_fmaf(-s.z[b][p], u[a][r], t[a][b][r]), acc[a][b][r]);
    }
  };

  if (wave < Q4_STEPS) {
    Q4Step sa, sb;
    load(wave, sa);
    for (int step = wave; step < Q4_STEPS; step += 2 * Q4_WAVES) {
      if (step + Q4_WAVES < Q4_STEPS) load(step + Q4_WAVES, sb);
      compute(sa);
      if (step + Q4_WAVES >= Q4_STEPS) break;
      if (step + 2 * Q4_WAVES < Q4_STEPS) load(step + 2 * Q4_WAVES, sa);
      compute(sb);
    }
  }
#pragma unroll
  for (int a = 0; a < Q4_MB; ++a)
#pragma unroll
    for (int b = 0; b < Q4_NT; ++b) red[wave][a * Q4_NT + b][lane] = acc[a][b];
  __syncthreads();
  for (int u = wave; u < Q4_MB * Q4_NT; u += Q4_WAVES) {
    kcg_f32x4 sum = red[0][u][lane];
#pragma unroll
    for (int w = 1; w < Q4_WAVES; ++w) sum += red[w][u][lane];
    const int n = n0 + (u % Q4_NT) * 16 + i;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = m0 + (u / Q4_NT) * 16 + g * 4 + r;
      if (n < Q4_N && m < M) Y[(long long)m * Q4_N + n] = (Q4_YT)(16.0f * sum[r]);
    }
  }
}
