// ---- low-rank adapters of many requests beside a shared projection ----
//   Z[t][n] = Y[t][n] + scale[r] * sum over j of B[r][n][j] * h[t][j],   h[t][j] = sum over k of A[r][j][k] * X[t][k],   r = which[t]
// A row whose adapter is none of the AD_ADAPTERS is Y's.  X, A and B in 16 bits, Y and Z in 16 or 32.
//
// Two launches, since every column needs all of h: adapters_down leaves h in fp32, in AD_KS parts of k; adapters_up adds the parts in order.
// Tokens come in any order, and a step's requests may have an adapter each or share one.  A tile is 16 tokens as they stand; each adapter that
// occurs in it (found by comparing lanes) is multiplied with the whole tile, and of the result only its own tokens are kept: rows of a
// matrix product do not touch one another.  A prompt's tiles have one adapter; a decoding step's have up to 16, which AD_S workgroups share.
// h is not rounded to 16 bits: it enters the second product as the sum of two 16-bit numbers, which the matrix instruction takes as 2 AD_RANK
// values of k with B's columns twice.  In half precision h is brought below 2^15 by a power of two of its row.
// Parameters: AD_NAME, AD_UP (this is adapters_up), AD_F16, AD_RANK, AD_K, AD_N, AD_XT, AD_YT, AD_ZT (strides of rows, elements), AD_YTYPE, AD_ALIGN (rows
// of Y and Z start on multiples of 16 bytes), AD_SCALE (0: no scales), AD_INPLACE, AD_KS, AD_S, AD_NS (workgroups along N).
typedef _Float16 ad_f16x8 __attribute__((ext_vector_type(8)));
#if AD_F16
typedef _Float16 ad_x;
#define AD_MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ad_f16x8, a), __builtin_bit_cast(ad_f16x8, b), c, 0, 0, 0)
#else
typedef __bf16 ad_x;
#define AD_MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(kcg_bf16x8, a), __builtin_bit_cast(kcg_bf16x8, b), c, 0, 0, 0)
#endif
typedef ad_x ad_v __attribute__((ext_vector_type(8)));
#define AD_JT ((AD_RANK + 15) / 16)                // tiles of the rank

// Calls each(r, mask of the tile's tokens) for the adapters of a tile that are this workgroup's.
template <class Each> __device__ __forceinline__ unsigned ad_adapters(const int* __restrict__ which, long long t0, long long T, long long adapters, int slot, Each each) {
  const int lane = threadIdx.x & 63;
  int mine = lane < 16 && t0 + lane < T ? which[t0 + lane] : -1;
  const unsigned with = (unsigned)__ballot(mine >= 0 && mine < adapters);
  unsigned todo = with;
  for (int n = 0; todo; ++n) {
    const int r = __builtin_amdgcn_readlane(mine, __builtin_ctz(todo));
    const unsigned same = (unsigned)__ballot(mine == r);
    todo &= ~same;
    if (n % AD_S == slot) each(r, same);
  }
  return with;
}

#if !AD_UP
extern "C" __global__ __launch_bounds__(256)
void AD_NAME(const ad_x* __restrict__ X, const ad_x* __restrict__ A, const int* __restrict__ which, long long T, long long adapters, float* __restrict__ part) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int ks = blockIdx.x % AD_KS, slot = blockIdx.x / AD_KS % AD_S;
  const long long t0 = (long long)(blockIdx.x / (AD_KS * AD_S)) * 16;
  __shared__ kcg_f32x4 red[4][AD_JT][64];
  const long long t = t0 + i < T ? t0 + i : T - 1;
  ad_adapters(which, t0, T, adapters, slot, [&](int r, unsigned same) {
    kcg_f32x4 acc[AD_JT];
#pragma unroll
    for (int j = 0; j < AD_JT; ++j) acc[j] = kcg_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const ad_x* x = X + t * AD_XT;
    const ad_x* a = A + (long long)r * AD_RANK * AD_K;
    for (int s = ks * 4 + wave; s < (AD_K + 31) / 32; s += AD_KS * 4) {
      const int k = s * 32 + g * 8;
      const bool in = AD_K % 32 == 0 || k < AD_K;
      kcg_u32x4 b = *(const kcg_u32x4*)(x + (in ? k : 0));
      if (!in) b = kcg_u32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < AD_JT; ++j) {
        const int row = j * 16 + i < AD_RANK ? j * 16 + i : AD_RANK - 1;
        kcg_u32x4 w = *(const kcg_u32x4*)(a + (long long)row * AD_K + (in ? k : 0));
        if (!in) w = kcg_u32x4{0, 0, 0, 0};
        acc[j] = AD_MFMA(w, b, acc[j]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < AD_JT; ++j) red[wave][j][lane] = acc[j];
    __syncthreads();
    for (int j = wave; j < AD_JT; j += 4) {
      const kcg_f32x4 sum = red[0][j][lane] + red[1][j][lane] + red[2][j][lane] + red[3][j][lane];
      const int at = j * 16 + g * 4;
      if ((same >> i & 1) && at < AD_RANK) *(kcg_f32x4*)(part + ((long long)ks * T + t) * AD_RANK + at) = sum;
    }
  });
}
#else
typedef AD_YTYPE ad_y;
typedef ad_y ad_y4 __attribute__((ext_vector_type(4)));
#define AD_CHUNKS (AD_RANK / 8)
#define AD_STEPS ((2 * AD_CHUNKS + 3) / 4)         // products: both halves of h

// Adds to 16 columns of a row.
__device__ __forceinline__ void ad_put(const ad_y* __restrict__ y, ad_y* __restrict__ z, int n, const kcg_f32x4 (&add)[4]) {
  if (AD_ALIGN && n + 16 <= AD_N) {
    ad_y4 v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = *(const ad_y4*)(y + n + q * 4);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[q][e] = (ad_y)((float)v[q][e] + add[q][e]);
      *(ad_y4*)(z + n + q * 4) = v[q];
    }
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + q * 4 + e < AD_N) z[n + q * 4 + e] = (ad_y)((float)y[n + q * 4 + e] + add[q][e]);
  }
}

extern "C" __global__ __launch_bounds__(256)
void AD_NAME(const float* __restrict__ part, const ad_y* Y, const ad_x* __restrict__ B, const int* __restrict__ which, const float* __restrict__ scale, long long T,
             long long adapters, ad_y* Z) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int ns = blockIdx.x % AD_NS, slot = blockIdx.x / AD_NS % AD_S;
  const long long t0 = (long long)(blockIdx.x / (AD_NS * AD_S)) * 16;
  const long long t = t0 + i < T ? t0 + i : T - 1;
  const ad_y* y = Y + t * AD_YT;
  ad_y* z = Z + t * AD_ZT;
  const unsigned with = ad_adapters(which, t0, T, adapters, slot, [&](int r, unsigned same) {
    float h[AD_STEPS][8], most = 0.0f;
#pragma unroll
    for (int s = 0; s < AD_STEPS; ++s) {
      const int c = (s * 4 + g) % AD_CHUNKS * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) h[s][e] = 0.0f;
#pragma unroll
      for (int p = 0; p < AD_KS; ++p) {
        const kcg_f32x4* at = (const kcg_f32x4*)(part + ((long long)p * T + t) * AD_RANK + c);
        const kcg_f32x4 one = at[0], two = at[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) h[s][e] += one[e], h[s][4 + e] += two[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, __builtin_fabsf(h[s][e]));
    }
    float up = 1.0f, down = 1.0f;
    if (AD_F16) {
      most = fmaxf(most, __shfl_xor(most, 16, 64));
      most = fmaxf(most, __shfl_xor(most, 32, 64));
      int e = (int)(__builtin_bit_cast(unsigned, most) >> 23) - 127;
      e = e < -100 ? -100 : e > 126 ? 126 : e;
      up = __builtin_bit_cast(float, (unsigned)(127 + 14 - e) << 23);
      down = __builtin_bit_cast(float, (unsigned)(127 - 14 + e) << 23);
    }
    kcg_u32x4 f[AD_STEPS];
#pragma unroll
    for (int s = 0; s < AD_STEPS; ++s) {
      const int q = s * 4 + g;
      ad_v v;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = h[s][e] * up;
        const ad_x high = (ad_x)a;
        const float left = a - (float)high;
        v[e] = q < AD_CHUNKS ? high : q < 2 * AD_CHUNKS && left - left == 0.0f ? (ad_x)left : (ad_x)0.0f;
      }
      f[s] = __builtin_bit_cast(kcg_u32x4, v);
    }
    const float by = (AD_SCALE ? scale[r] : 1.0f) * down;
    const ad_x* b = B + (long long)r * AD_N * AD_RANK;
    for (int nb = (ns * 4 + wave) * 64; nb < AD_N; nb += AD_NS * 256) {
      kcg_f32x4 acc[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = nb + (i >> 2) * 16 + q * 4 + (i & 3);
        const ad_x* row = b + (long long)(n < AD_N ? n : AD_N - 1) * AD_RANK;
        acc[q] = kcg_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < AD_STEPS; ++s) {
          const int c = s * 4 + g;
          kcg_u32x4 w = *(const kcg_u32x4*)(row + c % AD_CHUNKS * 8);
          if (c >= 2 * AD_CHUNKS) w = kcg_u32x4{0, 0, 0, 0};
          acc[q] = AD_MFMA(w, f[s], acc[q]);
        }
        acc[q] *= by;
      }
      if (same >> i & 1) ad_put(y, z, nb + g * 16, acc);
    }
  });
  if (!AD_INPLACE && slot == 0 && !(with >> i & 1) && t0 + i < T) {
    const kcg_f32x4 none[4] = {};
    for (int nb = (ns * 4 + wave) * 64; nb < AD_N; nb += AD_NS * 256) ad_put(y, z, nb + g * 16, none);
  }
}
#endif
