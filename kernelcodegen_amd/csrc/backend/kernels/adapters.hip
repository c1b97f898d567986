// ---- low-rank adapters of many requests beside a shared projection ----
//   Z[t][n] = Y[t][n] + scale[r] * sum over j of B[r][n][j] * h[t][j],   h[t][j] = sum over k of A[r][j][k] * X[t][k],   r = which[t]
// A row whose adapter is none of the AD_ADAPTERS is Y's.  X, A and B in 16 bits, Y and Z in 16 or 32.
//
// Two launches, since every column needs all of h: adapters_down leaves h in fp32, in AD_KS parts of k; adapters_up adds the parts in order.
// Tokens come in any order, and a step's requests may have an adapter each or share one.  A tile is 16 AD_TS tokens as they stand (of either launch its
// own AD_TS); each adapter that occurs in it (found by comparing lanes) is multiplied with the whole tile, and of the result only its own tokens
// are kept: rows of a matrix product do not touch one another.  Up to 1024 tokens, which may all have different ones, tiles have 16 tokens in the first launch and 16,
// 32 or 64 (ranks up to 16, up to 128, more) in the second, and workgroups share a tile's adapters; those that find none are the last of the launch.
// More tokens are prompts', whose tiles have one adapter or a few: 16 tokens, or 32 for ranks of 65 to 128, and 64.
// h is not rounded to 16 bits: it enters the second product as the sum of AD_PIECES 16-bit numbers, which the matrix instruction takes as AD_PIECES AD_RANK
// values of k with B's columns as often.  Two of half precision have 22 bits, three of bfloat16 all of fp32's 24.  (Two of bfloat16 have 16: of 262144
// results in bfloat16, 64 tokens with 40 adapters, 295 were not the nearest to the formula, of the formula in fp32 53, of this 24; 9.3 and 9.5 us.)  In half
// precision h is brought below 2^15 by a power of two of its row's finite numbers.
// Both products have the tokens as their columns, so that a lane has four neighbouring numbers of one token in each result.
// Reading and writing bound prompts: 5000 tokens, rank 64, K = N = 4096 in bfloat16 13.7 us (X, 3.0 TB/s, LDS under way 41 % of the time) and 22 (Y and Z, 3.7
// TB/s); 2600 tokens, rank 32, N = 11008 in fp32 11.5 and 50 (4.6 TB/s).  Of few tokens each launch is a chain: which adapter, its numbers, a sum over
// wavefronts, the store: one token 2.9 and 4.2 us, 64 tokens with 40 adapters between them 4.8 and 5.8.  Both in one launch, in which a workgroup has all
// of h for its columns, take as long for a tile alone (6.8) and lose from there on (64 tokens: 11.1).  Hundreds of tokens in any order with tens of adapters read a
// matrix once for each tile that has its adapter: 1000 tokens with 64 adapters of rank 16 54 us, where each matrix once would be 8.
// Parameters: AD_NAME, AD_UP (this is adapters_up), AD_F16, AD_PIECES, AD_RANK, AD_K, AD_N, AD_XT, AD_YT, AD_ZT (strides of rows, elements), AD_YTYPE,
// AD_YSIZE, AD_ALIGN (rows of Y and Z start on multiples of 16 bytes), AD_SCALE (0: no scales), AD_INPLACE, AD_TS, AD_KS, AD_DEPTH (steps of k under way), AD_MANY (a
// tile's adapters are shared out; between how many workgroups, and how many there are along N, are arguments), AD_ONCE (there are as many along N
// as have columns: each has one pass).  adapters_down has AD_F16, AD_RANK, AD_K, AD_XT, AD_TS, AD_KS, AD_DEPTH and AD_MANY of them.
typedef _Float16 ad_f16x8 __attribute__((ext_vector_type(8)));
#if AD_F16
typedef _Float16 ad_x;
#define AD_MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ad_f16x8, a), __builtin_bit_cast(ad_f16x8, b), c, 0, 0, 0)
#else
typedef __bf16 ad_x;
#define AD_MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(kcg_bf16x8, a), __builtin_bit_cast(kcg_bf16x8, b), c, 0, 0, 0)
#endif
typedef ad_x ad_v __attribute__((ext_vector_type(8)));
typedef unsigned long long ad_mask;
#define AD_JT ((AD_RANK + 15) / 16)                // tiles of the rank
#define AD_TILE (16 * AD_TS)

// The adapters of a tile that are this workgroup's, one after the other; `with`: the tile's tokens that have one.
struct AdTurns {
  int mine;
  ad_mask with, todo;
#if AD_MANY
  int turn, n, slots;
#endif
  __device__ __forceinline__ AdTurns(const int* __restrict__ which, long long t0, long long T, long long adapters, int slot, int slots_) {
    const int lane = threadIdx.x & 63;
    mine = lane < AD_TILE && t0 + lane < T ? which[t0 + lane] : -1;
    todo = with = __ballot(mine >= 0 && mine < adapters);
#if AD_MANY
    // tokens that are the first ones with their adapter: lane by lane further away compared
    int other = mine;
    bool again = false;
#pragma unroll
    for (int d = 1; d < AD_TILE; ++d) {
      other = __builtin_amdgcn_update_dpp(-1, other, 0x138, 0xf, 0xf, false);        // wave_shr 1
      again |= other == mine;
    }
    todo &= __ballot(!again);
    turn = __builtin_amdgcn_mbcnt_hi((unsigned)(todo >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)todo, 0));
    n = slot;
    slots = slots_;
#endif
  }
  // The next one's number and its tokens.
  __device__ __forceinline__ bool next(int& r, ad_mask& same) {
#if AD_MANY
    if (n >= __builtin_popcountll(todo)) return false;
    r = __builtin_amdgcn_readlane(mine, __builtin_ctzll(__ballot(turn == n) & todo));
    same = __ballot(mine == r);
    n += slots;
#else
    if (!todo) return false;
    r = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
    same = __ballot(mine == r);
    todo &= ~same;
#endif
    return true;
  }
};

#if !AD_UP
// A wavefront has its own part of k and brings it in whole lines, 64 k of eight rows a load: through LDS rows of its own, 16 bytes apart from a multiple
// of 128, from where a lane takes the chunks that the product wants (chunk l / 16 of row l % 16; straight from memory, neighbouring lanes touch
// different lines).
#define AD_STEPS ((AD_K + 63) / 64)
#define AD_SHARE ((AD_STEPS + 4 * AD_KS - 1) / (4 * AD_KS))       // of a wavefront
#define AD_ROWS (16 * (AD_TS + AD_JT))                            // of X, then of A
#define AD_PITCH 144
extern "C" __global__ __launch_bounds__(256)
void AD_NAME(const ad_x* __restrict__ X, const ad_x* __restrict__ A, const int* __restrict__ which, long long T, long long adapters, long long slots,
             float* __restrict__ part) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const unsigned tiles = (unsigned)((T + AD_TILE - 1) / AD_TILE);
  const int ks = blockIdx.x % AD_KS, slot = blockIdx.x / AD_KS / tiles;
  const long long t0 = (long long)(blockIdx.x / AD_KS % tiles) * AD_TILE;
  union Shared {
    __attribute__((aligned(16))) unsigned char rows[4][AD_ROWS * AD_PITCH];
    kcg_f32x4 red[4][AD_TS * AD_JT][64];
  };
  __shared__ Shared sh;
  unsigned char* mine = sh.rows[wave];
  const ad_x* x[AD_TS * 2];
#pragma unroll
  for (int c = 0; c < AD_TS * 2; ++c) {
    const long long t = t0 + c * 8 + lane / 8;
    x[c] = X + (t < T ? t : T - 1) * AD_XT;
  }
  const int first = (ks * 4 + wave) * AD_SHARE, end = first + AD_SHARE < AD_STEPS ? first + AD_SHARE : AD_STEPS;
  AdTurns turns(which, t0, T, adapters, slot, (int)slots);
  int r;
  ad_mask same;
  while (turns.next(r, same)) {
    kcg_f32x4 acc[AD_TS][AD_JT];
#pragma unroll
    for (int t = 0; t < AD_TS; ++t)
#pragma unroll
      for (int j = 0; j < AD_JT; ++j) acc[t][j] = kcg_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const ad_x* a = A + (long long)r * AD_RANK * AD_K;
    kcg_u32x4 next[AD_DEPTH][AD_ROWS / 8];
    auto fetch = [&](int s, kcg_u32x4 (&to)[AD_ROWS / 8]) {
      int k = (s < AD_STEPS ? s : 0) * 64 + lane % 8 * 8;
      if (AD_K % 64) k = k < AD_K ? k : 0;
#pragma unroll
      for (int c = 0; c < AD_TS * 2; ++c) to[c] = *(const kcg_u32x4*)(x[c] + k);
#pragma unroll
      for (int c = 0; c < AD_JT * 2; ++c) {
        const int row = c * 8 + lane / 8;
        to[AD_TS * 2 + c] = *(const kcg_u32x4*)(a + (AD_RANK % 16 && row >= AD_RANK ? AD_RANK - 1 : row) * (long long)AD_K + k);
      }
    };
#pragma unroll
    for (int d = 0; d < AD_DEPTH; ++d) fetch(first + d, next[d]);
#pragma unroll 1
    for (int s0 = first; s0 < end; s0 += AD_DEPTH) {
#pragma unroll
      for (int d = 0; d < AD_DEPTH; ++d) {
        const int s = s0 + d;
        // (k behind the last, and steps that are another wavefront's, take part as zeros)
        const bool in = s < end && (AD_K % 64 == 0 || s * 64 + lane % 8 * 8 < AD_K);
#pragma unroll
        for (int c = 0; c < AD_ROWS / 8; ++c)
          *(kcg_u32x4*)(mine + (c * 8 + lane / 8) * AD_PITCH + lane % 8 * 16) = in ? next[d][c] : kcg_u32x4{0, 0, 0, 0};
        fetch(s + AD_DEPTH, next[d]);
        __builtin_amdgcn_wave_barrier();        // (a wavefront's own accesses to LDS are carried out in order)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          kcg_u32x4 b[AD_TS];
#pragma unroll
          for (int t = 0; t < AD_TS; ++t) b[t] = *(const kcg_u32x4*)(mine + (t * 16 + i) * AD_PITCH + (h * 4 + g) * 16);
#pragma unroll
          for (int j = 0; j < AD_JT; ++j) {
            const kcg_u32x4 w = *(const kcg_u32x4*)(mine + ((AD_TS + j) * 16 + i) * AD_PITCH + (h * 4 + g) * 16);
#pragma unroll
            for (int t = 0; t < AD_TS; ++t) acc[t][j] = AD_MFMA(w, b[t], acc[t][j]);
          }
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < AD_TS; ++t)
#pragma unroll
      for (int j = 0; j < AD_JT; ++j) sh.red[wave][t * AD_JT + j][lane] = acc[t][j];
    __syncthreads();
    for (int u = wave; u < AD_TS * AD_JT; u += 4) {
      const kcg_f32x4 sum = sh.red[0][u][lane] + sh.red[1][u][lane] + sh.red[2][u][lane] + sh.red[3][u][lane];
      const int row = u / AD_JT * 16 + i, at = u % AD_JT * 16 + g * 4;
      if ((same >> row & 1) && at < AD_RANK) *(kcg_f32x4*)(part + ((long long)ks * T + t0 + row) * AD_RANK + at) = sum;
    }
    __syncthreads();
  }
}
#else
typedef AD_YTYPE ad_y;
#define AD_C (16 / AD_YSIZE)                       // columns of a lane, which lie beside one another: 16 bytes
#define AD_COLS (16 * AD_C)                        // and of a wavefront
typedef ad_y ad_yv __attribute__((ext_vector_type(AD_C)));
#if AD_ALIGN
typedef ad_yv ad_mem;
#else
typedef ad_y ad_mem __attribute__((ext_vector_type(AD_C), aligned(AD_YSIZE)));     // (rows may start anywhere)
#endif
#define AD_CHUNKS (AD_RANK / 8)
#define AD_STEPS ((AD_PIECES * AD_CHUNKS + 3) / 4)  // products: all numbers that h is the sum of
#define AD_OWN (AD_CHUNKS % 4 == 0 ? AD_CHUNKS / 4 : AD_STEPS)    // of which so many have other columns of B
#define AD_GROUPS (4 / AD_TS)                       // wavefronts beside one another along N; AD_TS of them have 16 tokens each
#define AD_STEP (AD_GROUPS * AD_COLS)              // columns of a workgroup
#define AD_EVEN (AD_N % AD_STEP == 0)               // no column is behind the last
#define AD_PITCH (AD_CHUNKS % 2 ? AD_RANK * 2 : AD_RANK * 2 + 16)  // of a row of B in LDS: an odd number of 16 bytes
#define AD_LOADS ((AD_STEP * AD_CHUNKS + 255) / 256)
#define AD_INSIDE (AD_EVEN && AD_STEP * AD_CHUNKS % 256 == 0)      // nor is a load's, whose lanes may pass the step's columns

// Columns n to n + AD_C of a row; elements of a vector that passes the row's end come one by one, all of them before any is put.
__device__ __forceinline__ ad_yv ad_get(const ad_y* y, int n) {
  ad_yv v = {};
  if (AD_N >= AD_C) v = *(const ad_mem*)(y + (AD_EVEN || n + AD_C <= AD_N ? n : 0));
  if (AD_N % AD_C && n < AD_N && n + AD_C > AD_N) {
#pragma unroll
    for (int e = 0; e < AD_C; ++e) v[e] = y[n + e < AD_N ? n + e : AD_N - 1];
  }
  return v;
}
__device__ __forceinline__ void ad_put(ad_y* z, int n, ad_yv v) {
  if (AD_EVEN || n + AD_C <= AD_N) {
    *(ad_mem*)(z + n) = v;
  } else if (AD_N % AD_C) {
#pragma unroll
    for (int e = 0; e < AD_C; ++e)
      if (n + e < AD_N) z[n + e] = v[e];
  }
}

// a as the sum of AD_PIECES 16-bit numbers of its sign, none of them 0 unless a is (or, in half precision, below 2^-23): an infinity of B times all of them
// is one, as times a.  Each is cut off, so that what is left has a's sign; where nothing is left, or nothing finite, halves of the first do (not of the last: a
// matrix instruction drops digits below those of fp32).
__device__ __forceinline__ void ad_split(float a, float (&p)[3]) {
#if AD_F16
  p[0] = (float)__builtin_amdgcn_cvt_pkrtz(a, a)[0];
  p[0] = (ad_x)(a - p[0]) == (ad_x)0.0f ? (float)(ad_x)(a * 0.5f) : p[0];
  p[1] = a - a == 0.0f ? a - p[0] : a;
#else
  auto cut = [](float v) { return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, v) & 0xffff0000u); };
  const float high = cut(a), half = a * 0.5f, left = __builtin_fabsf(a - high) > 0.0f ? a - high : half, rest = left - cut(left);
  p[0] = __builtin_fabsf(a - high) > 0.0f ? high : half;
  p[1] = cut(left);
  p[2] = __builtin_fabsf(rest) > 0.0f ? rest : p[0] * 0.5f;
  p[0] = __builtin_fabsf(rest) > 0.0f ? p[0] : p[0] * 0.5f;
#endif
}

// A wavefront takes AD_COLS columns of 16 tokens at a time: lane l gets columns (l % 16) AD_C on of tokens 4 (l / 16) to 4 (l / 16) + 3, whole lines of Y with
// its neighbours, when the columns of product q are every AD_C-th from q on.  B comes for the whole workgroup, in whole lines, and goes through LDS,
// rows put into the order in which the products take them; the next columns' B and Y, or the next adapter's, are under way meanwhile.
extern "C" __global__ __launch_bounds__(256)
void AD_NAME(const float* __restrict__ part, const ad_y* Y, const ad_x* __restrict__ B, const int* __restrict__ which, const float* __restrict__ scale, long long T,
             long long adapters, long long slots, long long NS_, ad_y* Z) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int sub = wave % AD_TS, group = wave / AD_TS;
  const unsigned NS = (unsigned)NS_, tiles = (unsigned)((T + AD_TILE - 1) / AD_TILE);
  const int ns = blockIdx.x % NS, slot = blockIdx.x / NS / tiles;
  const long long t0 = (long long)(blockIdx.x / NS % tiles) * AD_TILE, tw = t0 + sub * 16, step = (long long)NS * AD_STEP;
  __shared__ __attribute__((aligned(16))) unsigned char rows[AD_STEP * AD_PITCH];
  long long row[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) row[e] = tw + g * 4 + e < T ? tw + g * 4 + e : T - 1;
  AdTurns turns(which, t0, T, adapters, slot, (int)slots);
  int r;
  ad_mask same;
  kcg_u32x4 w[AD_LOADS], f[AD_STEPS];
  ad_yv v[4];
  float back = 1.0f, factor = 1.0f;
  // B of an adapter's columns from nb on, and its scale; Y of them
  auto fetch = [&](int r, int nb) {
    const ad_x* b = B + (long long)r * AD_N * AD_RANK;
#pragma unroll
    for (int c = 0; c < AD_LOADS; ++c) {
      const int u = c * 256 + threadIdx.x, n = nb + u / AD_CHUNKS;
      w[c] = *(const kcg_u32x4*)(b + (AD_INSIDE || n < AD_N ? (long long)n * AD_RANK + u % AD_CHUNKS * 8 : 0));
    }
    if (AD_SCALE) factor = scale[r];
  };
  auto fetch_y = [&](int nb) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = ad_get(Y + row[e] * AD_YT, nb + group * AD_COLS + i * AD_C);
  };
  bool more = turns.next(r, same);
  if (more) {
    fetch(r, ns * AD_STEP);
    fetch_y(ns * AD_STEP);
    // h of this wavefront's tokens in numbers of 16 bits
    const long long t = tw + i < T ? tw + i : T - 1;
    float h[AD_OWN][8], most = 0.0f;
#pragma unroll
    for (int s = 0; s < AD_OWN; ++s) {
      const int c = (s * 4 + g) % AD_CHUNKS * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) h[s][e] = 0.0f;
      kcg_f32x4 parts[AD_KS][2];
#pragma unroll
      for (int p = 0; p < AD_KS; ++p) {
        const kcg_f32x4* at = (const kcg_f32x4*)(part + ((long long)p * T + t) * AD_RANK + c);
        parts[p][0] = at[0];
        parts[p][1] = at[1];
      }
      __builtin_amdgcn_sched_barrier(0);        // (all on their way before the first is waited for)
#pragma unroll
      for (int p = 0; p < AD_KS; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) h[s][e] += parts[p][e / 4][e % 4];
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, __builtin_fabsf(h[s][e]) < __builtin_inff() ? __builtin_fabsf(h[s][e]) : 0.0f);        // (beside an infinity, the others)
    }
    float up = 1.0f;
    if (AD_F16) {
      most = fmaxf(most, __shfl_xor(most, 16, 64));
      most = fmaxf(most, __shfl_xor(most, 32, 64));
      int e = (int)(__builtin_bit_cast(unsigned, most) >> 23) - 127;
      e = e < -100 ? -100 : e > 126 ? 126 : e;
      up = __builtin_bit_cast(float, (unsigned)(127 + 14 - e) << 23);
      back = __builtin_bit_cast(float, (unsigned)(127 - 14 + e) << 23);
    }
#pragma unroll
    for (int s = 0; s < AD_OWN; ++s) {
      const int q = s * 4 + g;
      ad_v p[AD_STEPS / AD_OWN];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float of[3];
        ad_split(AD_F16 ? h[s][e] * up : h[s][e], of);
        if (AD_CHUNKS % 4) of[0] = q < AD_CHUNKS ? of[0] : q < 2 * AD_CHUNKS ? of[1] : q < AD_PIECES * AD_CHUNKS ? of[AD_PIECES - 1] : 0.0f;
#pragma unroll
        for (int n = 0; n < AD_STEPS / AD_OWN; ++n) p[n][e] = (ad_x)of[n];
      }
#pragma unroll
      for (int n = 0; n < AD_STEPS / AD_OWN; ++n) f[n * AD_OWN + s] = __builtin_bit_cast(kcg_u32x4, p[n]);
    }
  }
#pragma unroll 1
  while (more) {
    const unsigned mine = (unsigned)(same >> (sub * 16)) & 0xffffu;
    const float down = factor * back;
    kcg_f32x4 times;
#pragma unroll
    for (int e = 0; e < 4; ++e) times[e] = AD_F16 ? __shfl(down, g * 4 + e, 64) : down;
    int following = 0;
    more = turns.next(following, same);
#pragma unroll 1
    for (int nb = ns * AD_STEP; nb < AD_N; nb += NS * AD_STEP) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < AD_LOADS; ++c) {
        const int u = c * 256 + threadIdx.x, n = u / AD_CHUNKS;       // row n % AD_C of lane n / AD_C % 16 in product n % AD_C
        if (AD_STEP * AD_CHUNKS % 256 == 0 || n < AD_STEP)
          *(kcg_u32x4*)(rows + (n / AD_COLS * AD_COLS + n % AD_C * 16 + n % AD_COLS / AD_C) * AD_PITCH + u % AD_CHUNKS * 16) = w[c];
      }
      ad_yv now[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) now[e] = v[e];
      __syncthreads();
      // the next columns, or the next adapter's first
      if (!AD_ONCE && nb + step < AD_N) {
        fetch(r, nb + (int)step);
        fetch_y(nb + (int)step);
      } else if (more) {
        fetch(following, ns * AD_STEP);
        if (!AD_ONCE) fetch_y(ns * AD_STEP);
      }
      if (mine) {
        kcg_f32x4 acc[AD_C];
#pragma unroll
        for (int q = 0; q < AD_C; ++q) {
          const unsigned char* at = rows + (group * AD_COLS + q * 16 + i) * AD_PITCH;
          acc[q] = kcg_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          kcg_u32x4 c[AD_OWN];
#pragma unroll
          for (int s = 0; s < AD_OWN; ++s) {
            c[s] = *(const kcg_u32x4*)(at + (s * 4 + g) % AD_CHUNKS * 16);
            if (s * 4 + 3 >= AD_PIECES * AD_CHUNKS && s * 4 + g >= AD_PIECES * AD_CHUNKS) c[s] = kcg_u32x4{0, 0, 0, 0};        // (k behind all of them)
          }
#pragma unroll
          for (int s = 0; s < AD_STEPS; ++s) acc[q] = AD_MFMA(f[s], c[s % AD_OWN], acc[q]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ad_yv sum;
#pragma unroll
          for (int q = 0; q < AD_C; ++q) sum[q] = (ad_y)((float)now[e][q] + times[e] * acc[q][e]);
          if (mine >> (g * 4 + e) & 1) ad_put(Z + row[e] * AD_ZT, nb + group * AD_COLS + i * AD_C, sum);
        }
      }
      if (AD_ONCE) break;
    }
    r = following;
  }
  if (!AD_INPLACE && slot == 0) {
#pragma unroll 1
    for (int e = 0; e < 4; ++e) {
      if ((turns.with >> (sub * 16 + g * 4 + e) & 1) || tw + g * 4 + e >= T) continue;
      for (int n = ns * AD_STEP + group * AD_COLS + i * AD_C; n < AD_N; n += NS * AD_STEP)
        ad_put(Z + row[e] * AD_ZT, n, ad_get(Y + row[e] * AD_YT, n));
    }
  }
}
#endif
