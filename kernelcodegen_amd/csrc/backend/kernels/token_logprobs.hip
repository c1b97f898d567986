// ---- log probabilities of given tokens, entropies, and the likeliest alternatives ----
//   m = max x,  s = sum e^(x - m),  u = sum (x - m) e^(x - m)          over a row of logits
//   logprob = x[token] - m - ln s,  entropy = ln s - u / s,  and the LP_TOP largest x, ties to the lowest index, as x - m - ln s
// Rows without any token (all -inf): logprobs -inf, entropy 0.  A NaN or +inf in a row makes all its numbers NaN; among the largest a NaN
// counts as -inf.
//
// One pass over the row.  Each lane keeps m, s and u of what it has seen and brings s and u to a new maximum once for LP_U vectors:
//   s' = s e^(m - m'),  u' = (u + (m - m') s) e^(m - m')
// What a vector adds takes one instruction before its exponent: t = x log2 e - c with c = m log2 e rounded; what c lacks of it is known and divided out behind
// all of them.  From |m| = 2^30 on that would pass the exponent's range, and numbers that differ lie 64 or more apart: any other factor than log2 e does.
// m begins at the least finite number, not at -inf, so that x - m is never inf - inf for x = -inf.
// The alternatives need no second pass: the pass leaves the largest number of each segment of 16 vectors (a DPP row of lanes), and the LP_TOP
// largest numbers lie in the LP_TOP segments with the largest ones (ties to the lower segment, whose numbers come first), which are read again.
// Both times the largest of N keys are found the same way: the key holds value and index, so no two are equal; each thread takes its best one, of
// those of a wavefront the k-th is a bound, what reaches the highest bound is counted out against one another.
// Vectors are the aligned ones of memory, the first and the last of a row maybe with elements outside of it, which are left out.
// A row is a workgroup, or several parts (LP_SPLIT; how many is an argument), whose sums and segments logprobs_join (LP_JOIN) finishes.
// Reading bounds large calls, and their instructions nearly as much: 2000 rows of 32000 in bfloat16 26 us, 4.9 TB/s, vector instructions 88 % of the time; with
// 20 alternatives 35, of which the two picks take 8 (some 500 instructions of each wavefront, a chain of LDS accesses and three barriers each, while others
// read).  64 rows of 128000 in fp32 in 16 parts 8.4 us, 3.9 TB/s, and the join 2, or 5.9 with 20 alternatives.  One row of 32000 with 5 of them 7.0, a chain
// as well: four trips over the row, two picks, a trip between.  Of many equal numbers (a masked row's -inf) each wavefront finds its LP_TOP largest one after
// the other: 64 rows of 128000 with 8 left 24 us, not 13, 2000 of 32000 67, not 35.
// Parameters: LP_NAME, LP_V, LP_T, LP_ES (element bytes), LP_STRIDE (of rows, elements), LP_SHIFT (rows may start off a multiple of 16 bytes), LP_TOP,
// LP_SPLIT, LP_THREADS, LP_U, LP_JOIN.
typedef LP_T lp_t;
#define LP_VW (16 / LP_ES)
#define LP_VECTORS ((LP_V + (LP_SHIFT ? LP_VW - 1 : 0) + LP_VW - 1) / LP_VW)     // at most
#define LP_BLOCKS ((LP_VECTORS + 63) / 64)
#define LP_SEGMENTS (LP_BLOCKS * 4)
#define LP_WAVES (LP_THREADS / 64)
#define LP_LOW (-3.402823466e38f)
#define LP_LOG2E 1.4426950408889634f
#define LP_LN2 0.6931471805599453f
typedef lp_t lp_vec __attribute__((ext_vector_type(LP_VW)));
typedef double lp_key;

struct LpSum {
  float m, s, u;
};
__device__ __forceinline__ LpSum lp_add(LpSum a, LpSum b) {
  const float m = fmaxf(a.m, b.m), fa = __builtin_amdgcn_exp2f((a.m - m) * LP_LOG2E), fb = __builtin_amdgcn_exp2f((b.m - m) * LP_LOG2E);
  // (a difference that is no longer finite belongs to a factor of 0)
  return {m, fa * a.s + fb * b.s, fa * (a.u + fmaxf(a.m - m, -1e30f) * a.s) + fb * (b.u + fmaxf(b.m - m, -1e30f) * b.s)};
}
#define LP_DPP(old, v, control, rows) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old), __builtin_bit_cast(int, v), control, rows, 0xf, false))
// row_shr 1, 2, 4, 8, then a row's last lane into the next row, the second row's into the others: lane 63 has what is of all lanes
#define LP_LANES(STEP) STEP(0x111, 0xf) STEP(0x112, 0xf) STEP(0x114, 0xf) STEP(0x118, 0xf) STEP(0x142, 0xa) STEP(0x143, 0xc)
__device__ __forceinline__ float lp_last(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63)); }
// Of all lanes.
__device__ __forceinline__ LpSum lp_all(LpSum a) {
  float m = a.m, s, u;
#define LP_STEP(control, rows) m = fmaxf(m, LP_DPP(LP_LOW, m, control, rows));
  LP_LANES(LP_STEP)
#undef LP_STEP
  m = lp_last(m);
  const float d = a.m - m, f = __builtin_amdgcn_exp2f(d * LP_LOG2E);
  s = f * a.s;
  u = f * (a.u + fmaxf(d, -1e30f) * a.s);
#define LP_STEP(control, rows) s += LP_DPP(0.0f, s, control, rows); u += LP_DPP(0.0f, u, control, rows);
  LP_LANES(LP_STEP)
#undef LP_STEP
  return {m, lp_last(s), lp_last(u)};
}
// Elements of a row that lie in front of its first aligned vector's begin, as a number of that vector's elements.
__device__ __forceinline__ int lp_offset(const lp_t* x) { return LP_SHIFT ? (int)((size_t)x / LP_ES % LP_VW) : 0; }
// A vector of which parts may lie outside of the row: these are -inf.  (All loads are unconditional: one behind a branch would be waited for there.)
__device__ __forceinline__ void lp_edge(const lp_t* __restrict__ x, int at, float (&v)[LP_VW]) {
  lp_t raw[LP_VW];
#pragma unroll
  for (int i = 0; i < LP_VW; ++i) raw[i] = x[at + i < 0 ? 0 : at + i < LP_V ? at + i : LP_V - 1];
#pragma unroll
  for (int i = 0; i < LP_VW; ++i) v[i] = at + i >= 0 && at + i < LP_V ? (float)raw[i] : -__builtin_inff();
}

#if !LP_JOIN
// The sums of blocks [first, end) of a row, those of each wavefront; the segments' largest numbers.
__device__ __forceinline__ void lp_scan(const lp_t* __restrict__ x, int first, int end, LpSum* sums, float* segments) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, o = lp_offset(x);
  LpSum a = {LP_LOW, 0.0f, 0.0f};
  // Blocks that lie within the row are under way while those before them are counted; in the place of others the row's first whole vector is read.
  lp_vec next[LP_U] = {};
  auto inside = [&](int b) { return LP_V >= 2 * LP_VW && b < end && b * (64 * LP_VW) >= o && (b + 1) * (64 * LP_VW) - o <= LP_V; };
  auto fetch = [&](int b) {
    if (LP_V < 2 * LP_VW) return;
#pragma unroll
    for (int j = 0; j < LP_U; ++j) next[j] = *(const lp_vec*)(x + (inside(b + j) ? (b + j) * (64 * LP_VW) - o + lane * LP_VW : (LP_VW - o) % LP_VW));
  };
  fetch(first + wave * LP_U);
  for (int b = first + wave * LP_U; b < end; b += LP_WAVES * LP_U) {
    float v[LP_U][LP_VW], top[LP_U], most = a.m;
    bool whole = true;
#pragma unroll
    for (int j = 0; j < LP_U; ++j) whole = whole && inside(b + j);
    if (whole) {
#pragma unroll
      for (int j = 0; j < LP_U; ++j)
#pragma unroll
        for (int i = 0; i < LP_VW; ++i) v[j][i] = (float)next[j][i];
    } else {
#pragma unroll
      for (int j = 0; j < LP_U; ++j) {
#pragma unroll
        for (int i = 0; i < LP_VW; ++i) v[j][i] = inside(b + j) ? (float)next[j][i] : -__builtin_inff();
        if (b + j < end && !inside(b + j)) lp_edge(x, ((b + j) * 64 + lane) * LP_VW - o, v[j]);
      }
    }
    fetch(b + LP_WAVES * LP_U);
    asm volatile("" ::: "memory");        // (else the loads would be put where the next iteration begins)
#pragma unroll
    for (int j = 0; j < LP_U; ++j) {
      top[j] = v[j][0];
#pragma unroll
      for (int i = 1; i < LP_VW; ++i) top[j] = fmaxf(top[j], v[j][i]);
      most = fmaxf(most, top[j]);
    }
    const float change = a.m - most, factor = __builtin_amdgcn_exp2f(change * LP_LOG2E);
    const bool far = __builtin_fabsf(most) >= 1073741824.0f;
    const float by = far ? 1.0f : LP_LOG2E, c = most * by, rest = __builtin_fmaf(most, by, -c), back = __builtin_amdgcn_exp2f(-rest);
    float s = 0.0f, u = 0.0f;
#pragma unroll
    for (int j = 0; j < LP_U; ++j)
#pragma unroll
      for (int i = 0; i < LP_VW; ++i) {
        const float t = __builtin_fmaf(v[j][i], by, -c), e = __builtin_amdgcn_exp2f(t);
        s += e;
        u = __builtin_fmaf(fmaxf(t, -1e30f), e, u);          // (-inf times 0)
      }
    a.u = __builtin_fmaf(factor, a.u + fmaxf(change, -1e30f) * a.s, (u - rest * s) * (back * LP_LN2));
    a.s = __builtin_fmaf(factor, a.s, s * back);
    a.m = most;
#if LP_TOP
#pragma unroll
    for (int j = 0; j < LP_U; ++j) {
      float t = top[j];
#define LP_ROR(control) t = fmaxf(t, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, t), control, 0xf, 0xf, true)))
      LP_ROR(0x128);       // row_ror 8, 4, 2, 1: over the 16 lanes of a row
      LP_ROR(0x124);
      LP_ROR(0x122);
      LP_ROR(0x121);
#undef LP_ROR
      if (lane % 16 == 0 && b + j < end) segments[(b + j) * 4 + lane / 16] = t;
    }
#endif
  }
  a = lp_all(a);
  if (lane == 0) sums[wave] = a;
  __syncthreads();
}
#endif
// Of all wavefronts.
__device__ __forceinline__ LpSum lp_total(const LpSum* sums) {
  LpSum a = {sums[0].m, 0.0f, 0.0f};
#pragma unroll
  for (int i = 1; i < LP_WAVES; ++i) a.m = fmaxf(a.m, sums[i].m);
#pragma unroll
  for (int i = 0; i < LP_WAVES; ++i) {
    const float d = sums[i].m - a.m, f = __builtin_amdgcn_exp2f(d * LP_LOG2E);
    a.s += f * sums[i].s;
    a.u += f * (sums[i].u + fmaxf(d, -1e30f) * sums[i].s);
  }
  return a;
}

#if !LP_SPLIT || LP_JOIN
#if LP_TOP
// A value and an index below 2^19 as a number from 1 to 2, whose order is the values' and for equal ones the indices' backwards (comparing two of
// these takes one instruction of the ordinary rate); 0 is none.
__device__ __forceinline__ lp_key lp_order(float x, int index) {
  x = x != x ? -__builtin_inff() : x == 0.0f ? 0.0f : x;
  const unsigned b = __builtin_bit_cast(unsigned, x), up = b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
  return __builtin_bit_cast(double, 0x3ff0000000000000ULL | (unsigned long long)up << 19 | (0x7ffffu - (unsigned)index));
}
__device__ __forceinline__ float lp_value(lp_key k) {
  const unsigned up = (unsigned)(__builtin_bit_cast(unsigned long long, k) >> 19);
  return __builtin_bit_cast(float, up ^ (up >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int lp_index(lp_key k) { return 0x7ffff - (int)(__builtin_bit_cast(unsigned long long, k) & 0x7ffff); }
#define LP_LIST (LP_WAVES * LP_TOP > 256 ? LP_WAVES * LP_TOP : 256)               // keys that are counted out against one another
#define LP_E1 ((LP_SEGMENTS + LP_THREADS - 1) / LP_THREADS)                      // segments of a thread
#define LP_E2 ((LP_TOP * 16 + LP_THREADS - 1) / LP_THREADS)                      // and vectors, when they are read again
struct LpPick {
  lp_key list[2][LP_LIST + 32], found[2][LP_TOP];
  __attribute__((aligned(16))) float best[LP_THREADS / 2];
  float bound[LP_WAVES], share[LP_WAVES];
  int many[2];
};
#define LP_SWAP(v, control) __builtin_amdgcn_update_dpp(0, v, control, 0xf, 0xf, true)       // (quad_perm 1 0 3 2 is 0xb1, 2 3 0 1 is 0x4e)
// Least of the lanes' numbers, in lane 63.
__device__ __forceinline__ float lp_least(float v) {
#define LP_STEP(control, rows) v = fminf(v, LP_DPP(__builtin_inff(), v, control, rows));
  LP_LANES(LP_STEP)
#undef LP_STEP
  return v;
}
// The largest of the lanes' numbers, of their keys (first by the upper half).
__device__ __forceinline__ unsigned lp_most(unsigned v) {
#define LP_STEP(control, rows) { const unsigned o = __builtin_amdgcn_update_dpp(0, (int)v, control, rows, 0xf, false); v = v > o ? v : o; }
  LP_LANES(LP_STEP)
#undef LP_STEP
  return __builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ lp_key lp_most(lp_key v) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const unsigned high = lp_most((unsigned)(b >> 32)), low = lp_most((unsigned)(b >> 32) == high ? (unsigned)b : 0u);
  return __builtin_bit_cast(double, (unsigned long long)high << 32 | low);
}
// What LP_TOP of the workgroup's numbers reach (or all).  Of each wavefront's 32 pairs of lanes the LP_TOP-th largest is such a bound, the largest of these
// too; and so is the least of the wavefronts' LP_SHARE-th largest, which reach LP_TOP together: closer where the numbers are spread evenly (of 2000
// numbers 20 wanted, 8 wavefronts: about 40 reach it, 100 the first).
#define LP_SHARE ((LP_TOP + LP_WAVES - 1) / LP_WAVES)
__device__ __forceinline__ float lp_bound(LpPick& p, float best) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const float most = __builtin_inff(), pair = fmaxf(best, __builtin_bit_cast(float, LP_SWAP(__builtin_bit_cast(int, best), 0xb1)));
  p.best[threadIdx.x / 2] = pair;
  __builtin_amdgcn_wave_barrier();        // (a wavefront's own accesses to LDS are carried out in order)
  int r = 0;                               // pairs above this one; its lanes look at half of them each
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const kcg_f32x4 other = *(const kcg_f32x4*)(p.best + wave * 32 + lane % 2 * 16 + i * 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) r += other[e] > pair;
  }
  r += LP_SWAP(r, 0xb1);
  const float all = lp_least(r < LP_TOP ? pair : most), share = lp_least(r < LP_SHARE ? pair : most);
  if (lane == 63) {
    p.bound[wave] = all;
    p.share[wave] = share;
  }
  __syncthreads();
  float bound = -most, together = most;
#pragma unroll
  for (int w = 0; w < LP_WAVES; ++w) {
    bound = fmaxf(bound, p.bound[w]);
    together = fminf(together, p.share[w]);
  }
  return fmaxf(bound, together);
}
// The LP_TOP largest of the threads' numbers v[q] that are there (index(q) from 0 on) and not below the bound, by value and index, into p.found[turn]; all where
// they are fewer.  LP_TOP of the numbers (or all) reach the bound.  p.list and p.found are zeros before, p.many too.
template <int E, class Index> __device__ __forceinline__ void lp_pick(LpPick& p, int turn, const float (&v)[E], float bound, Index index) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  unsigned long long mask[E];
  int total = 0, at = 0;
#pragma unroll
  for (int q = 0; q < E; ++q) {
    mask[q] = __ballot(index(q) >= 0 && v[q] >= bound);
    total += __builtin_popcountll(mask[q]);
  }
  if (total) {
    if (lane == 0) at = atomicAdd(&p.many[turn], total);
    at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
    for (int q = 0; q < E; ++q) {
      const int mine = at + __builtin_amdgcn_mbcnt_hi((unsigned)(mask[q] >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask[q], 0));
      if ((mask[q] >> lane & 1) && mine < LP_LIST) p.list[turn][mine] = lp_order(v[q], index(q));
      at += __builtin_popcountll(mask[q]);
    }
  }
  __syncthreads();
  int n = p.many[turn];
  if (n > LP_LIST) {
    // many equal ones (of masked numbers, say), or the largest ones all in few threads: each wavefront's, one after the other
    n = LP_WAVES * LP_TOP;
    lp_key last = 2.0;
#pragma unroll 1
    for (int t = 0; t < LP_TOP; ++t) {
      lp_key best = 0.0;
#pragma unroll
      for (int q = 0; q < E; ++q) {
        const lp_key k = index(q) >= 0 ? lp_order(v[q], index(q)) : 0.0;
        best = k < last && k > best ? k : best;
      }
      last = lp_most(best);
      if (lane == 0) p.list[turn][wave * LP_TOP + t] = last;
    }
    for (int i = n + threadIdx.x; i < LP_LIST + 32; i += LP_THREADS) p.list[turn][i] = 0.0;
    __syncthreads();
  }
  // four lanes count how many are above one of them
#pragma unroll 1
  for (int i = threadIdx.x / 4; i < n; i += LP_THREADS / 4) {
    const lp_key k = p.list[turn][i];
    int r = 0;
#pragma unroll 1
    for (int j = 0; j < n; j += 32) {
      lp_key other[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) other[e] = p.list[turn][j + e * 4 + lane % 4];
#pragma unroll
      for (int e = 0; e < 8; ++e) r += other[e] > k;
    }
    r += LP_SWAP(r, 0xb1);
    r += LP_SWAP(r, 0x4e);
    if (r < LP_TOP && lane % 4 == 0) p.found[turn][r] = k;
  }
  __syncthreads();
}
#endif
// `sums`: gives the row's sums.
template <class Sums> __device__ __forceinline__ void lp_finish(const lp_t* __restrict__ x, long long row, Sums sums, const float* segments,
                                                                const long long* __restrict__ tokens, float* __restrict__ logprob, float* __restrict__ entropy,
                                                                float* __restrict__ values, long long* __restrict__ indices) {
  const float none = -__builtin_inff();
  const long long token = tokens[row];
  const float given = token >= 0 && token < LP_V ? (float)x[token] : none;
#if LP_TOP
  __shared__ LpPick p;
  const int o = lp_offset(x), count = ((LP_V + o + LP_VW - 1) / LP_VW + 15) / 16;          // segments of this row
  float v[LP_E1], best = none;
#pragma unroll
  for (int q = 0; q < LP_E1; ++q) {
    const int i = q * LP_THREADS + threadIdx.x;
    v[q] = segments[i < count ? i : 0];
    v[q] = i < count && v[q] == v[q] ? v[q] : none;
    best = fmaxf(best, v[q]);
  }
  for (int i = threadIdx.x; i < 2 * (LP_LIST + 32); i += LP_THREADS) p.list[0][i] = 0.0;
  if (threadIdx.x < 2 * LP_TOP) p.found[0][threadIdx.x] = 0.0;
  if (threadIdx.x < 2) p.many[threadIdx.x] = 0;
  lp_pick(p, 0, v, lp_bound(p, best), [&](int q) {
    const int i = q * LP_THREADS + (int)threadIdx.x;
    return i < count ? i : -1;
  });
  // their numbers
  int at[LP_E2];
  lp_vec raw[LP_E2];
#pragma unroll
  for (int q = 0; q < LP_E2; ++q) {
    const int i = q * LP_THREADS + threadIdx.x;
    const lp_key k = i < LP_TOP * 16 ? p.found[0][i < LP_TOP * 16 ? i / 16 : 0] : 0.0;
    at[q] = k > 0.0 ? (lp_index(k) * 16 + i % 16) * LP_VW - o : LP_V;
    if (LP_V >= 2 * LP_VW) raw[q] = *(const lp_vec*)(x + (at[q] >= 0 && at[q] + LP_VW <= LP_V ? at[q] : (LP_VW - o) % LP_VW));
  }
  LpSum a = {};
  float ln = 0.0f;
  if (__builtin_amdgcn_readfirstlane(threadIdx.x) < 64) {        // (the first wavefront, which gives the results)
    a = sums();
    ln = logf(a.s);
  }
  float w[LP_E2 * LP_VW];
  best = none;
#pragma unroll
  for (int q = 0; q < LP_E2; ++q) {
    float e[LP_VW];
#pragma unroll
    for (int j = 0; j < LP_VW; ++j) e[j] = LP_V >= 2 * LP_VW ? (float)raw[q][j] : none;
    if (at[q] < LP_V && (LP_V < 2 * LP_VW || at[q] < 0 || at[q] + LP_VW > LP_V)) lp_edge(x, at[q], e);
#pragma unroll
    for (int j = 0; j < LP_VW; ++j) {
      w[q * LP_VW + j] = e[j] == e[j] ? e[j] : none;
      best = fmaxf(best, at[q] < LP_V ? w[q * LP_VW + j] : none);
    }
  }
  // LP_TOP segments have one each that reaches the least of their largest ones; where there are not as many segments, a bound is found as for them
  const float bound = LP_V >= LP_TOP * 16 * LP_VW ? lp_value(p.found[0][LP_TOP - 1]) : lp_bound(p, best);
  lp_pick(p, 1, w, bound, [&](int q) {
    const int i = at[q / LP_VW] + q % LP_VW;
    return i < LP_V ? i : -1;                          // (or in front of the row)
  });
  if (threadIdx.x < LP_TOP) {
    const lp_key k = p.found[1][threadIdx.x];
    values[row * LP_TOP + threadIdx.x] = a.s == 0.0f ? none : lp_value(k) - a.m - ln;
    indices[row * LP_TOP + threadIdx.x] = lp_index(k);
  }
#else
  if (__builtin_amdgcn_readfirstlane(threadIdx.x) >= 64) return;
  const LpSum a = sums();
  const float ln = logf(a.s);
#endif
  if (threadIdx.x == 0) {
    const float h = ln - a.u / a.s;
    logprob[row] = a.s == 0.0f ? none : given - a.m - ln;
    entropy[row] = a.s == 0.0f || h < 0.0f ? 0.0f : h;
  }
}
#endif

extern "C" __global__ __launch_bounds__(LP_THREADS)
#if LP_JOIN
void LP_NAME(const float* __restrict__ part, const lp_t* __restrict__ logits, const long long* __restrict__ tokens, long long parts, float* __restrict__ logprob,
             float* __restrict__ entropy, float* __restrict__ values, long long* __restrict__ indices) {
  const long long row = blockIdx.x;
  const float* mine = part + row * (parts * 3 + (LP_TOP ? LP_SEGMENTS : 0));
  auto sums = [&] {
    // (each lane a part, or several)
    LpSum a = {LP_LOW, 0.0f, 0.0f};
    for (int i = threadIdx.x & 63; i < (int)parts; i += 64) a = lp_add(a, ((const LpSum*)mine)[i]);
    return lp_all(a);
  };
  lp_finish(logits + row * LP_STRIDE, row, sums, mine + parts * 3, tokens, logprob, entropy, values, indices);
#elif LP_SPLIT
void LP_NAME(const lp_t* __restrict__ logits, long long parts, float* __restrict__ part) {
  __shared__ LpSum sums[LP_WAVES];
  const unsigned n = (unsigned)parts, row = blockIdx.x / n, i = blockIdx.x % n, share = (LP_BLOCKS + n - 1) / n;
  const int first = (int)(i * share), end = first + (int)share < LP_BLOCKS ? first + (int)share : LP_BLOCKS;
  float* mine = part + row * (parts * 3 + (LP_TOP ? LP_SEGMENTS : 0));
  lp_scan(logits + row * LP_STRIDE, first, end, sums, mine + parts * 3);
  if (threadIdx.x == 0) ((LpSum*)mine)[i] = lp_total(sums);
#else
void LP_NAME(const lp_t* __restrict__ logits, const long long* __restrict__ tokens, float* __restrict__ logprob, float* __restrict__ entropy,
             float* __restrict__ values, long long* __restrict__ indices) {
  __shared__ LpSum sums[LP_WAVES];
#if LP_TOP
  __shared__ float segments[LP_SEGMENTS];
#else
  float* segments = nullptr;
#endif
  const long long row = blockIdx.x;
  lp_scan(logits + row * LP_STRIDE, 0, LP_BLOCKS, sums, segments);
  lp_finish(logits + row * LP_STRIDE, row, [&] { return lp_total(sums); }, segments, tokens, logprob, entropy, values, indices);
#endif
}
