// ---- log probabilities of given tokens, entropies, and the likeliest alternatives ----
//   m = max x,  s = sum e^(x - m),  u = sum (x - m) e^(x - m)          over a row of logits
//   logprob = x[token] - m - ln s,  entropy = ln s - u / s,  and the LP_TOP largest x, ties to the lowest index, as x - m - ln s
// Rows without any token (all -inf): logprobs -inf, entropy 0.  A NaN or +inf in a row makes all its numbers NaN; among the largest a NaN
// counts as -inf.
//
// One pass over the row.  Each lane keeps m, s and u of what it has seen and brings s and u to a new maximum once for LP_U vectors:
//   s' = s e^(m - m'),  u' = (u + (m - m') s) e^(m - m')
// m begins at the least finite number, not at -inf, so that x - m is never inf - inf for x = -inf.
// The alternatives need no second pass: the pass leaves the largest number of each segment of 16 vectors (a DPP row of lanes), and the LP_TOP
// largest numbers lie in the LP_TOP segments with the largest ones (ties to the lower segment, whose numbers come first), which are read again.
// Both times the largest of N keys are found the same way: the key holds value and index, so no two are equal; each thread takes its best one, of
// those of a wavefront the k-th is a bound, what reaches the highest bound is counted out against one another.
// Vectors are the aligned ones of memory, the first and the last of a row maybe with elements outside of it, which are left out.
// A row is a workgroup, or LP_PARTS of them, whose sums and segments logprobs_join (LP_JOIN) finishes.
// Parameters: LP_NAME, LP_V, LP_T, LP_ES (element bytes), LP_STRIDE (of rows, elements), LP_SHIFT (rows may start off a multiple of 16 bytes), LP_TOP,
// LP_PARTS, LP_THREADS, LP_U, LP_JOIN.
typedef LP_T lp_t;
#define LP_VW (16 / LP_ES)
#define LP_VECTORS ((LP_V + (LP_SHIFT ? LP_VW - 1 : 0) + LP_VW - 1) / LP_VW)     // at most
#define LP_BLOCKS ((LP_VECTORS + 63) / 64)
#define LP_SEGMENTS (LP_BLOCKS * 4)
#define LP_SHARE ((LP_BLOCKS + LP_PARTS - 1) / LP_PARTS)                         // blocks of a part
#define LP_WAVES (LP_THREADS / 64)
#define LP_LOW (-3.402823466e38f)
#define LP_LOG2E 1.4426950408889634f
typedef lp_t lp_vec __attribute__((ext_vector_type(LP_VW)));
typedef unsigned long long lp_key;

struct LpSum {
  float m, s, u;
};
__device__ __forceinline__ LpSum lp_add(LpSum a, LpSum b) {
  const float m = fmaxf(a.m, b.m), fa = __builtin_amdgcn_exp2f((a.m - m) * LP_LOG2E), fb = __builtin_amdgcn_exp2f((b.m - m) * LP_LOG2E);
  // (a difference that is no longer finite belongs to a factor of 0)
  return {m, fa * a.s + fb * b.s, fa * (a.u + fmaxf(a.m - m, -1e30f) * a.s) + fb * (b.u + fmaxf(b.m - m, -1e30f) * b.s)};
}
// Elements of a row that lie in front of its first aligned vector's begin, as a number of that vector's elements.
__device__ __forceinline__ int lp_offset(const lp_t* x) { return LP_SHIFT ? (int)((size_t)x / LP_ES % LP_VW) : 0; }
__device__ __forceinline__ void lp_load(const lp_t* __restrict__ x, int at, float (&v)[LP_VW]) {
  if (at >= 0 && at + LP_VW <= LP_V) {
    const lp_vec raw = *(const lp_vec*)(x + at);
#pragma unroll
    for (int i = 0; i < LP_VW; ++i) v[i] = (float)raw[i];
  } else {
#pragma unroll
    for (int i = 0; i < LP_VW; ++i) v[i] = at + i >= 0 && at + i < LP_V ? (float)x[at + i] : -__builtin_inff();
  }
}

#if !LP_JOIN
// The sums of blocks [first, end) of a row for the whole workgroup's threads; the segments' largest numbers.
__device__ __forceinline__ LpSum lp_scan(const lp_t* __restrict__ x, int first, int end, float* segments) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, o = lp_offset(x);
  LpSum a = {LP_LOW, 0.0f, 0.0f};
  for (int b = first + wave * LP_U; b < end; b += LP_WAVES * LP_U) {
    float v[LP_U][LP_VW], top[LP_U], most = a.m;
    if (b + LP_U <= end && b * (64 * LP_VW) >= o && (b + LP_U) * (64 * LP_VW) - o <= LP_V) {
      lp_vec raw[LP_U];
#pragma unroll
      for (int j = 0; j < LP_U; ++j) raw[j] = *(const lp_vec*)(x + ((b + j) * 64 + lane) * LP_VW - o);
#pragma unroll
      for (int j = 0; j < LP_U; ++j)
#pragma unroll
        for (int i = 0; i < LP_VW; ++i) v[j][i] = (float)raw[j][i];
    } else {
#pragma unroll
      for (int j = 0; j < LP_U; ++j) lp_load(x, b + j < end ? ((b + j) * 64 + lane) * LP_VW - o : LP_V, v[j]);
    }
#pragma unroll
    for (int j = 0; j < LP_U; ++j) {
      top[j] = v[j][0];
#pragma unroll
      for (int i = 1; i < LP_VW; ++i) top[j] = fmaxf(top[j], v[j][i]);
      most = fmaxf(most, top[j]);
    }
    const float change = a.m - most, factor = __builtin_amdgcn_exp2f(change * LP_LOG2E);
    a.u = factor * (a.u + fmaxf(change, -1e30f) * a.s);
    a.s *= factor;
    a.m = most;
#pragma unroll
    for (int j = 0; j < LP_U; ++j)
#pragma unroll
      for (int i = 0; i < LP_VW; ++i) {
        const float d = v[j][i] - most, e = __builtin_amdgcn_exp2f(d * LP_LOG2E);
        a.s += e;
        a.u = __builtin_fmaf(fmaxf(d, -1e30f), e, a.u);          // (-inf times 0)
      }
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
#pragma unroll
  for (int by = 32; by > 0; by >>= 1) a = lp_add(a, {__shfl_xor(a.m, by, 64), __shfl_xor(a.s, by, 64), __shfl_xor(a.u, by, 64)});
  __shared__ LpSum sums[LP_WAVES];
  if (lane == 0) sums[wave] = a;
  __syncthreads();
  a = sums[0];
#pragma unroll
  for (int w = 1; w < LP_WAVES; ++w) a = lp_add(a, sums[w]);
  return a;
}
#endif

#if LP_PARTS == 1 || LP_JOIN
#if LP_TOP
#define LP_Q1 ((LP_SEGMENTS + LP_THREADS - 1) / LP_THREADS)                      // segments of a thread
#define LP_Q2 ((LP_TOP * 16 + LP_THREADS - 1) / LP_THREADS)                      // and vectors, when they are read again
#define LP_MOST (LP_Q1 > LP_Q2 * LP_VW ? LP_Q1 : LP_Q2 * LP_VW)
__device__ __forceinline__ lp_key lp_order(float x, int index) {
  x = x != x ? -__builtin_inff() : x == 0.0f ? 0.0f : x;
  const unsigned b = __builtin_bit_cast(unsigned, x), up = b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
  return (lp_key)up << 32 | (0xffffffffu - (unsigned)index);
}
__device__ __forceinline__ float lp_value(lp_key k) {
  const unsigned up = (unsigned)(k >> 32);
  return __builtin_bit_cast(float, up ^ (up >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int lp_index(lp_key k) { return (int)(0xffffffffu - (unsigned)k); }
struct LpPick {
  lp_key best[LP_THREADS], bound[LP_WAVES], near[LP_WAVES * LP_TOP], list[LP_TOP * LP_MOST], found[LP_TOP], last;
  int many[2];
};
__device__ __forceinline__ int lp_rank(const lp_key* list, int n, lp_key k) {
  int r = 0;
#pragma unroll 8
  for (int i = 0; i < n; ++i) r += list[i] > k;
  return r;
}
// The LP_TOP largest of all threads' keys, or all where they are fewer, in order, into p.found; keys of 0 are none.
template <int Q> __device__ __forceinline__ void lp_pick(const lp_key (&keys)[Q], LpPick& p) {
  const int wave = threadIdx.x >> 6;
  lp_key best = keys[0];
#pragma unroll
  for (int q = 1; q < Q; ++q) best = keys[q] > best ? keys[q] : best;
  p.best[threadIdx.x] = best;
  if (threadIdx.x < LP_WAVES) p.bound[threadIdx.x] = 0;
  if (threadIdx.x < LP_TOP) p.found[threadIdx.x] = 0;
  if (threadIdx.x == 0) p.many[0] = p.many[1] = 0, p.last = 0;
  __syncthreads();
  if (best && lp_rank(p.best + wave * 64, 64, best) == LP_TOP - 1) p.bound[wave] = best;
  __syncthreads();
  lp_key bound = p.bound[0];
#pragma unroll
  for (int w = 1; w < LP_WAVES; ++w) bound = p.bound[w] > bound ? p.bound[w] : bound;
  const bool near = best && best >= bound;          // LP_TOP threads of a wavefront or fewer
  if (near) p.near[atomicAdd(&p.many[0], 1)] = best;
  __syncthreads();
  bool mine = false;
  if (near) {
    const int r = lp_rank(p.near, p.many[0], best);
    mine = r < LP_TOP;
    if (r == LP_TOP - 1) p.last = best;
  }
  __syncthreads();
  if (mine) {
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (keys[q] && keys[q] >= p.last) p.list[atomicAdd(&p.many[1], 1)] = keys[q];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.many[1]; i += LP_THREADS) {
    const int r = lp_rank(p.list, p.many[1], p.list[i]);
    if (r < LP_TOP) p.found[r] = p.list[i];
  }
  __syncthreads();
}
#endif
__device__ __forceinline__ void lp_finish(const lp_t* __restrict__ x, long long row, LpSum a, const float* segments, const long long* __restrict__ tokens,
                                          float* __restrict__ logprob, float* __restrict__ entropy, float* __restrict__ values, long long* __restrict__ indices) {
  const float none = -__builtin_inff(), ln = logf(a.s);
  if (threadIdx.x == 0) {
    const long long t = tokens[row];
    const float v = t >= 0 && t < LP_V ? (float)x[t] : none, h = ln - a.u / a.s;
    logprob[row] = a.s == 0.0f ? none : v - a.m - ln;
    entropy[row] = a.s == 0.0f || h < 0.0f ? 0.0f : h;
  }
#if LP_TOP
  __shared__ LpPick p;
  const int o = lp_offset(x), count = ((LP_V + o + LP_VW - 1) / LP_VW + 15) / 16;          // segments of this row
  lp_key one[LP_Q1];
#pragma unroll
  for (int q = 0; q < LP_Q1; ++q) {
    const int i = q * LP_THREADS + threadIdx.x;
    one[q] = i < count ? lp_order(segments[i], i) : 0;
  }
  lp_pick(one, p);
  lp_key two[LP_Q2 * LP_VW];
#pragma unroll
  for (int q = 0; q < LP_Q2; ++q) {
    const int i = q * LP_THREADS + threadIdx.x;
    const lp_key segment = i < LP_TOP * 16 ? p.found[i / 16] : 0;
    const int at = segment ? (lp_index(segment) * 16 + i % 16) * LP_VW - o : LP_V;
    float v[LP_VW];
    lp_load(x, at, v);
#pragma unroll
    for (int j = 0; j < LP_VW; ++j) two[q * LP_VW + j] = at + j >= 0 && at + j < LP_V ? lp_order(v[j], at + j) : 0;
  }
  __syncthreads();
  lp_pick(two, p);
  if (threadIdx.x < LP_TOP) {
    const lp_key k = p.found[threadIdx.x];
    values[row * LP_TOP + threadIdx.x] = a.s == 0.0f ? none : lp_value(k) - a.m - ln;
    indices[row * LP_TOP + threadIdx.x] = lp_index(k);
  }
#endif
}
#endif

extern "C" __global__ __launch_bounds__(LP_THREADS)
#if LP_JOIN
void LP_NAME(const float* __restrict__ part, const lp_t* __restrict__ logits, const long long* __restrict__ tokens, long long rows, float* __restrict__ logprob,
             float* __restrict__ entropy, float* __restrict__ values, long long* __restrict__ indices) {
  const long long row = blockIdx.x;
  const float* mine = part + row * (LP_PARTS * 3 + (LP_TOP ? LP_SEGMENTS : 0));
  LpSum a = {mine[0], mine[1], mine[2]};
#pragma unroll 4
  for (int i = 1; i < LP_PARTS; ++i) a = lp_add(a, {mine[3 * i], mine[3 * i + 1], mine[3 * i + 2]});
  lp_finish(logits + row * LP_STRIDE, row, a, mine + LP_PARTS * 3, tokens, logprob, entropy, values, indices);
#elif LP_PARTS > 1
void LP_NAME(const lp_t* __restrict__ logits, float* __restrict__ part) {
  const long long row = blockIdx.x / LP_PARTS;
  const int i = blockIdx.x % LP_PARTS, first = i * LP_SHARE, end = first + LP_SHARE < LP_BLOCKS ? first + LP_SHARE : LP_BLOCKS;
  float* mine = part + row * (LP_PARTS * 3 + (LP_TOP ? LP_SEGMENTS : 0));
  const LpSum a = lp_scan(logits + row * LP_STRIDE, first, end, mine + LP_PARTS * 3);
  if (threadIdx.x == 0) {
    mine[3 * i] = a.m;
    mine[3 * i + 1] = a.s;
    mine[3 * i + 2] = a.u;
  }
#else
void LP_NAME(const lp_t* __restrict__ logits, const long long* __restrict__ tokens, float* __restrict__ logprob, float* __restrict__ entropy,
             float* __restrict__ values, long long* __restrict__ indices) {
#if LP_TOP
  __shared__ float segments[LP_SEGMENTS];
#else
  float* segments = nullptr;
#endif
  const long long row = blockIdx.x;
  const LpSum a = lp_scan(logits + row * LP_STRIDE, 0, LP_BLOCKS, segments);
  lp_finish(logits + row * LP_STRIDE, row, a, segments, tokens, logprob, entropy, values, indices);
#endif
}
