// ---- attention of new tokens over a paged cache in 8 bits ----
//   s = scale * kscale[page, h] * (q . k8)        s = cap * tanh(s / cap)        s += slope[head] * (key - position)
//   o = sum_keys softmax(s) * vscale[page, h] * v8     over keys <= position, > position - window
// q, out [T][heads][D] in 16 bits; the caches hold e4m3 numbers [page][token][kv head][D] at any strides, with one scale per page
// and kv head; table[b] lists the pages of request b, lengths[b] its keys, starts[b] its first row of q.
//
// The rows that read the same keys (the CA_GS heads of a group, of CA_TOK tokens) form a tile, so that a key is read once for all of
// them.  A wavefront takes 32 keys a step, or with many rows 64.  K is the left operand of S^T = K Q^T as it lies in memory, in 8 bits:
// it is the queries that are converted, once, each row divided by a power of two and written as a sum of two e4m3 numbers (four bits each:
// all of a bfloat16's) or three (IEEE half), whose products are added; what that leaves out is below 2^-18 of the row's
// largest element.  The result's layout (a lane holds one row's scores of four neighbouring keys) is the layout in which the right
// operand of O^T = V^T P^T is read, when the eight keys of that product's lane are taken to be those that the lane has scores of.  V goes
// through LDS rows that belong to the wavefront alone, from which transposing reads give a lane its eight keys of one column, and is
// converted to IEEE half, exactly.  The probabilities are
// rounded to IEEE half (11 bits, they lie in [0, 2^(CA_LAZY + CA_HEAD)]), which leaves results in bfloat16, of 8 bits, about as exact as their own
// rounding does.  Results in half precision it would make 1.4 times less exact: there the rest of the rounding goes through a second product
// (CA_SPLIT), in every form, so that a row's bits do not go by the rows beside it.  Where the cache's bytes bound the launch that costs
// nothing, where rows share keys a fifth (1500 rows of 32 heads behind 6000 keys: 251 us, 209 without).
//
// A page's vscale goes into the exponent: P' = 2^(s - m) vscale = 2^(s + log2 vscale - m'), with m' the running maximum of that
// sum less CA_HEAD: half precision holds all bits of a P' down to 2^-23 of the largest, whatever the scales are.  Keys below add little to the
// result, but where their page's vscale is the small one they may have most of the weight: the sum of the probabilities takes
// P' / vscale before P' is rounded, in fp32.  (With the sum taken of the rounded P', pages with 2^-24 of another's scale did not count, and
// results came out twice what they should be.  The additions in place of two dot products are not seen in the time.)
//
// Work: the keys of a tile are cut into units of CA_UK = 32 CA_WAVES, one step of each wavefront of a workgroup.  All units of all tiles of a head
// stand in one line that is cut evenly between CA_PIECES workgroups (prefix sums of the units of each request, in closed form,
// taken by every workgroup); a tile cut between workgroups leaves partial results in `part`, which cache_join adds up.  So
// requests of any lengths fill the part.  CA_WHOLE: one workgroup for each tile, nothing to join.
// Measured, one token each, 32 heads over 8 of 128: 64 requests of up to 4096 keys 45 us and 4 for the join, 4.1 TB/s in the first; 4 of up to 131072,
// page by head, half precision: 91 and 5, 5.6 TB/s (a kernel that reads as many bytes only 6.3 and 6.6).  What is lost is between pieces of
// the ragged lengths and in rows of 128 bytes that lie 1 KiB apart.
// Parameters: CA_NAME, CA_D, CA_HKV, CA_G (heads per kv head), CA_GS, CA_PAGE, CA_F16, CA_SPLIT, CA_RB, CA_WAVES, CA_SHARE, CA_PIECES, CA_WHOLE, CA_JT, CA_MIN (least units of
// a workgroup), CA_SCALE, CA_CAP (0: none), CA_WINDOW (0: none), CA_SLOPES, CA_STARTS, CA_KP CA_KT CA_KH / CA_VP CA_VT CA_VH (strides of
// page, token, head), CA_QT CA_QH (of q), CA_JOIN (this is cache_join).
typedef _Float16 ca_f16x8 __attribute__((ext_vector_type(8)));
#if CA_F16
typedef _Float16 ca_q;
#define CA_PACK kcg_pack_f16x2
#define CA_QN 3                              // e4m3 numbers that a query's element is written as
#else
typedef __bf16 ca_q;
#define CA_PACK kcg_pack_bf16x2
#define CA_QN 2
#endif
#define CA_MFMA16(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ca_f16x8, a), __builtin_bit_cast(ca_f16x8, b), c, 0, 0, 0)
#define CA_CVT16(w, hi) __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, hi))
#define CA_NT (CA_D / 16)                    // tiles of 16 rows of O^T
#define CA_KR (CA_D / 16)                    // dwords of a lane's share of a key
#define CA_VL (CA_D / 32)                    // chunks of 16 bytes of a step's V that a lane brings
// Bytes of a key's V in LDS, an odd multiple of 32, the keys of the second half 16 bytes further: the 16 rows of 16 bytes that 32 lanes read
// together then meet all banks.
#define CA_VP_ ((CA_D + 31) / 64 * 64 + 32)
#define CA_VROW(key) ((key) * CA_VP_ + (key) / 16 * 16)
#define CA_KP_ (CA_D + 16)                   // of its K: eight lanes that read below one another meet all banks
#define CA_BLOCKS (CA_SHARE ? CA_RB * CA_WAVES : CA_RB)      // blocks of 16 rows of a tile
#define CA_ROWS (16 * CA_BLOCKS)
#define CA_TOK (CA_ROWS / CA_GS)             // tokens of a tile
#define CA_PARTS ((CA_G + CA_GS - 1) / CA_GS)    // tiles that the heads of a group are cut into
#define CA_HV (CA_HKV * CA_PARTS)
#define CA_UK (CA_SHARE ? 64 : 32 * CA_WAVES)
static_assert(0x7fff0000LL + 96 * CA_UK + 32 <= 0x7fffffff, "positions ahead of the last key of the longest request have 32 bits");
#define CA_LAZY 6.0f
#define CA_HEAD 9.0f
#define CA_TINY 1.17549435e-38f               // the least normal number: scales below count as zero
// What the logarithm of a scale of zero counts as: the keys of its page, which have weight but add nothing, then leave the running maximum, and so
// the bits of P', to those of pages with scales of 2^-50 and more; and up to 2^31 such keys leave their sum finite.
#define CA_NOTHING -80.0f
#define CA_SLOT (CA_ROWS * CA_D + 2 * CA_ROWS)   // floats of a partial result

struct CaRequest { int length, count, first; };       // keys, rows, first row

// Request b; b == B: the rows behind those of the last one, which see nothing.
__device__ __forceinline__ CaRequest ca_request(const int* __restrict__ lengths, const int* __restrict__ starts, int b, int B, int T, int most) {
  CaRequest r;
#if CA_STARTS
  const int s = starts[b], from = s < 0 ? 0 : (s > T ? T : s);
  int to = T;
  if (b < B) { to = starts[b + 1]; to = to > T ? T : to; }
  r.first = from;
  r.count = to > from ? to - from : 0;
#else
  r.first = b;
  r.count = b < B ? 1 : 0;
#endif
  const int n = b < B ? lengths[b] : 0;
  r.length = n < 0 ? 0 : (n > most ? most : n);
  return r;
}

// sum of the whole parts of (a i + b) / m over i < n (the steps of Euclid's algorithm on a and m); the sum and a n + b below 2^32
__device__ __forceinline__ unsigned ca_floor_sum(unsigned n, unsigned a, unsigned b, unsigned m) {
  unsigned sum = 0;
  while (n > 0) {
    sum += n * (n - 1) / 2 * (a / m) + n * (b / m);        // (a / m is not 0 in later rounds only, where n is small)
    a %= m;
    b %= m;
    const unsigned top = a * n + b;
    if (top < m) break;
    n = top / m;
    b = top % m;
    const unsigned t = m;
    m = a;
    a = t;
  }
  return sum;
}

__device__ __forceinline__ int ca_tokens(const CaRequest& r) { return r.count < CA_TOK ? (r.count > 0 ? r.count : 1) : CA_TOK; }
__device__ __forceinline__ int ca_tiles(const CaRequest& r) { return r.count <= CA_TOK ? (r.count > 0 ? 1 : 0) : (r.count + CA_TOK - 1) / CA_TOK; }
// The key that a request's first row stands at; negative where it has more rows than keys.
__device__ __forceinline__ int ca_base(const CaRequest& r) { return r.length - r.count; }
__device__ __forceinline__ int ca_low(const CaRequest& r, int tile) {     // first unit of a tile
#if CA_WINDOW
  const int p = ca_base(r) + tile * ca_tokens(r);
  return p >= CA_WINDOW ? (p - CA_WINDOW + 1) / CA_UK : 0;
#else
  return 0;
#endif
}
// A tile whose rows all stand before the first key counts one unit, in which there is nothing to do.
__device__ __forceinline__ int ca_units(const CaRequest& r, int tile) {
  const int whole = ca_base(r) + (tile + 1) * ca_tokens(r), end = whole < r.length ? whole : r.length;
  return end > 0 ? (end + CA_UK - 1) / CA_UK - ca_low(r, tile) : 1;
}
// Units of the tiles before `tile`: every tile ends with its last token's position, the last one of several with the last key.
__device__ __forceinline__ int ca_before(const CaRequest& r, int tile) {
  if (tile <= 1) return tile == 0 ? 0 : ca_units(r, 0);
  const int p = ca_base(r), t = ca_tokens(r);
  const bool cut = tile == ca_tiles(r);
  const int n = cut ? tile - 1 : tile, none = p < 0 ? -p / t : 0;       // (tiles before the first key)
  unsigned sum = cut ? ca_units(r, n) : 0;
  if (n <= none) return (int)sum + n;
  sum += none + ca_floor_sum(n - none, t, p + (none + 1) * t + CA_UK - 1, CA_UK);
#if CA_WINDOW
  const unsigned skip = p < CA_WINDOW ? (CA_WINDOW - 1u - p) / t + 1 : 0;       // tiles whose window begins with the first key
  if ((unsigned)n > skip) sum -= ca_floor_sum(n - skip, t, p + skip * t - CA_WINDOW + 1, CA_UK);
#endif
  return (int)sum;
}

// Sum over the lanes up to and including this one.
__device__ __forceinline__ int ca_scan(int v) {
#define CA_DPP(control, rows) v += __builtin_amdgcn_update_dpp(0, v, control, rows, 0xf, false)
  CA_DPP(0x111, 0xf);        // row_shr 1, 2, 4, 8: over the 16 lanes of a row
  CA_DPP(0x112, 0xf);
  CA_DPP(0x114, 0xf);
  CA_DPP(0x118, 0xf);
  CA_DPP(0x142, 0xa);        // a row's last lane into the next row, for the second and the fourth,
  CA_DPP(0x143, 0xc);        // the second row's into the third and the fourth
#undef CA_DPP
  return v;
}

// What the shares are cut by: units, or whole tiles where a workgroup takes one.
__device__ __forceinline__ int ca_cost(const CaRequest& r, int tile) { return CA_WHOLE ? tile : ca_before(r, tile); }

// What stands at the beginning of a workgroup's share.
struct CaPlace {
  int left, chunk;              // units of this share, and of every whole one
  CaRequest request;
  int b, tile, unit;
};
// The beginning of share `piece` of the units of a head; false where nothing is left.  Every wavefront finds it by itself, 64 requests to a
// round, or more to a lane: one read of the lengths, a sum over lanes, and reads of lanes.
__device__ __forceinline__ bool ca_locate(int piece, const int* __restrict__ lengths, const int* __restrict__ starts, int B, int T, int most, CaPlace& w) {
  const int requests = B + CA_STARTS, lane = threadIdx.x & 63;
  const int per = (requests + 63) / 64, b0 = lane * per, b1 = b0 + per < requests ? b0 + per : requests;
  CaRequest r = {0, 0, 0};
  int mine = 0;
  for (int i = b0; i < b1; ++i) {
    r = ca_request(lengths, starts, i, B, T, most);
    mine += ca_cost(r, ca_tiles(r));
  }
  const int through = ca_scan(mine), ahead = through - mine, all = __builtin_amdgcn_readlane(through, 63);
  const int even = (all + CA_PIECES - 1) / CA_PIECES;
  w.chunk = CA_WHOLE ? 1 : even < CA_MIN ? CA_MIN : even;
  if (piece >= (all + w.chunk - 1) / w.chunk) return false;
  const int f = piece * w.chunk;
  w.left = all - f < w.chunk ? all - f : w.chunk;
  int b = b0, tile = 0, unit = 0;
  const bool here = f >= ahead && f < through;
  if (here) {
    int at = ahead;
    for (; b < b1; ++b) {
      if (per > 1) r = ca_request(lengths, starts, b, B, T, most);
      const int tiles = ca_tiles(r), units = ca_cost(r, tiles);
      if (f < at + units) {
        int lo = 0, hi = tiles - 1;           // the last tile that begins at or before f
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (at + ca_cost(r, mid) <= f) lo = mid; else hi = mid - 1;
        }
        tile = lo;
        unit = f - at - ca_cost(r, lo);
        break;
      }
      at += units;
    }
  }
  const int who = __builtin_ctzll(__ballot(here));
  w.b = __builtin_amdgcn_readlane(b, who);
  w.tile = __builtin_amdgcn_readlane(tile, who);
  w.unit = __builtin_amdgcn_readlane(unit, who);
  w.request.length = __builtin_amdgcn_readlane(r.length, who);
  w.request.count = __builtin_amdgcn_readlane(r.count, who);
  w.request.first = __builtin_amdgcn_readlane(r.first, who);
  return true;
}

// The root of the factor that brings sums from one maximum to another: by two products with it, since a sum over pages with small scales is large
// and may stay where the factor itself is below the least number.
__device__ __forceinline__ float ca_root(float from, float to) { return __builtin_amdgcn_exp2f((from - to) * 0.5f); }

// kcg_fast_tanh's absolute error of 4e-7 is, times a cap of 64, 2^-15 of a probability.  Larger caps, which leave most scores nearly as they are, take
// the series where it is exact to fp32 (the next term is 1e-8 of the result), and 2e-6 of the result beyond
// (1500 rows of 32 heads behind 6000 keys: 314 us, 271 without the series; one row each of 64 requests the same time).
__device__ __forceinline__ float ca_tanh(float u) {
  const float far = kcg_fast_tanh(u);
  if (CA_CAP <= 64.0f) return far;
  const float v = u * u;
  const float near = u * __builtin_fmaf(v, __builtin_fmaf(v, __builtin_fmaf(v, __builtin_fmaf(v, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
  return __builtin_fabsf(u) < 0.25f ? near : far;
}

__device__ __forceinline__ float ca_cross(float v, bool max) {      // over the four lanes that hold a row
  auto a = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  const unsigned a0 = a[0], a1 = a[1];       // (the bits of an element of a vector have to be copied out of it first)
  const float x = __builtin_bit_cast(float, a0), y = __builtin_bit_cast(float, a1);
  v = max ? fmaxf(x, y) : x + y;
  auto b = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  const unsigned b0 = b[0], b1 = b[1];
  const float p = __builtin_bit_cast(float, b0), q = __builtin_bit_cast(float, b1);
  return max ? fmaxf(p, q) : p + q;
}

// One row block's tile of O^T to the rows of `out`, of `tokens` tokens from `first` on.
__device__ __forceinline__ void ca_store(ca_q* __restrict__ out, int first, int tokens, int hv, int rb, int tt, kcg_f32x4 o, float sum) {
  const int n = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4, row = rb * 16 + n;
  const int token = row / CA_GS, head = row - token * CA_GS, h = (hv / CA_PARTS) * CA_G + (hv % CA_PARTS) * CA_GS + head;
  if (token >= tokens || (hv % CA_PARTS) * CA_GS + head >= CA_G) return;
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);       // (a NaN stays one)
  ca_q* p = out + ((long long)(first + token) * (CA_HKV * CA_G) + h) * CA_D;
  *(kcg_u32x2*)(p + tt * 16 + g * 4) = kcg_u32x2{CA_PACK(o[0] * inv, o[1] * inv), CA_PACK(o[2] * inv, o[3] * inv)};
}

// What the workgroup of a share tells the join about the tile that its share begins inside of.
struct CaEnd { int first, tokens, parts, slot; };      // rows, parts (0: nothing to join, or an earlier share does), slot of the part before
#define CA_ENDS (4 * CA_HV * CA_PIECES)                // floats of all of them, in front of the parts

#if CA_JOIN
static_assert(CA_JT == 8 || CA_BLOCKS * CA_NT % CA_JT == 0, "wavefronts that share columns meet at barriers");
// A workgroup for every beginning of a share and CA_JT tiles of 16 rows and 16 columns of O; it has something to do where that is the first one
// inside of a tile of rows, and adds up the parts of the tile.  8 / CA_JT wavefronts take every so many-th part of the same columns: four
// in a decoding step, where a tile may have many parts; one, in a quarter of the workgroups, where tiles have 64 rows or more (1000 tokens
// of 32 heads: 67 us in all, 73 with four).
extern "C" __global__ __launch_bounds__(512)
void CA_NAME(const float* __restrict__ part, ca_q* __restrict__ out) {
  __shared__ kcg_f32x4 red[8][64];
  __shared__ float ml[8][16][2];
  const int hv = blockIdx.x % CA_HV, piece = blockIdx.x / CA_HV + 1, id = hv * CA_PIECES + piece;
  const CaEnd e = ((const CaEnd*)part)[id];
  if (e.parts == 0) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15;
  const int unit = wave % CA_JT, of16 = blockIdx.y * CA_JT + unit, rb = of16 / CA_NT, tt = of16 % CA_NT;
  if (rb >= CA_BLOCKS || rb * 16 >= e.tokens * CA_GS) return;      // (the last workgroup of a tile may have more wavefronts than there are columns)
  const int row = rb * 16 + n < e.tokens * CA_GS ? n : 0;                       // (rows that there are not were not written)
  const float* later = part + CA_ENDS + ((long long)id * 2 - 2) * CA_SLOT;       // part i > 0 is slot 0 of share id + i - 1
  const int at = CA_ROWS * CA_D + (rb * 16 + row) * 2, of = ((rb * CA_NT + tt) * 64 + lane - n + row) * 4;
  float m = -__builtin_inff(), l = 0.0f;
  kcg_f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int i = wave / CA_JT; i < e.parts; i += 8 / CA_JT) {
    const float* p = later + ((long long)i * 2 + (i ? 0 : e.slot)) * CA_SLOT;
    const kcg_f32x4 x = *(const kcg_f32x4*)(p + of);
    const float pm = p[at], pl = p[at + 1], to = fmaxf(m, pm), ref = to == -__builtin_inff() ? 0.0f : to;
    const float fa = ca_root(m, ref), fb = ca_root(pm, ref);
    o = o * (fa * fa) + x * (fb * fb);
    l = l * fa * fa + pl * fb * fb;
    m = to;
  }
  if (CA_JT < 8) {
    if (lane < 16) {
      ml[wave][n][0] = m;
      ml[wave][n][1] = l;
    }
    red[wave][lane] = o;
    __syncthreads();
    if (wave >= CA_JT) return;
    float top = m;
#pragma unroll
    for (int w = unit + CA_JT; w < 8; w += CA_JT) top = fmaxf(top, ml[w][n][0]);
    const float ref = top == -__builtin_inff() ? 0.0f : top;
    o = kcg_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    l = 0.0f;
#pragma unroll
    for (int w = unit; w < 8; w += CA_JT) {
      const float f = ca_root(ml[w][n][0], ref);
      o += red[w][lane] * (f * f);
      l += ml[w][n][1] * f * f;
    }
  }
  ca_store(out, e.first, e.tokens, hv, rb, tt, o, l);
}
#else

// A lane's part of a row of queries, and the same in 8 bits: a sum of CA_QN e4m3 numbers times the power of two that is returned.
typedef ca_q ca_q8 __attribute__((ext_vector_type(8)));
struct CaQuery { ca_q8 raw[CA_KR / 2]; };
__device__ __forceinline__ CaQuery ca_query_load(const ca_q* __restrict__ p) {
  CaQuery r;
#pragma unroll
  for (int i = 0; i < CA_KR / 2; ++i) r.raw[i] = *(const ca_q8*)(p + i * 8);
  return r;
}
__device__ __forceinline__ float ca_query(const CaQuery& r, unsigned (&qf)[CA_QN][CA_KR]) {
  const auto& raw = r.raw;
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < CA_KR * 4; ++i) top = fmaxf(top, __builtin_fabsf((float)raw[i / 8][i % 8]));
  top = ca_cross(top, true);
  // the least power of two whose 448-fold (1.75 * 2^8) reaches the row's largest element
  const unsigned bits = __builtin_bit_cast(unsigned, top);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < -100 ? -100 : e;
  const float inv = __builtin_bit_cast(float, (unsigned)(127 - e) << 23);
#pragma unroll
  for (int i = 0; i < CA_KR; ++i) {
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = (float)raw[i / 2][i % 2 * 4 + j] * inv;
#pragma unroll
    for (int c = 0; c < CA_QN; ++c) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], w, true);
      qf[c][i] = (unsigned)w;
      if (c + 1 < CA_QN) {
        f[0] -= __builtin_amdgcn_cvt_f32_fp8(w, 0);
        f[1] -= __builtin_amdgcn_cvt_f32_fp8(w, 1);
        f[2] -= __builtin_amdgcn_cvt_f32_fp8(w, 2);
        f[3] -= __builtin_amdgcn_cvt_f32_fp8(w, 3);
      }
    }
  }
  return __builtin_bit_cast(float, (unsigned)(e + 127) << 23);
}

// The scores of 16 keys, whose K is row `n` of `p`, and of row blocks with the queries `qf`.
template <int RB>
__device__ __forceinline__ void ca_scores(const unsigned char* p, const unsigned (&qf)[RB][CA_QN][CA_KR], kcg_f32x4 (&sc)[RB]) {
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) sc[rb] = kcg_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#if CA_D % 128 == 0
#pragma unroll
  for (int i = 0; i < CA_KR; i += 8) {
    const kcg_i32x4 k0 = *(const kcg_i32x4*)(p + i * 4), k1 = *(const kcg_i32x4*)(p + i * 4 + 16);
    const kcg_i32x8 kf = {k0[0], k0[1], k0[2], k0[3], k1[0], k1[1], k1[2], k1[3]};
#pragma unroll
    for (int c = 0; c < CA_QN; ++c)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const unsigned (&w)[CA_KR] = qf[rb][c];
        const kcg_i32x8 qv = {(int)w[i], (int)w[i + 1], (int)w[i + 2], (int)w[i + 3], (int)w[i + 4], (int)w[i + 5], (int)w[i + 6], (int)w[i + 7]};
        sc[rb] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kf, qv, sc[rb], 0, 0, 0, 0, 0, 0);
      }
  }
#else
#pragma unroll
  for (int i = 0; i < CA_KR; i += 2) {
    const long kf = *(const long*)(p + i * 4);
#pragma unroll
    for (int c = 0; c < CA_QN; ++c)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
        sc[rb] = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(kf, (long)((unsigned long)qf[rb][c][i + 1] << 32 | qf[rb][c][i]), sc[rb], 0, 0, 0);
  }
#endif
}

typedef __attribute__((address_space(3))) unsigned char* ca_lds;
typedef int ca_i32x2 __attribute__((ext_vector_type(2)));
// Eight keys of one column of V, by a transposing read, as IEEE half.
__device__ __forceinline__ kcg_u32x4 ca_columns(ca_lds p) {
  const ca_i32x2 raw = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) ca_i32x2*)p);
  const unsigned w0 = (unsigned)raw[0], w1 = (unsigned)raw[1];
  return kcg_u32x4{CA_CVT16(w0, false), CA_CVT16(w0, true), CA_CVT16(w1, false), CA_CVT16(w1, true)};
}
__device__ __forceinline__ unsigned ca_nan_bytes(unsigned w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u; }
// NaN for the rows (columns of `who`, 1.0 where the row sees the key) that see a key whose V is NaN (1.0 in `where`).
__device__ __forceinline__ void ca_spread_nan(kcg_u32x4 where, kcg_u32x4 who, kcg_f32x4& acc) {
  const kcg_f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
  kcg_f32x4 c = CA_MFMA16(where, who, none);          // how many such keys the row sees
  c *= 0x1p127f;
#pragma unroll
  for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf(c[r] * 0x1p127f, 0.0f, acc[r]);      // + 0, or infinity times 0
}

// The beginning of a workgroup's share, and what the join has to know of it; false where nothing is left.
__device__ __forceinline__ bool ca_begin(int id, int piece, float* __restrict__ part, const int* __restrict__ lengths, const int* __restrict__ starts, int B, int T,
                                         int most, CaPlace& w) {
  const bool some = ca_locate(piece, lengths, starts, B, T, most, w);
  if (threadIdx.x == 0) {
    CaEnd e = {0, 0, 0, 0};
    if (some && w.unit > 0 && w.unit <= w.chunk) {
      const int t = ca_tokens(w.request), at = w.tile * t;
      e.first = w.request.first + at;
      e.tokens = w.request.count - at < t ? w.request.count - at : t;
      e.parts = 1 + (ca_units(w.request, w.tile) - w.unit + w.chunk - 1) / w.chunk;
      e.slot = w.unit < w.chunk ? 1 : 0;          // the share before has it as its last piece, or as its only one
    }
    ((CaEnd*)part)[id] = e;
  }
  return some;
}

#if CA_SHARE
// Many rows: every wavefront has 16 CA_RB rows of the tile of its own, and all of them work on the same 64 keys a step, which they bring into two
// LDS buffers together; so a key is read once for 16 CA_RB CA_WAVES rows and nothing is added up between wavefronts.
// Measured: 1500 tokens of 32 heads over 8 of 128, behind 2 requests of up to 6000 keys, 160 us with the join, 625 TFLOP/s as 16-bit products
// would count; vector instructions are under way 55 % of the time (scores, exp2), matrix instructions 30 %.
// V is converted on its way into LDS, once for all wavefronts, as far as LDS holds two such workgroups (D up to 128).
#define CA_V16 (CA_D <= 128)
#define CA_VP16 (2 * CA_D + 32)              // bytes of a key's V in half precision: the eight rows of 32 bytes that 32 lanes read together meet all banks
#define CA_SL ((4 * CA_D + 64 * CA_WAVES - 1) / (64 * CA_WAVES))     // chunks of 16 bytes of a step's K, and of its V, that a lane brings
extern "C" __global__ __launch_bounds__(64 * CA_WAVES, CA_OCC)
void CA_NAME(const ca_q* __restrict__ q, const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc,
             const float* __restrict__ kscale, const float* __restrict__ vscale, const int* __restrict__ table,
             const int* __restrict__ lengths, const int* __restrict__ starts, const float* __restrict__ slopes,
             float* __restrict__ part, long long T_, long long B_, long long W_, long long table_row, long long pages_, ca_q* __restrict__ out) {
  struct Shared {
    __attribute__((aligned(16))) unsigned char k[2][64 * CA_KP_], v[2][CA_V16 ? 64 * CA_VP16 : CA_VROW(63) + CA_VP_];
    int nan[4];                  // whether a step has NaN in V where that matters, steps in turn
  };
  __shared__ Shared sh;
  const int T = (int)T_, B = (int)B_, most = (int)W_ * CA_PAGE, pages = (int)pages_;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int hv = blockIdx.x % CA_HV, requests = B + CA_STARTS, piece = blockIdx.x / CA_HV, id = hv * CA_PIECES + piece;
  CaPlace w;
  if (!ca_begin(id, piece, part, lengths, starts, B, T, most, w)) return;
  CaRequest rq = w.request;
  int b = w.b, tile = w.tile, unit = w.unit, left = w.left;
  bool begun = true;              // the first piece of this workgroup, if it is not a whole tile, goes to slot 0, a later one to slot 1
  if (threadIdx.x < 4) sh.nan[threadIdx.x] = 0;
  __syncthreads();
  unsigned koff[CA_SL], voff[CA_SL], kat[CA_SL], vat[CA_SL];
  int of[CA_SL];                  // key of the step that a chunk belongs to
#pragma unroll
  for (int u = 0; u < CA_SL; ++u) {
    int c = u * 64 * CA_WAVES + threadIdx.x;
    c = c < 4 * CA_D ? c : 4 * CA_D - 1;            // (behind the last chunk that one again)
    const int part16 = c % (CA_D / 16) * 16;
    of[u] = c / (CA_D / 16);
    koff[u] = (of[u] % 16) * (unsigned)CA_KT + part16;
    voff[u] = (of[u] % 16) * (unsigned)CA_VT + part16;
    kat[u] = of[u] * CA_KP_ + part16;
    vat[u] = CA_V16 ? of[u] * CA_VP16 + 2 * part16 : CA_VROW(of[u]) + part16;
  }
  auto stage = [&](unsigned char* vb, int u, const kcg_u32x4& x) __attribute__((always_inline)) {
#if CA_V16
    const unsigned x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3];
    *(kcg_u32x4*)(vb + vat[u]) = kcg_u32x4{CA_CVT16(x0, false), CA_CVT16(x0, true), CA_CVT16(x1, false), CA_CVT16(x1, true)};
    *(kcg_u32x4*)(vb + vat[u] + 16) = kcg_u32x4{CA_CVT16(x2, false), CA_CVT16(x2, true), CA_CVT16(x3, false), CA_CVT16(x3, true)};
#else
    *(kcg_u32x4*)(vb + vat[u]) = x;
#endif
  };
  // V of the keys that this lane has scores of, in column n of tile tt and half h of the step.  Of 16 bits a transposing read gives a lane four rows
  // of its column: lane 4 j + i of a group of 16 gives the address of quarter i of row j.
  const int key8 = n / 2 < 4 ? g * 4 + n / 2 : 16 + g * 4 + n / 2 - 4;        // the row that this lane gives the address of, of 8 bits
  const int vof = CA_V16 ? (g * 4 + n / 4) * CA_VP16 + n % 4 * 8 : CA_VROW(key8) + (n & 1) * 8;
  auto columns = [&](unsigned char* vb, int h, int tt) __attribute__((always_inline)) {
#if CA_V16
    typedef short ca_s16x4 __attribute__((ext_vector_type(4)));
    const ca_lds p = (ca_lds)vb + vof + h * 32 * CA_VP16 + tt * 32;
    const ca_s16x4 near = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ca_s16x4*)p);
    const ca_s16x4 far = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ca_s16x4*)(p + 16 * CA_VP16));
    return __builtin_bit_cast(kcg_u32x4, __builtin_shufflevector(near, far, 0, 1, 2, 3, 4, 5, 6, 7));
#else
    return ca_columns((ca_lds)vb + vof + h * CA_VROW(32) + tt * 16);
#endif
  };
  int count = 0;                  // steps so far

  while (left > 0) {
    const int t = ca_tokens(rq), tok0 = tile * t, tokens = rq.count - tok0 < t ? rq.count - tok0 : t;
    const int units = ca_units(rq, tile);
    const int until = left < units - unit ? unit + left : units;           // of this piece
    const int first = rq.length - rq.count + tok0;                         // position of the tile's first row
    const int hi = first + tokens > 0 ? first + tokens : 0;
    const int lo = CA_WINDOW && first - CA_WINDOW + 1 > 0 ? first - CA_WINDOW + 1 : 0;
    const int kvh = hv / CA_PARTS, head0 = kvh * CA_G + (hv % CA_PARTS) * CA_GS;
    const int base = ca_low(rq, tile) * CA_UK;
    int key = base + unit * CA_UK;
    const int end = base + until * CA_UK < hi ? base + until * CA_UK : hi;
    // tokens of this wavefront's rows; it has none where the first is not there
    const int t0 = wave * 16 * CA_RB / CA_GS, t1 = (wave * 16 * CA_RB + 16 * CA_RB - 1) / CA_GS;
    const bool mine = t0 < tokens;
    const int pos0 = first + t0, pos1 = first + (t1 < tokens ? t1 : tokens - 1);

    unsigned qf[CA_RB][CA_QN][CA_KR];
    float qs[CA_RB], slope[CA_RB], m[CA_RB], l[CA_RB];
    int pos[CA_RB];
    kcg_f32x4 acc[CA_RB][CA_NT];
#pragma unroll
    for (int rb = 0; rb < CA_RB; ++rb) {
      const int row = (wave * CA_RB + rb) * 16 + n, tk = row / CA_GS, hd = row - tk * CA_GS;
      const bool real = tk < tokens && (hv % CA_PARTS) * CA_GS + hd < CA_G;
      const int token = real ? tk : 0, head = real ? head0 + hd : head0;
      pos[rb] = first + token;
      slope[rb] = CA_SLOPES ? slopes[head] * 1.44269504088896340736f : 0.0f;
      qs[rb] = ca_query(ca_query_load(q + (long long)(rq.first + tok0 + token) * CA_QT + (long long)head * CA_QH + g * (CA_D / 4)), qf[rb]);
      m[rb] = -__builtin_inff();
      l[rb] = 0.0f;
#pragma unroll
      for (int i = 0; i < CA_NT; ++i) acc[rb][i] = kcg_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    if (key < end) {
      const int* row = table + (long long)b * table_row;
      // Pages and scales of the quarters of 16 steps, a lane each, read while the 16 steps before are worked on
      struct Block { int page; float ks, vs; };       // page -1: no such keys, or a page that there is none of
      auto pagesOf = [&](int from) {
        const int at = from + (lane >> 2) * CA_UK + (lane & 3) * 16;
        const int page = row[(at < hi ? at : hi - 1) / CA_PAGE];
        return at < hi && at + 16 > lo && (unsigned)page < (unsigned)pages ? page : -1;
      };
      auto scalesOf = [&](int page) {
        const long long at = (long long)(page < 0 ? 0 : page) * CA_HKV + kvh;       // (what is not there is read from somewhere that is)
        return Block{page, kscale[at], vscale[at]};
      };
      auto ready = [&](Block& x) {
        x.ks = x.page < 0 ? 0.0f : x.ks;
        x.vs = x.page < 0 || x.vs < CA_TINY ? -__builtin_inff() : __builtin_amdgcn_logf(x.vs);      // (scales of zero stand for pages of zeros)
      };
      kcg_u32x4 k[CA_SL], v[CA_SL];
      auto load = [&](int at, int step, const Block& x) {
#pragma unroll
        for (int u = 0; u < CA_SL; ++u) {
          int page = __shfl(x.page, step * 4 + of[u] / 16, 64);
          page = page < 0 ? 0 : page;
          const long long token = (at + of[u] / 16 * 16) % CA_PAGE;
          k[u] = *(const kcg_u32x4*)(kc + ((long long)page * CA_KP + token * CA_KT + (long long)kvh * CA_KH) + koff[u]);
          v[u] = *(const kcg_u32x4*)(vc + ((long long)page * CA_VP + token * CA_VT + (long long)kvh * CA_VH) + voff[u]);
        }
      };
      Block now = scalesOf(pagesOf(key)), soon;
      int later = pagesOf(key + 16 * CA_UK), step = 0;
      load(key, 0, now);
      ready(now);
#pragma unroll 1
      while (true) {
        if (step == 0) {
          soon = scalesOf(later);
          later = pagesOf(key + 32 * CA_UK);
        }
        float ks[4], lv[4], iv[4];
        bool there[4], zeros = false;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          there[h] = __builtin_amdgcn_readlane(now.page, 4 * step + h) >= 0;
          ks[h] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, now.ks), 4 * step + h));
          lv[h] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, now.vs), 4 * step + h));
          const bool zero = lv[h] == -__builtin_inff();
          zeros |= zero;
          if (zero) lv[h] = CA_NOTHING;
          iv[h] = __builtin_amdgcn_exp2f(-lv[h]);
        }
        unsigned char *kb = sh.k[count & 1], *vb = sh.v[count & 1];
        // not every row of the tile sees every key of the step, or a scale is zero
        bool flagged = false;
        if (key + 64 > first + 1 || (CA_WINDOW && key < first + tokens - CA_WINDOW) || zeros) {
          // V of keys that no row sees, which may be anything, counts as zero, and so does that of pages whose scale is zero, but for NaN
          unsigned nan = 0;
#pragma unroll
          for (int u = 0; u < CA_SL; ++u) {
            bool none = key + of[u] < lo || key + of[u] >= hi;
            if (zeros) {
              const float scale = __shfl(now.vs, step * 4 + of[u] / 16, 64);
              none |= __shfl(now.page, step * 4 + of[u] / 16, 64) < 0;
              if (scale == -__builtin_inff())
#pragma unroll
                for (int i = 0; i < 4; ++i) v[u][i] &= ca_nan_bytes(v[u][i]) * 0xffu;
            }
            if (none) v[u] = kcg_u32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) nan |= ca_nan_bytes(v[u][i]);
          }
          if (nan != 0) sh.nan[count & 3] = 1;
          __syncthreads();
          flagged = __builtin_amdgcn_readfirstlane(sh.nan[count & 3]) != 0;
        }
#pragma unroll
        for (int u = 0; u < CA_SL; ++u) {
          *(kcg_u32x4*)(kb + kat[u]) = k[u];
          kcg_u32x4 x = v[u];
          if (flagged)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = ca_nan_bytes(x[i]) * 0x38u;       // 1.0 where V is NaN, first
          stage(vb, u, x);
        }
        if (threadIdx.x == 0) sh.nan[(count + 2) & 3] = 0;                       // (read last two steps ago)
        const bool more = key + CA_UK < end;
        if (++step == 16) {
          step = 0;
          now = soon;
          ready(now);
        }
        if (more && !flagged) load(key + CA_UK, step, now);
        __syncthreads();           // the step is in LDS, and everybody has finished with the one before

        const bool work = mine && key <= pos1 && (!CA_WINDOW || key + 63 > pos0 - CA_WINDOW);
        unsigned pf[CA_RB][8];
#if CA_SPLIT
        unsigned pl[CA_RB][8];           // what the rounding of pf leaves
#endif
        kcg_f32x4 sc[CA_RB][4];
        if (work) {
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            kcg_f32x4 s[CA_RB];
            ca_scores<CA_RB>(kb + (h * 16 + n) * CA_KP_ + g * (CA_D / 4), qf, s);
#pragma unroll
            for (int rb = 0; rb < CA_RB; ++rb) sc[rb][h] = s[rb];
          }
          const bool masked = key + 64 > pos0 + 1 || (CA_WINDOW && key <= pos1 - CA_WINDOW) || zeros;
          const bool general = CA_HAS_CAP || CA_SLOPES || !(CA_SCALE > 0.0f) || masked || !(ks[0] > 0.0f && ks[1] > 0.0f && ks[2] > 0.0f && ks[3] > 0.0f);
#pragma unroll
          for (int rb = 0; rb < CA_RB; ++rb) {
            // the exponent of a score x is by * x + plus
            float by[4], plus[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              by[h] = ks[h] * (CA_SCALE * 1.44269504088896340736f) * qs[rb];
              plus[h] = lv[h];
            }
            if (general) {
#pragma unroll
              for (int h = 0; h < 4; ++h) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const int at = key + h * 16 + g * 4 + r;
                  float x = sc[rb][h][r];
#if CA_HAS_CAP
                  x = ca_tanh(x * (ks[h] * (CA_SCALE / CA_CAP) * qs[rb]));
                  x = __builtin_fmaf(x, CA_CAP * 1.44269504088896340736f, lv[h]);
#else
                  x = __builtin_fmaf(x, by[h], lv[h]);
#endif
                  if (CA_SLOPES) x = __builtin_fmaf(slope[rb], (float)(at - pos[rb]), x);
                  const bool seen = !masked || (at <= pos[rb] && (!CA_WINDOW || at > pos[rb] - CA_WINDOW) && there[h]);
                  sc[rb][h][r] = seen ? x : -__builtin_inff();
                }
                by[h] = 1.0f;
                plus[h] = 0.0f;
              }
            }
            float mx = -__builtin_inff();
#pragma unroll
            for (int h = 0; h < 4; ++h)
              mx = fmaxf(mx, __builtin_fmaf(fmaxf(fmaxf(sc[rb][h][0], sc[rb][h][1]), fmaxf(sc[rb][h][2], sc[rb][h][3])), by[h], plus[h]));
            mx = ca_cross(mx, true);
            if (__any(mx > m[rb] + CA_LAZY)) {
              const float to = fmaxf(m[rb], mx), f = to == -__builtin_inff() ? 1.0f : ca_root(m[rb], to);
              m[rb] = to;
              l[rb] = l[rb] * f * f;
#pragma unroll
              for (int i = 0; i < CA_NT; ++i) acc[rb][i] *= f * f;
            }
            const float ref = m[rb] == -__builtin_inff() ? 0.0f : m[rb] - CA_HEAD;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              float p[4];
#pragma unroll
              for (int r = 0; r < 4; ++r) p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[rb][h][r], by[h], plus[h] - ref));
              pf[rb][2 * h] = kcg_pack_f16x2(p[0], p[1]);
              pf[rb][2 * h + 1] = kcg_pack_f16x2(p[2], p[3]);
#if CA_SPLIT
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const kcg_f16x2 up = __builtin_bit_cast(kcg_f16x2, pf[rb][2 * h + j]);
                pl[rb][2 * h + j] = kcg_pack_f16x2(__builtin_fmaf((float)up[0], -1.0f, p[2 * j]), __builtin_fmaf((float)up[1], -1.0f, p[2 * j + 1]));
              }
#endif
              l[rb] = __builtin_fmaf((p[0] + p[1]) + (p[2] + p[3]), iv[h], l[rb]);
            }
          }
        }
        if (flagged) {
          // NaN where some rows see the key and some may not: it goes to those that do, by a product of where V is NaN and who sees
          if (work)
#pragma unroll
            for (int rb = 0; rb < CA_RB; ++rb)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                unsigned see[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  see[j] = (sc[rb][2 * h + j / 2][j % 2 * 2] != -__builtin_inff() ? 0x3c00u : 0u) | (sc[rb][2 * h + j / 2][j % 2 * 2 + 1] != -__builtin_inff() ? 0x3c000000u : 0u);
                const kcg_u32x4 who = {see[0], see[1], see[2], see[3]};
#pragma unroll
                for (int tt = 0; tt < CA_NT; ++tt) ca_spread_nan(columns(vb, h, tt), who, acc[rb][tt]);
              }
          __syncthreads();
#pragma unroll
          for (int u = 0; u < CA_SL; ++u) {
            kcg_u32x4 x = v[u];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] &= ~(ca_nan_bytes(x[i]) * 0xffu);
            stage(vb, u, x);
          }
          if (more) load(key + CA_UK, step, now);
          __syncthreads();
        }
        if (work) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int tt = 0; tt < CA_NT; ++tt) {
              const kcg_u32x4 vf = columns(vb, h, tt);
#pragma unroll
              for (int rb = 0; rb < CA_RB; ++rb) {
                const kcg_u32x4 p = {pf[rb][4 * h], pf[rb][4 * h + 1], pf[rb][4 * h + 2], pf[rb][4 * h + 3]};
                acc[rb][tt] = CA_MFMA16(vf, p, acc[rb][tt]);
#if CA_SPLIT
                const kcg_u32x4 q = {pl[rb][4 * h], pl[rb][4 * h + 1], pl[rb][4 * h + 2], pl[rb][4 * h + 3]};
                acc[rb][tt] = CA_MFMA16(vf, q, acc[rb][tt]);
#endif
              }
            }
        }
        ++count;
        if (!more) break;
        key += CA_UK;
      }
    }

    const bool whole = unit == 0 && until == units;
    float* slot = part + CA_ENDS + ((long long)id * 2 + (begun ? 0 : 1)) * CA_SLOT;
    begun = false;
#pragma unroll
    for (int rb = 0; rb < CA_RB; ++rb) {
      const int block = wave * CA_RB + rb, at = block * 16 + n;
      l[rb] = ca_cross(l[rb], false);
#pragma unroll
      for (int i = 0; i < CA_NT; ++i) {
        if (whole)
          ca_store(out, rq.first + tok0, tokens, hv, block, i, acc[rb][i], l[rb]);
        else
          *(kcg_f32x4*)(slot + ((block * CA_NT + i) * 64 + lane) * 4) = acc[rb][i];
      }
      if (!whole && g == 0) {
        slot[CA_ROWS * CA_D + at * 2] = m[rb];
        slot[CA_ROWS * CA_D + at * 2 + 1] = l[rb];
      }
    }
    left -= until - unit;
    unit = 0;
    if (left > 0 && ++tile >= ca_tiles(rq)) {      // the next tile that there is
      tile = 0;
      while (++b < requests) {
        rq = ca_request(lengths, starts, b, B, T, most);
        if (rq.count > 0) break;
      }
    }
  }
}
#else
extern "C" __global__ __launch_bounds__(64 * CA_WAVES, CA_OCC)
void CA_NAME(const ca_q* __restrict__ q, const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc,
             const float* __restrict__ kscale, const float* __restrict__ vscale, const int* __restrict__ table,
             const int* __restrict__ lengths, const int* __restrict__ starts, const float* __restrict__ slopes,
             float* __restrict__ part, long long T_, long long B_, long long W_, long long table_row, long long pages_, ca_q* __restrict__ out) {
  union Shared {
    kcg_f32x4 red[CA_WAVES][CA_NT][64];
    struct {
      __attribute__((aligned(16))) unsigned char v[CA_WAVES][CA_VROW(31) + CA_VP_], k[CA_WAVES][32 * CA_KP_];
    } tile;
  };
  __shared__ Shared sh;
  __shared__ float ml[CA_WAVES][CA_ROWS][2];
  const int T = (int)T_, B = (int)B_, most = (int)W_ * CA_PAGE, pages = (int)pages_;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;

  // neighbouring heads, whose rows of a token lie beside one another, walk over their keys at the same time, and a head's workgroups, which
  // have keys in common where there are many rows, lie on one XCD where the number of heads allows (workgroups are dealt to the eight in turn)
  const int hv = blockIdx.x % CA_HV;
  CaRequest rq;
  int b, tile, unit, left;                       // left: units this workgroup has to do
#if CA_WHOLE
  b = blockIdx.x / CA_HV;
  tile = unit = 0;
  left = 0x7fffffff;
#if CA_STARTS
  CaPlace w;
  if (!ca_locate(b, lengths, starts, B, T, most, w)) return;
  rq = w.request; b = w.b; tile = w.tile;
#else
  rq = ca_request(lengths, starts, b, B, T, most);
#endif
#else
  const int requests = B + CA_STARTS, piece = blockIdx.x / CA_HV, id = hv * CA_PIECES + piece;
  CaPlace w;
  if (!ca_begin(id, piece, part, lengths, starts, B, T, most, w)) return;
  rq = w.request; b = w.b; tile = w.tile; unit = w.unit; left = w.left;
  bool begun = true;              // the first piece of this workgroup, if it is not a whole tile, goes to slot 0, a later one to slot 1
#endif

  // What this workgroup has to do of a tile: rows, keys, and the keys that this wavefront begins with.
  struct Piece { CaRequest rq; int b, tile, unit, until, units, tok0, tokens, first, lo, hi, key, end; };
  const int kvh = hv / CA_PARTS, head0 = kvh * CA_G + (hv % CA_PARTS) * CA_GS;
  auto pieceOf = [&](const CaRequest& rq, int b, int tile, int unit, int left) {
    Piece s;
    s.rq = rq;
    s.b = b;
    s.tile = tile;
    s.unit = unit;
    const int t = ca_tokens(rq);
    s.tok0 = tile * t;
    s.tokens = rq.count - s.tok0 < t ? rq.count - s.tok0 : t;
    s.units = ca_units(rq, tile);
    s.until = left < s.units - unit ? unit + left : s.units;
    s.first = rq.length - rq.count + s.tok0;                             // position of the tile's first row
    s.hi = s.first + s.tokens > 0 ? s.first + s.tokens : 0;
    s.lo = CA_WINDOW && s.first - CA_WINDOW + 1 > 0 ? s.first - CA_WINDOW + 1 : 0;
    const int base = ca_low(rq, tile) * CA_UK;
    s.key = base + unit * CA_UK + wave * 32;
    s.end = base + s.until * CA_UK < s.hi ? base + s.until * CA_UK : s.hi;
    return s;
  };
  // Pages and scales of the halves of 32 steps, a lane each (lane 2 s + h half h of step s), read while the 32 steps before are worked on and
  // their pages while those before are: by vector loads, since a scalar load would be waited for by every LDS access.
  struct Block { int page; float ks, vs; };       // page -1: no such keys, or a page that there is none of
  auto pagesOf = [&](const Piece& s, int from) {
    const int at = from + (lane >> 1) * CA_UK + (lane & 1) * 16;
    const int page = table[(long long)(s.b < B ? s.b : 0) * table_row + (at < s.hi ? at : s.hi > 0 ? s.hi - 1 : 0) / CA_PAGE];
    return at < s.hi && at + 16 > s.lo && (unsigned)page < (unsigned)pages ? page : -1;
  };
  auto scalesOf = [&](int page) {
    const long long at = (long long)(page < 0 ? 0 : page) * CA_HKV + kvh;       // (what is not there is read from somewhere that is)
    return Block{page, kscale[at], vscale[at]};
  };
  // Addresses: a uniform base and an offset of the lane's
  // K and V go in chunks of 16 bytes, neighbouring lanes neighbouring chunks (read where a lane needs them, four neighbouring lanes touch
  // four lines)
  kcg_u32x4 k[CA_VL], v[CA_VL];
  unsigned koff[CA_VL], voff[CA_VL], kat[CA_VL], vat[CA_VL];
#pragma unroll
  for (int u = 0; u < CA_VL; ++u) {
    const int c = u * 64 + lane, key32 = c / (CA_D / 16), part16 = c % (CA_D / 16) * 16;
    koff[u] = (key32 % 16) * (unsigned)CA_KT + part16;
    voff[u] = (key32 % 16) * (unsigned)CA_VT + part16;
    kat[u] = key32 * CA_KP_ + part16;
    vat[u] = CA_VROW(key32) + part16;
  }
  // the half that a chunk's key lies in is the same for all lanes where 64 chunks are whole halves
#define CA_HALF(u) (CA_D % 64 == 0 ? (u) * 64 / CA_D : ((u) * 64 + lane) / CA_D)
  auto loadK = [&](int at, const int (&pg)[2]) {
    const unsigned char* kp[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      kp[h] = kc + ((long long)(pg[h] < 0 ? 0 : pg[h]) * CA_KP + (long long)((at + h * 16) % CA_PAGE) * CA_KT + (long long)kvh * CA_KH);
#pragma unroll
    for (int u = 0; u < CA_VL; ++u) k[u] = *(const kcg_u32x4*)((CA_HALF(u) ? kp[1] : kp[0]) + koff[u]);
  };
  auto loadV = [&](int at, const int (&pg)[2]) {
    const unsigned char* vp[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      vp[h] = vc + ((long long)(pg[h] < 0 ? 0 : pg[h]) * CA_VP + (long long)((at + h * 16) % CA_PAGE) * CA_VT + (long long)kvh * CA_VH);
#pragma unroll
    for (int u = 0; u < CA_VL; ++u) v[u] = *(const kcg_u32x4*)((CA_HALF(u) ? vp[1] : vp[0]) + voff[u]);
  };
  // A piece's pages are read while the piece before is worked on, its first keys and values, and its queries, while that one's results are added
  // up: what a short piece would wait for (64 requests of up to 4096 keys 54 us without, 50 with).  A wavefront that has no keys brings some
  // that nobody uses.
  CaQuery raw[CA_RB];
  Block now;
  int pg[2];
  auto queries = [&](const Piece& s) __attribute__((always_inline)) {
#pragma unroll
    for (int rb = 0; rb < CA_RB; ++rb) {
      const int row = rb * 16 + n, tk = row / CA_GS, hd = row - tk * CA_GS;
      const bool real = tk < s.tokens && (hv % CA_PARTS) * CA_GS + hd < CA_G;
      raw[rb] = ca_query_load(q + (long long)(s.rq.first + s.tok0 + (real ? tk : 0)) * CA_QT + (long long)(real ? head0 + hd : head0) * CA_QH + g * (CA_D / 4));
    }
  };
  // whether registers hold the next piece's first keys and values, and its queries, beside the results (at D 256 that spills: 16
  // requests of up to 8000 keys 49 us, not 47)
  constexpr bool AHEAD = CA_D <= 128;
  auto begin = [&](const Piece& s, int page) __attribute__((always_inline)) {
    if (AHEAD) queries(s);
    now = scalesOf(page);
    pg[0] = __builtin_amdgcn_readlane(page, 0);
    pg[1] = __builtin_amdgcn_readlane(page, 1);
    loadK(s.key, pg);
    loadV(s.key, pg);
  };
  Piece s = pieceOf(rq, b, tile, unit, left);
  int page = pagesOf(s, s.key), later = pagesOf(s, s.key + 32 * CA_UK);
  if (AHEAD) begin(s, page);

  while (true) {
    const int tokens = s.tokens, first = s.first, hi = s.hi, lo = s.lo, end = s.end;
    int key = s.key;
#if !CA_WHOLE
    left -= s.until - s.unit;
    Piece next = s;
    int nextPage = -1, nextLater = -1;
    auto follow = [&]() __attribute__((always_inline)) {      // the next tile that there is
      if (left <= 0) return;
      if (++tile >= ca_tiles(rq)) {
        tile = 0;
        while (++b < requests) {
          rq = ca_request(lengths, starts, b, B, T, most);
          if (rq.count > 0) break;
        }
      }
      next = pieceOf(rq, b, tile, 0, left);
      nextPage = pagesOf(next, next.key);
      nextLater = pagesOf(next, next.key + 32 * CA_UK);
    };
    if (AHEAD) follow();
#endif
    unsigned qf[CA_RB][CA_QN][CA_KR];
    float qs[CA_RB];               // the power of two that a row was divided by
    int pos[CA_RB];
    float slope[CA_RB];
    if (!AHEAD) queries(s);
#pragma unroll
    for (int rb = 0; rb < CA_RB; ++rb) {
      const int row = rb * 16 + n, tk = row / CA_GS, hd = row - tk * CA_GS;
      const bool real = tk < tokens && (hv % CA_PARTS) * CA_GS + hd < CA_G;
      pos[rb] = first + (real ? tk : 0);
      slope[rb] = CA_SLOPES ? slopes[real ? head0 + hd : head0] * 1.44269504088896340736f : 0.0f;
      qs[rb] = ca_query(raw[rb], qf[rb]);
    }
    if (!AHEAD) begin(s, page);

    kcg_f32x4 acc[CA_RB][CA_NT];
    float m[CA_RB], l[CA_RB];
#pragma unroll
    for (int rb = 0; rb < CA_RB; ++rb) {
      m[rb] = -__builtin_inff();
      l[rb] = 0.0f;
#pragma unroll
      for (int i = 0; i < CA_NT; ++i) acc[rb][i] = kcg_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    unsigned char *ks_ = sh.tile.k[wave], *vs = sh.tile.v[wave];
    // this lane's address for the transposing reads of tile 0: within each group of 16 lanes, lanes 2 j and 2 j + 1 give the two halves of row
    // j, and lane i receives column i of the eight rows.  The rows are the keys that lane group g has scores of.
    const int key8 = n / 2 < 4 ? g * 4 + n / 2 : 16 + g * 4 + n / 2 - 4;
    const ca_lds vread = (ca_lds)vs + CA_VROW(key8) + (n & 1) * 8;

    kcg_f32x4 sc[CA_RB][2];
    // `behind` is called when the registers of K are free
    auto scores = [&](auto behind) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < CA_VL; ++u) *(kcg_u32x4*)(ks_ + kat[u]) = k[u];
      behind();
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        kcg_f32x4 s[CA_RB];
        ca_scores<CA_RB>(ks_ + (h * 16 + n) * CA_KP_ + g * (CA_D / 4), qf, s);
#pragma unroll
        for (int rb = 0; rb < CA_RB; ++rb) sc[rb][h] = s[rb];
      }
    };
    // Scores to probabilities, and these into the sums; `masked`: not every row sees every key of the step, or a scale is zero.
    // `behind` is called when the registers of V are free.
    auto weigh = [&](int at, const bool (&there)[2], const bool (&zero)[2], const float (&ks)[2], const float (&lv)[2], const float (&iv)[2], bool masked,
                     auto behind) __attribute__((always_inline)) {
#pragma unroll
      for (int rb = 0; rb < CA_RB; ++rb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float x = sc[rb][h][r];
#if CA_HAS_CAP
            x = ca_tanh(x * (ks[h] * (CA_SCALE / CA_CAP) * qs[rb]));
            x = __builtin_fmaf(x, CA_CAP * 1.44269504088896340736f, lv[h]);
#else
            x = __builtin_fmaf(x, ks[h] * (CA_SCALE * 1.44269504088896340736f) * qs[rb], lv[h]);
#endif
            if (CA_SLOPES) x = __builtin_fmaf(slope[rb], (float)(at + h * 16 + g * 4 + r - pos[rb]), x);
            sc[rb][h][r] = x;
          }
        }
      if (masked) {
#pragma unroll
        for (int rb = 0; rb < CA_RB; ++rb)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int key16 = at + h * 16 + g * 4 + r;
              const bool seen = key16 <= pos[rb] && (!CA_WINDOW || key16 > pos[rb] - CA_WINDOW) && there[h];
              if (!seen) sc[rb][h][r] = -__builtin_inff();
            }
      }
      // running maximum: the sums are brought to a new one only where it is more than 2^CA_LAZY times the old
      unsigned pf[CA_RB][4];
#if CA_SPLIT
      unsigned pl[CA_RB][4];           // what the rounding of pf leaves
#endif
#pragma unroll
      for (int rb = 0; rb < CA_RB; ++rb) {
        float mx = fmaxf(fmaxf(fmaxf(sc[rb][0][0], sc[rb][0][1]), fmaxf(sc[rb][0][2], sc[rb][0][3])),
                         fmaxf(fmaxf(sc[rb][1][0], sc[rb][1][1]), fmaxf(sc[rb][1][2], sc[rb][1][3])));
        mx = ca_cross(mx, true);
        if (__any(mx > m[rb] + CA_LAZY)) {
          const float to = fmaxf(m[rb], mx), f = to == -__builtin_inff() ? 1.0f : ca_root(m[rb], to);
          m[rb] = to;
          l[rb] = l[rb] * f * f;
#pragma unroll
          for (int i = 0; i < CA_NT; ++i) acc[rb][i] *= f * f;
        }
        const float ref = m[rb] == -__builtin_inff() ? 0.0f : m[rb] - CA_HEAD;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float p[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) p[r] = __builtin_amdgcn_exp2f(sc[rb][h][r] - ref);
          pf[rb][2 * h] = kcg_pack_f16x2(p[0], p[1]);
          pf[rb][2 * h + 1] = kcg_pack_f16x2(p[2], p[3]);
#if CA_SPLIT
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const kcg_f16x2 up = __builtin_bit_cast(kcg_f16x2, pf[rb][2 * h + j]);
            pl[rb][2 * h + j] = kcg_pack_f16x2(__builtin_fmaf((float)up[0], -1.0f, p[2 * j]), __builtin_fmaf((float)up[1], -1.0f, p[2 * j + 1]));
          }
#endif
          l[rb] = __builtin_fmaf((p[0] + p[1]) + (p[2] + p[3]), iv[h], l[rb]);
        }
      }
      auto stage = [&]() __attribute__((always_inline)) {      // (a wavefront's own LDS accesses are carried out in order)
#pragma unroll
        for (int u = 0; u < CA_VL; ++u) *(kcg_u32x4*)(vs + vat[u]) = v[u];
        __builtin_amdgcn_wave_barrier();
      };
      if (masked) {
        // V of keys that no row sees, which may be anything, counts as zero, and so does that of pages whose scale is zero, but for NaN
        unsigned nan = 0;
#pragma unroll
        for (int u = 0; u < CA_VL; ++u) {
          const int key32 = (u * 64 + lane) / (CA_D / 16);
          if ((zero[0] || zero[1]) && (key32 < 16 ? zero[0] : zero[1]))
#pragma unroll
            for (int i = 0; i < 4; ++i) v[u][i] &= ca_nan_bytes(v[u][i]) * 0xffu;
          if (at + key32 < lo || at + key32 >= hi || !(key32 < 16 ? there[0] : there[1])) v[u] = kcg_u32x4{0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < 4; ++i) nan |= ca_nan_bytes(v[u][i]);
        }
        if (__any(nan != 0)) {
          // NaN where some rows see the key and some may not: it goes to those that do, by a product of where V is NaN and who sees
          kcg_u32x4 whole[CA_VL];
#pragma unroll
          for (int u = 0; u < CA_VL; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const unsigned bytes = ca_nan_bytes(v[u][i]);
              whole[u][i] = v[u][i] & ~(bytes * 0xffu);
              v[u][i] = bytes * 0x38u;               // 1.0
            }
          stage();
#pragma unroll
          for (int u = 0; u < CA_VL; ++u) v[u] = whole[u];
#pragma unroll
          for (int tt = 0; tt < CA_NT; ++tt) {
            const kcg_u32x4 where = ca_columns(vread + tt * 16);
#pragma unroll
            for (int rb = 0; rb < CA_RB; ++rb) {
              unsigned see[4];
#pragma unroll
              for (int j = 0; j < 4; ++j)
                see[j] = (sc[rb][j / 2][j % 2 * 2] != -__builtin_inff() ? 0x3c00u : 0u) | (sc[rb][j / 2][j % 2 * 2 + 1] != -__builtin_inff() ? 0x3c000000u : 0u);
              const kcg_u32x4 who = {see[0], see[1], see[2], see[3]};
              ca_spread_nan(where, who, acc[rb][tt]);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      stage();
      behind();
#pragma unroll
      for (int tt = 0; tt < CA_NT; ++tt) {
        const kcg_u32x4 vf = ca_columns(vread + tt * 16);
#pragma unroll
        for (int rb = 0; rb < CA_RB; ++rb) {
          const kcg_u32x4 p = {pf[rb][0], pf[rb][1], pf[rb][2], pf[rb][3]};
          acc[rb][tt] = CA_MFMA16(vf, p, acc[rb][tt]);
#if CA_SPLIT
          const kcg_u32x4 q = {pl[rb][0], pl[rb][1], pl[rb][2], pl[rb][3]};
          acc[rb][tt] = CA_MFMA16(vf, q, acc[rb][tt]);
#endif
        }
      }
    };

    if (key < end) {
      // The next step's keys are loaded when this one's scores are there, its values when this one's are in LDS: into the same registers, so
      // that many wavefronts fit.
      const int last = key + (end - 1 - key) / CA_UK * CA_UK;
      Block soon;
      int step = 0;
#pragma unroll 1
      while (true) {
        if (step == 0) {
          soon = scalesOf(later);
          later = pagesOf(s, key + 64 * CA_UK);
          // (scales of zero stand for pages of zeros)
          now.ks = now.page < 0 ? 0.0f : now.ks;
          now.vs = now.page < 0 || now.vs < CA_TINY ? -__builtin_inff() : __builtin_amdgcn_logf(now.vs);
        }
        bool there[2], zero[2];
        float ks[2], lv[2], iv[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          there[h] = pg[h] >= 0;
          ks[h] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, now.ks), 2 * step + h));
          lv[h] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, now.vs), 2 * step + h));
          zero[h] = lv[h] == -__builtin_inff();
          if (zero[h]) lv[h] = CA_NOTHING;
          iv[h] = __builtin_amdgcn_exp2f(-lv[h]);
        }
        const bool more = key < last;
        if (++step == 32) {
          step = 0;
          now = soon;
        }
        pg[0] = __builtin_amdgcn_readlane(now.page, 2 * step);
        pg[1] = __builtin_amdgcn_readlane(now.page, 2 * step + 1);
        scores([&]() { if (more) loadK(key + CA_UK, pg); });
        const bool masked = key + 32 > first + 1 || (CA_WINDOW && key < first + tokens - CA_WINDOW) || zero[0] || zero[1];
        weigh(key, there, zero, ks, lv, iv, masked, [&]() { if (more) loadV(key + CA_UK, pg); });
        if (!more) break;
        key += CA_UK;
      }
    }

#if !CA_WHOLE
    if (AHEAD && left > 0) begin(next, nextPage);
#endif
    // the wavefronts' results, added through LDS
#if CA_WHOLE
    const bool whole = true;
    float* slot = nullptr;
#else
    const bool whole = s.unit == 0 && s.until == s.units;
    float* slot = part + CA_ENDS + ((long long)id * 2 + (begun ? 0 : 1)) * CA_SLOT;
    begun = false;
#endif
#pragma unroll
    for (int rb = 0; rb < CA_RB; ++rb) {
      const int at = rb * 16 + n;
      l[rb] = ca_cross(l[rb], false);
      if (g == 0) {
        ml[wave][at][0] = m[rb];
        ml[wave][at][1] = l[rb];
      }
      if (CA_WAVES > 1) __syncthreads();           // (everybody has read the sums of the row block before, or V)
#pragma unroll
      for (int i = 0; i < CA_NT; ++i) sh.red[wave][i][lane] = acc[rb][i];
      if (CA_WAVES > 1) __syncthreads();
      float top = ml[0][at][0];
#pragma unroll
      for (int w = 1; w < CA_WAVES; ++w) top = fmaxf(top, ml[w][at][0]);
      const float ref = top == -__builtin_inff() ? 0.0f : top;
      float sum = 0.0f, f[CA_WAVES];
#pragma unroll
      for (int w = 0; w < CA_WAVES; ++w) {
        const float root = ca_root(ml[w][at][0], ref);
        f[w] = root * root;
        sum = __builtin_fmaf(ml[w][at][1] * root, root, sum);
      }
#pragma unroll
      for (int j = 0; j < (CA_NT + CA_WAVES - 1) / CA_WAVES; ++j) {
        const int i = j * CA_WAVES + wave;
        if (i >= CA_NT) break;
        kcg_f32x4 o = sh.red[0][i][lane] * f[0];
#pragma unroll
        for (int w = 1; w < CA_WAVES; ++w) o += sh.red[w][i][lane] * f[w];
        if (whole)
          ca_store(out, s.rq.first + s.tok0, tokens, hv, rb, i, o, sum);
        else if (at < tokens * CA_GS)        // (the join reads no others)
          *(kcg_f32x4*)(slot + ((rb * CA_NT + i) * 64 + lane) * 4) = o;
      }
      if (!whole && wave == 0 && g == 0) {
        slot[CA_ROWS * CA_D + at * 2] = top;
        slot[CA_ROWS * CA_D + at * 2 + 1] = sum;
      }
    }
#if CA_WHOLE
    break;
#else
    if (left <= 0) break;
    if (!AHEAD) follow();
    __syncthreads();
    s = next;
    page = nextPage;
    later = nextLater;
#endif
  }
}
#endif
#endif
