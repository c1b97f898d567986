// ---- attention of new tokens over a paged cache in 8 bits ----
//   s = scale * kscale[page, h] * (q . k8)        s = cap * tanh(s / cap)        s += slope[head] * (key - position)
//   o = sum_keys softmax(s) * vscale[page, h] * v8     over keys <= position, > position - window
// q, out [T][heads][D] in 16 bits; the caches hold e4m3 numbers [page][token][kv head][D] at any strides, with one scale per page
// and kv head; table[b] lists the pages of request b, lengths[b] its keys, starts[b] its first row of q.
//
// The rows that read the same keys (the CA_GS heads of a group, of CA_TOK tokens) form a tile of 16 * CA_RB rows, so that a key is
// read once for all of them.  A wavefront takes 32 keys a step, without LDS: K is the left operand of S^T = K Q^T, whose result layout
// (a lane holds one row's scores of four neighbouring keys) is the layout in which the right operand of O^T = V^T P^T is read, when the
// eight keys of that product's lane are taken to be those that the lane has scores of.  The order of the summed index is free in
// both products: K is read in runs of D / 4 bytes, V in runs of D / 16 of eight keys, which are turned into columns in registers
// by one v_perm each.  e4m3 numbers are exact in both 16-bit types, so the cache costs no rounding; the probabilities are
// rounded to IEEE half (11 bits, they lie in [0, 2^CA_LAZY]), whatever the type of q; for results in IEEE half, which that rounding would
// make 1.4 times less exact than their own does, the rest of the rounding goes through a second product (CA_SPLIT) where rows are few
// and the cache's bytes bound the launch.
//
// A page's vscale goes into the exponent: P' = 2^(s - m) vscale = 2^(s + log2 vscale - m'), with m' the running maximum of that
// sum, so P' keeps its bits whatever the scales are; the sum of the probabilities takes P' / vscale as rounded, in fp32, so that a
// rounding shifts weight between keys and does not scale the result (and two dot products replace four additions).
//
// Work: the keys of a tile are cut into units of CA_UK = 128, one step of each of the four wavefronts.  All units of all tiles, head
// after head, stand in one line that is cut evenly over CA_GRID workgroups (prefix sums of the units of each request, in closed form,
// taken by every workgroup); a tile cut between workgroups leaves partial results in `part`, which cache_join adds up.  So
// requests of any lengths fill the part.  CA_WHOLE: one workgroup for each tile of a request (one tile each), nothing to join.
// Parameters: CA_NAME, CA_D, CA_HKV, CA_G (heads per kv head), CA_GS, CA_PAGE, CA_F16, CA_SPLIT, CA_RB, CA_GRID, CA_WHOLE, CA_MIN (least units of
// a workgroup), CA_SCALE, CA_CAP (0: none), CA_WINDOW (0: none), CA_SLOPES, CA_STARTS, CA_KP CA_KT CA_KH / CA_VP CA_VT CA_VH (strides of
// page, token, head), CA_QT CA_QH (of q), CA_JOIN (this is cache_join).
typedef _Float16 ca_f16x8 __attribute__((ext_vector_type(8)));
#if CA_F16
typedef _Float16 ca_q;
#define CA_MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ca_f16x8, a), __builtin_bit_cast(ca_f16x8, b), c, 0, 0, 0)
#define CA_CVT(w, hi) __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, hi))
#define CA_PACK kcg_pack_f16x2
#else
typedef __bf16 ca_q;
#define CA_MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(kcg_bf16x8, a), __builtin_bit_cast(kcg_bf16x8, b), c, 0, 0, 0)
#define CA_CVT(w, hi) __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, hi))
#define CA_PACK kcg_pack_bf16x2
#endif
#define CA_MFMA16(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ca_f16x8, a), __builtin_bit_cast(ca_f16x8, b), c, 0, 0, 0)
#define CA_CVT16(w, hi) __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, hi))
#define CA_NT (CA_D / 16)                    // tiles of 16 rows of O^T
#define CA_KR (CA_D / 16)                    // dwords of a lane's share of a key
#define CA_N8 (CA_D / 128)                   // V: pieces of 8 bytes per lane,
#define CA_N4 ((CA_D % 128) / 64)            // of 4
#define CA_N2 ((CA_D % 64) / 32)             // and of 2
#define CA_VR (2 * CA_N8 + CA_N4 + CA_N2)    // dwords of a lane's share of a key
#define CA_ROWS (16 * CA_RB)
#define CA_TOK (CA_ROWS / CA_GS)             // tokens of a tile
#define CA_PARTS ((CA_G + CA_GS - 1) / CA_GS)    // tiles that the heads of a group are cut into
#define CA_HV (CA_HKV * CA_PARTS)
#define CA_UK 128
#define CA_LAZY 6.0f
#define CA_TINY 1.17549435e-38f               // the least normal number: scales below count as zero
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
__device__ __forceinline__ int ca_base(const CaRequest& r) { return r.length > r.count ? r.length - r.count : 0; }
__device__ __forceinline__ int ca_low(const CaRequest& r, int tile) {     // first unit of a tile
#if CA_WINDOW
  const int p = ca_base(r) + tile * ca_tokens(r) - CA_WINDOW + 1;
  return p > 0 && r.length >= r.count ? p / CA_UK : 0;        // (rows before the first key: from the start)
#else
  return 0;
#endif
}
__device__ __forceinline__ int ca_units(const CaRequest& r, int tile) {
  return (ca_base(r) + (tile + 1) * ca_tokens(r) + CA_UK - 1) / CA_UK - ca_low(r, tile);
}
// Units of the tiles before `tile`: every tile ends with its last token's position (the last tile of several counts as if it were whole).
__device__ __forceinline__ int ca_before(const CaRequest& r, int tile) {
  if (tile <= 1) return tile == 0 ? 0 : ca_units(r, 0);
  const int p = ca_base(r), t = ca_tokens(r);
  unsigned sum = ca_floor_sum(tile, t, p + t + CA_UK - 1, CA_UK);
#if CA_WINDOW
  int skip = 0;                            // tiles whose window begins with the first key
  if (r.length < r.count) skip = tile;
  else if (p < CA_WINDOW) skip = (CA_WINDOW - 1 - p) / t + 1;
  if (tile > skip) sum -= ca_floor_sum(tile - skip, t, p + skip * t - CA_WINDOW + 1, CA_UK);
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

// Where in the line of all units a workgroup's share begins.
struct CaPlace {
  long long at;                 // the place
  int all, chunk;               // units of one head, and of a workgroup
  int hv, b, tile, unit;        // what stands there
};
// The place where workgroup `piece` begins; false where there is none.  Every wavefront finds it by itself, 64 requests to a round, or
// more to a lane: a read of the lengths, a sum over lanes, and two reads of lanes.
__device__ __forceinline__ bool ca_locate(int piece, const int* __restrict__ lengths, const int* __restrict__ starts, int B, int T, int most, CaPlace& w) {
  const int requests = B + CA_STARTS, lane = threadIdx.x & 63;
  const int per = (requests + 63) / 64, b0 = lane * per, b1 = b0 + per < requests ? b0 + per : requests;
  int mine = 0;
  for (int i = b0; i < b1; ++i) {
    const CaRequest r = ca_request(lengths, starts, i, B, T, most);
    mine += ca_before(r, ca_tiles(r));
  }
  const int through = ca_scan(mine), ahead = through - mine;
  w.all = __builtin_amdgcn_readlane(through, 63);
  const long long total = (long long)w.all * CA_HV, even = (total + CA_GRID - 1) / CA_GRID;
  w.chunk = even < CA_MIN ? CA_MIN : (int)even;
  w.at = (long long)piece * w.chunk;
  if (w.at >= total) return false;
  w.hv = total >> 32 ? (int)(w.at / w.all) : (int)((unsigned)w.at / (unsigned)w.all);
  const int f = (int)(w.at - (long long)w.hv * w.all);
  int b = 0, tile = 0, unit = 0;
  const bool here = f >= ahead && f < through;
  if (here) {
    int at = ahead;
    for (int i = b0; i < b1; ++i) {
      const CaRequest r = ca_request(lengths, starts, i, B, T, most);
      const int tiles = ca_tiles(r), units = ca_before(r, tiles);
      if (f < at + units) {
        int lo = 0, hi = tiles - 1;           // the last tile that begins at or before f
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (at + ca_before(r, mid) <= f) lo = mid; else hi = mid - 1;
        }
        b = i;
        tile = lo;
        unit = f - at - ca_before(r, lo);
        break;
      }
      at += units;
    }
  }
  const int who = __builtin_ctzll(__ballot(here));
  w.b = __builtin_amdgcn_readlane(b, who);
  w.tile = __builtin_amdgcn_readlane(tile, who);
  w.unit = __builtin_amdgcn_readlane(unit, who);
  return true;
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

// Index in a row of O of element `r` of tile `tt`, of a lane of group g: the inverse of the order in which V is read.
__device__ __forceinline__ int ca_column(int tt, int g, int r) {
  const int w = tt / 4, e = tt % 4, m = g * 4 + r;
  if (w < 2 * CA_N8) return (w / 2) * 128 + m * 8 + (w & 1) * 4 + e;
  if (CA_N4 && w == 2 * CA_N8) return CA_N8 * 128 + m * 4 + e;
  return CA_N8 * 128 + CA_N4 * 64 + m * 2 + e;
}

// One row block's tile of O^T to the rows of `out`.
__device__ __forceinline__ void ca_store(ca_q* __restrict__ out, const CaRequest& rq, int hv, int tile, int rb, int tt, kcg_f32x4 o, float sum) {
  const int n = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4, row = rb * 16 + n;
  const int token = row / CA_GS, head = row - token * CA_GS, t = ca_tokens(rq);
  const int h = (hv / CA_PARTS) * CA_G + (hv % CA_PARTS) * CA_GS + head;
  if (token >= t || tile * t + token >= rq.count || (hv % CA_PARTS) * CA_GS + head >= CA_G) return;
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);       // (a NaN stays one)
  ca_q* p = out + ((long long)(rq.first + tile * t + token) * (CA_HKV * CA_G) + h) * CA_D;
#pragma unroll
  for (int r = 0; r < 4; ++r) p[ca_column(tt, g, r)] = (ca_q)(o[r] * inv);
}

#if CA_JOIN
// A workgroup for every end of a share, which has something to do where that is the first one inside of a tile: it adds up the parts of
// the tile, in order.  A wavefront takes every fourth tile of 16 columns of O.
extern "C" __global__ __launch_bounds__(256)
void CA_NAME(const float* __restrict__ part, const int* __restrict__ lengths, const int* __restrict__ starts, long long T_, long long B_,
             long long W_, ca_q* __restrict__ out) {
  const int T = (int)T_, B = (int)B_, most = (int)W_ * CA_PAGE, rb = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15;
  const int second = blockIdx.x + 1;
  CaPlace w;
  if (!ca_locate(second, lengths, starts, B, T, most, w) || w.unit == 0 || w.unit > w.chunk) return;
  const CaRequest rq = ca_request(lengths, starts, w.b, B, T, most);
  // the parts: of the workgroup before this end (its last piece, slot 1, unless its share begins with it), and of as many behind as
  // the tile goes on for
  const int count = 1 + (ca_units(rq, w.tile) - w.unit + w.chunk - 1) / w.chunk;
  const float* first = part + ((long long)(second - 1) * 2 + (w.unit < w.chunk ? 1 : 0)) * CA_SLOT;
  const float* later = part + (long long)second * 2 * CA_SLOT;
  // the largest maximum, and the sum: lane group g takes every fourth part
  const int at = CA_ROWS * CA_D + (rb * 16 + n) * 2;
  float m = -__builtin_inff(), l = 0.0f;
  for (int i = lane >> 4; i < count; i += 4) {
    const float* p = i ? later + (long long)(i - 1) * 2 * CA_SLOT : first;
    const float pm = p[at], to = fmaxf(m, pm), ref = to == -__builtin_inff() ? 0.0f : to;
    l = l * __builtin_amdgcn_exp2f(m - ref) + p[at + 1] * __builtin_amdgcn_exp2f(pm - ref);
    m = to;
  }
  const float top = ca_cross(m, true), ref = top == -__builtin_inff() ? 0.0f : top;
  const float sum = ca_cross(l * __builtin_amdgcn_exp2f(m - ref), false);
  for (int tt = wave; tt < CA_NT; tt += 4) {
    kcg_f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int i = 0; i < count; ++i) {
      const float* p = i ? later + (long long)(i - 1) * 2 * CA_SLOT : first;
      o += *(const kcg_f32x4*)(p + ((rb * CA_NT + tt) * 64 + lane) * 4) * __builtin_amdgcn_exp2f(p[at] - ref);
    }
    ca_store(out, rq, w.hv, w.tile, rb, tt, o, sum);
  }
}
#else

// What a step has beside its keys and values.
struct CaMeta {
  float ks[2], vs[2];      // scales of the pages of its two halves
  bool there[2];           // false: no such keys, or a page that there is none of
};

extern "C" __global__ __launch_bounds__(256, CA_OCC)
void CA_NAME(const ca_q* __restrict__ q, const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc,
             const float* __restrict__ kscale, const float* __restrict__ vscale, const int* __restrict__ table,
             const int* __restrict__ lengths, const int* __restrict__ starts, const float* __restrict__ slopes,
             float* __restrict__ part, long long T_, long long B_, long long W_, long long table_row, long long pages_, ca_q* __restrict__ out) {
  __shared__ kcg_f32x4 red[4][CA_NT][64];
  __shared__ float ml[4][CA_ROWS][2];
  const int T = (int)T_, B = (int)B_, most = (int)W_ * CA_PAGE, pages = (int)pages_;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;

  int hv, b, tile, unit;
  int left;                       // units this workgroup has to do
#if CA_WHOLE
  hv = blockIdx.x % CA_HV;
  b = blockIdx.x / CA_HV;
  tile = unit = 0;
  left = 0x7fffffff;
#else
  const int requests = B + CA_STARTS;
  // neighbouring shares, which have pages in common, on one XCD: workgroups are dealt to the eight in turn
  const int piece = (blockIdx.x & 7) * (CA_GRID / 8) + (blockIdx.x >> 3);
  CaPlace w;
  if (!ca_locate(piece, lengths, starts, B, T, most, w)) return;
  left = (long long)w.all * CA_HV - w.at < w.chunk ? (int)((long long)w.all * CA_HV - w.at) : w.chunk;
  hv = w.hv; b = w.b; tile = w.tile; unit = w.unit;
  bool begun = true;              // the first piece of this workgroup, if it is not a whole tile, goes to slot 0, a later one to slot 1
#endif

  while (left > 0) {
    const CaRequest rq = ca_request(lengths, starts, b, B, T, most);
    const int t = ca_tokens(rq), tok0 = tile * t, tokens = rq.count - tok0 < t ? rq.count - tok0 : t;
    const int units = ca_units(rq, tile);
    const int until = left < units - unit ? unit + left : units;      // of this piece
    const int first = rq.length - rq.count + tok0;                         // position of the tile's first row
    const int hi = first + tokens > 0 ? first + tokens : 0;
    const int lo = CA_WINDOW && first - CA_WINDOW + 1 > 0 ? first - CA_WINDOW + 1 : 0;
    const int kvh = hv / CA_PARTS, head0 = kvh * CA_G + (hv % CA_PARTS) * CA_GS;
    const int base = ca_low(rq, tile) * CA_UK;
    int key = base + unit * CA_UK + wave * 32;
    const int end = base + until * CA_UK < hi ? base + until * CA_UK : hi;

    // rows: query fragments, positions
    unsigned qf[CA_RB][CA_KR * 2];
    int pos[CA_RB];
    float slope[CA_RB];
#pragma unroll
    for (int rb = 0; rb < CA_RB; ++rb) {
      const int row = rb * 16 + n, tk = row / CA_GS, hd = row - tk * CA_GS;
      const bool real = tk < tokens && (hv % CA_PARTS) * CA_GS + hd < CA_G;
      const int token = real ? tk : 0, head = real ? head0 + hd : head0;
      pos[rb] = first + token;
      slope[rb] = CA_SLOPES ? slopes[head] * 1.44269504088896340736f : 0.0f;
      const ca_q* p = q + (long long)(rq.first + tok0 + token) * CA_QT + (long long)head * CA_QH + g * (CA_D / 4);
#pragma unroll
      for (int i = 0; i < CA_KR * 2; i += 4) *(kcg_u32x4*)&qf[rb][i] = *(const kcg_u32x4*)(p + i * 2);
    }

    kcg_f32x4 acc[CA_RB][CA_NT];
    float m[CA_RB], l[CA_RB];
#pragma unroll
    for (int rb = 0; rb < CA_RB; ++rb) {
      m[rb] = -__builtin_inff();
      l[rb] = 0.0f;
#pragma unroll
      for (int i = 0; i < CA_NT; ++i) acc[rb][i] = kcg_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const int* row = table + (long long)b * table_row;
    // Entries of the table for the two halves of a step.  What is wrong with them is looked at when they are used, a step later: until
    // then nobody waits for them.
    auto pagesOf = [&](int at, int (&page)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) page[h] = row[(at + h * 16 < hi ? at + h * 16 : hi - 1) / CA_PAGE];
    };
    // Addresses: a uniform base and an offset of the lane's
    const unsigned koff = n * (unsigned)CA_KT + g * (CA_D / 4), voff = g * 4 * (unsigned)CA_VT;
    unsigned k[2][CA_KR], v[8][CA_VR];
    // (what is not there is read from somewhere that is)
    auto loadMeta = [&](int at, const int (&page)[2], long long (&pg)[2], CaMeta& s) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s.there[h] = at + h * 16 < hi && at + h * 16 + 16 > lo && (unsigned)page[h] < (unsigned)pages;
        pg[h] = s.there[h] ? page[h] : 0;
        s.ks[h] = kscale[pg[h] * CA_HKV + kvh];
        s.vs[h] = vscale[pg[h] * CA_HKV + kvh];
      }
    };
    auto loadK = [&](int at, const long long (&pg)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned char* kp = kc + (pg[h] * CA_KP + (long long)((at + h * 16) % CA_PAGE) * CA_KT + (long long)kvh * CA_KH);
#if CA_KR % 4 == 0
#pragma unroll
        for (int i = 0; i < CA_KR; i += 4) *(kcg_u32x4*)&k[h][i] = *(const kcg_u32x4*)(kp + koff + i * 4);
#else
#pragma unroll
        for (int i = 0; i < CA_KR; i += 2) *(kcg_u32x2*)&k[h][i] = *(const kcg_u32x2*)(kp + koff + i * 4);
#endif
      }
    };
    auto loadV = [&](int at, const long long (&pg)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned char* vp = vc + (pg[h] * CA_VP + (long long)((at + h * 16) % CA_PAGE) * CA_VT + (long long)kvh * CA_VH);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const unsigned off = voff + r * (unsigned)CA_VT;
#pragma unroll
          for (int i = 0; i < CA_N8; ++i) *(kcg_u32x2*)&v[h * 4 + r][2 * i] = *(const kcg_u32x2*)(vp + off + (i * 128 + n * 8));
          if (CA_N4) v[h * 4 + r][2 * CA_N8] = *(const unsigned*)(vp + off + (CA_N8 * 128 + n * 4));
          if (CA_N2) v[h * 4 + r][2 * CA_N8 + CA_N4] = *(const unsigned short*)(vp + off + (CA_N8 * 128 + CA_N4 * 64 + n * 2));
        }
      }
    };

    float known = 1.0f;            // the last vscale that was not zero
    kcg_f32x4 sc[CA_RB][2];
    auto scores = [&]() {
#pragma unroll
      for (int rb = 0; rb < CA_RB; ++rb)
#pragma unroll
        for (int h = 0; h < 2; ++h) sc[rb][h] = kcg_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < CA_KR; i += 2) {
          const kcg_u32x4 kf = {CA_CVT(k[h][i], false), CA_CVT(k[h][i], true), CA_CVT(k[h][i + 1], false), CA_CVT(k[h][i + 1], true)};
#pragma unroll
          for (int rb = 0; rb < CA_RB; ++rb) {
            const kcg_u32x4 qv = {qf[rb][2 * i], qf[rb][2 * i + 1], qf[rb][2 * i + 2], qf[rb][2 * i + 3]};
            sc[rb][h] = CA_MFMA(kf, qv, sc[rb][h]);
          }
        }
    };
    // Scores to probabilities, and these into the sums; `masked`: not every row sees every key of the step, or a scale is zero.
    auto weigh = [&](int at, const CaMeta& s, bool masked) __attribute__((always_inline)) {
      // scales; those of zero stand for pages of zeros (or for pages that are not there)
      float ks[2], lv[2], iv[2];
      bool zero[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        zero[h] = masked && (!s.there[h] || s.vs[h] < CA_TINY);
        ks[h] = masked && !s.there[h] ? 0.0f : s.ks[h];
        if (!zero[h]) known = s.vs[h];
        lv[h] = __builtin_amdgcn_logf(known);
        iv[h] = __builtin_amdgcn_rcpf(known);
      }
#pragma unroll
      for (int rb = 0; rb < CA_RB; ++rb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float x = sc[rb][h][r];
#if CA_HAS_CAP
            x = kcg_fast_tanh(x * (ks[h] * (CA_SCALE / CA_CAP)));
            x = __builtin_fmaf(x, CA_CAP * 1.44269504088896340736f, lv[h]);
#else
            x = __builtin_fmaf(x, ks[h] * (CA_SCALE * 1.44269504088896340736f), lv[h]);
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
              const bool seen = key16 <= pos[rb] && (!CA_WINDOW || key16 > pos[rb] - CA_WINDOW) && s.there[h];
              if (!seen) sc[rb][h][r] = -__builtin_inff();
            }
        // V of keys that no row sees, which may be anything, and of pages whose scale is zero
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key16 = at + h * 16 + g * 4 + r;
            if (key16 < lo || key16 >= hi || zero[h])
#pragma unroll
              for (int w = 0; w < CA_VR; ++w) v[h * 4 + r][w] = 0;
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
          const float to = fmaxf(m[rb], mx), f = to == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m[rb] - to);
          m[rb] = to;
          l[rb] *= f;
#pragma unroll
          for (int i = 0; i < CA_NT; ++i) acc[rb][i] *= f;
        }
        const float ref = m[rb] == -__builtin_inff() ? 0.0f : m[rb];
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
            pl[rb][2 * h + j] = kcg_pack_f16x2(p[2 * j] - (float)up[0], p[2 * j + 1] - (float)up[1]);
          }
          const float sum = (p[0] + p[1]) + (p[2] + p[3]);
#else
          const kcg_f16x2 one = {(_Float16)1.0f, (_Float16)1.0f};
          const float sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(kcg_f16x2, pf[rb][2 * h]), one,
                                                   __builtin_amdgcn_fdot2(__builtin_bit_cast(kcg_f16x2, pf[rb][2 * h + 1]), one, 0.0f, false), false);
#endif
          l[rb] = __builtin_fmaf(sum, iv[h], l[rb]);
        }
      }
      if (masked) {
        // NaN in V where some rows see the key and some do not: it goes to those that do, by a product of where V is NaN and who sees
        unsigned any = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int w = 0; w < CA_VR; ++w) any |= ((v[k][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        if (__any(any != 0)) {
#pragma unroll
          for (int w = 0; w < CA_VR; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (w * 4 + e >= CA_NT) continue;
              unsigned x[4];             // 1.0 where column e of dword w is NaN
#pragma unroll
              for (int j = 0; j < 4; ++j)
                x[j] = ((v[2 * j][w] >> (8 * e) & 0x7f) == 0x7f ? 0x3c00u : 0u) | ((v[2 * j + 1][w] >> (8 * e) & 0x7f) == 0x7f ? 0x3c000000u : 0u);
              const kcg_u32x4 where = {x[0], x[1], x[2], x[3]};
#pragma unroll
              for (int rb = 0; rb < CA_RB; ++rb) {
                unsigned see[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  see[j] = (sc[rb][j / 2][j % 2 * 2] != -__builtin_inff() ? 0x3c00u : 0u) | (sc[rb][j / 2][j % 2 * 2 + 1] != -__builtin_inff() ? 0x3c000000u : 0u);
                const kcg_u32x4 who = {see[0], see[1], see[2], see[3]};
                const kcg_f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
                kcg_f32x4 c = CA_MFMA16(where, who, none);        // how many such keys the row sees
                c *= 0x1p127f;
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[rb][w * 4 + e][r] = __builtin_fmaf(c[r] * 0x1p127f, 0.0f, acc[rb][w * 4 + e][r]);      // + 0, or infinity times 0
              }
              __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
          for (int k8 = 0; k8 < 8; ++k8)
#pragma unroll
            for (int w = 0; w < CA_VR; ++w) v[k8][w] &= ~((((v[k8][w] & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u) * 0xffu);
        }
      }
#pragma unroll
      for (int w = 0; w < CA_VR; ++w)
#pragma unroll
        for (int e2 = 0; e2 < 2; ++e2) {
          const int tt = w * 4 + e2 * 2;
          if (tt >= CA_NT) continue;
          unsigned x[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = e2 ? CA_CVT16(v[k][w], true) : CA_CVT16(v[k][w], false);
          const kcg_u32x4 even = {__builtin_amdgcn_perm(x[1], x[0], 0x05040100u), __builtin_amdgcn_perm(x[3], x[2], 0x05040100u),
                                  __builtin_amdgcn_perm(x[5], x[4], 0x05040100u), __builtin_amdgcn_perm(x[7], x[6], 0x05040100u)};
          const kcg_u32x4 odd = {__builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u),
                                 __builtin_amdgcn_perm(x[5], x[4], 0x07060302u), __builtin_amdgcn_perm(x[7], x[6], 0x07060302u)};
#pragma unroll
          for (int rb = 0; rb < CA_RB; ++rb) {
            const kcg_u32x4 p = {pf[rb][0], pf[rb][1], pf[rb][2], pf[rb][3]};
            acc[rb][tt] = CA_MFMA16(even, p, acc[rb][tt]);
            acc[rb][tt + 1] = CA_MFMA16(odd, p, acc[rb][tt + 1]);
#if CA_SPLIT
            const kcg_u32x4 q = {pl[rb][0], pl[rb][1], pl[rb][2], pl[rb][3]};
            acc[rb][tt] = CA_MFMA16(even, q, acc[rb][tt]);
            acc[rb][tt + 1] = CA_MFMA16(odd, q, acc[rb][tt + 1]);
#endif
          }
        }
    };

    if (key < end) {
      // The next step's keys are loaded when this one's scores are there, its values when this one's sums are: into the same registers, so
      // that many wavefronts fit.  Pages are read two steps ahead.
      const int last = key + (end - 1 - key) / CA_UK * CA_UK;
      CaMeta meta;
      int next[2];
      long long pg[2];
      pagesOf(key, next);
      loadMeta(key, next, pg, meta);
      loadK(key, pg);
      loadV(key, pg);
      pagesOf(key + CA_UK < last ? key + CA_UK : last, next);
#pragma unroll 1
      while (true) {
        scores();
        const CaMeta now = meta;
        const bool more = key < last;
        if (more) {
          loadMeta(key + CA_UK, next, pg, meta);
          loadK(key + CA_UK, pg);
          pagesOf(key + 2 * CA_UK < last ? key + 2 * CA_UK : last, next);
        }
        weigh(key, now, key + 32 > first + 1 || (CA_WINDOW && key < first + tokens - CA_WINDOW) || !now.there[0] || !now.there[1] || now.vs[0] < CA_TINY || now.vs[1] < CA_TINY);
        if (!more) break;
        loadV(key + CA_UK, pg);
        key += CA_UK;
      }
    }

    // the four wavefronts' results, brought to one maximum and added through LDS
#pragma unroll
    for (int rb = 0; rb < CA_RB; ++rb) {
      l[rb] = ca_cross(l[rb], false);
      if (g == 0) {
        ml[wave][rb * 16 + n][0] = m[rb];
        ml[wave][rb * 16 + n][1] = l[rb];
      }
    }
    __syncthreads();
#if CA_WHOLE
    const bool whole = true;
    float* slot = nullptr;
#else
    const bool whole = unit == 0 && until == units;
    float* slot = part + ((long long)piece * 2 + (begun ? 0 : 1)) * CA_SLOT;
    begun = false;
#endif
#pragma unroll
    for (int rb = 0; rb < CA_RB; ++rb) {
      const int at = rb * 16 + n;
      const float top = fmaxf(fmaxf(ml[0][at][0], ml[1][at][0]), fmaxf(ml[2][at][0], ml[3][at][0]));
      const float ref = top == -__builtin_inff() ? 0.0f : top;
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) sum = __builtin_fmaf(ml[w][at][1], __builtin_amdgcn_exp2f(ml[w][at][0] - ref), sum);
      const float f = __builtin_amdgcn_exp2f(m[rb] - ref);
      if (rb) __syncthreads();
#pragma unroll
      for (int i = 0; i < CA_NT; ++i) red[wave][i][lane] = acc[rb][i] * f;
      __syncthreads();
      for (int i = wave; i < CA_NT; i += 4) {
        const kcg_f32x4 o = (red[0][i][lane] + red[1][i][lane]) + (red[2][i][lane] + red[3][i][lane]);
        if (whole)
          ca_store(out, rq, hv, tile, rb, i, o, sum);
        else
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
    __syncthreads();
    left -= until - unit;
    unit = 0;
    if (left > 0 && ++tile >= ca_tiles(rq)) {      // the next tile that there is: of a later request, or of the next head
      tile = 0;
      while (true) {
        if (++b >= requests) {
          b = 0;
          ++hv;
        }
        if (ca_request(lengths, starts, b, B, T, most).count > 0) break;
      }
    }
#endif
  }
}
#endif
