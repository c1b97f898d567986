// ---- new keys and values into a paged cache in 8 bits ----
//   a = largest finite magnitude among the new rows of a page and head, need = the least power of two with 448 need >= a (0 for a = 0)
//   scale = need where the page begins with these rows, else max(old scale, need); what the page holds is brought to it
//   cache = e4m3(x / scale), to the nearest, ties to even; infinities become +-448, or 0 where the scale is 0; a NaN stays one
// A scale that is a power of two costs a floating format range but no precision, and a page whose scale has to grow is converted
// without loss down to the format's least numbers.
//
// A wavefront for each head, keys or values, and CW_WIN consecutive tokens.  A token whose predecessor lies in another page leads: its
// wavefront takes the tokens behind it in that page too (slots of a page stand together and ascend), so nobody else touches the
// page and head, and no atomics are needed.  The slots of 64 tokens are one load, whose lanes give the window's leaders and how far their
// pages go; then rows and old scale are one more trip to memory, before the stores: what bounds a small step.
// A lane takes 8 elements, CW_RPP rows a pass; rows are held in registers between the two passes (magnitude, conversion) as far as CW_HOLD
// passes reach, else read again, from the caches.  Passes behind the last row read the last again, so that no load waits for a branch.
//
// With CW_ROT (the family cache_append) keys are turned by their tokens' positions on the way, and so are queries, which go to a tensor:
//   halves of a head's first CW_R numbers:   (x_i, x_{i + R/2}) -> (x_i c_i - x_{i + R/2} s_i, x_{i + R/2} c_i + x_i s_i)
//   neighbours (CW_PAIRS):                   (x_2i, x_2i+1) -> the same
// with c and s of row `position` of the table.  What becomes of a key jumps where 8 bits do, so it has to be the formula's: the two products
// are exact in fp64 and their sum is rounded there once; on the way to fp32 what is cut off leaves its trace in the last bit (rounding to odd), so the
// rounding to 8 bits is that of the 53-bit number, and so is the comparison with 448 that gives the scale.  Queries in fp32
// are summed in fp64 as well and rounded once (7206 tokens of 32 query heads, 8 others, 64 us, summed in fp32 68); those of 16 bits in fp32, off
// by 2^-24 of the product and of the sum before their own rounding (half precision 43 us; with sines in two parts, whose products are exact, 46; in fp64 79).
// Wavefronts behind those of the cache take a token's queries, CW_QN passes of CW_RPP heads for one reading of c and s.
// Half precision moves 163 MB in these 43 us, 3.7 TB/s, of which keys and values alone take about 23: the keys' turns in fp64 and their registers (two wavefronts a
// SIMD) bound it, not memory.  fp32 moves 310 MB at 4.8 TB/s.
// Measured, 8 heads of 128: 64 tokens of a page each 2.9 us (an empty launch 1.7); 9000 tokens of whole pages, half precision, 12.5 us, 4.4 TB/s.
// Parameters: CW_NAME, CW_H, CW_D, CW_PAGE, CW_T (input type), CW_ESIZE, CW_WIN, strides as in cache_attention: CW_KP .. CW_VH (bytes), CW_XKT
// CW_XKH CW_XVT CW_XVH (of k and v, elements); CW_ROT, and with it CW_R, CW_PAIRS, CW_HQ (heads of q), CW_QN, CW_XQT CW_XQH.
typedef CW_T cw_t;
#define CW_LPR (CW_D / 8)            // lanes per row
#define CW_RPP (64 / CW_LPR)         // rows per pass
#define CW_ALL ((CW_PAGE + CW_RPP - 1) / CW_RPP)          // passes of a whole page
#define CW_MOST (CW_ESIZE * 8 > 16 || CW_ROT ? 4 : 8)    // that registers hold
#define CW_NEAR (48 / CW_RPP)                            // whose rows' slots the lanes have
#define CW_HOLD (CW_ALL < CW_MOST ? (CW_ALL < CW_NEAR ? CW_ALL : CW_NEAR) : CW_MOST < CW_NEAR ? CW_MOST : CW_NEAR)
typedef cw_t cw_x8 __attribute__((ext_vector_type(8)));
#if CW_ROT
typedef float CW_ROW[8];             // a lane's part of a row
#define CW_QC ((CW_HQ + CW_QN * CW_RPP - 1) / (CW_QN * CW_RPP))      // wavefronts of a token's queries
#else
typedef cw_x8 CW_ROW;
#endif

// Largest of the lanes' numbers, none of which is negative.
__device__ __forceinline__ float cw_max(float v) {
#define CW_DPP(control, rows) v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), control, rows, 0xf, false)))
  CW_DPP(0x111, 0xf);        // row_shr 1, 2, 4, 8: over the 16 lanes of a row
  CW_DPP(0x112, 0xf);
  CW_DPP(0x114, 0xf);
  CW_DPP(0x118, 0xf);
  CW_DPP(0x142, 0xa);        // a row's last lane into the next row, for the second and the fourth,
  CW_DPP(0x143, 0xc);        // the second row's into the third and the fourth
#undef CW_DPP
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ float cw_finite(float a) { return a < __builtin_inff() ? a : 0.0f; }        // (a NaN is not less either)
__device__ __forceinline__ float cw_limit(float x) {
  return x != x ? x : fminf(fmaxf(x, -448.0f), 448.0f);
}
__device__ __forceinline__ kcg_u32x2 cw_encode(const float (&x)[8]) {
  int a = __builtin_amdgcn_cvt_pk_fp8_f32(cw_limit(x[0]), cw_limit(x[1]), 0, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(cw_limit(x[2]), cw_limit(x[3]), a, true);
  int b = __builtin_amdgcn_cvt_pk_fp8_f32(cw_limit(x[4]), cw_limit(x[5]), 0, false);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(cw_limit(x[6]), cw_limit(x[7]), b, true);
  return kcg_u32x2{(unsigned)a, (unsigned)b};
}

#if CW_ROT
// c and s of a lane's eight numbers, and what its chunk is: the first of its pairs, the second, neighbours, or not turned at all.
struct CwTurn {
  kcg_f32x4 t[4];
  bool turned, lost;           // lost: a position behind the table's last
};
#define CW_HALF (CW_R / 16)                              // chunks of half the turned numbers
// Where the other numbers of chunk c's pairs are.
__device__ __forceinline__ int cw_partner(int c) { return CW_PAIRS || c >= 2 * CW_HALF ? c : c < CW_HALF ? c + CW_HALF : c - CW_HALF; }
__device__ __forceinline__ CwTurn cw_turn(const float* __restrict__ table, int position, long long P, int c) {
  CwTurn w;
  w.turned = position >= 0 && c < 2 * CW_HALF;
  w.lost = position >= P;
  const int pair = !w.turned ? 0 : CW_PAIRS ? 4 * c : 8 * (c % CW_HALF);
  const float* at = table + (w.turned && !w.lost ? (long long)position * CW_R : 0) + pair;
  w.t[0] = *(const kcg_f32x4*)at;
  w.t[2] = *(const kcg_f32x4*)(at + CW_R / 2);
  if (!CW_PAIRS) {
    w.t[1] = *(const kcg_f32x4*)(at + 4);
    w.t[3] = *(const kcg_f32x4*)(at + CW_R / 2 + 4);
  }
  return w;
}
// To fp32, to odd.
__device__ __forceinline__ float cw_odd(double v) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const unsigned low = (unsigned)b, cut = (low & 0xe0000000u) | ((low & 0x1fffffffu) ? 0x20000000u : 0u);
  return (float)__builtin_bit_cast(double, (b & 0xffffffff00000000ULL) | cut);
}
// The chunk x, whose partner is y, turned: with a sum in fp64, rounded to odd (KEY) or to the nearest, or for 16 bits in fp32.
template <bool KEY> __device__ __forceinline__ void cw_apply(const CwTurn& w, const cw_x8& x, const cw_x8& y, int c, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float co = w.t[CW_PAIRS ? 0 : i / 4][CW_PAIRS ? i / 2 : i % 4], si = w.t[CW_PAIRS ? 2 : 2 + i / 4][CW_PAIRS ? i / 2 : i % 4];
    const float a = (float)x[i], b = (float)(CW_PAIRS ? x[i ^ 1] : y[i]);
    const bool first = CW_PAIRS ? i % 2 == 0 : c < CW_HALF;
    float v;
    if (KEY || CW_ESIZE > 2) {
      const double p = (double)b * si, sum = (double)a * co + (first ? -p : p);
      v = KEY ? cw_odd(sum) : (float)sum;
    } else {
      const float p = b * si;
      v = __builtin_fmaf(a, co, first ? -p : p);
    }
    f[i] = w.turned ? w.lost ? __builtin_nanf("") : v : a;
  }
}
#endif

extern "C" __global__ __launch_bounds__(256)
void CW_NAME(const cw_t* __restrict__ k, const cw_t* __restrict__ v, unsigned char* __restrict__ kc, unsigned char* __restrict__ vc,
             float* __restrict__ ks, float* __restrict__ vs, const long long* __restrict__ slots, long long T_, long long pages
#if CW_ROT
             , const cw_t* __restrict__ q, const int* __restrict__ positions, const float* __restrict__ table, long long P, cw_t* __restrict__ out
#endif
) {
  const int T = (int)T_, lane = threadIdx.x & 63;
  const long long job = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = (int)(job % (2 * CW_H)), h = part >> 1;
  const long long win = job / (2 * CW_H);
#if CW_ROT
  const long long first = ((long long)T + CW_WIN - 1) / CW_WIN * (2 * CW_H);
  if (job >= first) {
    const int c = lane % CW_LPR, rr = lane / CW_LPR;
    const long long t = (job - first) / CW_QC;
    const int h0 = (int)((job - first) % CW_QC) * (CW_QN * CW_RPP) + rr;
    if (t >= T) return;
    const cw_t* x = q + t * CW_XQT + (long long)h0 * CW_XQH;
    const CwTurn w = cw_turn(table, positions[t], P, c);
    cw_x8 a[CW_QN], b[CW_QN];
#pragma unroll
    for (int j = 0; j < CW_QN; ++j) {
      const int h = j * CW_RPP;
      const cw_t* at = x + (h0 + h < CW_HQ ? h : 0) * CW_XQH;
      if (h0 >= CW_HQ) at = q + t * CW_XQT;
      a[j] = *(const cw_x8*)(at + c * 8);
      if (!CW_PAIRS) b[j] = *(const cw_x8*)(at + cw_partner(c) * 8);
    }
#pragma unroll
    for (int j = 0; j < CW_QN; ++j) {
      const int h = h0 + j * CW_RPP;
      float f[8];
      cw_apply<false>(w, a[j], b[CW_PAIRS ? 0 : j], c, f);
      cw_x8 o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = (cw_t)f[i];
      if (h < CW_HQ && rr < CW_RPP) *(cw_x8*)(out + (t * CW_HQ + h) * CW_D + c * 8) = o;
    }
    return;
  }
#endif
  if (win * CW_WIN >= T) return;
  const bool values = part & 1;
  const cw_t* x = (values ? v : k) + (long long)h * (values ? CW_XVH : CW_XKH);
  unsigned char* cache = (values ? vc : kc) + (long long)h * (values ? CW_VH : CW_KH);
  float* scales = values ? vs : ks;
  const long long xt = values ? CW_XVT : CW_XKT, cp = values ? CW_VP : CW_KP, ct = values ? CW_VT : CW_KT;
  const int rr = lane / CW_LPR, c = lane % CW_LPR;
  const long long limit = pages * CW_PAGE;
  // slots of the token before the window and of those from its first one on
  const int t0 = (int)(win * CW_WIN), mine = t0 - 1 + lane;
  const long long slot = slots[mine < 0 ? 0 : mine < T ? mine : T - 1];
  const int page = mine >= 0 && mine < T && slot >= 0 && slot < limit ? (int)(slot / CW_PAGE) : -1, place = (int)(slot % CW_PAGE);
#if CW_ROT
  const int position = positions[mine < 0 ? 0 : mine < T ? mine : T - 1], partner = cw_partner(c);
#endif
  const int before = __builtin_amdgcn_update_dpp(-1, page, 0x138, 0xf, 0xf, false);        // wave_shr 1
  unsigned long long todo = __ballot(lane >= 1 && lane <= CW_WIN && page >= 0 && page != before);        // the tokens that lead
  while (todo) {
    const int l = __builtin_ctzll(todo), t = t0 - 1 + l;
    todo &= todo - 1;
    const int p = __builtin_amdgcn_readlane(page, l), kept = __builtin_amdgcn_readlane(place, l);        // rows of the page that stay
    const unsigned long long same = __ballot(page == p) >> l;
    int run = __builtin_ctzll(~same);                        // tokens of this page (l is 1 or more)
    if (l + run == 64) {
      for (;;) {
        const int u = t + run + lane;
        const long long s = slots[u < T ? u : T - 1];
        const unsigned long long more = __ballot(u < T && s >= 0 && s < limit && s / CW_PAGE == p);
        const int n = more == ~0ULL ? 64 : __builtin_ctzll(~more);
        run += n;
        if (n < 64 || run >= CW_PAGE) break;
      }
    }
    run = run < CW_PAGE ? run : CW_PAGE;
    // magnitude
    const cw_t* rows = x + t * xt + c * 8;
    const float there = scales[(long long)p * CW_H + h];
    float top = 0.0f;
#if CW_ROT
    float held[CW_HOLD][8];
    cw_x8 raws[CW_HOLD], others[CW_HOLD];
    CwTurn turns[CW_HOLD];
#pragma unroll
    for (int j = 0; j < CW_HOLD; ++j) {
      const int r = j * CW_RPP + rr, u = r < run ? r : run - 1;
      raws[j] = *(const cw_x8*)(rows + u * xt);
      if (!values) {
        others[j] = *(const cw_x8*)(rows + u * xt + (partner - c) * 8);
        turns[j] = cw_turn(table, __builtin_amdgcn_ds_bpermute((l + u) * 4, position), P, c);
      }
    }
#pragma unroll
    for (int j = 0; j < CW_HOLD; ++j)
      if (values) {
#pragma unroll
        for (int i = 0; i < 8; ++i) held[j][i] = (float)raws[j][i];
      } else if (j == 0 || j * CW_RPP < run) {
        cw_apply<true>(turns[j], raws[j], others[j], c, held[j]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) held[j][i] = 0.0f;
      }
    // a row that registers do not hold
    auto again = [&](int r, float (&f)[8]) {
      const cw_x8 raw = *(const cw_x8*)(rows + r * xt);
      if (values) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)raw[i];
      } else {
        cw_apply<true>(cw_turn(table, positions[t + r], P, c), raw, *(const cw_x8*)(rows + r * xt + (partner - c) * 8), c, f);
      }
    };
#else
    cw_x8 held[CW_HOLD];
#pragma unroll
    for (int j = 0; j < CW_HOLD; ++j) {
      const int r = j * CW_RPP + rr;
      held[j] = *(const cw_x8*)(rows + (r < run ? r : run - 1) * xt);
    }
    auto again = [&](int r, cw_x8& raw) { raw = *(const cw_x8*)(rows + r * xt); };
#endif
#pragma unroll
    for (int j = 0; j < CW_HOLD; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, cw_finite(__builtin_fabsf((float)held[j][i])));
    for (int r = CW_HOLD * CW_RPP + rr; CW_HOLD < CW_ALL && r < run && rr < CW_RPP; r += CW_RPP) {
      CW_ROW raw;
      again(r, raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, cw_finite(__builtin_fabsf((float)raw[i])));
    }
    top = cw_max(top);
    const unsigned bits = __builtin_bit_cast(unsigned, top);
    int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);       // 448 = 1.75 * 2^8
    e = e < -126 ? -126 : e;
    const float need = top > 0.0f ? __builtin_bit_cast(float, (unsigned)(e + 127) << 23) : 0.0f;
    const float old = kept ? there : 0.0f;
    const float scale = fmaxf(old, need);
    unsigned char* base = cache + p * cp;
    if (kept && scale != old) {
      const float ratio = old / scale;
      for (int r = rr; r < kept; r += CW_RPP) {
        if (rr >= CW_RPP) break;
        kcg_u32x2* at = (kcg_u32x2*)(base + r * ct + c * 8);
        const kcg_u32x2 w = *at;
        float f[8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          f[4 * j + 0] = __builtin_amdgcn_cvt_f32_fp8(w[j], 0) * ratio;
          f[4 * j + 1] = __builtin_amdgcn_cvt_f32_fp8(w[j], 1) * ratio;
          f[4 * j + 2] = __builtin_amdgcn_cvt_f32_fp8(w[j], 2) * ratio;
          f[4 * j + 3] = __builtin_amdgcn_cvt_f32_fp8(w[j], 3) * ratio;
        }
        *at = cw_encode(f);
      }
    }
    // (a scale that is no power of two can only be one that was there before)
    const bool power = (__builtin_bit_cast(unsigned, scale) & 0x7fffffu) == 0;
    const float inv = scale > 0.0f ? 1.0f / scale : 0.0f;
    auto put = [&](const CW_ROW& raw, int at) {
      float f[8];
      if (power) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)raw[i] * inv;
        if (scale == 0.0f) {         // (nothing finite but zeros)
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = raw[i] != raw[i] ? f[i] : 0.0f;
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < 8; ++i) f[i] = (float)raw[i] / scale;
      }
      *(kcg_u32x2*)(base + at * ct + c * 8) = cw_encode(f);
    };
#pragma unroll
    for (int j = 0; j < CW_HOLD; ++j) {
      if (j * CW_RPP >= run) break;
      const int r = j * CW_RPP + rr, at = __builtin_amdgcn_ds_bpermute((l + r) * 4, place);
      if (r < run && rr < CW_RPP) put(held[j], at);
    }
    for (int r = CW_HOLD * CW_RPP + rr; CW_HOLD < CW_ALL && r < run && rr < CW_RPP; r += CW_RPP) {
      CW_ROW raw;
      again(r, raw);
      put(raw, (int)(slots[t + r] % CW_PAGE));
    }
    if (lane == 0) scales[(long long)p * CW_H + h] = scale;
  }
}
