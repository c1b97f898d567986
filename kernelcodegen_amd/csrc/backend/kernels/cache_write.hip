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
// Measured, 8 heads of 128: 64 tokens of a page each 2.9 us (an empty launch 1.7); 9000 tokens of whole pages, half precision, 12.5 us, 4.4 TB/s.
// Parameters: CW_NAME, CW_H, CW_D, CW_PAGE, CW_T (input type), CW_ESIZE, CW_WIN, strides as in cache_attention: CW_KP .. CW_VH (bytes), CW_XKT
// CW_XKH CW_XVT CW_XVH (of k and v, elements).
typedef CW_T cw_t;
#define CW_LPR (CW_D / 8)            // lanes per row
#define CW_RPP (64 / CW_LPR)         // rows per pass
#define CW_ALL ((CW_PAGE + CW_RPP - 1) / CW_RPP)          // passes of a whole page
#define CW_MOST (CW_ESIZE * 8 > 16 ? 4 : 8)              // that registers hold
#define CW_NEAR (48 / CW_RPP)                            // whose rows' slots the lanes have
#define CW_HOLD (CW_ALL < CW_MOST ? (CW_ALL < CW_NEAR ? CW_ALL : CW_NEAR) : CW_MOST < CW_NEAR ? CW_MOST : CW_NEAR)
typedef cw_t cw_x8 __attribute__((ext_vector_type(8)));

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

extern "C" __global__ __launch_bounds__(256)
void CW_NAME(const cw_t* __restrict__ k, const cw_t* __restrict__ v, unsigned char* __restrict__ kc, unsigned char* __restrict__ vc,
             float* __restrict__ ks, float* __restrict__ vs, const long long* __restrict__ slots, long long T_, long long pages) {
  const int T = (int)T_, lane = threadIdx.x & 63;
  const long long job = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = (int)(job % (2 * CW_H)), h = part >> 1;
  const long long win = job / (2 * CW_H);
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
    cw_x8 held[CW_HOLD];
#pragma unroll
    for (int j = 0; j < CW_HOLD; ++j) {
      const int r = j * CW_RPP + rr;
      held[j] = *(const cw_x8*)(rows + (r < run ? r : run - 1) * xt);
    }
    const float there = scales[(long long)p * CW_H + h];
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < CW_HOLD; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, cw_finite(__builtin_fabsf((float)held[j][i])));
    for (int r = CW_HOLD * CW_RPP + rr; CW_HOLD < CW_ALL && r < run && rr < CW_RPP; r += CW_RPP) {
      const cw_x8 raw = *(const cw_x8*)(rows + r * xt);
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
    auto put = [&](const cw_x8& raw, int at) {
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
    for (int r = CW_HOLD * CW_RPP + rr; CW_HOLD < CW_ALL && r < run && rr < CW_RPP; r += CW_RPP)
      put(*(const cw_x8*)(rows + r * xt), (int)(slots[t + r] % CW_PAGE));
    if (lane == 0) scales[(long long)p * CW_H + h] = scale;
  }
}
