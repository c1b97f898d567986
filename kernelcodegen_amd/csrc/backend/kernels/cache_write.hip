// ---- new keys and values into a paged cache in 8 bits ----
//   a = largest finite magnitude among the new rows of a page and head, need = the least power of two with 448 need >= a (0 for a = 0)
//   scale = need where the page begins with these rows, else max(old scale, need); what the page holds is brought to it
//   cache = e4m3(x / scale), to the nearest, ties to even; infinities become +-448, a NaN stays one
// A scale that is a power of two costs a floating format range but no precision, and a page whose scale has to grow is converted
// without loss down to the format's least numbers.
//
// A wavefront for each head, keys or values, and CW_WIN consecutive tokens.  A token whose predecessor lies in another page leads: its
// wavefront takes the tokens behind it in that page too (slots of a page stand together and ascend), so nobody else touches the
// page and head, and no atomics are needed.  A lane takes 8 elements, CW_RPP rows a pass; rows are held in registers between the two
// passes (magnitude, conversion) as far as CW_HOLD passes reach, else read again, from the caches.
// Parameters: CW_NAME, CW_H, CW_D, CW_PAGE, CW_T (input type), CW_ESIZE, CW_WIN, strides as in cache_attention: CW_KP .. CW_VH (bytes), CW_XKT
// CW_XKH CW_XVT CW_XVH (of k and v, elements).
typedef CW_T cw_t;
#define CW_LPR (CW_D / 8)            // lanes per row
#define CW_RPP (64 / CW_LPR)         // rows per pass
#define CW_HOLD 4
typedef cw_t cw_x8 __attribute__((ext_vector_type(8)));

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
  auto pageOf = [&](int t) -> long long {
    if (t < 0 || t >= T) return -1;
    const long long s = slots[t];
    return s >= 0 && s < limit ? s / CW_PAGE : -1;
  };
  auto row = [&](int t, float (&f)[8]) {
    const cw_x8 raw = *(const cw_x8*)(x + t * xt + c * 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)raw[i];
  };
  // the tokens of the window that lead
  const int t0 = (int)(win * CW_WIN);
  bool lead = false;
  if (lane < CW_WIN && t0 + lane < T) {
    const long long p = pageOf(t0 + lane);
    lead = p >= 0 && (t0 + lane == 0 || pageOf(t0 + lane - 1) != p);
  }
  unsigned long long todo = __ballot(lead);
  while (todo) {
    const int t = t0 + __builtin_ctzll(todo);
    todo &= todo - 1;
    const long long slot = slots[t], page = slot / CW_PAGE;
    const int kept = (int)(slot - page * CW_PAGE);           // rows of the page that stay
    int run = 1;                                             // tokens of this page
    for (int i = 1; i < CW_PAGE; i += 64) {
      const unsigned long long same = __ballot(i + lane < CW_PAGE && pageOf(t + i + lane) == page);
      const int n = same == ~0ULL ? 64 : __builtin_ctzll(~same);
      run += n;
      if (n < 64) break;
    }
    // magnitude
    cw_x8 held[CW_HOLD];
    float top = 0.0f;
    for (int i = 0, r = rr; i * CW_RPP < run; ++i, r += CW_RPP) {
      if (rr >= CW_RPP || r >= run) continue;
      const cw_x8 raw = *(const cw_x8*)(x + (t + r) * xt + c * 8);
#pragma unroll
      for (int j = 0; j < CW_HOLD; ++j)
        if (j == i) held[j] = raw;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, cw_finite(__builtin_fabsf((float)raw[j])));
    }
    top = kcg_wave_max(top);
    const unsigned bits = __builtin_bit_cast(unsigned, top);
    int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);       // 448 = 1.75 * 2^8
    e = e < -126 ? -126 : e;
    const float need = top > 0.0f ? __builtin_bit_cast(float, (unsigned)(e + 127) << 23) : 0.0f;
    const float old = kept ? scales[page * CW_H + h] : 0.0f;
    const float scale = fmaxf(old, need);
    unsigned char* base = cache + page * cp;
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
    for (int i = 0, r = rr; i * CW_RPP < run; ++i, r += CW_RPP) {
      if (rr >= CW_RPP || r >= run) continue;
      cw_x8 raw;
      if (i < CW_HOLD) {
#pragma unroll
        for (int j = 0; j < CW_HOLD; ++j)
          if (j == i) raw = held[j];
      } else {
        raw = *(const cw_x8*)(x + (t + r) * xt + c * 8);
      }
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = power ? (float)raw[j] * inv : (float)raw[j] / scale;
      const int at = (int)(slots[t + r] - page * CW_PAGE);
      *(kcg_u32x2*)(base + at * ct + c * 8) = cw_encode(f);
    }
    if (lane == 0) scales[page * CW_H + h] = scale;
  }
}
