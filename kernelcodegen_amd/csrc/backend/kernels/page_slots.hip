// ---- page tables and slots of one step's tokens ----
//   before_b = ceil(length_b / page), after_b = ceil((length_b + added_b) / page); request b takes after_b - before_b pages off the list
//   of free ones, those of earlier requests first, and its table is continued with them; its new tokens get the positions from
//   length_b on and the slots table[position / page] * page + position % page (-1 where there is no page)
// Every workgroup takes the prefix sums of all requests (PS_BLOCK at a time) and then its share of the pages and tokens, each found in the
// sums in LDS: a step of any shape is one launch.  Bound by what waits for one another: the lengths, the sums, the table or the
// list, the stores.
// Measured: 64 requests of one token each 2.8 us (an empty launch 1.7), 200 of up to 700 8.
// Lengths, places and sums are counted without a sign, so that length + added may use all bits of a positive number, and a place is compared
// with its table without one: sums that pass 32 bits give wrong slots, but no access out of range.
// Parameters: PS_NAME, PS_BLOCK, PS_PAGE.
struct PsSums { unsigned pages[PS_BLOCK + 1], tokens[PS_BLOCK + 1], lengths[PS_BLOCK], waves[2][PS_BLOCK / 64]; };

__device__ __forceinline__ unsigned ps_pages(unsigned tokens) { return tokens / PS_PAGE + (tokens % PS_PAGE ? 1 : 0); }

// Sum over the lanes up to and including this one.
__device__ __forceinline__ int ps_scan(int v) {
#define PS_DPP(control, rows) v += __builtin_amdgcn_update_dpp(0, v, control, rows, 0xf, false)
  PS_DPP(0x111, 0xf);        // row_shr 1, 2, 4, 8: over the 16 lanes of a row
  PS_DPP(0x112, 0xf);
  PS_DPP(0x114, 0xf);
  PS_DPP(0x118, 0xf);
  PS_DPP(0x142, 0xa);        // a row's last lane into the next row, for the second and the fourth,
  PS_DPP(0x143, 0xc);        // the second row's into the third and the fourth
#undef PS_DPP
  return v;
}

extern "C" __global__ __launch_bounds__(PS_BLOCK)
void PS_NAME(const int* __restrict__ lengths, const int* __restrict__ added, int* __restrict__ table, const int* __restrict__ free_pages,
             long long B_, long long T_, long long W_, long long table_row, long long F_, long long* __restrict__ slots,
             int* __restrict__ positions, int* __restrict__ starts, int* __restrict__ lengths_out, int* __restrict__ used) {
  __shared__ PsSums s;
  const int B = (int)B_;
  const unsigned T = (unsigned)T_, W = (unsigned)W_, F = F_ < 0x7fffffff ? (unsigned)F_ : 0x7fffffffu;
  constexpr unsigned page = PS_PAGE;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned first = blockIdx.x * PS_BLOCK + threadIdx.x, step = gridDim.x * PS_BLOCK;
  unsigned pages0 = 0, tokens0 = 0;            // of the requests before this round's
  for (int b0 = 0; b0 < B; b0 += PS_BLOCK) {
    const int b = b0 + threadIdx.x, n = B - b0 < PS_BLOCK ? B - b0 : PS_BLOCK;
    unsigned len = 0, add = 0;
    if (b < B) {
      len = lengths[b] > 0 ? lengths[b] : 0;
      add = added[b] > 0 ? added[b] : 0;
    }
    const unsigned p = ps_scan(ps_pages(len + add) - ps_pages(len)), t = ps_scan(add);
    if (lane == 63) { s.waves[0][wave] = p; s.waves[1][wave] = t; }
    __syncthreads();
    unsigned pb = 0, tb = 0;
#pragma unroll
    for (int w = 0; w < PS_BLOCK / 64 - 1; ++w) {
      const unsigned pw = s.waves[0][w], tw = s.waves[1][w];
      pb += w < wave ? pw : 0;
      tb += w < wave ? tw : 0;
    }
    s.lengths[threadIdx.x] = len;
    s.pages[threadIdx.x + 1] = pb + p;
    s.tokens[threadIdx.x + 1] = tb + t;
    if (threadIdx.x == 0) s.pages[0] = s.tokens[0] = 0;
    __syncthreads();
    if (blockIdx.x == 0 && b < B) {
      starts[b + 1] = tokens0 + s.tokens[threadIdx.x + 1];
      lengths_out[b] = len + add;
    }
    // Which request of this round: the last whose sum before it is not over `i`.  Of eight parts at a time, since the reads of one step are
    // under way together: a round of 256 takes three.
    auto find = [&](const unsigned* sums, unsigned i) {
      int lo = 0;
#pragma unroll
      for (int part = PS_BLOCK > 512 ? 512 : 64; part > 0; part /= 8) {
        const int from = lo;
#pragma unroll
        for (int j = 1; j < 8 && j * part < PS_BLOCK; ++j) {
          const int at = from + j * part;
          lo = sums[at < n ? at : n] <= i && at < n ? at : lo;
        }
      }
      return lo;
    };
    // page i off the list and token i: both numbers' loads, from some length where there is none, then the stores
    const unsigned pages = s.pages[n], tokens = s.tokens[n];
    const unsigned freed = pages0 < F ? F - pages0 : 0, rows = tokens0 < T ? T - tokens0 : 0;        // what there is room for (below 2^31)
    const unsigned some = pages < freed ? pages : freed, rest = tokens < rows ? tokens : rows, most = some > rest ? some : rest;
    for (unsigned i = first; i < most; i += step) {
      const int rp = find(s.pages, i);
      const unsigned place = ps_pages(s.lengths[rp]) + i - s.pages[rp];
      const bool put = i < some && place < W;
      const int fresh = *(put ? free_pages + pages0 + i : lengths);
      const int r = find(s.tokens, i);
      const unsigned have = s.lengths[r], at = have + i - s.tokens[r], before = ps_pages(have), column = at / page;
      const unsigned k = pages0 + s.pages[r] + column - before;
      const bool token = i < rest, old = column < before, page_there = token && column < W && (old || k < F);
      const int id = *(!page_there ? lengths : old ? table + (long long)(b0 + r) * table_row + column : free_pages + k);
      if (put) table[(long long)(b0 + rp) * table_row + place] = fresh;
      if (token) {
        slots[tokens0 + i] = !page_there || id < 0 ? -1 : (long long)id * page + (at - column * page);
        positions[tokens0 + i] = at;
      }
    }
    pages0 += pages;
    tokens0 += tokens;
    __syncthreads();
  }
  for (long long i = (long long)tokens0 + first; i < T; i += step) {
    slots[i] = -1;
    positions[i] = -1;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    starts[0] = 0;
    used[0] = pages0 < F ? pages0 : F;
  }
}
