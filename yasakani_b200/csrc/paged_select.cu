// Choice of the blocks that a row attends to (sm_100a): a score for every complete page, then the highest ones.
//
// Mathematics: score(b) = max over the heads h of a kv-head's group of sum_c q_h[c] mean_b[c].  The choice is the one that fp64 sums make.  Products of two 16-bit values are
// exact there (22 bits at most), and so is a sum of 256 of them, in any order, while those that are not zero lie within a factor of 2^23 (fp16) or 2^29 (bf16, 16 bits) of one another.  Beyond that a sum
// is off by 2^-42 of the largest product at most (eight sums of a lane, five over lanes), and blocks whose scores differ by less than 2^-41 of it stand in the order that exact_key's sums give them: four to eight channels a
// lane in turn, then lanes 16, 8, 4, 2 and 1 apart.  Equal mean keys have equal scores always.  fp64 sums of everything
// were fp64-bound, though (16 rows of 7 heads over 65,536 tokens: 28 us for 15 MB of mean keys).  So:
//   1. scores on the tensor cores: exact products, fp32 sums, off by at most e = HD 2^-21 * max over blocks and heads of sum_c |q_h[c] mean_b[c]|, which a second
//      product yields (HD / 16 instructions of 16 products and a sum each, truncated at 2^-23 of the largest: (17/16) HD 2^-23 of that sum; a factor of about four is margin);
//   2. with t the (take - 1)-th highest of them: what is above t + 2e is among the chosen, what is below t - 2e is not, for at least take - 1 exact scores are
//      t - e or more, and at most take - 2 are above t + e; what lies between, a block or two, is scored in fp64.
// Where a score or e is not finite everything is scored in fp64, as are scores that are all equal: by one thread block a (row, kv-head), 198 us for 2,048 blocks of eight heads of 128 channels
// and 1.66 ms for 16,383, in place of 13 and 17.
//
// Bound: the mean keys, 2 HD bytes a page and kv-head, read once per row; in practice latency: from one launch to the next a chain of five dependent reads (position, table,
// means; scores, page) and six block-wide steps.  2,048 blocks of one row: scores 3.7 us, choice 7 us (with fp64 scores of all blocks and a choice by 8-bit digits: 31 and 14 us for
// 16 rows over 65,536 tokens in place of 5.4 and 8).
#include "paged_common.cuh"

namespace kv4 {
namespace paged {
namespace {

typedef unsigned long long u64;

struct SelectP {
  Rows R; int rows, g, nh;
  const uint16_t* q; long long qs; const uint16_t* kmean;
  float2* approx; u64* exact;                // [row][kv-head][block]: score and sum of |q mean| (negative: no page); fp64 score as a sortable key, where it is needed
  int take; int* ids;
  int scored;                                // the launch in front of the choice is the scores'
};

// A warp takes sixteen blocks.  The contraction's order is free, so lane (g, j) reads channels 64 s + 16 j .. + 15 of its two blocks and of its head as they lie, 32 bytes
// at a time, and takes two pairs of them for each of four instructions.
constexpr int SCORE_WARPS = 4;
template <int HD, bool BF, int NT>
__global__ void __launch_bounds__(SCORE_WARPS * 32) paged_score_kernel(const SelectP P) {
  constexpr int S = HD / 64;
  pdl_wait();
  pdl_launch();
  const int row = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 31, g8 = lane >> 2, j = lane & 3;
  const int b0 = ((int)blockIdx.x * SCORE_WARPS + (int)(threadIdx.x >> 5)) * 16;
  uint4 q[NT][S][2];
  #pragma unroll
  for (int n = 0; n < NT; ++n) {
    const uint4* src = reinterpret_cast<const uint4*>(P.q + row * P.qs + (size_t)(h * P.g + min(8 * n + g8, P.g - 1)) * HD + 16 * j);
    #pragma unroll
    for (int s = 0; s < S; ++s) { q[n][s][0] = src[8 * s]; q[n][s][1] = src[8 * s + 1]; }
  }
  const Place w = place_of(P.R, row);
  const int n_cand = w.seq >= 0 && w.vis > 0 ? (w.vis - 1) >> P.R.lp : 0;          // candidates: blocks in front of the last
  if (b0 >= n_cand) return;
  const int mine = b0 + (lane & 15) < n_cand ? page_of(P.R, w.seq, b0 + (lane & 15)) : -1;
  uint4 a[2][S][2];
  #pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int page = max(0, __shfl_sync(0xffffffffu, mine, g8 + 8 * r));           // no page: any, the result is not used
    const uint4* src = reinterpret_cast<const uint4*>(P.kmean + ((size_t)page * P.R.kvh + h) * HD + 16 * j);
    #pragma unroll
    for (int s = 0; s < S; ++s) { a[r][s][0] = src[8 * s]; a[r][s][1] = src[8 * s + 1]; }
  }
  float c[NT][4], m[NT][4];                  // scores; sums of the products' magnitudes
  #pragma unroll
  for (int n = 0; n < NT; ++n)
    #pragma unroll
    for (int e = 0; e < 4; ++e) c[n][e] = m[n][e] = 0.f;
  constexpr uint32_t ABS = 0x7fff7fffu;
  #pragma unroll
  for (int s = 0; s < S; ++s)
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t x[4] = {a[0][s][i].x, a[0][s][i].y, a[0][s][i].z, a[0][s][i].w}, y[4] = {a[1][s][i].x, a[1][s][i].y, a[1][s][i].z, a[1][s][i].w};
      #pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 b = q[n][s][i];
        mma<BF>(c[n], x[0], y[0], x[1], y[1], b.x, b.y);
        mma<BF>(m[n], x[0] & ABS, y[0] & ABS, x[1] & ABS, y[1] & ABS, b.x & ABS, b.y & ABS);
        mma<BF>(c[n], x[2], y[2], x[3], y[3], b.z, b.w);
        mma<BF>(m[n], x[2] & ABS, y[2] & ABS, x[3] & ABS, y[3] & ABS, b.z & ABS, b.w & ABS);
      }
    }
  #pragma unroll
  for (int r = 0; r < 2; ++r) {
    float best = -INFINITY, mag = 0.f;       // mag: infinity where a head's sum is no number, or beyond fp32 (then its magnitudes are too)
    #pragma unroll
    for (int n = 0; n < NT; ++n)
      #pragma unroll
      for (int e = 0; e < 2; ++e)
        if (8 * n + 2 * j + e < P.g) { best = fmaxf(best, c[n][2 * r + e]); mag = m[n][2 * r + e] < INFINITY ? fmaxf(mag, m[n][2 * r + e]) : INFINITY; }
    #pragma unroll
    for (int d = 1; d < 4; d <<= 1) { best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, d)); mag = fmaxf(mag, __shfl_xor_sync(0xffffffffu, mag, d)); }
    const int i = g8 + 8 * r, page = __shfl_sync(0xffffffffu, mine, i);
    if (j == 0 && b0 + i < n_cand)
      P.approx[((size_t)row * P.R.kvh + h) * P.R.blocks + b0 + i] = page < 0 ? make_float2(0.f, -1.f) : mag < INFINITY ? make_float2(best, mag) : make_float2(0.f, INFINITY);
  }
}

// Bits of a number as an unsigned integer of the same order, above 1; 1 for what is not a number.
__device__ __forceinline__ u64 key_of(double x) {
  if (x != x) return 1ull;
  const long long b = __double_as_longlong(x + 0.0);                    // -0 counts as 0
  return b < 0 ? ~(u64)b : (u64)b | 0x8000000000000000ull;
}
__device__ __forceinline__ uint32_t key_of(float x) {                  // finite; never 0
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float float_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

constexpr int CT = 512, WARPS = CT / 32, BINS = 2048, LIST = 256;
constexpr unsigned ALL = 0xffffffffu;
struct Shared {
  uint4 range[WARPS];                        // of each warp: highest and lowest key, number of keys, largest sum of magnitudes
  alignas(16) int hist[BINS];                // zero between its uses
  u64 list[LIST], hi[WARPS], lo[WARPS], cut;
  int warps[WARPS], bin, left, count, n, at[LIST];
};
static_assert(BINS == 4 * CT && WARPS == 16, "four bins a thread; half a warp looks at all warps");

// What the warps in front of this one hold, and all of them: v of every warp in sh.warps.
__device__ __forceinline__ int ahead_of(const Shared& sh, int warp, int lane) { return __reduce_add_sync(ALL, lane < warp ? sh.warps[lane & 15] : 0); }
__device__ __forceinline__ int of_all(const Shared& sh, int lane) { return __reduce_add_sync(ALL, lane < WARPS ? sh.warps[lane & 15] : 0); }
__device__ __forceinline__ int upto_lane(int v, int lane) {             // sum of the lanes up to this one
  #pragma unroll
  for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(ALL, v, d); if (lane >= d) v += o; }
  return v;
}

// The bin that holds the `left`-th highest of the keys counted in sh.hist (zero again behind it), and how many of its keys are among the first `left`.
__device__ __forceinline__ int border_bin(Shared& sh, int& left) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __syncthreads();
  int4* h4 = reinterpret_cast<int4*>(sh.hist) + (BINS / 4 - 1 - tid);   // thread t: bins BINS - 1 - 4t and the three below
  const int4 c = *h4;
  *h4 = make_int4(0, 0, 0, 0);
  const int c4[4] = {c.w, c.z, c.y, c.x}, mine = c.x + c.y + c.z + c.w, upto = upto_lane(mine, lane);
  if (lane == 31) sh.warps[warp] = upto;
  __syncthreads();
  int above = ahead_of(sh, warp, lane) + upto - mine;
  #pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (above < left && above + c4[e] >= left) { sh.bin = BINS - 1 - 4 * tid - e; sh.left = left - above; sh.count = c4[e]; }
    above += c4[e];
  }
  __syncthreads();
  left = sh.left;
  return sh.bin;
}

// The `left`-th highest of the n 64-bit keys (0: no key), and in `left` how many keys of its height are among the first `left`; all keys: 0.  The keys' range is cut into
// 2,048 bins at a time, from the highest bit in which they differ on.
__device__ u64 border(Shared& sh, const u64* keys, int n, int& left) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  u64 hi = 0, lo = ~0ull;
  int count = 0;
  for (int i = tid; i < n; i += CT) { const u64 k = keys[i]; if (k) { hi = k > hi ? k : hi; lo = k < lo ? k : lo; ++count; } }
  #pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const u64 a = __shfl_xor_sync(ALL, hi, d), b = __shfl_xor_sync(ALL, lo, d);
    hi = a > hi ? a : hi; lo = b < lo ? b : lo;
  }
  count = __reduce_add_sync(ALL, count);
  if (lane == 0) { sh.hi[warp] = hi; sh.lo[warp] = lo; sh.warps[warp] = count; }
  __syncthreads();
  for (int i = 0; i < WARPS; ++i) { hi = sh.hi[i] > hi ? sh.hi[i] : hi; lo = sh.lo[i] < lo ? sh.lo[i] : lo; }
  count = of_all(sh, lane);
  __syncthreads();
  if (count <= left) return 0;
  int top = hi == lo ? 0 : 64 - __clzll((long long)(hi ^ lo));          // the keys that are still looked at have `fixed` from bit `top` on
  u64 fixed = top < 64 ? hi >> top : 0ull;
  while (top > 0) {
    const int shift = max(0, top - 11);
    for (int i = tid; i < n; i += CT) {
      const u64 k = keys[i];
      if (k && (top < 64 ? k >> top : 0ull) == fixed) atomicAdd(&sh.hist[(int)(k >> shift) & ((1 << (top - shift)) - 1)], 1);
    }
    fixed = fixed << (top - shift) | (u64)border_bin(sh, left);
    top = shift;
  }
  return fixed;
}

// fp64 score of block b as a key, by one warp; 0 without a page.  Eight heads at a time, whose sums are folded over the warp together: at each step a lane gives
// away half of what it holds.
template <int HD, bool BF> __device__ u64 exact_key(const SelectP& P, const Place& w, int row, int h, int b, int lane) {
  constexpr int C = HD / 32, GP = 8;
  const int page = page_of(P.R, w.seq, b);
  if (page < 0) return 0ull;
  const uint32_t* src = reinterpret_cast<const uint32_t*>(P.kmean + ((size_t)page * P.R.kvh + h) * HD + C * lane);
  uint32_t u[C / 2];
  #pragma unroll
  for (int e = 0; e < C / 2; ++e) u[e] = src[e];
  u64 best = 1ull;
  for (int g0 = 0; g0 < P.g; g0 += GP) {
    double s[GP];
    #pragma unroll
    for (int i = 0; i < GP; ++i) {
      const uint32_t* qp = reinterpret_cast<const uint32_t*>(P.q + row * P.qs + (size_t)(h * P.g + min(g0 + i, P.g - 1)) * HD + C * lane);
      s[i] = 0.0;
      #pragma unroll
      for (int e = 0; e < C / 2; ++e) {
        const float2 x = unpack16<BF>(u[e]), y = unpack16<BF>(qp[e]);
        s[i] = fma((double)x.x, (double)y.x, s[i]); s[i] = fma((double)x.y, (double)y.y, s[i]);
      }
    }
    #pragma unroll
    for (int d = 16, c = GP / 2; c >= 1; d >>= 1, c >>= 1) {            // 8 -> 4 -> 2 -> 1 sums a lane
      const bool up = (lane & d) != 0;
      #pragma unroll
      for (int i = 0; i < GP / 2; ++i)
        if (i < c) { const double give = up ? s[i] : s[i + c], keep = up ? s[i + c] : s[i]; s[i] = keep + __shfl_xor_sync(ALL, give, d); }
    }
    double t = s[0];                                                    // head g0 + lane / 4, repeated heads among them
    t += __shfl_xor_sync(ALL, t, 2);
    t += __shfl_xor_sync(ALL, t, 1);
    const u64 k = key_of(t);
    best = k > best ? k : best;
  }
  #pragma unroll
  for (int d = 16; d >= 4; d >>= 1) { const u64 o = __shfl_xor_sync(ALL, best, d); best = o > best ? o : best; }
  return best;
}

// The choice, a thread block a (row, kv-head).  PER blocks a thread stay in registers: 8, or 32 where a table has more than 4,096 (16,383 blocks of one row read again for each walk: with
// scores and attention 44.5 us, kept 30.5; 32 of 256 channels in bf16 leave 96 bytes of a thread outside its registers).
template <int HD, bool BF, int PER>
__global__ void __launch_bounds__(CT, 1) paged_choose_kernel(const SelectP P) {
  __shared__ Shared sh;
  const int row = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // Ahead of the wait, where the scores are: their kernel lets this one start when all of its blocks have seen what lies in front of them finished
  Place w{-1, 0};
  if (P.scored) w = place_of<true>(P.R, row);
  pdl_wait();
  pdl_launch();
  if (!P.scored) w = place_of(P.R, row);
  const size_t pair = (size_t)row * P.R.kvh + h;
  const float2* approx = P.approx + pair * P.R.blocks;
  u64* exact = P.exact + pair * P.R.blocks;
  int* ids = P.ids + pair * P.take;
  // A warp has 32 PER blocks in a row, x[e] of a lane is the block at 32 e + lane of them: loads of whole lines, and an order that ballots keep.  Up to PER * CT blocks are
  // read once (few of them beside the row's place), and stay; more are read again for each walk.
  float2 x[PER];
  const int mine0 = warp * (32 * PER) + lane;
  const unsigned below = (1u << lane) - 1u;
  auto read = [&](int i0, int end) {
    #pragma unroll
    for (int e = 0; e < PER; ++e) { const int i = i0 + mine0 + 32 * e; x[e] = i < end ? approx[i] : make_float2(0.f, -1.f); }
  };
  if (PER == 8) read(0, P.R.blocks - 1);
  reinterpret_cast<int4*>(sh.hist)[tid] = make_int4(0, 0, 0, 0);
  if (tid == 0) sh.n = 0;
  if (w.seq < 0) return;
  const int last = w.vis > 0 ? (w.vis - 1) >> P.R.lp : -1, n = last > 0 ? last : 0;
  if (PER == 8) {
    #pragma unroll
    for (int e = 0; e < PER; ++e) if (mine0 + 32 * e >= n) x[e] = make_float2(0.f, -1.f);     // behind the candidates nothing has been written
  } else read(0, n);                                                    // a wide table may be of short rows: not ahead of the place
  auto each = [&](auto f) {
    for (int i0 = 0; i0 < n; i0 += PER * CT) {
      if (n > PER * CT) read(i0, n);
      #pragma unroll
      for (int e = 0; e < PER; ++e) f(i0 + mine0 + 32 * e, x[e]);
    }
  };
  // ---- the scores' range, the largest sum of magnitudes
  uint32_t khi = 0, klo = ALL, big = 0;
  int count = 0;
  each([&](int, const float2& f) {
    if (f.y >= 0.f) {
      const uint32_t k = key_of(f.x);
      khi = max(khi, k); klo = min(klo, k); ++count;
      big = max(big, __float_as_uint(f.y));                             // not negative: sorts like its bits
    }
  });
  khi = __reduce_max_sync(ALL, khi); klo = __reduce_min_sync(ALL, klo); count = __reduce_add_sync(ALL, count); big = __reduce_max_sync(ALL, big);
  if (lane == 0) sh.range[warp] = make_uint4(khi, klo, (uint32_t)count, big);
  __syncthreads();
  const uint4 r = sh.range[lane & 15];
  khi = __reduce_max_sync(ALL, r.x); klo = __reduce_min_sync(ALL, r.y); big = __reduce_max_sync(ALL, r.w);
  count = __reduce_add_sync(ALL, lane < WARPS ? (int)r.z : 0);
  // the sum of magnitudes is itself rounded; products below fp32's range (bf16) may count as zero
  const double e2 = 2.0 * ((HD * 0x1p-21) * 1.01 * (double)__uint_as_float(big) + HD * 0x1p-120);
  const bool wild = !(e2 < (double)INFINITY), all = count <= P.take - 1;                     // all: no more candidates than places

  // ---- the bin that holds the border, and what may be on either side of it
  float lo = -INFINITY, hi = INFINITY;                                  // scored in fp64: what is neither above hi nor below lo (rounded outwards)
  if (!wild && !all) {
    const float flo = float_of(klo), fhi = float_of(khi), scale = (float)BINS / (fhi - flo);
    lo = __double2float_rd((double)flo - e2); hi = __double2float_ru((double)fhi + e2);
    if (fhi - flo < INFINITY && scale < INFINITY) {                     // else all are unsure: scores that are as good as equal, or a range beyond fp32
      each([&](int, const float2& f) { if (f.y >= 0.f) atomicAdd(&sh.hist[min(BINS - 1, (int)((f.x - flo) * scale))], 1); });
      int left = P.take - 1;
      const double bin = (double)border_bin(sh, left), step = 1.0 / (double)scale;
      // a score's bin is rounded by less than 2^-9 of a bin
      lo = __double2float_rd(fmax((double)flo, (double)flo + (bin - 0.01) * step) - e2);
      hi = __double2float_ru(fmin((double)fhi, (double)flo + (bin + 1.01) * step) + e2);
    }
  }
  auto unsure = [&](const float2& f) { return f.y >= 0.f && !(f.x > hi) && !(f.x < lo); };
  // ---- how many are chosen for sure, how many are unsure, and which those are
  int sure = 0, many = 0;
  if (!all) {
    if (n <= PER * CT) {                                                // one walk: places are known with the counts
      int mine = 0;                                                     // sure ones, and unsure ones << 16
      #pragma unroll
      for (int e = 0; e < PER; ++e) if (x[e].y >= 0.f && !(x[e].x < lo)) mine += x[e].x > hi ? 1 : 1 << 16;
      mine = __reduce_add_sync(ALL, mine);
      if (lane == 0) sh.warps[warp] = mine;
      __syncthreads();
      const int before = ahead_of(sh, warp, lane), total = of_all(sh, lane);
      sure = total & 0xffff; many = total >> 16;
      if (many <= P.take - 1 - sure) {                                  // the unsure ones are all chosen, as mostly: the border itself and nothing else
        int at = (before & 0xffff) + (before >> 16);
        #pragma unroll
        for (int e = 0; e < PER; ++e) {
          const bool t = x[e].y >= 0.f && !(x[e].x < lo);
          const unsigned b = __ballot_sync(ALL, t);
          if (b == 0) continue;
          if (t) ids[at + __popc(b & below)] = mine0 + 32 * e;
          at += __popc(b);
        }
        if (tid == 0) ids[sure + many] = last;
        for (int i = sure + many + 1 + tid; i < P.take; i += CT) ids[i] = -1;
        return;
      }
    }
    int s2 = 0;                                                         // more blocks than 16 bits count, or a choice to be made among the unsure ones: which they are
    __syncthreads();
    each([&](int i, const float2& f) {
      if (unsure(f)) { const int at = atomicAdd(&sh.n, 1); if (at < LIST) sh.at[at] = i; }
      else if (f.y >= 0.f && f.x > hi) ++s2;
    });
    s2 = __reduce_add_sync(ALL, s2);
    if (lane == 0) sh.warps[warp] = s2;
    __syncthreads();
    sure = of_all(sh, lane);
    many = sh.n;
  }
  int left = P.take - 1 - sure;                                         // places for the unsure ones
  u64 cut = 0;                                                          // of these: above `cut`, and the first `left` equal to it
  const bool need = !all && many > left, listed = need && many <= LIST && n <= 32 * BINS;
  if (listed) {
    for (int i = warp; i < many; i += WARPS) { const u64 k = exact_key<HD, BF>(P, w, row, h, sh.at[i], lane); if (lane == 0) sh.list[i] = k; }
    __syncthreads();
    if (tid < many) {                                                   // how many come before this one: the higher, and of equal ones the lower blocks
      const u64 k = sh.list[tid];
      const int at = sh.at[tid];
      int before = 0;
      for (int i = 0; i < many; ++i) before += sh.list[i] > k || (sh.list[i] == k && sh.at[i] < at);
      if (before < left) atomicOr(&sh.hist[at >> 5], 1 << (at & 31));   // a bit for each block
    }
  } else if (need) {
    for (int i = warp; i < n; i += WARPS) {
      u64 k = 0;
      if (unsure(approx[i])) k = exact_key<HD, BF>(P, w, row, h, i, lane);
      if (lane == 0) exact[i] = k;
    }
    __syncthreads();
    cut = border(sh, exact, n, left);
  }
  __syncthreads();
  // ---- one walk in rising order
  int at = 0, equal = 0;                                                // taken so far; keys equal to the border so far
  for (int i0 = 0; i0 < n; i0 += PER * CT) {
    if (n > PER * CT) read(i0, n);
    uint32_t taken = 0, same = 0;                                       // bit e: x[e] is taken; is equal to the border
    int mine = 0;                                                       // of the warp: taken ones, and equal ones << 16
    #pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int i = i0 + mine0 + 32 * e;
      const float2 f = x[e];
      bool t = false, q = false;
      if (f.y >= 0.f) {
        if (all || f.x > hi) t = true;
        else if (unsure(f)) {
          if (!need) t = true;
          else if (listed) t = (sh.hist[i >> 5] >> (i & 31)) & 1;
          else { const u64 k = exact[i]; t = k > cut; q = k && k == cut; }
        }
      }
      taken |= (uint32_t)t << e; same |= (uint32_t)q << e;
      mine += __popc(__ballot_sync(ALL, t)) + (__popc(__ballot_sync(ALL, q)) << 16);
    }
    if (lane == 0) sh.warps[warp] = mine;
    __syncthreads();
    const int ahead = ahead_of(sh, warp, lane), total = of_all(sh, lane);
    int e0 = equal + (ahead >> 16), place = at + (ahead & 0xffff) + min(e0, left) - min(equal, left);
    #pragma unroll
    for (int e = 0; e < PER; ++e) {
      const bool q = (same >> e) & 1;
      const unsigned bq = __ballot_sync(ALL, q);
      const bool t = ((taken >> e) & 1) || (q && e0 + __popc(bq & below) < left);
      const unsigned bt = __ballot_sync(ALL, t);
      if (t) ids[place + __popc(bt & below)] = i0 + mine0 + 32 * e;
      place += __popc(bt); e0 += __popc(bq);
    }
    at += (total & 0xffff) + min(equal + (total >> 16), left) - min(equal, left);
    equal += total >> 16;
    if (i0 + PER * CT < n) __syncthreads();
  }
  if (tid == 0 && last >= 0) ids[at] = last;
  if (last >= 0) ++at;
  for (int i = at + tid; i < P.take; i += CT) ids[i] = -1;
}

template <int HD, bool BF> int launch(const SelectP& P, cudaStream_t st) {
  if (P.R.blocks > 1) {
    auto score = P.g <= 8 ? paged_score_kernel<HD, BF, 1> : paged_score_kernel<HD, BF, 2>;
    constexpr int per = 16 * SCORE_WARPS;
    if (int rc = launch_pdl("paged_score_kernel", score, dim3((unsigned)((P.R.blocks - 1 + per - 1) / per), (unsigned)P.R.kvh, (unsigned)P.rows), SCORE_WARPS * 32, 0, st, P))
      return rc;
  }
  auto choose = P.R.blocks <= 8 * CT ? paged_choose_kernel<HD, BF, 8> : paged_choose_kernel<HD, BF, 32>;
  return launch_pdl("paged_choose_kernel", choose, dim3((unsigned)P.R.kvh, (unsigned)P.rows), CT, 0, st, P);
}

}  // namespace
}  // namespace paged

size_t paged_select_bytes(const yskn_paged_cache& c, int rows, int blocks) { return (size_t)rows * c.kvh * blocks * 16; }

int launch_paged_select(const yskn_paged_cache& c, const yskn_paged_rows& r, const yskn_paged_select_args& a, cudaStream_t st) {
  using namespace paged;
  const size_t n = (size_t)r.rows * c.kvh * r.blocks;
  SelectP P{rows_of(c, r, 0), r.rows, a.nh / c.kvh, a.nh, static_cast<const uint16_t*>(a.q), (long long)a.q_stride, static_cast<const uint16_t*>(c.kmean),
            static_cast<float2*>(a.workspace), reinterpret_cast<u64*>(static_cast<float2*>(a.workspace) + n), a.take, a.ids, r.blocks > 1 ? 1 : 0};
  const bool bf = c.dtype == YSKN_KV4_BF16;
  return c.hd == 256 ? (bf ? launch<256, true>(P, st) : launch<256, false>(P, st)) : (bf ? launch<128, true>(P, st) : launch<128, false>(P, st));
}

}  // namespace kv4
