// Choice of the blocks that a row attends to (sm_100a): a score for every complete page, then the highest ones.
//
// Mathematics: score(b) = max over the heads h of a kv-head's group of sum_c q_h[c] mean_b[c].  Products of two 16-bit values are exact in fp32, and all the more so in
// fp64, and a sum of HD of them in fp64 is exact or off by 2^-52 of its largest part: the choice does not depend on the order of the sum, and two builds, or a
// plain program, agree on every block.  fp32 sums differ by 2^-24, which decides between neighbours every few thousand rows.
//
// Bound: the mean keys, 2 HD bytes a page and kv-head, read once per row, and fp64 products beside them, which B200 does at half the rate of fp32.
// Two launches: scores as 64-bit keys that sort like the score (workspace); the choice, a block a (row, kv-head).
#include "paged_common.cuh"

namespace kv4 {
namespace paged {
namespace {

struct SelectP {
  Rows R; int rows, g, nh;
  const uint16_t* q; long long qs; const uint16_t* kmean;
  unsigned long long* keys; int take; int* ids;
};

// A number's bits as an unsigned integer of the same order; 0 for what is no candidate, 1 for a score that is not a number.
__device__ __forceinline__ unsigned long long key_of(double x) {
  if (x != x) return 1ull;
  const long long b = __double_as_longlong(x + 0.0);                    // -0 counts as 0
  return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | 0x8000000000000000ull;
}

constexpr int SCORE_WARPS = 8;
// A warp takes a block at a time, HD / 32 channels a lane; a lane keeps its channels of up to eight heads in registers (fp64; from shared memory they would be the
// bound: eight bytes a product).  The heads' sums are folded over the warp together: at each step a lane gives away half of what it holds.  Pages and
// mean keys are asked for four blocks ahead of their use.
template <int HD, bool BF>
__global__ void __launch_bounds__(SCORE_WARPS * 32) paged_score_kernel(const SelectP P, int per_warp) {
  constexpr int C = HD / 32, GP = 8, AHEAD = 4;
  pdl_wait();
  pdl_launch();
  const int row = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b0 = ((int)blockIdx.x * SCORE_WARPS + warp) * per_warp;
  const Place w = place_of(P.R, row);
  const int n = w.seq >= 0 && w.vis > 0 ? (w.vis - 1) >> P.R.lp : 0;    // candidates: blocks in front of the last
  const int b1 = min(n, b0 + per_warp);
  if (b0 >= b1) return;
  unsigned long long* keys = P.keys + ((size_t)row * P.R.kvh + h) * P.R.blocks;
  for (int g0 = 0; g0 < P.g; g0 += GP) {                                // more than eight heads: in two walks
    const int gn = min(GP, P.g - g0);
    double q[GP][C];
    #pragma unroll
    for (int i = 0; i < GP; ++i) {
      const uint16_t* src = P.q + row * P.qs + (size_t)(h * P.g + g0 + min(i, gn - 1)) * HD + C * lane;
      #pragma unroll
      for (int e = 0; e < C / 2; ++e) { const float2 f = unpack16<BF>(reinterpret_cast<const uint32_t*>(src)[e]); q[i][2 * e] = f.x; q[i][2 * e + 1] = f.y; }
    }
    for (int bb = b0; bb < b1; bb += 32) {
      const int mine = bb + lane < b1 ? page_of(P.R, w.seq, bb + lane) : -1;
      const int m = min(32, b1 - bb);
      uint32_t u[AHEAD][C / 2];
      auto ask = [&](int i, uint32_t (&x)[C / 2]) {
        const int page = __shfl_sync(0xffffffffu, mine, i & 31);
        const uint16_t* src = P.kmean + ((size_t)max(page, 0) * P.R.kvh + h) * HD + C * lane;          // no page: any, its key is overwritten
        if constexpr (C == 8) { const uint4 v = *reinterpret_cast<const uint4*>(src); x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
        else { const uint2 v = *reinterpret_cast<const uint2*>(src); x[0] = v.x; x[1] = v.y; }
      };
      #pragma unroll
      for (int i = 0; i < AHEAD; ++i) ask(i, u[i]);
      for (int i0 = 0; i0 < m; i0 += AHEAD) {
        #pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
          double x[C], s[GP];
          #pragma unroll
          for (int e = 0; e < C / 2; ++e) { const float2 f = unpack16<BF>(u[a][e]); x[2 * e] = f.x; x[2 * e + 1] = f.y; }
          ask(i0 + a + AHEAD, u[a]);
          #pragma unroll
          for (int i = 0; i < GP; ++i) {
            s[i] = 0.0;
            if (i < gn) {
              #pragma unroll
              for (int e = 0; e < C; ++e) s[i] = fma(q[i][e], x[e], s[i]);
            }
          }
          // 8 -> 4 -> 2 -> 1 sums a lane; lane bits 4, 3, 2 are then the head, and two more steps finish its sum
          #pragma unroll
          for (int d = 16, c = GP / 2; c >= 1; d >>= 1, c >>= 1) {
            const bool up = (lane & d) != 0;
            #pragma unroll
            for (int i = 0; i < GP / 2; ++i)
              if (i < c) { const double give = up ? s[i] : s[i + c], keep = up ? s[i + c] : s[i]; s[i] = keep + __shfl_xor_sync(0xffffffffu, give, d); }
          }
          double t = s[0];
          t += __shfl_xor_sync(0xffffffffu, t, 2);
          t += __shfl_xor_sync(0xffffffffu, t, 1);
          unsigned long long key = (lane >> 2) < gn ? key_of(t) : 0ull;
          #pragma unroll
          for (int d = 16; d >= 4; d >>= 1) { const unsigned long long o = __shfl_xor_sync(0xffffffffu, key, d); key = o > key ? o : key; }
          const int i = i0 + a, page = __shfl_sync(0xffffffffu, mine, i & 31);
          if (lane == 0 && i < m) {
            if (g0 > 0) { const unsigned long long o = keys[bb + i]; key = o > key ? o : key; }
            keys[bb + i] = page < 0 ? 0ull : key;
          }
        }
      }
    }
  }
}

// The choice.  The highest keys' range is cut into 2,048 bins at a time, from the highest bit in which the keys differ on: the bin that holds the last place, then, where it holds
// few keys, the place in it by counting for each how many come before it; otherwise its bins in turn.  Keys of equal height are taken from the lowest block on.
// Then one walk writes the chosen blocks in rising order.
constexpr int CT = 512, BINS = 2048, LIST = 256;
__global__ void __launch_bounds__(CT) paged_choose_kernel(const SelectP P) {
  __shared__ unsigned long long s_hi[CT / 32], s_lo[CT / 32], list[LIST], s_cut;
  __shared__ int hist[BINS], warps[CT / 32], s_bin, s_left, s_count, s_n;
  pdl_wait();
  pdl_launch();
  const int row = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Place w = place_of(P.R, row);
  if (w.seq < 0) return;
  const size_t pair = (size_t)row * P.R.kvh + h;
  const unsigned long long* keys = P.keys + pair * P.R.blocks;
  int* ids = P.ids + pair * P.take;
  const int last = w.vis > 0 ? (w.vis - 1) >> P.R.lp : -1, n = last > 0 ? last : 0;

  // ---- highest and lowest candidate, and how many there are
  unsigned long long hi = 0, lo = ~0ull;
  int count = 0;
  #pragma unroll 4
  for (int i = tid; i < n; i += CT) { const unsigned long long k = keys[i]; if (k) { hi = k > hi ? k : hi; lo = k < lo ? k : lo; ++count; } }
  #pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const unsigned long long a = __shfl_xor_sync(0xffffffffu, hi, d), b = __shfl_xor_sync(0xffffffffu, lo, d);
    hi = a > hi ? a : hi; lo = b < lo ? b : lo; count += __shfl_xor_sync(0xffffffffu, count, d);
  }
  if (lane == 0) { s_hi[warp] = hi; s_lo[warp] = lo; warps[warp] = count; }
  __syncthreads();
  count = 0;
  #pragma unroll
  for (int i = 0; i < CT / 32; ++i) { hi = s_hi[i] > hi ? s_hi[i] : hi; lo = s_lo[i] < lo ? s_lo[i] : lo; count += warps[i]; }
  __syncthreads();

  // ---- the border: keys above `cut` are taken, and of those equal to it the first `left`
  unsigned long long cut = 0;
  int left = P.take - 1;
  if (count > left && hi == lo) cut = hi;                               // all alike
  else if (count > left) {
    int top = 64 - __clzll((long long)(hi ^ lo));                       // the keys that are still looked at have `fixed` from bit `top` on
    unsigned long long fixed = top < 64 ? hi >> top : 0ull;
    auto looked = [&](unsigned long long k) { return k && (top < 64 ? k >> top : 0ull) == fixed; };
    for (;;) {
      const int shift = max(0, top - 11);
      for (int i = tid; i < BINS; i += CT) hist[i] = 0;
      if (tid == 0) s_n = 0;
      __syncthreads();
      for (int i = tid; i < n; i += CT) {
        const unsigned long long k = keys[i];
        if (looked(k)) atomicAdd(&hist[(int)(k >> shift) & ((1 << (top - shift)) - 1)], 1);
      }
      __syncthreads();
      // thread t has bins BINS - 1 - 4t and the three below: how many keys lie above them
      int c4[4], mine = 0;
      #pragma unroll
      for (int e = 0; e < 4; ++e) { c4[e] = hist[BINS - 1 - 4 * tid - e]; mine += c4[e]; }
      int upto = mine;
      #pragma unroll
      for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(0xffffffffu, upto, d); if (lane >= d) upto += o; }
      if (lane == 31) warps[warp] = upto;
      __syncthreads();
      for (int i = 0; i < warp; ++i) upto += warps[i];
      int above = upto - mine;
      #pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (above < left && above + c4[e] >= left) { s_bin = BINS - 1 - 4 * tid - e; s_left = left - above; s_count = c4[e]; }
        above += c4[e];
      }
      __syncthreads();
      left = s_left;
      fixed = fixed << (top - shift) | (unsigned long long)s_bin;
      top = shift;
      const int in_bin = s_count;
      if (shift == 0) { cut = fixed; break; }                           // equal keys
      if (in_bin <= LIST) {
        for (int i = tid; i < n; i += CT) { const unsigned long long k = keys[i]; if (looked(k)) list[atomicAdd(&s_n, 1)] = k; }
        __syncthreads();
        if (tid < in_bin) {                                             // the `left`-th of the list from the top; of equal keys any thread may say it
          const unsigned long long k = list[tid];
          int more = 0, same = 0;
          for (int i = 0; i < in_bin; ++i) { more += list[i] > k; same += list[i] == k; }
          if (more < left && more + same >= left) { s_cut = k; s_left = left - more; }
        }
        __syncthreads();
        cut = s_cut; left = s_left;
        break;
      }
      __syncthreads();
    }
  }
  __syncthreads();
  // ---- one walk in rising order, four blocks a thread
  int at = 0, equal = 0;                                                // taken so far; keys equal to the border so far
  for (int i0 = 0; i0 < n; i0 += 4 * CT) {
    unsigned long long k4[4];
    int mine = 0;                                                       // keys above the border, and equal ones << 16
    #pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + 4 * tid + e;
      k4[e] = i < n ? keys[i] : 0ull;
      mine += k4[e] > cut ? 1 : k4[e] && k4[e] == cut ? 1 << 16 : 0;
    }
    int upto = mine;
    #pragma unroll
    for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(0xffffffffu, upto, d); if (lane >= d) upto += o; }
    if (lane == 31) warps[warp] = upto;
    __syncthreads();
    int before = upto - mine, all = 0;
    #pragma unroll
    for (int i = 0; i < CT / 32; ++i) { const int v = warps[i]; if (i < warp) before += v; all += v; }
    int a = before & 0xffff, e0 = equal + (before >> 16);
    #pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool eq = k4[e] && k4[e] == cut, take = k4[e] > cut || (eq && e0 < left);
      if (take) ids[at + a + min(e0, left) - min(equal, left)] = i0 + 4 * tid + e;
      a += k4[e] > cut; e0 += eq;
    }
    at += (all & 0xffff) + min(equal + (all >> 16), left) - min(equal, left);
    equal += all >> 16;
    __syncthreads();
  }
  if (tid == 0 && last >= 0) ids[at] = last;
  if (last >= 0) ++at;
  for (int i = at + tid; i < P.take; i += CT) ids[i] = -1;
}

}  // namespace
}  // namespace paged

size_t paged_select_bytes(const yskn_paged_cache& c, int rows, int blocks) { return (size_t)rows * c.kvh * blocks * 8; }

int launch_paged_select(const yskn_paged_cache& c, const yskn_paged_rows& r, const yskn_paged_select_args& a, cudaStream_t st) {
  using namespace paged;
  const bool bf = c.dtype == YSKN_KV4_BF16;
  const int g = a.nh / c.kvh;
  SelectP P{rows_of(c, r, 0), r.rows, g, a.nh, static_cast<const uint16_t*>(a.q), (long long)a.q_stride, static_cast<const uint16_t*>(c.kmean),
            static_cast<unsigned long long*>(a.workspace), a.take, a.ids};
  auto score = c.hd == 256 ? (bf ? paged_score_kernel<256, true> : paged_score_kernel<256, false>)
                           : (bf ? paged_score_kernel<128, true> : paged_score_kernel<128, false>);
  if (r.blocks > 1) {
    // blocks of a warp: as many as leave two CTAs an SM, since a CTA's start (its queries as fp64) costs what eight blocks do
    int per = 4;
    while (per < 64 && (long long)r.rows * c.kvh * ((r.blocks - 1) / (SCORE_WARPS * 2 * per)) >= 2 * SMS) per *= 2;
    const int cta = SCORE_WARPS * per;
    if (int rc = launch_pdl("paged_score_kernel", score, dim3((unsigned)((r.blocks - 1 + cta - 1) / cta), (unsigned)c.kvh, (unsigned)r.rows), SCORE_WARPS * 32, 0, st, P, per))
      return rc;
  }
  return launch_pdl("paged_choose_kernel", paged_choose_kernel, dim3((unsigned)c.kvh, (unsigned)r.rows), CT, 0, st, P);
}

}  // namespace kv4
