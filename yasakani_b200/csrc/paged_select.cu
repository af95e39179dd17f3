// Choice of the blocks that a row attends to (sm_100a): a score for every complete page, then the highest ones.
//
// Mathematics: score(b) = max over the heads h of a kv-head's group of sum_c q_h[c] mean_b[c].  Products of two 16-bit values are exact in fp32, and all the more so in
// fp64, and a sum of HD of them in fp64 is exact or off by 2^-52 of its largest part: the choice does not depend on the order of the sum, and two builds, or a
// plain program, agree on every block.  fp32 sums differ by 2^-24, which decides between neighbours every few thousand rows.
//
// Bound: the mean keys, 2 HD bytes a page and kv-head, read once per row.  B200 does fp64 at half the rate of fp32, so the G products a channel run beside the loads.
// Two launches: scores as 64-bit keys that sort like the score (workspace); the choice, a block a (row, kv-head): digits of the keys counted from the highest
// on until the border is found, then one walk that writes the chosen blocks in rising order.
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

constexpr int SCORE_BLOCKS = 64;             // blocks of one CTA
// A warp takes a block at a time: lane l has channels 8l .. 8l + 7 (hd 128: half a warp a block).  Queries in shared memory as fp64.
template <int HD, bool BF>
__global__ void __launch_bounds__(256) paged_score_kernel(const SelectP P) {
  constexpr int LPB = HD / 8, BPW = 32 / LPB;
  extern __shared__ double qs[];                                        // [g][HD], channel c of lane l at (c % 8) * LPB + l: lanes side by side
  pdl_wait();
  pdl_launch();
  const int row = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place w = place_of(P.R, row);
  if (w.seq < 0) return;
  const int n = w.vis > 0 ? (w.vis - 1) >> P.R.lp : 0;                  // candidates: blocks in front of the last
  const int b0 = (int)blockIdx.x * SCORE_BLOCKS;
  if (b0 >= n) return;
  for (int i = threadIdx.x; i < P.g * (HD / 2); i += 256) {
    const int gi = i / (HD / 2), c = 2 * (i % (HD / 2));
    const float2 f = unpack16<BF>(*reinterpret_cast<const uint32_t*>(P.q + row * P.qs + (size_t)(h * P.g + gi) * HD + c));
    double* d = qs + gi * HD + c / 8;
    d[(c & 7) * LPB] = f.x; d[((c & 7) + 1) * LPB] = f.y;
  }
  __syncthreads();
  const int l = lane % LPB;
  #pragma unroll 1
  for (int i = warp * BPW + lane / LPB; i < SCORE_BLOCKS; i += 8 * BPW) {
    const int b = b0 + i;
    const int page = b < n ? page_of(P.R, w.seq, b) : -1;
    double x[8];
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (page >= 0) u = *reinterpret_cast<const uint4*>(P.kmean + ((size_t)page * P.R.kvh + h) * HD + 8 * l);
    const uint32_t u4[4] = {u.x, u.y, u.z, u.w};
    #pragma unroll
    for (int e = 0; e < 4; ++e) { const float2 f = unpack16<BF>(u4[e]); x[2 * e] = f.x; x[2 * e + 1] = f.y; }
    double best = 0.0;
    bool any = false;
    for (int gi = 0; gi < P.g; ++gi) {
      const double* q = qs + gi * HD + l;
      double a = 0.0, b2 = 0.0;
      #pragma unroll
      for (int e = 0; e < 8; e += 2) { a = fma(q[e * LPB], x[e], a); b2 = fma(q[(e + 1) * LPB], x[e + 1], b2); }
      a += b2;
      #pragma unroll
      for (int d = LPB / 2; d > 0; d >>= 1) a += __shfl_xor_sync(0xffffffffu, a, d);
      if (a == a) { best = any ? fmax(best, a) : a; any = true; }
    }
    if (l == 0 && b < n) P.keys[((size_t)row * P.R.kvh + h) * P.R.blocks + b] = page < 0 ? 0ull : any ? key_of(best) : 1ull;
  }
}

// The choice.  Keys of equal height are taken from the lowest block on.  Digits of 8 bits from the top: how many keys share the digits so far, until what is left to
// take is all of them or the digits are used up.
__global__ void __launch_bounds__(256) paged_choose_kernel(const SelectP P) {
  __shared__ int hist[256], warps[8], s_digit, s_left, s_all;
  pdl_wait();
  pdl_launch();
  const int row = blockIdx.y, h = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place w = place_of(P.R, row);
  if (w.seq < 0) return;
  const size_t pair = (size_t)row * P.R.kvh + h;
  const unsigned long long* keys = P.keys + pair * P.R.blocks;
  int* ids = P.ids + pair * P.take;
  const int last = w.vis > 0 ? (w.vis - 1) >> P.R.lp : -1, n = last > 0 ? last : 0;
  // ---- the border: keys above `low` are taken, and of those equal to it the first `left`
  unsigned long long prefix = 0, mask = 0;
  int left = P.take - 1;
  bool all = n <= left;                                                 // every candidate
  for (int shift = 56; shift >= 0 && !all; shift -= 8) {
    hist[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 256) {
      const unsigned long long k = keys[i];
      if ((k & mask) == prefix && k != 0) atomicAdd(&hist[(int)(k >> shift) & 255], 1);
    }
    __syncthreads();
    // thread t stands for digit 255 - t: keys of higher digits in front
    const int mine = hist[255 - threadIdx.x];
    int upto = mine;
    #pragma unroll
    for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(0xffffffffu, upto, d); if (lane >= d) upto += o; }
    if (lane == 31) warps[warp] = upto;
    if (threadIdx.x == 0) s_all = 0;
    __syncthreads();
    for (int i = 0; i < warp; ++i) upto += warps[i];
    if (upto - mine < left && upto >= left) { s_digit = 255 - threadIdx.x; s_left = left - (upto - mine); s_all = upto == left ? 1 : 0; }
    if (threadIdx.x == 255 && upto < left) s_all = 2;                   // fewer candidates than places: all of them
    __syncthreads();
    if (s_all == 2) { all = true; break; }
    prefix |= (unsigned long long)s_digit << shift; mask |= 255ull << shift;
    left = s_left;
    const bool done = s_all == 1;                                       // all keys with these digits are taken
    __syncthreads();
    if (done) break;
  }
  // ---- one walk in rising order
  int at = 0;                                                           // taken so far; `equal` of them with the border's digits
  int equal = 0;
  for (int i0 = 0; i0 < n; i0 += 256) {
    const int i = i0 + (int)threadIdx.x;
    const unsigned long long k = i < n ? keys[i] : 0ull;
    const bool eq = !all && k != 0 && (k & mask) == prefix;
    const bool above = k != 0 && (all || (k & mask) > prefix);
    const unsigned be = __ballot_sync(0xffffffffu, eq), ba = __ballot_sync(0xffffffffu, above), under = (1u << lane) - 1u;
    if (lane == 0) warps[warp] = __popc(be) << 16 | __popc(ba);
    __syncthreads();
    int e = equal, a = 0, te = 0, ta = 0;
    #pragma unroll
    for (int x = 0; x < 8; ++x) { const int v = warps[x]; if (x < warp) { e += v >> 16; a += v & 0xffff; } te += v >> 16; ta += v & 0xffff; }
    e += __popc(be & under); a += __popc(ba & under);
    const int eq_before = min(e, left) - min(equal, left);              // equal keys taken among this walk's lower ones
    if ((eq && e < left) || above) ids[at + a + eq_before] = i;
    at += ta + min(equal + te, left) - min(equal, left);
    equal += te;
    __syncthreads();
  }
  if (threadIdx.x == 0 && last >= 0) ids[at] = last;
  if (last >= 0) ++at;
  for (int i = at + (int)threadIdx.x; i < P.take; i += 256) ids[i] = -1;
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
  if (r.blocks > 1)
    if (int rc = launch_pdl("paged_score_kernel", score, dim3((unsigned)((r.blocks - 1 + SCORE_BLOCKS - 1) / SCORE_BLOCKS), (unsigned)c.kvh, (unsigned)r.rows), 256,
                            (size_t)g * c.hd * 8, st, P)) return rc;
  return launch_pdl("paged_choose_kernel", paged_choose_kernel, dim3((unsigned)c.kvh, (unsigned)r.rows), 256, 0, st, P);
}

}  // namespace kv4
