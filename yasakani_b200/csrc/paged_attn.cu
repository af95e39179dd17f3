// Attention of single rows over a paged 16-bit cache (sm_100a): batched decode, attention over chosen blocks, the rows' own part behind a shared prefix.
//
// Mathematics: o = sum_j p_j v_j / sum_j p_j, p_j = 2^(s q.k_j log2 e - m), m the running maximum; a tile of 64 tokens at a time, one pass over K and V.
// p is rounded to the cache's type for the product with V, its sum stays fp32.  fp16 has no numbers between 0 and 2^-24 and less than 11 bits below 2^-14, and a long tail of
// such weights may carry a channel in which the largest weight's value is zero: there m is the maximum less 15, so that p lies in (0, 2^15] and is rounded by half a step of its own down to 2^-29 of
// the largest, by 2^-40 of that below.  It cancels in the quotient, and the merge takes (m, l, O) as it takes others.
//
// Bound: HBM.  A token of a kv-head costs 4 HD bytes and 2 G HD multiply-adds for the G <= 16 heads that share it, which is what warp-level tensor-core
// tiles are for: S^T[16 tokens x 8 heads] = K Q^T, O^T[16 channels x 8 heads] += V^T P^T, keys and values straight from the swizzled tiles (ldmatrix).
//
// Work split.  The tiles of all (row, kv-head) pairs form one line, row after row, which the CTAs of a grid that fills the GPU share out evenly, whatever the lengths
// are.  A pair's start and end cost what a tile does, so in the line it is a step longer than its tiles (64 rows of 1 to 1,500 tokens in four kv-heads: CTAs took
// 23 to 36 us, by the number of their pairs).  A CTA's run covers parts of one or several pairs.  A pair that lies in one CTA is finished there; of a
// pair that lies on several each CTA writes (m, l, O) to the piece number (CTA + pair), which is unique because along the line either number only grows, and
// the merge kernel adds the pieces up.  Every CTA derives the line from the positions itself (a scan over at most ROWS rows).
//
// A CTA: one producer warp, four compute warps.  The producer asks for the tiles' pages by TMA (a box of min(page, 64) rows, 128-byte swizzle) into a ring of six
// half stages, K and V in turn, ahead of the compute warps and across the borders of pairs; page numbers come 32 at a time.  The compute warps take 16 tokens
// each for S, share the tile's maxima and weights through shared memory (two named barriers a tile), and take HD / 4 channels each for O, so no warp holds a copy of O.
// hd 256: one CTA an SM (192 KB in flight); hd 128: two.
//
// Measured (bf16, 24 / 4 heads of 256): eight rows over 2,048 .. 131,072 tokens 231 us with the merge, 6.4 TB/s of the 6.56 that a copy has; 48,000 tokens 40 us for a floor of
// 30, in one row or in 64: 4 us from the launch to the first tile (positions, table, copy), 1 us from the last tile to the merge's start, 2 us of merge, and a
// tail in which SMs that take in their bytes 15 % more slowly than others are left.  The tail's bytes are bound by HBM all the same: shares of the line handed out as CTAs
// came to an end (a quarter of it, by clusterlaunchcontrol) changed 231 us to 237 and 52 to 58 (33 rows of 28 heads), for the pieces and lookups that it added.
//
// Tokens that a row does not see: absent blocks are read outside the tensor map (zeros); what a page holds behind the sequence's end leaves the fragments of V by a mask
// (a weight of 0 times an infinity would be none; zeroed in shared memory it cost each row's last tile 1 us); scores are masked by selection.
// Every wait is bounded; one that runs out sets the status word (8) and all warps walk to the end without waiting again.
#include "paged_common.cuh"
#include <algorithm>
#include <cstring>

namespace kv4 {
namespace paged {

__device__ int g_attn_status = 0;            // 0 ok; 8 = a bounded wait ran out

namespace {

constexpr int ROWS = 224;                    // rows of one launch (a multiple of 32; what shared memory leaves beside the ring)
constexpr int NSLOT = 6;                     // half stages of the ring: K, V, K, V, K, V
constexpr int CW = 4, NT_ = (CW + 1) * 32;   // compute warps; threads
template <bool BF> constexpr float ABOVE = BF ? 0.f : 15.f;            // log2 of the largest weight

struct AttnP {
  Rows R; int rows, g, nh;
  const uint16_t* q; long long qs; float cs; // cs = qscale * log2(e)
  uint16_t* o16;
  int shared; const int* ids; int take;
  int2* span; float2* ml; float* pacc;       // first and last CTA of a pair; its pieces: maxima and sums, O
  const float2* qml; const float* qacc; int splits;     // partials over the shared prefix
  int beside;                                // the launch in front is the prefix kernel of this call
};

template <int HD, int NT> struct Lay {
  // Queries of pairs that have been asked for: of pairs of a tile or two their number is what the ring's depth is of long ones
  static constexpr int NQ = NT == 1 ? 4 : 2;
  static constexpr int HALF = TILE * HD * 2, QP = HD * 2 + 16, PP = TILE * 2 + 16;   // bytes: a half stage; a row of Q; a row of P (paddings: eight rows on different banks)
  static constexpr int OFF_Q = NSLOT * HALF, OFF_P = OFF_Q + NQ * NT * 8 * QP, OFF_MAX = OFF_P + 2 * NT * 8 * PP, OFF_L = OFF_MAX + 2 * CW * NT * 8 * 4;
  static constexpr int OFF_BASE = OFF_L + 2 * CW * NT * 8 * 4, OFF_BAR = OFF_BASE + 3 * 4 * 4, OFF_PLACE = OFF_BAR + 20 * 8 + 8, OFF_FIRST = OFF_PLACE + ROWS * 8;
  static constexpr int TOTAL = OFF_FIRST + (ROWS + 1) * 4;
  static constexpr int CTAS = HD == 256 ? 1 : 2;
  static_assert(HALF % 1024 == 0 && OFF_BASE % 16 == 0 && OFF_BAR % 8 == 0 && CTAS * (TOTAL + 1024) <= 228 * 1024, "shared memory");
};

__device__ __forceinline__ void ldm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void stm2t(uint32_t a, uint32_t x, uint32_t y) {
  asm volatile("stmatrix.sync.aligned.m8n8.x2.trans.shared.b16 [%0], {%1,%2};" ::"r"(a), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Tokens of a row that this kernel attends to by position: [start, vis); a row that has all of the shared prefix leaves that to the prefix kernel.
__device__ __forceinline__ int start_of(const Place& w, int shared) { return shared > 0 && w.vis >= shared ? shared : 0; }
__device__ __forceinline__ int tiles_of(const AttnP& P, const Place& w) {
  if (w.vis <= 0) return 0;
  if (P.ids) return (int)((((long long)P.take << P.R.lp) + TILE - 1) / TILE);
  return (w.vis - start_of(w, P.shared) + TILE - 1) / TILE;
}

template <int HD, int NT, bool BF>
__global__ void __launch_bounds__(NT_, Lay<HD, NT>::CTAS)
paged_attn_kernel(const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV, const AttnP P) {
  using L = Lay<HD, NT>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sb = s_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t b_full = sb + L::OFF_BAR, b_empty = b_full + 8 * NSLOT, b_qfull = b_empty + 8 * NSLOT, b_qempty = b_qfull + 8 * L::NQ;
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + L::OFF_BAR + 20 * 8);
  int* first = reinterpret_cast<int*>(smem + L::OFF_FIRST);
  Place* places = reinterpret_cast<Place*>(smem + L::OFF_PLACE);
  if (threadIdx.x == 0) {
    for (int i = 0; i < NSLOT; ++i) { bar_init(b_full + 8 * i, 1); bar_init(b_empty + 8 * i, CW); }
    for (int i = 0; i < L::NQ; ++i) { bar_init(b_qfull + 8 * i, 1); bar_init(b_qempty + 8 * i, CW); }
    *s_abort = sb & 1023u ? 1 : 0;           // the swizzled tiles need a base of 1 KB
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mapK) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mapV) : "memory");
  }
  __syncthreads();
  // Behind the prefix kernel there is nothing to wait for: it lets this one start when all of its blocks have seen what lies in front of it finished, and this one
  // reads nothing that it writes, so the two run side by side where there is room.  The wait comes at the end: the merge waits for this grid, and thereby for both.
  if (!P.beside) pdl_wait();
  pdl_launch();

  // ---- the line: first[r] = steps of one kv-head ahead of row r; a row's are one, without a tile, and its tiles.  Every warp finds it for itself (all write the same): no barrier between the positions and the first copy
  int steps_of_all;
  {
    int below = 0;
    for (int r0 = 0; r0 < P.rows; r0 += 32) {
      const int r = r0 + lane;
      int mine = 0;
      if (r < P.rows) { const Place w = place_of<true>(P.R, r); places[r] = w; const int nt = tiles_of(P, w); mine = nt > 0 ? nt + 1 : 0; }
      int upto = mine;
      #pragma unroll
      for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(0xffffffffu, upto, d); if (lane >= d) upto += o; }
      first[r] = below + upto - mine;
      below += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) first[P.rows] = below;
    steps_of_all = below;
    __syncwarp();
  }
  const int kvh = P.R.kvh, total = steps_of_all * kvh, grid = min((int)gridDim.x, total), cta = (int)blockIdx.x;       // every CTA below `grid` has a step at least
  if (cta >= grid) { if (P.beside) pdl_wait(); return; }
  const int u0 = (int)((long long)total * cta / grid), u1 = (int)((long long)total * (cta + 1) / grid);

  int row = 0;                               // the row that holds step u0: the last whose first step is not behind it
  for (int hi = P.rows - 1; row < hi; ) { const int mid = (row + hi + 1) >> 1; if (first[mid] * kvh <= u0) row = mid; else hi = mid - 1; }
  const int lc = min(P.R.lp, 6), chunk = 1 << lc, npt = TILE >> lc;    // rows of a box, boxes of a tile

  if (warp == CW) {
    // =========================================================================================== producer
    const int none = (P.R.pages * kvh) << P.R.lp;                      // a row outside the arrays: zeros
    // Boxes come 32 at a time, one a lane, looked up a batch ahead and across the borders of pairs: the lookups' latency (place, chosen block, table) is never
    // waited for.  A box: its row in the arrays, the position of its first token, its pair.
    struct Box { int at, base, pair; };
    int base_row = row;                                                // of the steps that are looked up: they lie a few rows on at most
    auto box_of = [&](int u, int j) {                                  // box j of step u; of a step without a tile: pair -1
      Box x{none, NO_TOKEN, -1};
      if (u >= u1) return x;
      int row = base_row;
      #pragma unroll 1
      while (first[row + 1] * kvh <= u) ++row;
      const int steps = first[row + 1] - first[row], in = u - first[row] * kvh, head = in / steps, t = in - head * steps - 1;
      if (t < 0) return x;
      const Place w = places[row];
      x.pair = row * kvh + head;
      const int ci = t * npt + j;
      int b = -1, sub = 0;
      if (P.ids) {
        const int cpp = P.R.lp - lc, e = ci >> cpp;                    // log2 of a page's boxes; entry
        if (e < P.take) b = P.ids[(size_t)x.pair * P.take + e];
        sub = (ci & ((1 << cpp) - 1)) << lc;
      } else {
        const long long tok = start_of(w, P.shared) + ((long long)ci << lc);
        if (tok < w.vis) { b = (int)(tok >> P.R.lp); sub = (int)tok & (P.R.page - 1); }
      }
      if (b < 0 || b >= P.R.blocks || ((long long)b << P.R.lp) + sub >= w.vis) return x;
      const int pg = page_of<true>(P.R, w.seq, b);
      if (pg < 0) return x;
      x.at = ((pg * kvh + head) << P.R.lp) + sub;
      x.base = (b << P.R.lp) + sub;
      return x;
    };
    int k = 0, pair = -1, issued = 0, queries = 0;                     // tiles so far; the pair they belong to; half stages and queries asked for
    bool ok = *s_abort == 0;
    const int tpb = 32 / npt, jl = lane & (npt - 1), tl = lane / npt;  // tiles of a batch; this lane's box and tile in it
    Box now{}, next{};
    for (int u = u0; u < u1 && ok; ++u) {
      int i = u - u0;
      const int in = i % tpb;
      if (i == 0 || in == 4) {                                         // the first batch; the one behind this, once the ring is full (in one place: every line of cold code counts)
        const Box x = box_of(i == 0 ? u0 + tl : u - in + tpb + tl, jl);
        if (i == 0) now = x; else next = x;
      }
      if (i > 0 && in == 0) { now = next; while (first[base_row + 1] * kvh <= u) ++base_row; }
      i = in * npt + jl;
      const int at = __shfl_sync(0xffffffffu, now.at, i), base = __shfl_sync(0xffffffffu, now.base, i), pr = __shfl_sync(0xffffffffu, now.pair, i);
      if (pr < 0) continue;
      if (pr != pair) {                                                // queries of the next pair
        pair = pr;
        const int qb = queries % L::NQ;
        if (queries >= L::NQ && !__all_sync(0xffffffffu, bar_wait(b_qempty + 8 * qb, (queries / L::NQ - 1) & 1))) { ok = false; break; }
        if (lane == 0) bar_expect_tx(b_qfull + 8 * qb, P.g * HD * 2);
        __syncwarp();
        ++queries;
        const int row = pair / kvh, head = pair - row * kvh;
        if (lane < P.g) bulk_1d(sb + L::OFF_Q + (qb * NT * 8 + lane) * L::QP, P.q + row * P.qs + (size_t)(head * P.g + lane) * HD, HD * 2, b_qfull + 8 * qb);
      }
      #pragma unroll
      for (int v = 0; v < 2; ++v) {                                    // keys, values
        const int it = 2 * k + v, slot = it % NSLOT;
        if (it >= NSLOT && !__all_sync(0xffffffffu, bar_wait(b_empty + 8 * slot, (it / NSLOT - 1) & 1))) ok = false;
        if (*s_abort) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (v == 0 && lane < npt) reinterpret_cast<int*>(smem + L::OFF_BASE)[(k % 3) * 4 + lane] = base;
        __syncwarp();
        if (lane == 0) bar_expect_tx(b_full + 8 * slot, L::HALF);      // whole boxes, rows outside the arrays among them
        __syncwarp();
        ++issued;
        if (lane < npt) tma_3d(sb + slot * L::HALF + lane * (chunk * HD * 2), v ? &mapV : &mapK, 0, at, 0, b_full + 8 * slot);
      }
      ++k;
    }
    if (!ok) {                                                         // give up; the copies under way land before the block ends
      if (lane == 0) { atomicExch(&g_attn_status, 8); *s_abort = 1; }
      for (int it = max(0, issued - NSLOT); it < issued; ++it) bar_wait(b_full + 8 * (it % NSLOT), (it / NSLOT) & 1);
      for (int it = max(0, queries - L::NQ); it < queries; ++it) bar_wait(b_qfull + 8 * (it % L::NQ), (it / L::NQ) & 1);
    }
    if (P.beside) pdl_wait();
    return;
  }

  // ============================================================================================= compute warps
  const int g8 = lane >> 2, j = lane & 3;
  const float cs = P.cs;
  float* smax = reinterpret_cast<float*>(smem + L::OFF_MAX);
  float* sl = reinterpret_cast<float*>(smem + L::OFF_L);
  constexpr int MT = HD / CW / 16;                                     // 16-channel tiles of O of this warp
  bool ok = true;
  auto wait = [&](uint32_t bar, int n) {                               // phase n of a barrier
    if (ok && (*s_abort || !bar_wait(bar, n & 1))) { atomicExch(&g_attn_status, 8); *s_abort = 1; ok = false; }
    __syncwarp();                                                      // each lane has polled for itself, and what follows wants the warp together
  };
  int k = 0, sg = 0, steps = first[row + 1] - first[row], head = (u0 - first[row] * kvh) / steps, at = u0 - first[row] * kvh - head * steps;
  for (int u = u0; ; ) {                                               // tiles [t0, t1) of the nt tiles of (row, kv-head)
    const int to = min(steps, at + (u1 - u)), nt = steps - 1, t0 = max(0, at - 1), t1 = to - 1;
    u += to - at;
    if (t1 > t0) {                                                     // else the step without a tile, and this CTA's last
    const Place w = places[row];
    uint32_t qf[NT][HD / 16][2];
    const int qb = sg % L::NQ;
    wait(b_qfull + 8 * qb, sg / L::NQ);
    #pragma unroll
    for (int n = 0; n < NT; ++n)
      #pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        uint32_t r[4];
        ldm4(sb + L::OFF_Q + (qb * NT * 8 + n * 8 + (lane & 7)) * L::QP + (4 * i + (lane >> 3)) * 16, r);
        qf[n][2 * i][0] = r[0]; qf[n][2 * i][1] = r[1]; qf[n][2 * i + 1][0] = r[2]; qf[n][2 * i + 1][1] = r[3];
      }
    __syncwarp();
    if (lane == 0) bar_arrive(b_qempty + 8 * qb);

    float o[NT][MT][4], m[NT][2], l[NT][2];
    #pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY; l[n][0] = l[n][1] = 0.f;
      #pragma unroll
      for (int x = 0; x < MT; ++x) o[n][x][0] = o[n][x][1] = o[n][x][2] = o[n][x][3] = 0.f;
    }
    for (int t = t0; t < t1; ++t, ++k) {
      const int ik = 2 * k, kslot = ik % NSLOT, iv = ik + 1, vslot = iv % NSLOT, buf = k & 1;
      // ---- S^T of this warp's 16 tokens
      wait(b_full + 8 * kslot, ik / NSLOT);
      const int tok = 16 * warp, cb = tok >> lc, rr = tok & (chunk - 1);                    // its chunk, first row there
      const int4 b4 = *reinterpret_cast<const int4*>(smem + L::OFF_BASE + (k % 3) * 16);    // read before the half stage is handed back: the next tile's come then
      auto base_of = [&](int i) { return box_base(i == 0 ? b4.x : i == 1 ? b4.y : i == 2 ? b4.z : b4.w, w.vis); };
      const int base = base_of(cb);
      float c[NT][2][4];                                                                    // two sums, so that products do not wait for one another
      #pragma unroll
      for (int n = 0; n < NT; ++n)
        #pragma unroll
        for (int x = 0; x < 4; ++x) c[n][0][x] = c[n][1][x] = 0.f;
      {
        const int r = rr + (lane & 7) + ((lane >> 3) & 1) * 8;
        const uint32_t a0 = sb + kslot * L::HALF + cb * (chunk * HD * 2) + r * 128;
        #pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          const int cc = 2 * ks + (lane >> 4);
          uint32_t a[4];
          ldm4(a0 + (cc >> 3) * (chunk * 128) + (((cc & 7) ^ (r & 7)) << 4), a);
          #pragma unroll
          for (int n = 0; n < NT; ++n) mma<BF>(c[n][ks & 1], a[0], a[1], a[2], a[3], qf[n][ks][0], qf[n][ks][1]);
        }
      }
      // tokens of the tile that the row sees: lane row g8 and g8 + 8 of this warp's
      const bool see0 = base + rr + g8 < w.vis, see1 = base + rr + g8 + 8 < w.vis;
      float x[NT][4];
      #pragma unroll
      for (int n = 0; n < NT; ++n) {
        #pragma unroll
        for (int e = 0; e < 4; ++e) x[n][e] = (e < 2 ? see0 : see1) ? (c[n][0][e] + c[n][1][e]) * cs : -INFINITY;
        #pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v = fmaxf(x[n][e], x[n][e + 2]);
          #pragma unroll
          for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
          if (lane < 4) smax[(buf * CW + warp) * (NT * 8) + n * 8 + 2 * j + e] = v - ABOVE<BF>;
        }
      }
      __syncwarp();
      if (lane == 0) bar_arrive(b_empty + 8 * kslot);
      compute_sync();
      float alpha[NT][2];
      #pragma unroll
      for (int n = 0; n < NT; ++n) {
        float2 top = make_float2(m[n][0], m[n][1]);
        #pragma unroll
        for (int i = 0; i < CW; ++i) {
          const float2 f = *reinterpret_cast<const float2*>(smax + (buf * CW + i) * (NT * 8) + n * 8 + 2 * j);
          top.x = fmaxf(top.x, f.x); top.y = fmaxf(top.y, f.y);
        }
        const float r0 = top.x == -INFINITY ? 0.f : top.x, r1 = top.y == -INFINITY ? 0.f : top.y;      // nothing seen so far: any reference does
        alpha[n][0] = ex2(m[n][0] - r0); alpha[n][1] = ex2(m[n][1] - r1);
        m[n][0] = top.x; m[n][1] = top.y;
        const float p0 = ex2(x[n][0] - r0), p1 = ex2(x[n][1] - r1), p2 = ex2(x[n][2] - r0), p3 = ex2(x[n][3] - r1);
        l[n][0] = l[n][0] * alpha[n][0] + (p0 + p2); l[n][1] = l[n][1] * alpha[n][1] + (p1 + p3);
        stm2t(sb + L::OFF_P + (buf * NT * 8 + n * 8 + (lane & 7)) * L::PP + (tok + 8 * ((lane >> 3) & 1)) * 2, pack_weights<BF>(p0, p1), pack_weights<BF>(p2, p3));
      }
      // ---- O^T of this warp's channels
      wait(b_full + 8 * vslot, iv / NSLOT);
      const uint32_t sv = sb + vslot * L::HALF;
      compute_sync();
      #pragma unroll
      for (int n = 0; n < NT; ++n)
        #pragma unroll
        for (int y = 0; y < MT; ++y) { o[n][y][0] *= alpha[n][0]; o[n][y][1] *= alpha[n][1]; o[n][y][2] *= alpha[n][0]; o[n][y][3] *= alpha[n][1]; }
      #pragma unroll
      for (int h = 0; h < 2; ++h) {                                                         // 32 tokens
        uint32_t pf[NT][4];
        #pragma unroll
        for (int n = 0; n < NT; ++n) ldm4(sb + L::OFF_P + (buf * NT * 8 + n * 8 + (lane & 7)) * L::PP + (4 * h + (lane >> 3)) * 16, pf[n]);
        #pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const int t16 = 32 * h + 16 * ks, ch = t16 >> lc, r16 = t16 & (chunk - 1), r = r16 + (lane & 7) + ((lane >> 4) & 1) * 8;
          // of these 16 tokens the row sees the first n16 (no block: none, and what was read is zero); a lane's registers hold tokens 2j, 2j + 1 and the eight behind them
          const int n16 = w.vis - base_of(ch) - r16 - 2 * j;
          const uint32_t keep0 = keep_pair(n16), keep1 = keep_pair(n16 - 8);
          #pragma unroll
          for (int y = 0; y < MT; ++y) {
            const int cc = warp * (2 * MT) + 2 * y + ((lane >> 3) & 1);
            uint32_t a[4];
            ldm4t(sv + ch * (chunk * HD * 2) + (cc >> 3) * (chunk * 128) + r * 128 + (((cc & 7) ^ (r & 7)) << 4), a);
            a[0] &= keep0; a[1] &= keep0; a[2] &= keep1; a[3] &= keep1;
            #pragma unroll
            for (int n = 0; n < NT; ++n) mma<BF>(o[n][y], a[0], a[1], a[2], a[3], pf[n][2 * ks], pf[n][2 * ks + 1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) bar_arrive(b_empty + 8 * vslot);
    }
    // ---- this CTA's part of the pair
    #pragma unroll
    for (int n = 0; n < NT; ++n)
      #pragma unroll
      for (int e = 0; e < 2; ++e) {
        #pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
        if (lane < 4) sl[((sg & 1) * CW + warp) * (NT * 8) + n * 8 + 2 * j + e] = l[n][e];
      }
    compute_sync();
    const bool direct = t1 - t0 == nt && start_of(w, P.shared) == 0;
    const int pair = row * kvh + head;
    const size_t piece = (size_t)cta + pair;
    if (threadIdx.x == 0) { if (t0 == 0) P.span[pair].x = cta; if (t1 == nt) P.span[pair].y = cta; }
    #pragma unroll
    for (int n = 0; n < NT; ++n)
      #pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = n * 8 + 2 * j + e;
        float sum = 0.f;
        #pragma unroll
        for (int i = 0; i < CW; ++i) sum += sl[((sg & 1) * CW + i) * (NT * 8) + h];
        if (h >= P.g || !ok) continue;
        if (direct) {
          uint16_t* dst = P.o16 + ((size_t)row * P.nh + head * P.g + h) * HD + warp * (HD / CW);
          const float inv = sum == 0.f ? 0.f : 1.f / sum;                                   // nothing seen: zeros
          #pragma unroll
          for (int y = 0; y < MT; ++y) {
            const uint32_t v = pack16<BF>(sum == 0.f ? 0.f : o[n][y][e] * inv, sum == 0.f ? 0.f : o[n][y][e + 2] * inv);
            dst[16 * y + g8] = (uint16_t)v; dst[16 * y + g8 + 8] = (uint16_t)(v >> 16);
          }
        } else {
          float* dst = P.pacc + (piece * (NT * 8) + h) * HD + warp * (HD / CW);
          #pragma unroll
          for (int y = 0; y < MT; ++y) { dst[16 * y + g8] = o[n][y][e]; dst[16 * y + g8 + 8] = o[n][y][e + 2]; }
          if (warp == 0 && g8 == 0) P.ml[piece * (NT * 8) + h] = make_float2(m[n][e], sum);
        }
      }
    ++sg;
    }
    if (u >= u1) break;
    at = 0;                                                            // the next pair
    if (++head == kvh) { head = 0; do ++row; while (row < P.rows && first[row + 1] == first[row]); steps = row < P.rows ? first[row + 1] - first[row] : 1; }
  }
  if (P.beside) pdl_wait();
}

// Joins what the parts of a (row, head) hold: partials over the shared prefix, then pieces of CTAs.  W warps for 128 channels of a (row, head), four a lane: each looks at all
// parts' maxima and sums by itself, a lane a part, and adds up every W-th part's O, U of them asked for together.
constexpr int MERGE_THREADS = 256;
template <int HD, bool BF, int W, int U>
__global__ void __launch_bounds__(MERGE_THREADS) paged_merge_kernel(const AttnP P, int slot_rows) {
  constexpr int V = HD / 128;
  __shared__ float4 part[W][W > 1 ? 32 : 1];
  const int lane = threadIdx.x & 31, wid = (int)(blockIdx.x * (MERGE_THREADS / 32) + (threadIdx.x >> 5)), xv = wid / W, x = xv / V, v = xv % V, wi = wid % W;
  if (x >= P.rows * P.nh) return;            // the same for the whole block where W is its number of warps
  const int row = x / P.nh, head = x - row * P.nh, h = head / P.g, hh = head - h * P.g, pair = row * P.R.kvh + h;
  // Ahead of the wait: the attention kernel lets this one start when all of its blocks have seen what lies in front of them finished, and writes no positions
  const Place w = place_of<true>(P.R, row);
  pdl_wait();
  pdl_launch();
  if (w.seq < 0) return;
  const int2 span = P.span[pair];            // of a row without tiles nobody has written it, and nobody looks at it
  const bool prefix = start_of(w, P.shared) > 0, own = tiles_of(P, w) > 0;
  if (!prefix && own && span.x == span.y) return;                      // finished where it was computed
  const int np = prefix ? P.splits : 0, n = np + (own ? span.y - span.x + 1 : 0);
  const float2* qml = P.qml + (size_t)row * P.splits * P.nh + head;
  const float* qacc = P.qacc + ((size_t)row * P.splits * P.nh + head) * HD + 128 * v;
  const size_t piece0 = ((size_t)span.x + pair) * slot_rows + hh;      // piece c of the pair: + c * slot_rows
  auto ml_at = [&](int i) { return i < np ? qml[(size_t)i * P.nh] : P.ml[piece0 + (size_t)(i - np) * slot_rows]; };
  auto o_at = [&](int i) { return i < np ? qacc + (size_t)i * P.nh * HD : P.pacc + (piece0 + (size_t)(i - np) * slot_rows) * HD + 128 * v; };
  constexpr int PC = U * W;                  // parts that all W warps ask for together
  auto ml_or = [&](int i) { return i < n ? ml_at(i) : make_float2(-INFINITY, 0.f); };
  float4 o[U];
  auto ask = [&](int c) {                    // O of this warp's parts c + wi + W u: beside the maxima and sums, not behind them
    #pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = c + wi + W * u;
      if (i < n) o[u] = reinterpret_cast<const float4*>(o_at(i))[lane];
    }
  };
  float2 f0 = ml_or(lane), f1 = ml_or(32 + lane);
  ask(0);
  float top = fmaxf(f0.y != 0.f ? f0.x : -INFINITY, f1.y != 0.f ? f1.x : -INFINITY);
  for (int i = 64 + lane; i < n; i += 32) { const float2 f = ml_at(i); if (f.y != 0.f) top = fmaxf(top, f.x); }
  #pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (top == -INFINITY) top = 0.f;
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c = 0; c < n; c += PC) {
    if (c > 0) { f0 = ml_or(c + lane); f1 = PC > 32 ? ml_or(c + 32 + lane) : f1; ask(c); }
    const float w0 = lane < PC && f0.y != 0.f ? ex2(f0.x - top) : 0.f, w1 = PC > 32 && f1.y != 0.f ? ex2(f1.x - top) : 0.f;
    if (lane < PC && f0.y != 0.f) sum += f0.y * w0;
    if (PC > 32 && f1.y != 0.f) sum += f1.y * w1;
    #pragma unroll
    for (int u = 0; u < U; ++u) {
      const float wk = __shfl_sync(0xffffffffu, W * u < 32 ? w0 : w1, (wi + W * u) & 31);
      if (wk != 0.f) { acc.x += wk * o[u].x; acc.y += wk * o[u].y; acc.z += wk * o[u].z; acc.w += wk * o[u].w; }      // a part without weight may hold anything
    }
  }
  #pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (W > 1) {
    part[wi][W > 1 ? lane : 0] = acc;
    __syncthreads();
    if (wi > 0) return;
    #pragma unroll
    for (int i = 1; i < W; ++i) { const float4 f = part[i][W > 1 ? lane : 0]; acc.x += f.x; acc.y += f.y; acc.z += f.z; acc.w += f.w; }
  }
  const float inv = 1.f / sum;
  uint2 y;
  y.x = sum == 0.f ? 0u : pack16<BF>(acc.x * inv, acc.y * inv);
  y.y = sum == 0.f ? 0u : pack16<BF>(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(P.o16 + (size_t)x * HD + 128 * v + 4 * lane) = y;
}

template <int HD, int W, int U> int launch_merge(const AttnP& P, bool bf, int slot_rows, cudaStream_t st) {
  auto kern = bf ? paged_merge_kernel<HD, true, W, U> : paged_merge_kernel<HD, false, W, U>;
  const long long warps = (long long)P.rows * P.nh * (HD / 128) * W;
  return launch_pdl("paged_merge_kernel", kern, dim3((unsigned)((warps + 7) / 8)), MERGE_THREADS, 0, st, P, slot_rows);
}

int ctas_of(int hd) { return SMS * (hd == 256 ? 1 : 2); }
int slot_rows_of(int g) { return g <= 8 ? 8 : 16; }

Work carve(void* ws, const yskn_paged_cache& c, int rows, int nh, size_t prefix_parts) {
  const int chunk = std::min(rows, ROWS), sr = slot_rows_of(nh / c.kvh);
  const size_t pieces = (size_t)ctas_of(c.hd) + (size_t)chunk * c.kvh, parts = prefix_parts * nh;
  size_t at = 0;
  auto take = [&](size_t n) { const size_t x = at; at = (at + n + 255) / 256 * 256; return static_cast<uint8_t*>(ws) + x; };
  Work w;
  w.span = reinterpret_cast<int2*>(take((size_t)chunk * c.kvh * 8));
  w.ml = reinterpret_cast<float2*>(take(pieces * sr * 8));
  w.pacc = reinterpret_cast<float*>(take(pieces * sr * c.hd * 4));
  w.qml = reinterpret_cast<float2*>(take(parts * 8));
  w.qacc = reinterpret_cast<float*>(take(parts * c.hd * 4));
  w.bytes = at;
  return w;
}

template <int HD, int NT, bool BF>
int launch(const yskn_paged_cache& c, const AttnP& P, cudaStream_t st) {
  using L = Lay<HD, NT>;
  auto kern = paged_attn_kernel<HD, NT, BF>;
  static std::atomic<unsigned long long> attr{0};
  if (int rc = allow_smem(attr, kern, L::TOTAL)) return rc;
  CUtensorMap mk, mv;
  memcpy(&mk, c.maps[0], sizeof(mk)); memcpy(&mv, c.maps[1], sizeof(mv));
  return launch_pdl("paged_attn_kernel", kern, dim3((unsigned)ctas_of(HD)), NT_, L::TOTAL, st, mk, mv, P);
}
template <int HD>
int dispatch(const yskn_paged_cache& c, const AttnP& P, cudaStream_t st) {
  const bool bf = c.dtype == YSKN_KV4_BF16;
  if (P.g <= 8) return bf ? launch<HD, 1, true>(c, P, st) : launch<HD, 1, false>(c, P, st);
  return bf ? launch<HD, 2, true>(c, P, st) : launch<HD, 2, false>(c, P, st);
}

}  // namespace

int attn_status_fetch(int* out) {
  int v = 0;
  KV4_CUDA(cudaMemcpyFromSymbol(&v, g_attn_status, sizeof(int)));
  const int zero = 0;
  KV4_CUDA(cudaMemcpyToSymbol(g_attn_status, &zero, sizeof(int)));
  *out = v; return 0;
}

}  // namespace paged

size_t paged_attention_bytes(const yskn_paged_cache& c, int rows, int nh, int shared) {
  return paged::carve(nullptr, c, rows, nh, shared > 0 ? paged_prefix_parts(rows, nh / c.kvh, c.kvh, shared) : 0).bytes;
}

int launch_paged_attention(const yskn_paged_cache& c, const yskn_paged_rows& r, const yskn_paged_attn_args& a, cudaStream_t st) {
  using namespace paged;
  const int g = a.nh / c.kvh, splits = a.shared > 0 ? paged_prefix_splits(r.rows, g, c.kvh, a.shared) : 0;
  const Work w = carve(a.workspace, c, r.rows, a.nh, (size_t)r.rows * splits);
  if (splits > 0) if (int rc = launch_paged_prefix(c, r, a, splits, w, st)) return rc;
  for (int first = 0; first < r.rows; first += ROWS) {
    const int rows = std::min(ROWS, r.rows - first);
    const size_t part = (size_t)first * splits * a.nh;
    AttnP P{rows_of(c, r, first), rows, g, a.nh, static_cast<const uint16_t*>(a.q) + first * a.q_stride, (long long)a.q_stride, a.qscale * LOG2E,
            static_cast<uint16_t*>(a.o16) + (size_t)first * a.nh * c.hd, splits > 0 ? a.shared : 0, a.ids ? a.ids + (size_t)first * c.kvh * a.take : nullptr, a.take,
            w.span, w.ml, w.pacc, w.qml + part, w.qacc + part * c.hd, splits, splits > 0 && first == 0 ? 1 : 0};
    if (int rc = c.hd == 256 ? dispatch<256>(c, P, st) : dispatch<128>(c, P, st)) return rc;
    // Few rows have many parts: eight warps each, a block an SM at most, since blocks of this launch lie beside the attention kernel's from early on and a second wave of them
    // would start when all is over (five rows of 24 heads over 48 blocks with their choice 31.8 us, 240 blocks of 256 channels' halves, and 25.7 with 30).  Between events of a graph, eight warps and one, rows of 28 heads of 128 over 1,000 tokens: 28 items 7.3 us and 8.2, 140 8.7 and 9.7, and beyond the border 168 8.8 and
    // 9.7, 224 9.2 and 9.7, 280 10.2 and 10.1, 336 13.4 and 11.4; over 8,000 tokens 28 items 10.5 and 18.1, 140 21.8 and 23.0, 280 34.5 and 35.2, 336 41.4 and 40.0.  More have few parts:
    // a warp, which asks for eight at once where there are SMs for all of them (16 rows of 28 heads over 33 blocks 33.6 us, four at once 34.7), and for
    // four where its registers count (200 rows of 28 heads behind 5,216 tokens 62.4 us, eight 63.7)
    const bool bf = c.dtype == YSKN_KV4_BF16;
    const long long items = (long long)rows * a.nh * (c.hd / 128);
    const int sr = slot_rows_of(g), rc =
        items <= SMS ? (c.hd == 256 ? launch_merge<256, 8, 8>(P, bf, sr, st) : launch_merge<128, 8, 8>(P, bf, sr, st))
        : items <= 8 * SMS ? (c.hd == 256 ? launch_merge<256, 1, 8>(P, bf, sr, st) : launch_merge<128, 1, 8>(P, bf, sr, st))
                           : (c.hd == 256 ? launch_merge<256, 1, 4>(P, bf, sr, st) : launch_merge<128, 1, 4>(P, bf, sr, st));
    if (rc) return rc;
  }
  return 0;
}

}  // namespace kv4
