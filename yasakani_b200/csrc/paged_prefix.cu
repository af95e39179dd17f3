// Attention of many rows over one shared prefix of a paged 16-bit cache, on the 5th-generation tensor cores (tcgen05 + TMEM, sm_100a).
//
// Mathematics: partial (m, l, O) of every (row, head) over a run of the prefix's tokens, p = 2^(s q.k log2 e - m): no mask, since all rows see the whole prefix; the runs
// and what each row has behind the prefix are joined by the merge kernel (paged_attn.cu).
//
// Bound: the tensor cores from about 250 (row, head) pairs a kv-head on (2 HD multiply-adds per 2 HD * 2 bytes and pair), the prefix's bytes below.
//
// A pair of CTAs (a cluster of two, cta_group::2) takes 256 (row, head) pairs of one kv-head, 128 each, and one run of the tokens in tiles of 128.  Per CTA:
//   warps 0-7   two warpgroups that take the tiles in turn, a thread a row: scores from tensor memory, running maximum, weights back over the scores just read
//   warps 8, 10 TMA: its half of every K tile (64 tokens), of every V tile (HD/2 channels), a box of min(page, 64) rows x 64 channels a copy, NK and NV stages.  A
//               warp each, since a stage of V is free two tiles later than one of K: asked for in turn, K came a tile ahead of its use and the tensor pipe waited 780
//               cycles a tile for it
//   warp 9      (leader) issues S = Q K^T (M256 N128) into one of two or three buffers of tensor memory and O += P V (M256 N = HD, P from tensor memory)
// Each CTA stages half a tile because an SM takes in 40 to 50 bytes a clock from L2, and a whole tile a CTA would want 64.  S of a later tile is issued
// behind P V of this one, so the tensor pipe works while the weights are computed; O is rescaled only where a maximum has grown by more than 2^8.
//
// Weights are rounded to the cache's type, their sum stays fp32.  In fp16 m is the maximum less 7: weights reach 2^15, with what the maximum may have grown, and are rounded by half a step of
// their own down to 2^-21 of that maximum's weight, by 2^-32 of it below, so that a tail of small ones beside a large one is neither lost nor coarse.
//
// Measured (bf16, 64 rows of 24 / 4 heads of 256 over 32,768 tokens, nine runs): 53 us, 51.5 GFLOP at 970 TFLOP/s; 29 tiles of 1.36 us (2,057 cycles of tensor work at 1.9 GHz
// are 1.08), 4 us in front of them and 4 behind (O out).  96 of a CTA's 128 rows hold queries there: 16 rows of six heads, shared out evenly over two pairs.
//
// 44 to 48 bytes of a thread lie outside its registers, read or written once in a tile or less (25,000 stores and 12,500 loads of a warp in the launch above, 0.2 % of what L1 takes).
//
// Tokens of the last tile beyond the prefix are read outside the tensor map (zeros) and their scores masked.  Every wait is bounded; one that runs out sets
// the status word (9) and the CTA frees its tensor memory and returns.
#include "paged_common.cuh"
#include <algorithm>
#include <cstring>

namespace kv4 {
namespace paged {

__device__ int g_prefix_status = 0;          // 0 ok; 9 = a bounded wait ran out

namespace {

constexpr int BN = 128;                      // tokens of a tile
constexpr int SW = 8, THREADS = 384;         // softmax warps; threads (three warpgroups of 168 registers: 2 x 208 and 88 after the split)
constexpr int MAX_SPLITS = 64;
// log2 of the weight of the maximum that m was taken from; of what a maximum may grow by before O is rescaled.  A smaller margin would leave more room above and cost rescales of the first
// tiles (f16, 8 rows behind 4,096 tokens: 12.1 us as it is and without any room, 12.3 with a margin of 7, 12.6 with 6, 12.8 with 4)
template <bool BF> constexpr float ABOVE = BF ? 0.f : 7.f;
constexpr float MARGIN = 8.f;

template <int HD> struct Lay {
  static constexpr int KBLK = HD / 64, VBLK = HD / 128;                // 64-channel blocks of a K half tile, of a V half tile
  static constexpr int Q_BLOCK = 128 * 128, K_BLOCK = 64 * 128, V_BLOCK = BN * 128;      // bytes: [row][128 B]
  static constexpr int K_HALF = KBLK * K_BLOCK, V_HALF = VBLK * V_BLOCK;
  // 128 channels: a third buffer of scores, so that S of the next tile but one does not wait for P V of this one, whose softmax takes as long as the tile's products
  // (200 rows of 28 heads behind 5,216 tokens, with their own parts, 63.3 -> 62.1 us)
  static constexpr int NB = HD == 128 ? 3 : 2, NK = NB + 1, NV = NB;
  static constexpr int OFF_K = KBLK * Q_BLOCK, OFF_V = OFF_K + NK * K_HALF, OFF_BAR = OFF_V + NV * V_HALF;
  static constexpr int OFF_XCH = OFF_BAR + 256;                        // float [2][128] maxima, [2][128] sums; u16 [2][128] tags
  static constexpr int TOTAL = OFF_XCH + 4 * 128 * 4 + 2 * 128 * 2;
  static constexpr uint32_t TM_O = NB * BN;                            // tensor memory: the score buffers, 128 columns each, then O
  static constexpr int PITCH = HD * 4 + 16;                            // a row of O on its way out (eight lanes' 16 bytes on different banks)
  static_assert(TOTAL <= 227 * 1024 && 128 * PITCH <= OFF_BAR && NB * BN + HD <= 512 && NK <= 4 && NV <= 4 && NB <= 3, "shared memory, tensor memory");
};

struct PrefixP {
  Rows R; int rows, G, tpc, nh, splits, per, tiles, shared;            // tpc rows of a CTA; per tiles of a split
  const uint16_t* q; long long qs; float cs; uint32_t flip;            // |qscale| log2 e; its sign, as sign bits of two queries
  float2* qml; float* qacc;
};

__device__ __forceinline__ bool elect_one() {
  uint32_t p; asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p)); return p != 0;
}
__device__ __forceinline__ uint32_t leader_addr(uint32_t local) { uint32_t r; asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(local)); return r; }
__device__ __forceinline__ void arrive_cluster(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void cluster_sync_all() { asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// A copy into this CTA's shared memory that reports to a barrier of the pair's leader.
__device__ __forceinline__ void tma_pair(uint32_t dst, const CUtensorMap* m, int x, int y, int z, uint32_t lead_bar) {
  asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(m), "r"(x), "r"(y), "r"(z), "r"(lead_bar) : "memory");
}
// 128-byte swizzle.  K-major: atoms of eight 128-byte rows, `sbo` between them.  MN-major: `lbo` between 64-element blocks, `sbo` between groups of eight k.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16: A and B both fp16 or both bf16, fp32 sums, A K-major.
__host__ __device__ constexpr uint32_t instr_desc(int M, int N, bool b_mn, bool bf) {
  return (1u << 4) | ((bf ? 1u : 0u) << 7) | ((bf ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(acc) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(acc) : "memory");
}
__device__ __forceinline__ void commit_pair(uint32_t bar) {            // arrives in both CTAs once all MMAs so far are done
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_ld32(uint32_t a, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                 "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                 "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]) : "r"(a) : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t a, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
               ::"r"(a), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
                 "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
                 "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t a, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               ::"r"(a), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
                 "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ float2 fma2(float2 a, float b, float c) {   // two fp32 operations in one instruction, each rounded as the single one
  float2 d;
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %4};\n mov.b64 c, {%5, %5};\n fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

template <int HD, bool BF>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
paged_prefix_kernel(const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV, const PrefixP P) {
  using L = Lay<HD>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sb = s_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)blockIdx.x & 1;                                // the leader (rank 0) issues the MMAs
  const int G = P.G, nquad = (P.tpc * G + 31) / 32;                    // quadrants of 32 rows that hold queries
  // the leader's copy alone: kfull[NK] vfull[NV] phalf[NB] pready[NB] q; each CTA's: kempty[NK] vempty[NV] sready[NB] pvdone[NB]
  const uint32_t b0 = sb + L::OFF_BAR;
  const uint32_t b_kfull = b0, b_kempty = b0 + 32, b_vfull = b0 + 64, b_vempty = b0 + 96, b_sready = b0 + 128, b_pvdone = b0 + 152, b_phalf = b0 + 176,
                 b_pready = b0 + 200, b_q = b0 + 224;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::OFF_BAR + 232);
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + L::OFF_BAR + 236);
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::NK; ++i) { bar_init(b_kfull + 8 * i, 1); bar_init(b_kempty + 8 * i, 1); }
    for (int i = 0; i < L::NV; ++i) { bar_init(b_vfull + 8 * i, 1); bar_init(b_vempty + 8 * i, 1); }
    for (int i = 0; i < L::NB; ++i) {
      bar_init(b_sready + 8 * i, 1); bar_init(b_pvdone + 8 * i, 1);
      bar_init(b_phalf + 8 * i, 2 * nquad); bar_init(b_pready + 8 * i, 2 * nquad);          // the warps with queries of the tile's warpgroup, both CTAs
    }
    bar_init(b_q, 2 * SW);
    *s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x < 128) reinterpret_cast<volatile uint32_t*>(smem + L::OFF_XCH + 4 * 128 * 4)[threadIdx.x] = 0;
  if (warp == SW + 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sb + L::OFF_BAR + 232), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  cluster_sync_all();
  fence_after();
  // an allocation of all 512 columns starts at column 0: the addresses below are constants
  const bool bad = *tmem_slot != 0 || (sb & 1023u);                    // the same for the CTA; the other one's waits run out
  if (bad && threadIdx.x == 0) { atomicExch(&g_prefix_status, 9); *s_abort = 1; }
  pdl_wait();
  pdl_launch();

  const int kvh = blockIdx.z, split = blockIdx.y, row0 = (int)blockIdx.x * P.tpc;
  const int j0 = split * P.per, n = min(P.tiles, j0 + P.per) - j0;

  int issued = 0;                                                      // stages that a producer has asked for
  auto fail = [&]() { atomicExch(&g_prefix_status, 9); *s_abort = 1; };

  auto role_producer = [&](const bool is_v) {
    const int lc = min(P.R.lp, 6), chunk = 1 << lc, npt = BN >> lc;    // rows of a box; boxes of a tile's tokens
    const int none = (P.R.pages * P.R.kvh) << P.R.lp;                  // a row outside the arrays: zeros
    // The first row that has the whole prefix: its table names the pages.  Where no row has, zeros are taken and nothing is kept.
    int seq = -1;
    for (int r0 = 0; r0 < P.rows && seq < 0; r0 += 32) {
      Place w{-1, 0};
      if (r0 + lane < P.rows) w = place_of(P.R, r0 + lane);
      const unsigned found = __ballot_sync(0xffffffffu, w.vis >= P.shared);
      if (found) seq = __shfl_sync(0xffffffffu, w.seq, __ffs(found) - 1);
    }
    auto row_at = [&](int ci) {                                        // chunk ci of the prefix as a row of the arrays
      const long long tok = (long long)ci << lc;
      if (tok >= P.shared || seq < 0) return none;
      const int pg = page_of(P.R, seq, (int)(tok >> P.R.lp));
      return pg < 0 ? none : ((pg * P.R.kvh + kvh) << P.R.lp) + (int)(tok & (P.R.page - 1));
    };
    const int tpb = 32 / npt, blks = is_v ? L::VBLK : L::KBLK, boxes = is_v ? npt : npt / 2, stages = is_v ? L::NV : L::NK;
    const int box = lane / blks, blk = lane % blks;                    // this lane's copy: tokens, 64 channels
    const uint32_t full = is_v ? b_vfull : b_kfull, empty = is_v ? b_vempty : b_kempty, lead = leader_addr(full), bytes = is_v ? L::V_HALF : L::K_HALF;
    const uint32_t dst = sb + (is_v ? L::OFF_V + blk * L::V_BLOCK : L::OFF_K + blk * L::K_BLOCK) + box * (chunk * 128);
    const int z = is_v ? L::VBLK * rank + blk : blk, from = (is_v ? 0 : rank * boxes) + min(box, boxes - 1);
    const CUtensorMap* map = is_v ? &mapV : &mapK;
    int at0 = row_at(j0 * npt + lane), at1 = at0;                      // 32 boxes, one a lane, and the 32 behind them
    for (int i = 0; i < n; ++i) {
      const int in = i % tpb, st = i % stages;
      if (i > 0 && in == 0) at0 = at1;
      const int at = __shfl_sync(0xffffffffu, at0, in * npt + from);
      bool ok = i < stages || bar_wait(empty + 8 * st, (i / stages - 1) & 1);
      ok = __all_sync(0xffffffffu, ok && !*s_abort);
      if (!ok) { if (lane == 0) fail(); break; }
      if (rank == 0 && lane == 0) bar_expect_tx(full + 8 * st, 2 * bytes);
      ++issued;
      if (box < boxes) tma_pair(dst + st * bytes, map, 0, at, z, lead + 8 * st);
      if (in == min(2, tpb - 1)) at1 = row_at((j0 + i - in + tpb) * npt + lane);            // once the stages are full
    }
  };

  auto role_mma = [&]() {
    constexpr uint32_t ID_S = instr_desc(256, BN, false, BF), ID_PV = instr_desc(256, HD, true, BF);
    const bool leader = elect_one();
    bool ok = true;
    auto wait = [&](uint32_t bar, int phase) {
      if (ok && !__all_sync(0xffffffffu, bar_wait(bar, phase & 1))) { if (leader) fail(); ok = false; }
      return ok;
    };
    const uint64_t qd = smem_desc(sb, 16, 1024), kd0 = smem_desc(sb + L::OFF_K, 16, 1024), vd0 = smem_desc(sb + L::OFF_V, L::V_BLOCK, 1024);
    auto issue_s = [&](int i) {
      if (!wait(b_kfull + 8 * (i % L::NK), i / L::NK)) return;
      fence_after();
      const uint64_t kd = kd0 + (uint64_t)((i % L::NK * L::K_HALF) >> 4);
      if (leader) {
        #pragma unroll
        for (int x = 0; x < HD / 16; ++x)
          mma_ss(i % L::NB * BN, qd + (uint64_t)(((x >> 2) * L::Q_BLOCK + (x & 3) * 32) >> 4), kd + (uint64_t)(((x >> 2) * L::K_BLOCK + (x & 3) * 32) >> 4), ID_S, x > 0);
        commit_pair(b_sready + 8 * (i % L::NB));
        commit_pair(b_kempty + 8 * (i % L::NK));
      }
      __syncwarp();
    };
    auto issue_pv = [&](int i) {                                       // weights of tokens 0-63 while the others are still being computed
      if (!wait(b_phalf + 8 * (i % L::NB), i / L::NB) || !wait(b_vfull + 8 * (i % L::NV), i / L::NV)) return;
      fence_after();
      const uint64_t vd = vd0 + (uint64_t)((i % L::NV * L::V_HALF) >> 4);
      const uint32_t p = i % L::NB * BN;
      #pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == 1) { if (!wait(b_pready + 8 * (i % L::NB), i / L::NB)) return; fence_after(); }
        if (leader) {
          #pragma unroll
          for (int x = 0; x < 4; ++x) mma_ts(L::TM_O, p + 64 * h + 8 * x, vd + (uint64_t)(((4 * h + x) * 2048) >> 4), ID_PV, i > 0 || h + x > 0);
        }
        __syncwarp();
      }
      if (leader) { commit_pair(b_pvdone + 8 * (i % L::NB)); commit_pair(b_vempty + 8 * (i % L::NV)); }
      __syncwarp();
    };
    wait(b_q, 0);
    fence_after();
    for (int i = 0; i < L::NB && i < n && ok; ++i) issue_s(i);
    for (int i = 0; i < n && ok; ++i) {
      issue_pv(i);
      if (ok && i + L::NB < n) issue_s(i + L::NB);                     // over the scores that P V of tile i has read its weights from: the pipe runs in order
    }
  };

  auto role_softmax = [&]() {
    const int quad = warp & 3, hf = warp >> 2, rho = quad * 32 + lane; // quadrant of tensor memory; warpgroup; row of the tile
    const int row = row0 + rho / G, head = kvh * G + rho % G;
    // ---- queries into the swizzled blocks
    {
      constexpr int N = 128 * (HD / 8) / (32 * SW);                    // 16-byte pieces a thread, all asked for together
      uint4 u[N];
      #pragma unroll
      for (int x = 0; x < N; ++x) {
        const int it = threadIdx.x + x * 32 * SW, r = it / (HD / 8), w = it % (HD / 8), t = r / G;
        u[x] = make_uint4(0u, 0u, 0u, 0u);
        if (t < P.tpc && row0 + t < P.rows) u[x] = *reinterpret_cast<const uint4*>(P.q + (row0 + t) * P.qs + (size_t)(kvh * G + r - t * G) * HD + 8 * w);
      }
      #pragma unroll
      for (int x = 0; x < N; ++x) {
        const int it = threadIdx.x + x * 32 * SW, r = it / (HD / 8), w = it % (HD / 8);
        sts128(sb + (w >> 3) * L::Q_BLOCK + r * 128 + (((w & 7) ^ (r & 7)) << 4), make_uint4(u[x].x ^ P.flip, u[x].y ^ P.flip, u[x].z ^ P.flip, u[x].w ^ P.flip));
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) arrive_cluster(leader_addr(b_q));
    if (quad >= nquad) return;
    const bool valid = rho < P.tpc * G && row < P.rows && place_of(P.R, row).vis >= P.shared;
    const uint32_t trow = (uint32_t)(quad * 32) << 16, lead_half = leader_addr(b_phalf), lead_ready = leader_addr(b_pready);
    // What passes between a row's two threads: the running maximum, tile by tile, and at the end the sums; a value, then a tag that the other polls (bounded).
    volatile float* xval = reinterpret_cast<volatile float*>(smem + L::OFF_XCH);
    volatile uint16_t* xtag = reinterpret_cast<volatile uint16_t*>(smem + L::OFF_XCH + 4 * 128 * 4);
    auto tag_wait = [&](int slot, int tag) {
      for (uint32_t it = 0; it < WAIT_LIMIT; ++it)
        if ((uint16_t)(xtag[slot * 128 + rho] - (uint16_t)tag) < 0x8000u) { __threadfence_block(); return true; }
      return false;
    };
    const float cs = P.cs;
    float m = -INFINITY, mown = -INFINITY, l = 0.f;                    // the row's maximum; the one that this thread's l refers to
    bool ok = true;
    #pragma unroll 1
    for (int i = hf; i < n; i += 2) {
      const int sbuf = i % L::NB;            // of three buffers a warpgroup sees every other phase; the one between is over, since S of this warpgroup's tile before came behind it
      const uint32_t sc = trow + sbuf * BN;
      if (!bar_wait(b_sready + 8 * sbuf, (i / L::NB) & 1)) { fail(); ok = false; }
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      fence_after();
      uint32_t xr[128];
      #pragma unroll
      for (int c = 0; c < 4; ++c) tm_ld32(sc + 32 * c, xr + 32 * c);
      tm_wait_ld();
      float x[128];
      #pragma unroll
      for (int k = 0; k < 128; ++k) x[k] = __uint_as_float(xr[k]);
      if ((j0 + i + 1) * BN > P.shared) {                              // the prefix ends inside this tile
        const int end = P.shared - (j0 + i) * BN;
        #pragma unroll
        for (int k = 0; k < 128; ++k) x[k] = k < end ? x[k] : -INFINITY;
      }
      float t4[4] = {x[0], x[1], x[2], x[3]};
      #pragma unroll
      for (int k = 4; k < 128; k += 4)
        #pragma unroll
        for (int e = 0; e < 4; ++e) t4[e] = fmaxf(t4[e], x[k + e]);
      const float raw = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * cs;
      const bool far = !BF && fabsf(raw) >= 0x1p22f;                   // scores whose own steps would add to the weights' 2^15: as near to 1 as they come
      const float top = raw - (far ? 0.f : ABOVE<BF>);
      if (i > 0) {                                                     // the tile before this one is the other warpgroup's
        if (!tag_wait(hf ^ 1, i)) { fail(); ok = false; }
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        m = xval[(hf ^ 1) * 128 + rho];
      }
      const bool bump = valid && top > m + (far ? 0.f : MARGIN);
      const float alpha = bump ? ex2(m - top) : 1.f;
      if (bump) m = top;
      xval[hf * 128 + rho] = m;
      __threadfence_block();
      xtag[hf * 128 + rho] = (uint16_t)(i + 1);
      if (mown != m) { l *= ex2(mown - m); mown = m; }
      if (__any_sync(0xffffffffu, bump && i > 0)) {                    // rows whose maximum stays multiply by exactly 1
        if (!bar_wait(b_pvdone + 8 * ((i - 1) % L::NB), ((i - 1) / L::NB) & 1)) { fail(); ok = false; }
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        fence_after();
        #pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tm_ld32(trow + L::TM_O + 32 * c, o);
          tm_wait_ld();
          #pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
          tm_st32(trow + L::TM_O + 32 * c, o);
        }
      }
      const float nm = m == -INFINITY ? 0.f : -m;                      // nothing but -inf so far: any reference does
      float2 s0 = make_float2(0.f, 0.f), s1 = s0;
      #pragma unroll
      for (int c = 0; c < 4; ++c) {                                    // 32 tokens; weights over the scores that this thread has read
        uint32_t pk[16];
        #pragma unroll
        for (int k = 0; k < 32; k += 4) {
          float2 a = fma2(make_float2(x[32 * c + k], x[32 * c + k + 1]), cs, nm), b = fma2(make_float2(x[32 * c + k + 2], x[32 * c + k + 3]), cs, nm);
          a.x = ex2(a.x); a.y = ex2(a.y); b.x = ex2(b.x); b.y = ex2(b.y);
          s0 = add2(s0, a); s1 = add2(s1, b);
          pk[k / 2] = valid ? pack_weights<BF>(a.x, a.y) : 0u; pk[k / 2 + 1] = valid ? pack_weights<BF>(b.x, b.y) : 0u;
        }
        tm_st16(sc + 64 * (c >> 1) + 16 * (c & 1), pk);
        if (c & 1) {
          tm_wait_st();
          fence_before();
          __syncwarp();
          if (lane == 0) arrive_cluster((c == 1 ? lead_half : lead_ready) + 8 * sbuf);
        }
      }
      l += (s0.x + s0.y) + (s1.x + s1.y);
    }
    // ---- the row's maximum and sum; then O, half of the channels a thread, through shared memory so that a warp stores whole lines
    if (ok) {
      if (((n - 1) & 1) != hf) { ok = tag_wait(hf ^ 1, n); if (ok) m = xval[(hf ^ 1) * 128 + rho]; }
      if (mown != m) l *= ex2(mown - m);
      xval[256 + hf * 128 + rho] = l;
      __threadfence_block();
      xtag[hf * 128 + rho] = (uint16_t)(n + 1);
      if (ok) ok = tag_wait(hf ^ 1, n + 1);
      l = xval[256 + rho] + xval[256 + 128 + rho];
    }
    // one barrier a score buffer: its phase before this is tile n - 1 - NB's, over since S of tile n - 1 came behind that P V and a tag of that S was seen
    if (ok && !bar_wait(b_pvdone + 8 * ((n - 1) % L::NB), ((n - 1) / L::NB) & 1)) ok = false;
    if (!ok) fail();
    if (!__all_sync(0xffffffffu, ok && !*s_abort)) return;
    fence_after();
    const size_t part = ((size_t)row * P.splits + split) * P.nh + head;
    if (valid && hf == 0) P.qml[part] = make_float2(m, l);
    __syncwarp();
    constexpr int LPR = HD / 8;                                        // lanes that cover half a row
    #pragma unroll 1
    for (int c = hf * (HD / 64); c < (hf + 1) * (HD / 64); ++c) {
      uint32_t o[32];
      tm_ld32(trow + L::TM_O + 32 * c, o);
      tm_wait_ld();
      #pragma unroll
      for (int k = 0; k < 8; ++k) sts128(sb + rho * L::PITCH + 128 * c + 16 * k, make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]));
    }
    __syncwarp();
    #pragma unroll 4
    for (int r0 = 0; r0 < 32; r0 += 32 / LPR) {
      const int r = r0 + lane / LPR, off = hf * 2 * HD + 16 * (lane % LPR);
      const long long to = __shfl_sync(0xffffffffu, valid ? (long long)part : -1ll, r);
      const uint4 v = lds128(sb + (quad * 32 + r) * L::PITCH + off);
      if (to >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(P.qacc) + (size_t)to * (4 * HD) + off) = v;
    }
  };

  if (warp < SW) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    if (!bad) role_softmax();
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (bad) {}
    else if (warp == SW) role_producer(false);
    else if (warp == SW + 2) role_producer(true);
    else if (warp == SW + 1 && rank == 0) role_mma();
  }
  fence_before();
  __syncthreads();
  if (rank == 0 && *s_abort) {                                         // copies of both CTAs that are still under way land before the pair ends
    if (warp == SW) for (int i = max(0, issued - L::NK); i < issued; ++i) bar_wait(b_kfull + 8 * (i % L::NK), (i / L::NK) & 1);
    if (warp == SW + 2) for (int i = max(0, issued - L::NV); i < issued; ++i) bar_wait(b_vfull + 8 * (i % L::NV), (i / L::NV) & 1);
  }
  __syncwarp();
  cluster_sync_all();                                                  // neither CTA's memory is in use by the other any more
  if (warp == SW + 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(0u), "n"(512) : "memory");
}

int tiles_of(int shared) { return (shared + BN - 1) / BN; }

template <int HD, bool BF>
int launch(const yskn_paged_cache& c, const PrefixP& P, int pairs, cudaStream_t st) {
  using L = Lay<HD>;
  auto kern = paged_prefix_kernel<HD, BF>;
  static std::atomic<unsigned long long> attr{0};
  if (int rc = allow_smem(attr, kern, L::TOTAL)) return rc;
  CUtensorMap mk, mv;
  memcpy(&mk, c.maps[2], sizeof(mk)); memcpy(&mv, c.maps[3], sizeof(mv));
  return launch_pdl("paged_prefix_kernel", kern, dim3(2u * pairs, (unsigned)P.splits, (unsigned)c.kvh), THREADS, L::TOTAL, st, mk, mv, P);
}

int most_runs(int tiles) { return (tiles + 1) / 2; }
int pairs_of(int rows, int g) { const int tok = 128 / g; return (rows + 2 * tok - 1) / (2 * tok); }

}  // namespace

int prefix_status_fetch(int* out) {
  int v = 0;
  KV4_CUDA(cudaMemcpyFromSymbol(&v, g_prefix_status, sizeof(int)));
  const int zero = 0;
  KV4_CUDA(cudaMemcpyToSymbol(g_prefix_status, &zero, sizeof(int)));
  *out = v; return 0;
}

}  // namespace paged

// Runs of the prefix for so many pairs of CTAs a kv-head: one wave of them where that goes, else what fills the waves best, a run's start and end counted as a
// twentieth of a prefix.  It depends on the prefix only in that a run has two tiles at least, so that a workspace for many rows and tokens serves fewer.  Both rules are compromises:
//   two tiles  (2 to 100 rows, 200 tokens of their own, us with one / two / three tiles at least) gains where one tile a run takes the SMs from the rows' own part beside it, loses a little where it
//              leaves them idle, and from 8,192 tokens (256 channels) or 16,384 (128) on nothing of it is felt: 28 heads of 128, eight rows: behind 512 tokens 10.1 / 10.8 / 10.8, behind 2,048 16.0 / 11.7 / 12.4, behind
//              4,096 17.0 / 16.9 / 16.1; 24 heads of 256, 32 rows: behind 512 25.2 / 25.3 / 25.0, behind 2,048 30.0 / 26.8 / 27.6, behind 4,096 31.7 / 31.5 / 29.2
//   a twentieth (64 heads over eight of 128 channels, us with 1 / 2 / 3 / 4 runs) is about right for long prefixes, too little for short ones: 80 pairs of CTAs (four by the rule) behind 16,384 tokens
//              275 / 230 / 221 / 225, behind 2,048 87 / 89 / 95 / 108; 128 (one) 311 / 324 / 342 / 335 and 117 / 133 / 149 / 165; 192 (three) 484 / 501 / 492 / 530 and 174 / 199 / 214 / 246
static int prefix_runs(long long pairs, int kvh) {
  const long long items = pairs * kvh, slots = paged::SMS / 2;
  if (items <= slots) return (int)std::min<long long>(paged::MAX_SPLITS, slots / items);
  int best = 1;
  double cost = 0.0;
  for (int s = 1; s <= 4; ++s) {
    const double x = (double)((items * s + slots - 1) / slots) * (1.0 / s + 0.05);
    if (s == 1 || x < cost) { cost = x; best = s; }
  }
  return best;
}

int paged_prefix_splits(int rows, int g, int kvh, int shared) {
  using namespace paged;
  const int nt = tiles_of(shared), s = std::min(prefix_runs(pairs_of(rows, g), kvh), most_runs(nt)), per = (nt + s - 1) / s;
  return (nt + per - 1) / per;
}

// Partials (row, run) of any call with up to so many rows and shared tokens.
size_t paged_prefix_parts(int rows, int g, int kvh, int shared) {
  using namespace paged;
  size_t most = 0;
  const int tok = 128 / g, pairs = pairs_of(rows, g);
  for (int p = 1; p <= pairs; ++p) most = std::max(most, (size_t)std::min<long long>(rows, 2ll * tok * p) * std::min(prefix_runs(p, kvh), most_runs(tiles_of(shared))));
  return most;
}

int launch_paged_prefix(const yskn_paged_cache& c, const yskn_paged_rows& r, const yskn_paged_attn_args& a, int splits, const paged::Work& w, cudaStream_t st) {
  using namespace paged;
  const int g = a.nh / c.kvh, pairs = pairs_of(r.rows, g), tpc = (r.rows + 2 * pairs - 1) / (2 * pairs), nt = tiles_of(a.shared);
  const float cs = a.qscale == 0.f ? 1.17549435e-38f : a.qscale * LOG2E;          // not 0: masked scores are -inf times it
  PrefixP P{rows_of(c, r, 0), r.rows, g, tpc, a.nh, splits, (nt + splits - 1) / splits, nt, a.shared, static_cast<const uint16_t*>(a.q), (long long)a.q_stride,
            cs < 0.f ? -cs : cs, cs < 0.f ? 0x80008000u : 0u, w.qml, w.qacc};
  const bool bf = c.dtype == YSKN_KV4_BF16;
  return c.hd == 256 ? (bf ? launch<256, true>(c, P, pairs, st) : launch<256, false>(c, P, pairs, st))
                     : (bf ? launch<128, true>(c, P, pairs, st) : launch<128, false>(c, P, pairs, st));
}

}  // namespace kv4
