// Rows of several sequences into a paged 16-bit cache (sm_100a): keys and queries rotated at each row's position on the way, and the mean key of every
// page that a row completes.
//
// Mathematics: channels (c, c + rd/2), c < rd/2, of a head turn by the angle of (position, c): (a, b) -> (a cos - b sin, b cos + a sin), fp32, rounded once.
// Mean of a page: fp32 sum of its `page` rows in a fixed order, times 1 / page (a power of two, exact), rounded once.
//
// Bound: bytes.  Every row is read and written once, 16 bytes a lane; a warp holds whole heads (hd 256: one, hd 128: two), so the other channel of a pair
// is in another lane of the same warp and comes by a shuffle.  8,192 rows of 24 + 2 * 4 heads of 256 channels: 52.6 us, 5.2 TB/s of 6.6 that a copy has.  What that
// took: nobody reads the inputs again, and of a prompt nobody the rows before L2 has let them go, so both pass as streaming data (57.2 us without either hint, 56.7 with
// one); 32 warps an SM with four loads each (two loads a lane 71 us, eight 76; a loop over items with the next one's loads ahead 65); the means' blocks first, since
// they bring the keys into L2 (last 61 us, between the others 64).
//
// The means are taken in the same launch, by blocks of their own: of a page's rows those that this call brings are turned again from the call's inputs, as their
// places in the cache are being written at the same time, and the others are read from the cache.  A launch behind the first one took a
// call of eight rows from 8.9 to 11.3 us, most of it on the host.  Where the rows in front of a page's last one are the page's, as in a prompt, they are found at once; else every row of the call is looked at
// for each completed page and kv-head (8,192 rows of 64 sequences: one after the other 58 us between events, in any order 65, interleaved by position, so that one block meets 32 completed pages, 271).
#include "paged_common.cuh"

namespace kv4 {
namespace paged {
namespace {

struct AppendP {
  Rows R; int rows;
  const uint16_t* k_in; const uint16_t* v_in; const uint16_t* q_in; uint16_t* q_out;
  long long ks, vs, qs;
  const float* rope; int rope_rows, rd, nh;
  uint16_t* k; uint16_t* v; uint16_t* kmean;
  int mean_blocks;                           // blocks in front of the others, one for 32 rows and a kv-head; 0: no means
  int spr;                                   // slots (256 channels) of a row: heads of q, k, v one after the other
  int wpr;                                   // warps that share a row
};

constexpr int SLOTS = 4;                     // 16-byte loads a lane has in flight: 4 KB a warp

// Two channels' worth of a 32-bit word, a, turned with the other channels of their pairs, d: a cos + d sin, the sine's sign being that of the channel's half.
template <bool BF> __device__ __forceinline__ uint32_t turn(uint32_t aw, uint32_t dw, const float4& t) {
  const float2 a = unpack16<BF>(aw), d = unpack16<BF>(dw);
  return pack16<BF>(fmaf(d.x, t.y, a.x * t.x), fmaf(d.y, t.w, a.y * t.z));
}
template <bool BF> __device__ __forceinline__ uint4 turn8(const uint4& a, const uint4& d, const float4 (&t)[4]) {
  return make_uint4(turn<BF>(a.x, d.x, t[0]), turn<BF>(a.y, d.y, t[1]), turn<BF>(a.z, d.z, t[2]), turn<BF>(a.w, d.w, t[3]));
}
// (cos, sin) of channels ch .. ch + 7 at a position, ch < rd; -sin in the first half of the rotated channels.
__device__ __forceinline__ void angles(const AppendP& P, int pos, int ch, float4 (&t)[4]) {
  const int half = P.rd / 2;
  const bool lower = ch < half;
  const float4* src = reinterpret_cast<const float4*>(P.rope + ((size_t)pos * half + (lower ? ch : ch - half)) * 2);
  #pragma unroll
  for (int e = 0; e < 4; ++e) { const float4 f = src[e]; t[e] = lower ? make_float4(f.x, -f.y, f.z, -f.w) : f; }
}
// The page of a row, -1 where the row is left out; `at` its position.
__device__ __forceinline__ int page_of_row(const AppendP& P, int row, int& at) {
  const int s = P.R.seq[row];
  at = P.R.pos[row];
  if (s < 0 || s >= P.R.seqs || at < 0 || (P.rd > 0 && at >= P.rope_rows) || (at >> P.R.lp) >= P.R.blocks) return -1;
  return page_of(P.R, s, at >> P.R.lp);
}

// Mean keys: a block looks at 32 rows and one kv-head; most rows complete no page.
template <int HD, bool BF>
__device__ void page_means(const AppendP& P, int r0, int h) {
  constexpr int LPH = HD / 8, GROUPS = 256 / LPH;                      // lanes of a row; rows in flight
  __shared__ float part[GROUPS][HD];
  __shared__ int from[128];                                            // the row of this call that holds a token of the page; -1: the cache does
  const int tid = threadIdx.x, lane = tid & 31;
  int pos = 0, page = -1;
  if (r0 + lane < P.rows) { page = page_of_row(P, r0 + lane, pos); if ((pos & (P.R.page - 1)) != P.R.page - 1) page = -1; }
  unsigned todo = __ballot_sync(0xffffffffu, page >= 0);               // the same in every warp of the block
  while (todo) {
    const int which = __ffs(todo) - 1, pg = __shfl_sync(0xffffffffu, page, which), end = __shfl_sync(0xffffffffu, pos, which), first = end - P.R.page + 1;
    const int seq = P.R.seq[r0 + which];
    todo &= todo - 1;
    if (tid < P.R.page) from[tid] = -1;
    __syncthreads();
    // Where the rows in front of this one are the page's other tokens, as in a prompt, that is all; else every row of the call is looked at
    bool there = true;
    if (tid < P.R.page) {
      const int r = r0 + which - (P.R.page - 1 - tid);
      there = r >= 0 && P.R.seq[r] == seq && P.R.pos[r] == first + tid;
      if (there) from[tid] = r;
    }
    if (!__syncthreads_and(there)) {
      #pragma unroll 4
      for (int r = tid; r < P.rows; r += 256) {
        const int p = P.R.pos[r];
        if (p >= first && p <= end && P.R.seq[r] == seq) from[p - first] = r;
      }
    }
    __syncthreads();
    const int grp = tid / LPH, ch = 8 * (tid % LPH), half = P.rd / 2;
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    #pragma unroll 2
    for (int t = grp; t < P.R.page; t += GROUPS) {
      const int r = from[t];
      uint4 u;
      if (r < 0) u = *reinterpret_cast<const uint4*>(P.k + ((((size_t)pg * P.R.kvh + h) << P.R.lp) + t) * HD + ch);
      else {
        const uint16_t* src = P.k_in + r * P.ks + (size_t)h * HD;
        u = *reinterpret_cast<const uint4*>(src + ch);
        if (ch < P.rd) {
          float4 cs[4];
          angles(P, first + t, ch, cs);
          u = turn8<BF>(u, *reinterpret_cast<const uint4*>(src + (ch < half ? ch + half : ch - half)), cs);
        }
      }
      const uint32_t u4[4] = {u.x, u.y, u.z, u.w};
      #pragma unroll
      for (int e = 0; e < 4; ++e) { const float2 f = unpack16<BF>(u4[e]); sum[2 * e] += f.x; sum[2 * e + 1] += f.y; }
    }
    #pragma unroll
    for (int e = 0; e < 8; ++e) part[grp][ch + e] = sum[e];
    __syncthreads();
    if (2 * tid < HD) {
      const int x = 2 * tid;
      float a = 0.f, b = 0.f;
      #pragma unroll
      for (int i = 0; i < GROUPS; ++i) { a += part[i][x]; b += part[i][x + 1]; }
      const float inv = 1.f / (float)P.R.page;
      *reinterpret_cast<uint32_t*>(P.kmean + ((size_t)pg * P.R.kvh + h) * HD + x) = pack16<BF>(a * inv, b * inv);
    }
    __syncthreads();
  }
}

// One warp per SLOTS * 256 channels of a row.  The rows' own loads do not wait for the position; the table entry does.
template <int HD, bool BF>
__global__ void __launch_bounds__(256, 4) paged_append_kernel(const AppendP P) {
  constexpr int LPH = HD / 8;                // lanes of a head
  pdl_wait();
  pdl_launch();
  const int block = (int)blockIdx.x - P.mean_blocks;                   // the blocks for the means come first: theirs is the longer way
  if (block < 0) { page_means<HD, BF>(P, (int)blockIdx.x / P.R.kvh * 32, (int)blockIdx.x % P.R.kvh); return; }
  const int w = (int)((block * 256u + threadIdx.x) >> 5), lane = threadIdx.x & 31;
  const int row = w / P.wpr, s0 = (w - row * P.wpr) * SLOTS;
  if (row >= P.rows) return;
  const int nq = P.q_in ? P.nh : 0, kvh = P.R.kvh, heads = nq + 2 * kvh;
  const int c = lane % LPH, ch = 8 * c;      // this lane's channels
  uint4 x[SLOTS];
  int vh[SLOTS];
  #pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int h = (s0 + i) * (256 / HD) + lane / LPH;
    vh[i] = s0 + i < P.spr && h < heads ? h : -1;
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    if (vh[i] >= 0) {
      const uint16_t* src = h < nq ? P.q_in + row * P.qs + (size_t)h * HD : h < nq + kvh ? P.k_in + row * P.ks + (size_t)(h - nq) * HD
                                                                                       : P.v_in + row * P.vs + (size_t)(h - nq - kvh) * HD;
      x[i] = __ldcs(reinterpret_cast<const uint4*>(src + ch));
    }
  }
  const int s = P.R.seq[row], pos = P.R.pos[row];
  if (s < 0 || s >= P.R.seqs || pos < 0 || (P.rd > 0 && pos >= P.rope_rows)) return;          // the same for the whole warp
  const int b = pos >> P.R.lp;
  const int page = b < P.R.blocks ? page_of(P.R, s, b) : -1;
  const int half = P.rd / 2, lh = half / 8;                            // lanes of half the rotated channels
  float4 cs[4];
  if (ch < P.rd) angles(P, pos, ch, cs);
  const int partner = ch < half ? lane + lh : ch < P.rd ? lane - lh : lane;
  uint16_t* const q_row = P.q_out + (size_t)row * P.nh * HD + ch;
  const size_t place = (((size_t)page * kvh) << P.R.lp) + (pos & (P.R.page - 1));            // of kv-head 0; the others a page's rows further each
  #pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int h = vh[i];
    uint4 y = x[i];
    if (P.rd > 0 && (s0 + i) * (256 / HD) < nq + kvh) {                // not a slot of values alone: the same for the whole warp
      uint4 o;
      o.x = __shfl_sync(0xffffffffu, y.x, partner); o.y = __shfl_sync(0xffffffffu, y.y, partner);
      o.z = __shfl_sync(0xffffffffu, y.z, partner); o.w = __shfl_sync(0xffffffffu, y.w, partner);
      if (ch < P.rd && h < nq + kvh) y = turn8<BF>(y, o, cs);
    }
    if (h < 0 || (h >= nq && page < 0)) continue;
    uint16_t* dst;
    if (h < nq) dst = q_row + h * HD;
    else {
      const int j = h - nq, jj = j < kvh ? j : j - kvh;
      dst = (j < kvh ? P.k : P.v) + (place + ((size_t)jj << P.R.lp)) * HD + ch;
    }
    __stcs(reinterpret_cast<uint4*>(dst), y);
  }
}

}  // namespace
}  // namespace paged

int launch_paged_append(const yskn_paged_cache& c, const yskn_paged_rows& r, const yskn_paged_append_args& a, cudaStream_t st) {
  using namespace paged;
  const bool bf = c.dtype == YSKN_KV4_BF16;
  AppendP P{rows_of(c, r, 0), r.rows, static_cast<const uint16_t*>(a.k_in), static_cast<const uint16_t*>(a.v_in), static_cast<const uint16_t*>(a.q_in),
            static_cast<uint16_t*>(a.q_out), a.k_stride, a.v_stride, a.q_stride, a.rope, a.rope_rows, a.rd, a.nh,
            static_cast<uint16_t*>(c.k), static_cast<uint16_t*>(c.v), static_cast<uint16_t*>(c.kmean), 0, 0, 0};
  const long long heads = (a.q_in ? a.nh : 0) + 2ll * c.kvh;
  P.spr = (int)((heads * c.hd + 255) / 256);
  P.wpr = (P.spr + SLOTS - 1) / SLOTS;
  const long long means = c.kmean ? (long long)((r.rows + 31) / 32) * c.kvh : 0, blocks = means + ((long long)r.rows * P.wpr + 7) / 8;
  if (blocks >= 1ll << 23) KV4_REJECT("yskn_kv4_paged_append: too many rows (%d) for one call", r.rows);
  P.mean_blocks = (int)means;
  auto kern = c.hd == 256 ? (bf ? paged_append_kernel<256, true> : paged_append_kernel<256, false>)
                          : (bf ? paged_append_kernel<128, true> : paged_append_kernel<128, false>);
  return launch_pdl("paged_append_kernel", kern, dim3((unsigned)blocks), 256, 0, st, P);
}

}  // namespace kv4
