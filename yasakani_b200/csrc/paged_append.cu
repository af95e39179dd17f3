// Rows of several sequences into a paged 16-bit cache (sm_100a): keys and queries rotated at each row's position on the way, and the mean key of every
// page that a row completes.
//
// Mathematics: channels (c, c + rd/2), c < rd/2, of a head turn by the angle of (position, c): (a, b) -> (a cos - b sin, b cos + a sin), fp32, rounded once.
// Mean of a page: fp32 sum of its `page` rows in a fixed order, times 1 / page (a power of two, exact), rounded once.
//
// Bound: bytes.  Every row is read and written once, 16 bytes a lane; a warp holds whole heads (hd 256: one, hd 128: two), so the other channel of a pair
// is in another lane of the same warp and comes by a shuffle.
#include "paged_common.cuh"

namespace kv4 {
namespace paged {
namespace {

struct AppendP {
  Rows R; int rows;
  const uint16_t* k_in; const uint16_t* v_in; const uint16_t* q_in; uint16_t* q_out;
  long long ks, vs, qs;
  const float* rope; int rope_rows, rd, nh;
  uint16_t* k; uint16_t* v;
  int spr;                                   // slots (256 channels) of a row: heads of q, k, v one after the other
  int wpr;                                   // warps that share a row
};

constexpr int SLOTS = 4;                     // 16-byte loads a lane has in flight: 4 KB a warp

// One warp per SLOTS * 256 channels of a row.  The rows' own loads do not wait for the position; the table entry does.
template <int HD, bool BF>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendP P) {
  constexpr int LPH = HD / 8;                // lanes of a head
  pdl_wait();
  pdl_launch();
  const int w = (int)((blockIdx.x * 256u + threadIdx.x) >> 5), lane = threadIdx.x & 31;
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
      x[i] = *reinterpret_cast<const uint4*>(src + ch);
    }
  }
  const int s = P.R.seq[row], pos = P.R.pos[row];
  if (s < 0 || s >= P.R.seqs || pos < 0 || (P.rd > 0 && pos >= P.rope_rows)) return;          // the same for the whole warp
  const int b = pos >> P.R.lp;
  const int page = b < P.R.blocks ? page_of(P.R, s, b) : -1;
  const int half = P.rd / 2, lh = half / 8;                            // lanes of half the rotated channels
  float cs[8], sn[8];
  if (ch < P.rd) {
    const float4* t = reinterpret_cast<const float4*>(P.rope + ((size_t)pos * half + (ch < half ? ch : ch - half)) * 2);
    #pragma unroll
    for (int e = 0; e < 4; ++e) { const float4 f = t[e]; cs[2 * e] = f.x; sn[2 * e] = f.y; cs[2 * e + 1] = f.z; sn[2 * e + 1] = f.w; }
  }
  const int partner = ch < half ? lane + lh : ch < P.rd ? lane - lh : lane;
  #pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    uint4 y = x[i];
    if (P.rd > 0) {
      uint4 o;
      o.x = __shfl_sync(0xffffffffu, y.x, partner); o.y = __shfl_sync(0xffffffffu, y.y, partner);
      o.z = __shfl_sync(0xffffffffu, y.z, partner); o.w = __shfl_sync(0xffffffffu, y.w, partner);
      if (ch < P.rd && vh[i] < nq + kvh) {
        const uint32_t a4[4] = {y.x, y.y, y.z, y.w}, b4[4] = {o.x, o.y, o.z, o.w};
        uint32_t r[4];
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 a = unpack16<BF>(a4[e]), d = unpack16<BF>(b4[e]);
          const float sx = ch < half ? -sn[2 * e] : sn[2 * e], sy = ch < half ? -sn[2 * e + 1] : sn[2 * e + 1];
          r[e] = pack16<BF>(fmaf(d.x, sx, a.x * cs[2 * e]), fmaf(d.y, sy, a.y * cs[2 * e + 1]));
        }
        y = make_uint4(r[0], r[1], r[2], r[3]);
      }
    }
    if (vh[i] < 0) continue;
    uint16_t* dst;
    if (vh[i] < nq) dst = P.q_out + ((size_t)row * P.nh + vh[i]) * HD;
    else {
      if (page < 0) continue;
      const int h = vh[i] - nq;
      const size_t at = (((size_t)page * kvh + (h < kvh ? h : h - kvh)) << P.R.lp) + (pos & (P.R.page - 1));
      dst = (h < kvh ? P.k : P.v) + at * HD;
    }
    *reinterpret_cast<uint4*>(dst + ch) = y;
  }
}

// Mean keys.  A block looks at 32 rows and one kv-head; most rows complete no page.  The warps take the page's rows in turn, 16 bytes a lane; their sums
// go through shared memory.
template <int HD, bool BF>
__global__ void __launch_bounds__(128) paged_mean_kernel(const AppendP P, uint16_t* kmean) {
  constexpr int LPH = HD / 8, GROUPS = 128 / LPH;                      // lanes of a row; rows in flight
  __shared__ float part[GROUPS][HD];
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, h = blockIdx.y, r0 = (int)blockIdx.x * 32;
  int page = -1;
  if (r0 + lane < P.rows) {
    const int s = P.R.seq[r0 + lane], pos = P.R.pos[r0 + lane];
    if (s >= 0 && s < P.R.seqs && pos >= 0 && !(P.rd > 0 && pos >= P.rope_rows) && ((pos + 1) & (P.R.page - 1)) == 0 && (pos >> P.R.lp) < P.R.blocks)
      page = page_of(P.R, s, pos >> P.R.lp);
  }
  unsigned todo = __ballot_sync(0xffffffffu, page >= 0);                // the same in every warp of the block
  while (todo) {
    const int pg = __shfl_sync(0xffffffffu, page, __ffs(todo) - 1);
    todo &= todo - 1;
    const int grp = threadIdx.x / LPH, ch = 8 * (threadIdx.x % LPH);
    const uint16_t* src = P.k + (((size_t)pg * P.R.kvh + h) << P.R.lp) * HD + ch;
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    #pragma unroll 4
    for (int t = grp; t < P.R.page; t += GROUPS) {
      const uint4 u = *reinterpret_cast<const uint4*>(src + (size_t)t * HD);
      const uint32_t u4[4] = {u.x, u.y, u.z, u.w};
      #pragma unroll
      for (int e = 0; e < 4; ++e) { const float2 f = unpack16<BF>(u4[e]); sum[2 * e] += f.x; sum[2 * e + 1] += f.y; }
    }
    #pragma unroll
    for (int e = 0; e < 8; ++e) part[grp][ch + e] = sum[e];
    __syncthreads();
    for (int x = 2 * (int)threadIdx.x; x < HD; x += 256) {
      float a = 0.f, b = 0.f;
      #pragma unroll
      for (int i = 0; i < GROUPS; ++i) { a += part[i][x]; b += part[i][x + 1]; }
      const float inv = 1.f / (float)P.R.page;
      *reinterpret_cast<uint32_t*>(kmean + ((size_t)pg * P.R.kvh + h) * HD + x) = pack16<BF>(a * inv, b * inv);
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace paged

int launch_paged_append(const yskn_paged_cache& c, const yskn_paged_rows& r, const yskn_paged_append_args& a, cudaStream_t st) {
  using namespace paged;
  const bool bf = c.dtype == YSKN_KV4_BF16;
  AppendP P{rows_of(c, r, 0), r.rows, static_cast<const uint16_t*>(a.k_in), static_cast<const uint16_t*>(a.v_in), static_cast<const uint16_t*>(a.q_in),
            static_cast<uint16_t*>(a.q_out), a.k_stride, a.v_stride, a.q_stride, a.rope, a.rope_rows, a.rd, a.nh,
            static_cast<uint16_t*>(c.k), static_cast<uint16_t*>(c.v), 0, 0};
  const long long heads = (a.q_in ? a.nh : 0) + 2ll * c.kvh;
  P.spr = (int)((heads * c.hd + 255) / 256);
  P.wpr = (P.spr + SLOTS - 1) / SLOTS;
  const long long blocks = ((long long)r.rows * P.wpr + 7) / 8;
  if (blocks >= 1ll << 23) KV4_REJECT("yskn_kv4_paged_append: too many rows (%d) for one call", r.rows);
  auto kern = c.hd == 256 ? (bf ? paged_append_kernel<256, true> : paged_append_kernel<256, false>)
                          : (bf ? paged_append_kernel<128, true> : paged_append_kernel<128, false>);
  if (int rc = launch_pdl("paged_append_kernel", kern, dim3((unsigned)blocks), 256, 0, st, P)) return rc;
  if (!c.kmean) return 0;
  auto mean = c.hd == 256 ? (bf ? paged_mean_kernel<256, true> : paged_mean_kernel<256, false>)
                          : (bf ? paged_mean_kernel<128, true> : paged_mean_kernel<128, false>);
  return launch_pdl("paged_mean_kernel", mean, dim3((unsigned)((r.rows + 31) / 32), (unsigned)c.kvh), 128, 0, st, P, static_cast<uint16_t*>(c.kmean));
}

}  // namespace kv4
