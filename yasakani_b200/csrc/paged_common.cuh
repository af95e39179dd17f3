// Declarations shared by the kernels of the paged 16-bit cache (paged_append.cu, paged_select.cu, paged_attn.cu, paged_prefix.cu).
#pragma once
#include "kv4_common.cuh"
#include <cuda.h>

namespace kv4 {
namespace paged {

constexpr int SMS = 148;
constexpr int TILE = 64;                     // tokens of one step of the attention kernel
constexpr float LOG2E = 1.4426950408889634f;

// What every kernel needs of the cache and of the call's rows.
struct Rows {
  const int* table; int seqs, blocks;        // page of block b of sequence s at table[s * blocks + b]
  const int* seq; const int* pos;            // of each row
  int pages, kvh, page, lp;                  // page = 1 << lp tokens
};

// A row's place: sequence, and how many tokens it sees.  seq < 0: the row is padding.
// PAST_L1: for kernels that read places and pages without a wait of their own, behind one that has waited; what an SM holds from before is then not dropped for them.
struct Place { int seq, vis; };
template <bool PAST_L1 = false> __device__ __forceinline__ int read_index(const int* p) { return PAST_L1 ? __ldcg(p) : *p; }
template <bool PAST_L1 = false> __device__ __forceinline__ Place place_of(const Rows& R, int row) {
  const int s = read_index<PAST_L1>(R.seq + row), p = read_index<PAST_L1>(R.pos + row);
  Place w;
  w.seq = s >= 0 && s < R.seqs ? s : -1;
  const long long cap = (long long)R.blocks << R.lp;
  w.vis = w.seq < 0 || p < 0 ? 0 : (long long)p + 1 < cap ? p + 1 : (int)cap;
  return w;
}
// Page of block b of sequence s; -1 where the table names none.
template <bool PAST_L1 = false> __device__ __forceinline__ int page_of(const Rows& R, int s, int b) {
  const int p = read_index<PAST_L1>(R.table + (size_t)s * R.blocks + b);
  return p >= 0 && p < R.pages ? p : -1;
}

// A box's first token for a row that sees `vis` tokens.  One without a token of the row's (NO_TOKEN among them) stands at `vis`, so that offsets into it can be added.
constexpr int NO_TOKEN = 0x7fffffff;
__host__ __device__ __forceinline__ int box_base(int base, int vis) { return base < vis ? base : vis; }
// Of two 16-bit values in a register, tokens 0 and 1 of the n that the row still sees from there: those that it sees.
__host__ __device__ __forceinline__ uint32_t keep_pair(int n) { return (n > 0 ? 0xffffu : 0u) | (n > 1 ? 0xffff0000u : 0u); }

// ---------------------------------------------------------------------------------------------------------------- PTX
constexpr uint32_t WAIT_LIMIT = 1u << 22;    // polls before a wait gives up
__device__ __forceinline__ uint32_t s_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void bar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {          // bounded; false = gave up
  for (uint32_t i = 0; i < WAIT_LIMIT; ++i) if (bar_try(bar, parity)) return true;
  return false;
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* m, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(m), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void bulk_1d(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
template <bool BF> __device__ __forceinline__ uint32_t pack16(float lo, float hi) {        // two values rounded to the 16-bit type
  uint32_t d;
  if (BF) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// Two weights of a softmax rounded to the 16-bit type.  fp16's largest number stands for what is beyond it, as only scores have whose own steps are of that size.
template <bool BF> __device__ __forceinline__ uint32_t pack_weights(float lo, float hi) {
  if (BF) return pack16<true>(lo, hi);
  uint32_t d;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
template <bool BF> __device__ __forceinline__ float2 unpack16(uint32_t w) {
  if (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  const __half2 h = *reinterpret_cast<const __half2*>(&w);
  return __half22float2(h);
}
// D[16 x 8] += A[16 x 16] B[16 x 8] of 16-bit operands, fp32 sums: one warp.
template <bool BF> __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF) asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
              : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
           : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v; asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory"); return v;
}
__device__ __forceinline__ void sts128(uint32_t a, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Workspace of one attention call.  Of (row, kv-head) pairs that lie on several CTAs: the first and the last, and a piece from each, (m, l) and O of the pair's heads.
// Partials over the shared prefix, [row][split][head].
struct Work {
  int2* span; float2* ml; float* pacc; float2* qml; float* qacc;
  size_t bytes;
};

}  // namespace paged

int launch_paged_append(const yskn_paged_cache& c, const yskn_paged_rows& r, const yskn_paged_append_args& a, cudaStream_t st);
int launch_paged_select(const yskn_paged_cache& c, const yskn_paged_rows& r, const yskn_paged_select_args& a, cudaStream_t st);
int launch_paged_attention(const yskn_paged_cache& c, const yskn_paged_rows& r, const yskn_paged_attn_args& a, cudaStream_t st);
size_t paged_attention_bytes(const yskn_paged_cache& c, int rows, int nh, int shared);
size_t paged_select_bytes(const yskn_paged_cache& c, int rows, int blocks);
int paged_prefix_splits(int rows, int g, int kvh, int shared);
size_t paged_prefix_parts(int rows, int g, int kvh, int shared);
int launch_paged_prefix(const yskn_paged_cache& c, const yskn_paged_rows& r, const yskn_paged_attn_args& a, int splits, const paged::Work& w, cudaStream_t st);

namespace paged {
inline Rows rows_of(const yskn_paged_cache& c, const yskn_paged_rows& r, int first) {
  int lp = 0;
  while ((1 << lp) < c.page) ++lp;
  return Rows{r.table, r.seqs, r.blocks, r.seq + first, r.pos + first, c.pages, c.kvh, c.page, lp};
}
}  // namespace paged
}  // namespace kv4
