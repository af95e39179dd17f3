// extern "C" surface of the paged 16-bit cache: argument checks, the tensor maps of a cache.
#include "paged_common.cuh"
#include <algorithm>
#include <cstring>

namespace kv4 {
namespace paged {
namespace {

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr; cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// [rows][hd] as (64 channels, rows, hd / 64 blocks): a box of (64, box_rows, box_blocks) lands as [block][row][128 bytes], 128-byte swizzle.
bool encode(uint64_t* out, void* base, const yskn_paged_cache& c, int box_rows, int box_blocks) {
  EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {64, (cuuint64_t)c.pages * c.kvh * c.page, (cuuint64_t)(c.hd / 64)}, strides[2] = {(cuuint64_t)c.hd * 2, 128};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, (cuuint32_t)box_blocks}, es[3] = {1, 1, 1};
  alignas(64) CUtensorMap m;
  static_assert(sizeof(m) == sizeof(uint64_t) * 16, "yskn_paged_cache.maps");
  const bool ok = fn(&m, c.dtype == YSKN_KV4_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims, strides, box, es,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  if (ok) memcpy(out, &m, sizeof(m));
  return ok;
}

bool odd16(const void* p) { return ((uintptr_t)p & 15) != 0; }

int check_cache(const yskn_paged_cache* c, const char* who) {
  if (!c || !c->k || !c->v) KV4_REJECT("%s: null cache array", who);
  if (c->hd != 128 && c->hd != 256) KV4_REJECT("%s: head_dim %d is neither 128 nor 256", who, c->hd);
  if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128) KV4_REJECT("%s: page of %d tokens (16, 32, 64 or 128)", who, c->page);
  if (c->dtype != YSKN_KV4_F16 && c->dtype != YSKN_KV4_BF16) KV4_REJECT("%s: the cache's rows are F16 or BF16", who);
  // rows are addressed by a 32-bit coordinate, and a tile of rows outside the arrays has to lie below its limit too
  if (c->pages <= 0 || c->kvh <= 0 || c->kvh > 4096 || (long long)c->pages * c->kvh > (0x7fffffffll - 1024) / c->page)
    KV4_REJECT("%s: bad shape (pages %d, kvh %d, page %d)", who, c->pages, c->kvh, c->page);
  if (odd16(c->k) || odd16(c->v) || odd16(c->kmean)) KV4_REJECT("%s: cache arrays must be 16-byte aligned", who);
  return 0;
}

int check_rows(const yskn_paged_cache* c, const yskn_paged_rows* r, const char* who) {
  if (int rc = check_cache(c, who)) return rc;
  if (!c->ready) KV4_REJECT("%s: yskn_kv4_paged_init has not been called for this cache", who);
  if (!r) KV4_REJECT("%s: null argument struct", who);
  if (r->rows < 0) KV4_REJECT("%s: rows %d", who, r->rows);
  if (r->rows == 0) return 0;
  if (!r->table || !r->seq || !r->pos) KV4_REJECT("%s: null buffer", who);
  if (r->seqs <= 0 || r->blocks <= 0 || (long long)r->blocks * c->page > 0x7fffffffll - 1024)
    KV4_REJECT("%s: bad table (%d sequences of %d blocks)", who, r->seqs, r->blocks);
  return 0;
}

int check_heads(const yskn_paged_cache* c, const yskn_paged_rows* r, const void* q, int64_t q_stride, int nh, const char* who) {
  if (nh <= 0 || nh % c->kvh || nh / c->kvh > 16) KV4_REJECT("%s: %d heads over %d kv-heads (a multiple, at most 16 times)", who, nh, c->kvh);
  if (!q) KV4_REJECT("%s: null buffer", who);
  if (odd16(q) || q_stride % 8 || q_stride < (int64_t)nh * c->hd) KV4_REJECT("%s: q must be 16-byte aligned, its rows %lld elements apart at least and a multiple of 8",
                                                                            who, (long long)nh * c->hd);
  if (r->rows > 65535) KV4_REJECT("%s: %d rows (at most 65535)", who, r->rows);
  return 0;
}

}  // namespace
}  // namespace paged
}  // namespace kv4

using namespace kv4;
using namespace kv4::paged;

extern "C" {

int yskn_kv4_paged_init(yskn_paged_cache* c) {
  if (c) c->ready = 0;
  if (int rc = check_cache(c, "yskn_kv4_paged_init")) return rc;
  const int chunk = std::min(c->page, 64);
  if (!encode(c->maps[0], c->k, *c, chunk, c->hd / 64) || !encode(c->maps[1], c->v, *c, chunk, c->hd / 64) || !encode(c->maps[2], c->k, *c, chunk, 1) ||
      !encode(c->maps[3], c->v, *c, chunk, 1))
    KV4_REJECT("yskn_kv4_paged_init: cuTensorMapEncodeTiled failed or is unavailable");
  c->ready = 1;
  return 0;
}

int yskn_kv4_paged_append(const yskn_paged_cache* c, const yskn_paged_rows* r, const yskn_paged_append_args* a, void* cuda_stream) {
  const char* who = "yskn_kv4_paged_append";
  if (int rc = check_rows(c, r, who)) return rc;
  if (!a) KV4_REJECT("%s: null argument struct", who);
  if (r->rows == 0) return 0;
  if (!a->k_in || !a->v_in || (a->q_in && !a->q_out)) KV4_REJECT("%s: null buffer", who);
  if (a->rd < 0 || a->rd > c->hd || a->rd % 16) KV4_REJECT("%s: rotary width %d is no multiple of 16 up to %d", who, a->rd, c->hd);
  if (a->rd > 0 && (!a->rope || a->rope_rows <= 0)) KV4_REJECT("%s: rotary width %d needs a rope table", who, a->rd);
  const int64_t kv = (int64_t)c->kvh * c->hd;
  if (odd16(a->k_in) || odd16(a->v_in) || odd16(a->q_in) || odd16(a->q_out) || odd16(a->rope) || a->k_stride % 8 || a->v_stride % 8 || a->k_stride < kv || a->v_stride < kv)
    KV4_REJECT("%s: rows and rope table must be 16-byte aligned, rows %lld elements apart at least and a multiple of 8", who, (long long)kv);
  if (a->q_in && (a->nh <= 0 || a->nh > 65536 || a->q_stride % 8 || a->q_stride < (int64_t)a->nh * c->hd))
    KV4_REJECT("%s: bad queries (%d heads, rows %lld elements apart)", who, a->nh, (long long)a->q_stride);
  return launch_paged_append(*c, *r, *a, (cudaStream_t)cuda_stream);
}

int yskn_kv4_paged_select(const yskn_paged_cache* c, const yskn_paged_rows* r, const yskn_paged_select_args* a, void* cuda_stream) {
  const char* who = "yskn_kv4_paged_select";
  if (int rc = check_rows(c, r, who)) return rc;
  if (!a) KV4_REJECT("%s: null argument struct", who);
  if (!c->kmean) KV4_REJECT("%s: the cache keeps no mean keys", who);
  if (r->rows == 0) return 0;
  if (int rc = check_heads(c, r, a->q, a->q_stride, a->nh, who)) return rc;
  if (!a->ids) KV4_REJECT("%s: null buffer", who);
  if (a->take < 2 || a->take > 1024) KV4_REJECT("%s: take %d (2 to 1024)", who, a->take);
  const size_t need = paged_select_bytes(*c, r->rows, r->blocks);
  if (!a->workspace || a->workspace_bytes < need) KV4_REJECT("%s: workspace of %zu bytes needed, %zu given", who, need, a->workspace ? a->workspace_bytes : (size_t)0);
  if ((uintptr_t)a->workspace & 255) KV4_REJECT("%s: the workspace must be 256-byte aligned", who);
  return launch_paged_select(*c, *r, *a, (cudaStream_t)cuda_stream);
}

int yskn_kv4_paged_attention(const yskn_paged_cache* c, const yskn_paged_rows* r, const yskn_paged_attn_args* a, void* cuda_stream) {
  const char* who = "yskn_kv4_paged_attention";
  if (int rc = check_rows(c, r, who)) return rc;
  if (!a) KV4_REJECT("%s: null argument struct", who);
  if (r->rows == 0) return 0;
  if (int rc = check_heads(c, r, a->q, a->q_stride, a->nh, who)) return rc;
  if (!a->o16 || odd16(a->o16)) KV4_REJECT("%s: o16 must be 16-byte aligned", who);
  if (a->shared < 0 || a->shared % c->page || a->shared > (long long)r->blocks * c->page)
    KV4_REJECT("%s: a shared part of %d tokens is no multiple of the page (%d) within the table", who, a->shared, c->page);
  if (a->ids && a->shared > 0) KV4_REJECT("%s: chosen blocks and a shared part exclude one another", who);
  if (a->ids && (a->take <= 0 || (long long)a->take * c->page > 0x7fffffffll - 1024)) KV4_REJECT("%s: take %d", who, a->take);
  const long long tiles = (((a->ids ? (long long)a->take : (long long)r->blocks) * c->page) + TILE - 1) / TILE + 1;         // and a step without a tile
  if (tiles * std::min(r->rows, 224) * c->kvh > 0x7fffffffll) KV4_REJECT("%s: %d rows of up to %lld tokens are too many for one call", who, r->rows, tiles * TILE);
  const size_t need = paged_attention_bytes(*c, r->rows, a->nh, a->shared);
  if (!a->workspace || a->workspace_bytes < need) KV4_REJECT("%s: workspace of %zu bytes needed, %zu given", who, need, a->workspace ? a->workspace_bytes : (size_t)0);
  if ((uintptr_t)a->workspace & 255) KV4_REJECT("%s: the workspace must be 256-byte aligned", who);
  return launch_paged_attention(*c, *r, *a, (cudaStream_t)cuda_stream);
}

size_t yskn_kv4_paged_workspace_bytes(const yskn_paged_cache* c, int rows, int nh, int shared, int blocks) {
  if (check_cache(c, "yskn_kv4_paged_workspace_bytes")) return 0;
  if (rows <= 0 || rows > 65535 || nh <= 0 || nh % c->kvh || nh / c->kvh > 16 || shared < 0 || shared % c->page || blocks < 0) {
    set_error("yskn_kv4_paged_workspace_bytes: bad shape (rows %d, nh %d, shared %d, blocks %d)", rows, nh, shared, blocks);
    return 0;
  }
  const size_t n = paged_attention_bytes(*c, rows, nh, shared);
  return blocks > 0 ? std::max(n, paged_select_bytes(*c, rows, blocks)) : n;
}

}  // extern "C"
