#include "paged_common.cuh"
namespace kv4 {
namespace paged { int prefix_status_fetch(int* out) { *out = 0; return 0; } }
int paged_prefix_splits(int, int, int, int) { return 0; }
int launch_paged_prefix(const yskn_paged_cache&, const yskn_paged_rows&, const yskn_paged_attn_args&, int, const paged::Work&, cudaStream_t) { return 0; }
}
