// The attention over a paged key / value cache for __nv_bfloat16.
#include "paged_attention_core.cuh"

namespace oslo {
int paged_attention_bf16(PagedAttnParams& p, int block_rows, PagedAttnPlan& plan, bool run, void* ws, cudaStream_t st) {
  return paged_attention_type<__nv_bfloat16>(p, block_rows, plan, run, ws, st);
}
}  // namespace oslo
