// The attention over a paged key / value cache for __half.
#include "paged_attention_core.cuh"

namespace oslo {
int paged_attention_f16(PagedAttnParams& p, int block_rows, PagedAttnPlan& plan, bool run, void* ws, cudaStream_t st) {
  return paged_attention_type<__half>(p, block_rows, plan, run, ws, st);
}
}  // namespace oslo
