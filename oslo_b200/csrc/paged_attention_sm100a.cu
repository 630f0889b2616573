// Entry points of the attention over a paged key / value cache; the kernels are in paged_attention_core.cuh, and their 16-bit forms
// are compiled beside this file.
#include "paged_attention_core.cuh"
#include "step_args.h"

namespace oslo {
int paged_attention_f32(PagedAttnParams& p, int block_rows, PagedAttnPlan& plan, bool run, void* ws, cudaStream_t st) {
  return paged_attention_type<float>(p, block_rows, plan, run, ws, st);
}
}  // namespace oslo

extern "C" {

static bool paged_attention_params(const OsloPagedAttentionArgs* a, oslo::PagedAttnParams& p) {
  if (a->hkv <= 0 || a->group <= 0 || a->d <= 0 || a->d > 256 || a->d % 8 || a->page_size <= 0 || a->page_size % 16) return false;
  if (a->b > 0x3fffffff || a->s > 0x3fffffff || a->group > 0x3fffffff || a->s * a->group > 0x3fffffff) return false;
  if (a->hkv > 0x3fffffff || a->b * a->hkv > 0x3fffffff) return false;
  const bool together = a->mask_len < 0 || a->mask_s == 0;  // the query tokens of a sequence share what they see but for the last ones
  const long long rows = together ? a->s * a->group : a->group, groups = a->b * a->hkv * (together ? 1 : a->s);
  const long long most = oslo::paged_attention_rows(a->dtype, a->d, rows, groups),
                  tiles = (rows + most - 1) / most;
  if (a->b * a->s > 0x3fffffff || a->max_pages * a->page_size > 0x3fffffff || groups * tiles * 8 > 0x3fffffff) return false;
  p.q = reinterpret_cast<const void*>(a->q), p.k = reinterpret_cast<const void*>(a->k_pages), p.v = reinterpret_cast<const void*>(a->v_pages);
  p.mask = reinterpret_cast<const float*>(a->mask), p.out = reinterpret_cast<void*>(a->out);
  p.table = reinterpret_cast<const int*>(a->table), p.lens = reinterpret_cast<const int*>(a->lens);
  p.status = reinterpret_cast<int*>(a->status);
  p.q_sb = a->q_b, p.q_ss = a->q_s, p.q_sh = a->q_h, p.k_page = a->k_page, p.k_head = a->k_head, p.v_page = a->v_page;
  p.v_head = a->v_head, p.table_stride = a->table_row, p.m_sb = a->mask_b, p.m_ss = a->mask_s;
  p.b = a->b, p.s = a->s, p.hkv = a->hkv, p.group = a->group, p.d = a->d, p.page_size = a->page_size, p.max_pages = a->max_pages;
  p.num_pages = a->num_pages, p.mask_len = a->mask_len, p.scale = static_cast<float>(a->scale), p.row_tiles = static_cast<int>(tiles);
  p.queries = together ? 1 : static_cast<int>(a->s), p.rows = static_cast<int>(rows);
  return true;
}

static int paged_attention_call(const OsloPagedAttentionArgs* a, oslo::PagedAttnPlan& plan, bool run) {
  using namespace oslo;
  PagedAttnParams p{};
  if (!paged_attention_params(a, p)) return -1;
  const int rows = paged_attention_rows(a->dtype, a->d, p.rows, static_cast<long long>(p.b) * p.queries * p.hkv);
  void* ws = reinterpret_cast<void*>(a->workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a->stream);
  if (a->dtype == 0) return paged_attention_f32(p, rows, plan, run, ws, st);
  if (a->dtype == 1) return paged_attention_f16(p, rows, plan, run, ws, st);
  if (a->dtype == 2) return paged_attention_bf16(p, rows, plan, run, ws, st);
  return -1;
}

// Bytes of workspace that the call needs on the current device; negative: an error.
long long oslo_paged_attention_workspace_bytes(const OsloPagedAttentionArgs* a) {
  if (a->b <= 0 || a->s <= 0) return 0;
  oslo::PagedAttnPlan plan{};
  const int rc = paged_attention_call(a, plan, false);
  return rc ? rc : plan.bytes;
}

int oslo_paged_attention(const OsloPagedAttentionArgs* a) {
  if (a->b <= 0 || a->s <= 0) return 0;
  oslo::PagedAttnPlan plan{};
  return paged_attention_call(a, plan, true);
}
}
