// Argument structs of the decoding step's entry points: eight bytes a field, so that Python can pack them with one format and
// csrc/torch/step_calls.cpp fills them directly.  Addresses may be 0 where a comment says so; strides are in elements.
#pragma once

extern "C" {

struct OsloPagedAppendArgs {
  long long q, k, v, q_out, k_pages, v_pages, table, start, count, cosb, sinb, status, stream;  // q and count may be 0
  long long q_b, q_s, q_h, k_b, k_s, k_h, v_b, v_s, v_h, k_page, k_head, v_page, v_head, table_row;
  long long b, s, hq, hkv, d, rot, neox, positions, page_size, max_pages, num_pages, dtype;  // rot = 0: no rotation
};

struct OsloPagedAttentionArgs {
  long long q, k_pages, v_pages, table, lens, mask, out, workspace, status, stream;
  long long q_b, q_s, q_h, k_page, k_head, v_page, v_head, table_row, mask_b, mask_s;
  long long b, s, hkv, group, d, page_size, max_pages, num_pages, mask_len, dtype;  // mask_len < 0: no mask (an empty one has no address)
  double scale;
};

struct OsloProcessLogitsArgs {
  long long x, y, tokens, token_lens, prompt_lens, rep, pres, freq, bias, allowed, stream;  // from tokens on they may be 0
  long long x_stride, y_stride, tok_stride, bias_stride, allowed_stride, rows, vocab, history, tok64, dtype;
  double rep_s, pres_s, freq_s;
};

}  // extern "C"
