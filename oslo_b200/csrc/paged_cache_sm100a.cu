// Storing new tokens in a paged key / value cache.
//
//   oslo_paged_kv_append   q' = R(p) q,  k' = R(p) k  (rotary embedding at the token's own position p), then k' and v go to row
//                          p % page_size of page table[b, p / page_size].  One pass: every input is read once and every
//                          output written once, so the kernel is bound by HBM for prompts and by launch latency for single
//                          tokens.
//
// Pools are [pages, kv_heads, page_size, head_dim]: the tokens of one head inside a page are contiguous, which is what the
// attention over the pages streams.  A thread moves 16 bytes of one head; the half-rotation partner (rot / 2 elements away) is
// read by a second 16-byte load that hits L1, because the warp that owns those elements loads them too.
#include "common.cuh"

namespace oslo {

struct PagedAppendParams {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;  // [b, s, hq, d] contiguous
  void* k_pages;
  void* v_pages;
  const int* table;
  const int* start;
  const int* count;  // null: all s tokens are real
  const float* cosb;  // [positions, rot / 2]; null: no rotation
  const float* sinb;
  int* status;
  long long q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;  // element strides of batch, token, head
  long long kp_page, kp_head, vp_page, vp_head, table_stride;
  int b, s, hq, hkv, d, rot, neox, positions, page_size, max_pages, num_pages;
};

template <typename T>
struct PagedVec {  // 16 bytes of T
  static constexpr int E = 16 / sizeof(T);
  T v[E];
};
OSLO_DEVINL float pg_f(float x) { return x; }
OSLO_DEVINL float pg_f(__half x) { return __half2float(x); }
OSLO_DEVINL float pg_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
OSLO_DEVINL T pg_t(float x);
template <>
OSLO_DEVINL float pg_t<float>(float x) { return x; }
template <>
OSLO_DEVINL __half pg_t<__half>(float x) { return __float2half_rn(x); }
template <>
OSLO_DEVINL __nv_bfloat16 pg_t<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T>
OSLO_DEVINL PagedVec<T> pg_ld(const T* p) {
  PagedVec<T> r;
  *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
  return r;
}
template <typename T>
OSLO_DEVINL void pg_st(T* p, const PagedVec<T>& r) { *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r); }

// Elements [c * E, c * E + E) of one head, rotated.  `x` points at the head's element 0.
template <typename T>
OSLO_DEVINL PagedVec<T> rotate_chunk(const T* x, int c, const float* cs, const float* sn, int rot, bool neox) {
  constexpr int E = PagedVec<T>::E;
  PagedVec<T> own = pg_ld(x + c * E);
  const int d0 = c * E;
  if (d0 >= rot) return own;
  PagedVec<T> out = own;
  const int half = rot / 2;
  if (!neox) {  // pairs (2j, 2j + 1) lie inside the chunk
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const int dim = d0 + e;
      if (dim < rot) {
        const float a = pg_f(own.v[e]), b = pg_f(own.v[e + 1]), cc = cs[dim / 2], ss = sn[dim / 2];
        out.v[e] = pg_t<T>(a * cc - b * ss);
        out.v[e + 1] = pg_t<T>(b * cc + a * ss);
      }
    }
    return out;
  }
  if (half % E == 0) {  // the partners are one aligned chunk too
    const bool low = d0 < half;
    const PagedVec<T> other = pg_ld(x + (low ? d0 + half : d0 - half));
    const int j = low ? d0 : d0 - half;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float a = pg_f(own.v[e]), b = pg_f(other.v[e]), cc = cs[j + e], ss = sn[j + e];
      out.v[e] = pg_t<T>(low ? a * cc - b * ss : a * cc + b * ss);
    }
    return out;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int dim = d0 + e;
    if (dim < rot) {
      const bool low = dim < half;
      const int j = low ? dim : dim - half;
      const float a = pg_f(own.v[e]), b = pg_f(x[low ? dim + half : dim - half]);
      out.v[e] = pg_t<T>(low ? a * cs[j] - b * sn[j] : a * cs[j] + b * sn[j]);
    }
  }
  return out;
}

// Block (token, part): the rows (heads of q, then k, then v) of one token, cut into 16-byte chunks.
template <typename T>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedAppendParams p, int parts) {
  constexpr int E = PagedVec<T>::E;
  const int token = blockIdx.x / parts, part = blockIdx.x % parts;
  const int b = token / p.s, i = token % p.s;
  const int cpr = p.d / E;
  const int chunks = (p.hq + 2 * p.hkv) * cpr;
  const bool real = p.count == nullptr || i < p.count[b];
  const long long pos = static_cast<long long>(p.start[b]) + i;
  bool ok = real;
  int page = 0;
  if (real) {
    const long long at = pos / p.page_size;
    ok = pos >= 0 && at < p.max_pages && (p.cosb == nullptr || pos < p.positions);
    if (ok) {
      page = p.table[b * p.table_stride + at];
      ok = page >= 0 && page < p.num_pages;
    }
    if (!ok && threadIdx.x == 0) atomicCAS(p.status, kStatusOk, kStatusPageRange);
  }
  const int row_in_page = ok ? static_cast<int>(pos % p.page_size) : 0;
  const float* cs = p.cosb != nullptr && ok ? p.cosb + pos * (p.rot / 2) : nullptr;
  const float* sn = p.cosb != nullptr && ok ? p.sinb + pos * (p.rot / 2) : nullptr;
  const int rot = p.cosb != nullptr ? p.rot : 0;
  for (int idx = part * blockDim.x + threadIdx.x; idx < chunks; idx += parts * blockDim.x) {
    const int row = idx / cpr, c = idx - row * cpr;
    if (row < p.hq) {
      T* dst = static_cast<T*>(p.q_out) + (static_cast<long long>(token) * p.hq + row) * p.d + c * E;
      if (ok) {
        const T* src = static_cast<const T*>(p.q) + b * p.q_sb + i * p.q_ss + row * p.q_sh;
        pg_st(dst, rotate_chunk(src, c, cs, sn, rot, p.neox != 0));
      } else {
        *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
      }
    } else if (ok) {
      const int h = row - p.hq;
      if (h < p.hkv) {
        const T* src = static_cast<const T*>(p.k) + b * p.k_sb + i * p.k_ss + h * p.k_sh;
        T* dst = static_cast<T*>(p.k_pages) + page * p.kp_page + h * p.kp_head + static_cast<long long>(row_in_page) * p.d + c * E;
        pg_st(dst, rotate_chunk(src, c, cs, sn, rot, p.neox != 0));
      } else {
        const T* src = static_cast<const T*>(p.v) + b * p.v_sb + i * p.v_ss + (h - p.hkv) * p.v_sh;
        T* dst =
            static_cast<T*>(p.v_pages) + page * p.vp_page + (h - p.hkv) * p.vp_head + static_cast<long long>(row_in_page) * p.d + c * E;
        pg_st(dst, pg_ld(src + c * E));
      }
    }
  }
}

}  // namespace oslo

// Everything a call needs, eight bytes each.  Strides in elements.
struct OsloPagedAppendArgs {
  long long q, k, v, q_out, k_pages, v_pages, table, start, count, cosb, sinb, status, stream;  // addresses; q, count, cosb may be 0
  long long q_b, q_s, q_h, k_b, k_s, k_h, v_b, v_s, v_h, k_page, k_head, v_page, v_head, table_row;
  long long b, s, hq, hkv, d, rot, neox, positions, page_size, max_pages, num_pages, dtype;
};

extern "C" int oslo_paged_kv_append(const OsloPagedAppendArgs* a) {
  using namespace oslo;
  if (a->b <= 0 || a->s <= 0) return 0;
  if (a->hkv <= 0 || a->d <= 0 || a->d % 8 || a->page_size <= 0 || a->rot < 0 || a->rot > a->d || a->rot % 2) return -1;
  PagedAppendParams p;
  p.q = reinterpret_cast<const void*>(a->q), p.k = reinterpret_cast<const void*>(a->k), p.v = reinterpret_cast<const void*>(a->v);
  p.q_out = reinterpret_cast<void*>(a->q_out), p.k_pages = reinterpret_cast<void*>(a->k_pages);
  p.v_pages = reinterpret_cast<void*>(a->v_pages), p.table = reinterpret_cast<const int*>(a->table);
  p.start = reinterpret_cast<const int*>(a->start), p.count = reinterpret_cast<const int*>(a->count);
  p.cosb = reinterpret_cast<const float*>(a->rot ? a->cosb : 0), p.sinb = reinterpret_cast<const float*>(a->rot ? a->sinb : 0);
  p.status = reinterpret_cast<int*>(a->status);
  p.q_sb = a->q_b, p.q_ss = a->q_s, p.q_sh = a->q_h, p.k_sb = a->k_b, p.k_ss = a->k_s, p.k_sh = a->k_h;
  p.v_sb = a->v_b, p.v_ss = a->v_s, p.v_sh = a->v_h;
  p.kp_page = a->k_page, p.kp_head = a->k_head, p.vp_page = a->v_page, p.vp_head = a->v_head, p.table_stride = a->table_row;
  p.b = a->b, p.s = a->s, p.hq = a->q ? a->hq : 0, p.hkv = a->hkv, p.d = a->d, p.rot = a->rot, p.neox = a->neox;
  p.positions = a->positions, p.page_size = a->page_size, p.max_pages = a->max_pages, p.num_pages = a->num_pages;
  const int e = a->dtype == 0 ? 4 : 8;
  const long long chunks = static_cast<long long>(p.hq + 2 * p.hkv) * (p.d / e);
  const long long parts = (chunks + 255) / 256;
  if (a->b * a->s * parts > 0x7fffffffll) return -1;
  const unsigned grid = static_cast<unsigned>(a->b * a->s * parts);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a->stream);
  if (a->dtype == 0) paged_append_kernel<float><<<grid, 256, 0, st>>>(p, static_cast<int>(parts));
  else if (a->dtype == 1) paged_append_kernel<__half><<<grid, 256, 0, st>>>(p, static_cast<int>(parts));
  else if (a->dtype == 2) paged_append_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p, static_cast<int>(parts));
  else return -1;
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
