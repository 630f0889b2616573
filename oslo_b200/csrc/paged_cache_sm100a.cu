// Storing new tokens in a paged key / value cache.
//
//   oslo_paged_kv_append   q' = R(p) q,  k' = R(p) k  (rotary embedding at the token's own position p), then k' and v go to row
//                          p % page_size of page table[b, p / page_size].  One pass: every input is read once and every
//                          output written once, so the kernel is bound by HBM for prompts (8 x 1999 tokens, 32 heads of
//                          128, 591 MB in 100 us: 92% of the copy bandwidth) and by launch latency for single tokens
//                          (2.8 us for one, 3.6 us for 256).
//
// Pools are [pages, kv_heads, page_size, head_dim]: the tokens of one head inside a page are contiguous, which is what the
// attention over the pages streams.
#include "common.cuh"
#include "step_args.h"

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

// How the 16-byte chunks of a head pair up under the rotation.
enum : int {
  kRotateHalves = 0,  // chunk c with chunk c + rot / (2 E): a thread takes both, and turns every head by the same angles
  kRotateInside = 1,  // neighbouring elements, or no rotation: a chunk is on its own
  kRotateElements = 2,  // halves that no 16-byte chunk boundary separates: partners are read one by one
};

template <typename T, int MODE>
struct HeadTurn {
  static constexpr int E = PagedVec<T>::E;
  static constexpr int N = MODE == kRotateHalves ? 2 : 1;  // chunks of a thread
  PagedVec<T> x[N];

  static OSLO_DEVINL int columns(int d, int rot) { return MODE == kRotateHalves ? (d - rot / 2) / E : d / E; }
  // first element of column c's chunk n; halves: columns below rot / 2 are pairs, the others chunks behind the rotated part
  static OSLO_DEVINL int dim(int c, int n, int rot) { return MODE != kRotateHalves ? c * E : c * E < rot / 2 ? c * E + n * (rot / 2) : c * E + rot / 2; }
  static OSLO_DEVINL int chunks(int c, int rot) { return MODE == kRotateHalves && c * E < rot / 2 ? 2 : 1; }

  OSLO_DEVINL void load(const T* head, int c, int rot) {
    x[0] = pg_ld(head + dim(c, 0, rot));
    if constexpr (N == 2) {
      if (chunks(c, rot) == 2) x[N - 1] = pg_ld(head + dim(c, 1, rot));
    }
  }
  OSLO_DEVINL void turn(const T* head, int c, int rot, const float (&cs)[E], const float (&sn)[E], const float* cos_row, const float* sin_row) {
    if constexpr (MODE == kRotateHalves) {
      if (chunks(c, rot) == 1) return;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float a = pg_f(x[0].v[e]), b = pg_f(x[N - 1].v[e]);
        x[0].v[e] = pg_t<T>(a * cs[e] - b * sn[e]);
        x[N - 1].v[e] = pg_t<T>(b * cs[e] + a * sn[e]);
      }
    } else if constexpr (MODE == kRotateInside) {  // pair j of the chunk turns by angle j
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        if (c * E + e >= rot) break;
        const float a = pg_f(x[0].v[e]), b = pg_f(x[0].v[e + 1]);
        x[0].v[e] = pg_t<T>(a * cs[e / 2] - b * sn[e / 2]);
        x[0].v[e + 1] = pg_t<T>(b * cs[e / 2] + a * sn[e / 2]);
      }
    } else {
      const int half = rot / 2;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = c * E + e;
        if (i >= rot) break;
        const bool low = i < half;
        const int j = low ? i : i - half;
        const float a = pg_f(x[0].v[e]), b = pg_f(head[low ? i + half : i - half]);
        x[0].v[e] = pg_t<T>(low ? a * cos_row[j] - b * sin_row[j] : a * cos_row[j] + b * sin_row[j]);
      }
    }
  }
  OSLO_DEVINL void store(T* head, int c, int rot) const {
    pg_st(head + dim(c, 0, rot), x[0]);
    if constexpr (N == 2) {
      if (chunks(c, rot) == 2) pg_st(head + dim(c, 1, rot), x[N - 1]);
    }
  }
};

// Small blocks: 8 prompts of up to 1999 tokens, 32 heads of 128, take 100 us with 64 or 128 threads a block, 110 us with 256 and
// 169 us with 512 (the copy bandwidth gives 92 us); with 8 key heads of 64 and neighbouring pairs 34, 39, 67 and 123 us.
constexpr int kAppendThreads = 64;
constexpr int kAppendRows = 2;  // heads of a thread in flight

// Block (token, part of its heads).  A thread keeps one column (chunk or pair of chunks) and walks over the heads of queries and
// keys, so it reads its angles once; the values are copied in the same way.  The chain start -> page -> store is three
// trips to memory: the first heads and values of a real token are read before it, the angles beside it.
template <typename T, int MODE>
__global__ void __launch_bounds__(kAppendThreads, MODE == kRotateElements ? 12 : 16) paged_append_kernel(const PagedAppendParams p, int parts) {
  using H = HeadTurn<T, MODE>;
  constexpr int E = PagedVec<T>::E;
  const int token = blockIdx.x / parts, part = blockIdx.x - token * parts;
  const int b = token / p.s, i = token - b * p.s;
  const int start = p.start[b], count = p.count ? p.count[b] : p.s;
  const T* q = static_cast<const T*>(p.q) + b * p.q_sb + i * p.q_ss;
  const T* k = static_cast<const T*>(p.k) + b * p.k_sb + i * p.k_ss;
  const T* v = static_cast<const T*>(p.v) + b * p.v_sb + i * p.v_ss;
  T* q_out = static_cast<T*>(p.q_out) + static_cast<long long>(token) * p.hq * p.d;
  const int rot = p.cosb != nullptr ? p.rot : 0, rows = p.hq + p.hkv;
  const auto source = [&](int r) { return r < p.hq ? q + r * p.q_sh : k + (r - p.hq) * p.k_sh; };

  const int columns = H::columns(p.d, rot), r0 = threadIdx.x / columns, c = threadIdx.x - r0 * columns;
  const int step = kAppendThreads / columns, stride = parts * step;
  const bool real = i < count;
  int r = r0 < step && real ? part * step + r0 : rows;
  H h[kAppendRows];
#pragma unroll
  for (int j = 0; j < kAppendRows; ++j)
    if (r + j * stride < rows) h[j].load(source(r + j * stride), c, rot);
  const int v_columns = p.d / E, v_r0 = threadIdx.x / v_columns, v_c = threadIdx.x - v_r0 * v_columns;
  const int v_step = kAppendThreads / v_columns, v_stride = parts * v_step;
  int vr = v_r0 < v_step && real ? part * v_step + v_r0 : p.hkv;
  PagedVec<T> x[kAppendRows];
#pragma unroll
  for (int j = 0; j < kAppendRows; ++j)
    if (vr + j * v_stride < p.hkv) x[j] = pg_ld(v + (vr + j * v_stride) * p.v_sh + v_c * E);

  // a real token needs a page, a row and a rotation; one without them is reported and treated as padding
  const long long pos = static_cast<long long>(start) + i;
  const long long at = pos / p.page_size;
  const bool known = real && pos >= 0 && at < p.max_pages && (rot == 0 || pos < p.positions);
  const int page = known ? p.table[b * p.table_stride + at] : -1;
  const float* cos_row = rot && known ? p.cosb + pos * (rot / 2) : nullptr;
  const float* sin_row = rot && known ? p.sinb + pos * (rot / 2) : nullptr;
  float cs[E], sn[E];
  if (cos_row) {
    if constexpr (MODE == kRotateHalves) {
      if (c * E < rot / 2) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
          *reinterpret_cast<float4*>(cs + e) = *reinterpret_cast<const float4*>(cos_row + c * E + e);
          *reinterpret_cast<float4*>(sn + e) = *reinterpret_cast<const float4*>(sin_row + c * E + e);
        }
      }
    } else if constexpr (MODE == kRotateInside) {
#pragma unroll
      for (int e = 0; e < E / 2; ++e)
        if (c * E + 2 * e < rot) cs[e] = cos_row[c * E / 2 + e], sn[e] = sin_row[c * E / 2 + e];
    }
  }
  if (page < 0 || page >= p.num_pages) {
    if (real && threadIdx.x == 0) atomicCAS(p.status, kStatusOk, kStatusPageRange);
    const int n = p.hq * (p.d / E);
    for (int y = part * kAppendThreads + threadIdx.x; y < n; y += parts * kAppendThreads)
      *reinterpret_cast<uint4*>(q_out + static_cast<long long>(y) * E) = make_uint4(0, 0, 0, 0);
    return;
  }
  const long long in_page = (pos - at * p.page_size) * p.d;
  T* kd = static_cast<T*>(p.k_pages) + page * p.kp_page + in_page;
  T* vd = static_cast<T*>(p.v_pages) + page * p.vp_page + in_page;
  while (r < rows) {
#pragma unroll
    for (int j = 0; j < kAppendRows; ++j) {
      const int rr = r + j * stride;
      if (rr < rows) {
        h[j].turn(source(rr), c, rot, cs, sn, cos_row, sin_row);
        h[j].store(rr < p.hq ? q_out + rr * p.d : kd + (rr - p.hq) * p.kp_head, c, rot);
      }
    }
    r += stride * kAppendRows;
#pragma unroll
    for (int j = 0; j < kAppendRows; ++j)
      if (r + j * stride < rows) h[j].load(source(r + j * stride), c, rot);
  }
  while (vr < p.hkv) {
#pragma unroll
    for (int j = 0; j < kAppendRows; ++j)
      if (vr + j * v_stride < p.hkv) pg_st(vd + (vr + j * v_stride) * p.vp_head + v_c * E, x[j]);
    vr += v_stride * kAppendRows;
#pragma unroll
    for (int j = 0; j < kAppendRows; ++j)
      if (vr + j * v_stride < p.hkv) x[j] = pg_ld(v + (vr + j * v_stride) * p.v_sh + v_c * E);
  }
}

template <typename T>
int paged_append_launch(const PagedAppendParams& p, cudaStream_t st) {
  constexpr int E = PagedVec<T>::E;
  const int rot = p.cosb ? p.rot : 0;
  int mode = kRotateInside;
  if (rot && p.neox) {
    const bool whole = rot % (2 * E) == 0 && ((reinterpret_cast<uintptr_t>(p.cosb) | reinterpret_cast<uintptr_t>(p.sinb)) & 15) == 0;
    mode = whole ? kRotateHalves : kRotateElements;
  }
  const long long tokens = static_cast<long long>(p.b) * p.s;
  // A token's heads are cut over several blocks only as far as there are too few tokens to fill the GPU.
  const int columns = mode == kRotateHalves ? (p.d - rot / 2) / E : p.d / E;
  const long long rounds = (static_cast<long long>(p.hq + p.hkv) * columns + kAppendThreads - 1) / kAppendThreads;
  const long long parts = tokens >= 592 ? 1 : (592 + tokens - 1) / tokens < rounds ? (592 + tokens - 1) / tokens : rounds;
  if (tokens * parts > 0x7fffffffll) return -1;
  const unsigned grid = static_cast<unsigned>(tokens * parts);
  const int n = static_cast<int>(parts);
  if (mode == kRotateHalves) paged_append_kernel<T, kRotateHalves><<<grid, kAppendThreads, 0, st>>>(p, n);
  else if (mode == kRotateInside) paged_append_kernel<T, kRotateInside><<<grid, kAppendThreads, 0, st>>>(p, n);
  else paged_append_kernel<T, kRotateElements><<<grid, kAppendThreads, 0, st>>>(p, n);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace oslo

extern "C" int oslo_paged_kv_append(const OsloPagedAppendArgs* a) {
  using namespace oslo;
  if (a->b <= 0 || a->s <= 0) return 0;
  if (a->hkv <= 0 || a->d <= 0 || a->d % 8 || a->page_size <= 0 || a->rot < 0 || a->rot > a->d || a->rot % 2) return -1;
  PagedAppendParams p;
  p.q = reinterpret_cast<const void*>(a->q), p.k = reinterpret_cast<const void*>(a->k), p.v = reinterpret_cast<const void*>(a->v);
  p.q_out = reinterpret_cast<void*>(a->q_out), p.k_pages = reinterpret_cast<void*>(a->k_pages);
  p.v_pages = reinterpret_cast<void*>(a->v_pages), p.table = reinterpret_cast<const int*>(a->table);
  p.start = reinterpret_cast<const int*>(a->start), p.count = reinterpret_cast<const int*>(a->count);
  // tables without positions have no address: another one stands for them, nothing is read there
  p.cosb = reinterpret_cast<const float*>(a->rot == 0 ? 0 : a->positions > 0 ? a->cosb : a->status);
  p.sinb = reinterpret_cast<const float*>(a->rot == 0 ? 0 : a->positions > 0 ? a->sinb : a->status);
  p.status = reinterpret_cast<int*>(a->status);
  p.q_sb = a->q_b, p.q_ss = a->q_s, p.q_sh = a->q_h, p.k_sb = a->k_b, p.k_ss = a->k_s, p.k_sh = a->k_h;
  p.v_sb = a->v_b, p.v_ss = a->v_s, p.v_sh = a->v_h;
  p.kp_page = a->k_page, p.kp_head = a->k_head, p.vp_page = a->v_page, p.vp_head = a->v_head, p.table_stride = a->table_row;
  p.b = a->b, p.s = a->s, p.hq = a->q ? a->hq : 0, p.hkv = a->hkv, p.d = a->d, p.rot = a->rot, p.neox = a->neox;
  p.positions = a->positions, p.page_size = a->page_size, p.max_pages = a->max_pages, p.num_pages = a->num_pages;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a->stream);
  if (a->b * a->s > 0x7fffffffll || p.d / 4 > kAppendThreads) return -1;
  if (a->dtype == 0) return paged_append_launch<float>(p, st);
  if (a->dtype == 1) return paged_append_launch<__half>(p, st);
  if (a->dtype == 2) return paged_append_launch<__nv_bfloat16>(p, st);
  return -1;
}
