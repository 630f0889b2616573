// Attention of the newest tokens over a paged key / value cache.
//
//   o = softmax(scale * q K^T + mask) V   over the tokens of the sequence's pages that the query sees; a query that sees none
//   gives zeros.
//
// Every key and value is used by `group` query heads only, so HBM bounds it: 4 * head_dim bytes a token and key head against
// 4 * group * head_dim operations.
//
// Work is cut into units of 64 tokens (32 for fp32) of one (query token, key head, block of query heads), a "segment" being all
// units of one such triple.  As many blocks as the GPU holds at once take equal, contiguous ranges of units, found on the
// device from the lengths: one long sequence occupies every SM, a ragged batch leaves none idle, and the host needs to know
// no length.  Inside a block each of four warps walks every fourth 16-token tile (8 for fp32) with its own running maximum,
// sum and output; the four are joined when the segment or the range ends.  Segments that several blocks share are joined by a
// second kernel, launched programmatically so that its start overlaps the first one's end; the parts are added in block order,
// so results do not depend on timing.
//
// The tiles go from HBM straight into the registers in the layout that mma.sync wants as its B operand, 16 bytes per load and
// without shared memory, because the order of the summed index is free as long as both operands share it:
//   scores   lane (r, q) = (lane / 4, lane % 4) holds 16 contiguous bytes of key r; Q is loaded with the same pattern.
//   output   the accumulator columns of the scores (tokens 2q, 2q + 1) are the A operand's summed index, so lane (r, q) loads
//            the values of exactly those tokens, 16 bytes at head dim r * E of each 8 E wide block.
// The probabilities enter the second product as the sum of two 16-bit numbers (high part and remainder), which keeps 16 bits
// and more of each; fp32 inputs are split in the same way into tf32 parts (three products), which keeps 21 bits.
#include "common.cuh"

namespace oslo {

struct PagedAttnParams {
  const void* q;
  const void* k;
  const void* v;
  const float* mask;  // additive, [b, s, mask_len] by strides; null: none
  void* out;          // [b, s, hq, d] contiguous
  const int* table;
  const int* lens;
  int* status;
  long long q_sb, q_ss, q_sh, k_page, k_head, v_page, v_head, table_stride, m_sb, m_ss;
  float* part_o;   // [grid, 2, RT, DP] unnormalised outputs of shared segments: 0 = begun by an earlier block, 1 = begun here
  float2* part_ml;  // [grid, 2, RT] their maxima and sums
  int4* shared_seg;  // [grid] of the segment begun earlier that ends here: (first block, query, key head, first row); x < 0: none
  int b, s, hkv, group, d, page_size, max_pages, num_pages, mask_len, row_tiles;
  float scale;
};

//: units a block takes at least
constexpr int kMinUnits = 2;

constexpr float kLog2e = 1.4426950408889634f;

OSLO_DEVINL uint4 ldg16(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
OSLO_DEVINL float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
struct Mma16;  // D[16 x 8] += A[16 x 16] B[16 x 8], 16-bit operands
template <>
struct Mma16<__nv_bfloat16> {
  static OSLO_DEVINL void run(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static OSLO_DEVINL uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(r);
  }
  static OSLO_DEVINL float low(uint32_t r) { return __uint_as_float(r << 16); }
  static OSLO_DEVINL float high(uint32_t r) { return __uint_as_float(r & 0xffff0000u); }
};
template <>
struct Mma16<__half> {
  static OSLO_DEVINL void run(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static OSLO_DEVINL uint32_t pack(float lo, float hi) {
    const __half2 r = __floats2half2_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(r);
  }
  static OSLO_DEVINL float low(uint32_t r) { return __low2float(reinterpret_cast<const __half2&>(r)); }
  static OSLO_DEVINL float high(uint32_t r) { return __high2float(reinterpret_cast<const __half2&>(r)); }
};
// D[16 x 8] += A[16 x 8] B[8 x 8], tf32 operands
OSLO_DEVINL void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
OSLO_DEVINL uint32_t tf32_hi(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
OSLO_DEVINL uint32_t tf32_lo(float x, uint32_t hi) { return tf32_hi(x - __uint_as_float(hi)); }
// a * b with both split: the product of the two remainders (2^-22 relative) is left out
OSLO_DEVINL void mma_3xtf32(float (&c)[4], const float (&a)[4], float b0, float b1) {
  const uint32_t h0 = tf32_hi(a[0]), h1 = tf32_hi(a[1]), h2 = tf32_hi(a[2]), h3 = tf32_hi(a[3]);
  const uint32_t g0 = tf32_hi(b0), g1 = tf32_hi(b1);
  mma_tf32(c, tf32_lo(a[0], h0), tf32_lo(a[1], h1), tf32_lo(a[2], h2), tf32_lo(a[3], h3), g0, g1);
  mma_tf32(c, h0, h1, h2, h3, tf32_lo(b0, g0), tf32_lo(b1, g1));
  mma_tf32(c, h0, h1, h2, h3, g0, g1);
}

// s / l, zeros where nothing was seen
OSLO_DEVINL void pa_store(float* dst, float4 s, float l) {
  const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
  *reinterpret_cast<float4*>(dst) = make_float4(s.x * inv, s.y * inv, s.z * inv, s.w * inv);
}
template <typename T>
OSLO_DEVINL void pa_store(T* dst, float4 s, float l) {
  const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
  uint2 r;
  r.x = Mma16<T>::pack(s.x * inv, s.y * inv), r.y = Mma16<T>::pack(s.z * inv, s.w * inv);
  *reinterpret_cast<uint2*>(dst) = r;
}

// T: element type; DP: head_dim rounded up to 64, 128 or 256; WIDE: 9 to 16 query heads per block instead of up to 8
template <typename T, int DP, bool WIDE, bool MASK>
struct PagedAttn {
  static constexpr int E = 16 / sizeof(T);           // elements of one load
  static constexpr int TT = sizeof(T) == 2 ? 16 : 8;  // tokens of one tile
  static constexpr int NT = TT / 8;
  static constexpr int KC = DP / (4 * E);   // loads per key and lane
  static constexpr int VC = DP / (8 * E);   // loads per value and lane
  static constexpr int VT = TT / 4;         // value tokens of a lane
  static constexpr int RT = WIDE ? 16 : 8;  // query rows
  static constexpr int ROW = DP + 4;        // padded row of the joining buffer
  static constexpr int WARPS = 4;
  // Blocks an SM should hold: enough loads in flight to cover HBM's latency (8 KB a warp and tile) without spilling.
  static constexpr int BLOCKS = DP == 64 ? (sizeof(T) == 2 ? 4 : 2) : DP == 128 && sizeof(T) == 2 && !WIDE ? 3 : 2;
  static constexpr size_t kSmem = sizeof(float) * (WARPS * RT * ROW + 2 * WARPS * RT);

  uint4 q0[KC], q1[WIDE ? KC : 1];
  float o[VC][E][WIDE ? 4 : 2];
  float m0, m1, l0, l1;

  OSLO_DEVINL void load_q(const PagedAttnParams& p, const T* q, int row0) {
    const int r = (threadIdx.x & 31) >> 2, quad = threadIdx.x & 3;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int dim = c * 4 * E + quad * E;
      q0[c] = row0 + r < p.group && dim < p.d ? ldg16(q + (row0 + r) * p.q_sh + dim) : make_uint4(0, 0, 0, 0);
      if constexpr (WIDE)
        q1[c] = row0 + r + 8 < p.group && dim < p.d ? ldg16(q + (row0 + r + 8) * p.q_sh + dim) : make_uint4(0, 0, 0, 0);
    }
  }
  OSLO_DEVINL void clear() {
    m0 = m1 = -INFINITY;
    l0 = l1 = 0.f;
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int x = 0; x < (WIDE ? 4 : 2); ++x) o[j][e][x] = 0.f;
  }

  // One tile: its TT tokens start at `token`; the tile's keys and values at k, v; tokens at or past `limit` are not seen.
  OSLO_DEVINL void tile(const PagedAttnParams& p, const T* k, const T* v, int token, int limit, const float* mask) {
    const int lane = threadIdx.x & 31, r = lane >> 2, quad = lane & 3;
    uint4 kr[NT][KC], vr[VT][VC];
    float add[NT][2];
    bool seen[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int t = token + n * 8 + quad * 2 + x;
        seen[n][x] = t < limit;
        add[n][x] = 0.f;
        if constexpr (MASK) {
          if (seen[n][x]) add[n][x] = mask[t];
          seen[n][x] = seen[n][x] && add[n][x] != -INFINITY;
        }
      }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const int dim = c * 4 * E + quad * E;
        kr[n][c] = dim < p.d ? ldg16(k + (n * 8 + r) * p.d + dim) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
    for (int t = 0; t < VT; ++t)
#pragma unroll
      for (int c = 0; c < VC; ++c) {
        const int dim = c * 8 * E + r * E;
        // a token that is not seen may hold anything: its values never enter the product
        vr[t][c] = dim < p.d && seen[t >> 1][t & 1] ? ldg16(v + ((t >> 1) * 8 + quad * 2 + (t & 1)) * p.d + dim) : make_uint4(0, 0, 0, 0);
      }
    float sc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint4 qa = q0[c], qb = WIDE ? q1[WIDE ? c : 0] : make_uint4(0, 0, 0, 0);
        if constexpr (sizeof(T) == 2) {
          Mma16<T>::run(sc[n], qa.x, qb.x, qa.y, qb.y, kr[n][c].x, kr[n][c].y);
          Mma16<T>::run(sc[n], qa.z, qb.z, qa.w, qb.w, kr[n][c].z, kr[n][c].w);
        } else {
          const float a[4] = {__uint_as_float(qa.x), __uint_as_float(qb.x), __uint_as_float(qa.y), __uint_as_float(qb.y)};
          const float b[4] = {__uint_as_float(qa.z), __uint_as_float(qb.z), __uint_as_float(qa.w), __uint_as_float(qb.w)};
          mma_3xtf32(sc[n], a, __uint_as_float(kr[n][c].x), __uint_as_float(kr[n][c].y));
          mma_3xtf32(sc[n], b, __uint_as_float(kr[n][c].z), __uint_as_float(kr[n][c].w));
        }
      }
    }
    float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        sc[n][x] = seen[n][x] ? score(p, sc[n][x], add[n][x]) : -INFINITY;
        t0 = fmaxf(t0, sc[n][x]);
        if constexpr (WIDE) {
          sc[n][2 + x] = seen[n][x] ? score(p, sc[n][2 + x], add[n][x]) : -INFINITY;
          t1 = fmaxf(t1, sc[n][2 + x]);
        }
      }
    t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
    t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2));
    if constexpr (WIDE) {
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
    }
    if (__any_sync(0xffffffffu, t0 > m0 || (WIDE && t1 > m1))) {  // a new maximum: what was summed is scaled to it
      const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
      const float f0 = weight(m0, n0), f1 = WIDE ? weight(m1, n1) : 0.f;
      m0 = n0, m1 = n1;
      l0 *= f0, l1 *= f1;
#pragma unroll
      for (int j = 0; j < VC; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          o[j][e][0] *= f0, o[j][e][1] *= f0;
          if constexpr (WIDE) o[j][e][2] *= f1, o[j][e][3] *= f1;
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        sc[n][x] = weight(sc[n][x], m0);
        l0 += sc[n][x];
        if constexpr (WIDE) {
          sc[n][2 + x] = weight(sc[n][2 + x], m1);
          l1 += sc[n][2 + x];
        }
      }
    if constexpr (sizeof(T) == 2) {
      uint32_t hi[4], lo[4];  // A operand: rows r / r + 8 of tokens 2q.. and 8 + 2q..
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int x = 0; x < (WIDE ? 2 : 1); ++x) {
          const float a = sc[n][2 * x], b = sc[n][2 * x + 1];
          const uint32_t h = Mma16<T>::pack(a, b);
          hi[2 * n + x] = h;
          lo[2 * n + x] = Mma16<T>::pack(a - Mma16<T>::low(h), b - Mma16<T>::high(h));
        }
      if constexpr (!WIDE) hi[1] = hi[3] = lo[1] = lo[3] = 0;
#pragma unroll
      for (int j = 0; j < VC; ++j) {
        const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&vr[0][j]);
        const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&vr[1][j]);
        const uint32_t* w2 = reinterpret_cast<const uint32_t*>(&vr[2][j]);
        const uint32_t* w3 = reinterpret_cast<const uint32_t*>(&vr[3][j]);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t sel = e & 1 ? 0x7632 : 0x5410;
          const uint32_t b0 = __byte_perm(w0[e / 2], w1[e / 2], sel), b1 = __byte_perm(w2[e / 2], w3[e / 2], sel);
          float c[4] = {o[j][e][0], o[j][e][1], WIDE ? o[j][e][WIDE ? 2 : 0] : 0.f, WIDE ? o[j][e][WIDE ? 3 : 0] : 0.f};
          Mma16<T>::run(c, hi[0], hi[1], hi[2], hi[3], b0, b1);
          Mma16<T>::run(c, lo[0], lo[1], lo[2], lo[3], b0, b1);
          o[j][e][0] = c[0], o[j][e][1] = c[1];
          if constexpr (WIDE) o[j][e][2] = c[2], o[j][e][3] = c[3];
        }
      }
    } else {
      const float a[4] = {sc[0][0], WIDE ? sc[0][2] : 0.f, sc[0][1], WIDE ? sc[0][3] : 0.f};
#pragma unroll
      for (int j = 0; j < VC; ++j) {
        const float* w0 = reinterpret_cast<const float*>(&vr[0][j]);
        const float* w1 = reinterpret_cast<const float*>(&vr[1][j]);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float c[4] = {o[j][e][0], o[j][e][1], WIDE ? o[j][e][WIDE ? 2 : 0] : 0.f, WIDE ? o[j][e][WIDE ? 3 : 0] : 0.f};
          mma_3xtf32(c, a, w0[e], w1[e]);
          o[j][e][0] = c[0], o[j][e][1] = c[1];
          if constexpr (WIDE) o[j][e][2] = c[2], o[j][e][3] = c[3];
        }
      }
    }
  }

  // With a mask the scores stay in natural units: a mask of the type's lowest value times log2(e) would leave its range.
  static OSLO_DEVINL float score(const PagedAttnParams& p, float s, float add) {
    return MASK ? fmaf(s, p.scale, add) : s * (p.scale * kLog2e);
  }
  // exp(x - m); m = -inf: nothing was seen yet
  static OSLO_DEVINL float weight(float x, float m) {
    const float mm = m == -INFINITY ? 0.f : m;
    return ex2(MASK ? (x - mm) * kLog2e : x - mm);
  }

  // Joins the warps' sums.  Afterwards every thread may read row sums / maxima (ml) and the output (buf, unnormalised).
  OSLO_DEVINL void join(float* buf, float* ml) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, quad = lane & 3;
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    if (quad == 0) {
      ml[warp * RT + r] = m0;
      if constexpr (WIDE) ml[warp * RT + 8 + r] = m1;
    }
    __syncthreads();
    float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      top0 = fmaxf(top0, ml[w * RT + r]);
      if constexpr (WIDE) top1 = fmaxf(top1, ml[w * RT + 8 + r]);
    }
    const float f0 = weight(m0, top0), f1 = WIDE ? weight(m1, top1) : 0.f;
    if (quad == 0) {
      ml[WARPS * RT + warp * RT + r] = l0 * f0;
      if constexpr (WIDE) ml[WARPS * RT + warp * RT + 8 + r] = l1 * f1;
    }
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int x = 0; x < (WIDE ? 4 : 2); ++x) {
        float* dst = buf + (warp * RT + r + (x >> 1) * 8) * ROW + j * 8 * E + (quad * 2 + (x & 1)) * E;
        const float f = x >> 1 ? f1 : f0;
#pragma unroll
        for (int e = 0; e < E; e += 4)
          *reinterpret_cast<float4*>(dst + e) = make_float4(o[j][e][x] * f, o[j][e + 1][x] * f, o[j][e + 2][x] * f, o[j][e + 3][x] * f);
      }
    __syncthreads();
  }
};

// The tokens a query sees, as far as the table (and the mask) reach.
template <bool MASK>
OSLO_DEVINL int query_limit(const PagedAttnParams& p, int query, bool report) {
  const int b = query / p.s, i = query - b * p.s;
  const long long limit = static_cast<long long>(p.lens[b]) - p.s + 1 + i;
  const int cap = MASK ? min(p.mask_len, p.max_pages * p.page_size) : p.max_pages * p.page_size;
  if (limit > cap && report) atomicCAS(p.status, kStatusOk, kStatusPageRange);
  return static_cast<int>(min(max(limit, 0ll), static_cast<long long>(cap)));
}

template <typename T, int DP, bool WIDE, bool MASK>
__global__ void __launch_bounds__(128, PagedAttn<T, DP, WIDE, MASK>::BLOCKS) paged_attention_kernel(const PagedAttnParams p) {
  using A = PagedAttn<T, DP, WIDE, MASK>;
  constexpr int UNIT = A::WARPS * A::TT;
  extern __shared__ float4 smem4[];
  __shared__ long long scan[A::WARPS + 2];
  float* buf = reinterpret_cast<float*>(smem4);
  float* ml = buf + A::WARPS * A::RT * A::ROW;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // This block's range of units: an exclusive prefix sum of the queries' units over the block's threads, each of which owns a
  // contiguous run of queries.  A query without tokens is one unit, so that its zeros are written.
  const int queries = p.b * p.s, run = (queries + 127) / 128;
  const int first = min(queries, static_cast<int>(threadIdx.x) * run), last = min(queries, first + run);
  long long mine = 0;
  for (int i = first; i < last; ++i) mine += max(1, (query_limit<MASK>(p, i, false) + UNIT - 1) / UNIT);
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long n = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += n;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  long long before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < A::WARPS; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  const int heads = p.hkv * p.row_tiles;  // segments of a query
  const long long units = total * heads;
  const long long blocks = min(static_cast<long long>(gridDim.x), max(1ll, units / kMinUnits));
  if (threadIdx.x == 0) p.shared_seg[blockIdx.x] = make_int4(-1, 0, 0, 0);
  if (blockIdx.x >= blocks) return;
  long long u = units * blockIdx.x / blocks;
  const long long u_end = units * (blockIdx.x + 1) / blocks;
  const long long at = u / heads;
  __syncthreads();
  if (mine > 0 && at >= before && at < before + mine) {
    int i = first;
    long long n;
    while (at >= before + (n = max(1, (query_limit<MASK>(p, i, false) + UNIT - 1) / UNIT))) before += n, ++i;
    scan[0] = i;
    scan[1] = before;
  }
  __syncthreads();
  int query = static_cast<int>(scan[0]);
  long long base = scan[1] * heads;  // first unit of the query
  int limit = query_limit<MASK>(p, query, threadIdx.x == 0);
  int n_units = max(1, (limit + UNIT - 1) / UNIT);

  while (u < u_end) {
    if (u >= base + static_cast<long long>(n_units) * heads) {
      base += static_cast<long long>(n_units) * heads;
      ++query;
      limit = query_limit<MASK>(p, query, threadIdx.x == 0);
      n_units = max(1, (limit + UNIT - 1) / UNIT);
    }
    const int seg = static_cast<int>((u - base) / n_units);
    const int a = static_cast<int>((u - base) - static_cast<long long>(seg) * n_units);
    const int e = static_cast<int>(min(static_cast<long long>(n_units), a + (u_end - u)));
    const int h = seg / p.row_tiles, row0 = (seg - h * p.row_tiles) * A::RT;
    const int b = query / p.s, i = query - b * p.s;

    A acc;
    acc.load_q(p, static_cast<const T*>(p.q) + b * p.q_sb + i * p.q_ss + static_cast<long long>(h) * p.group * p.q_sh, row0);
    acc.clear();
    const float* mask = MASK ? p.mask + b * p.m_sb + i * p.m_ss : nullptr;
    const int* table = p.table + b * p.table_stride;
    const int end = min(limit, e * UNIT);
    int t = a * UNIT + warp * A::TT;
    int page = t < end ? table[t / p.page_size] : 0;
    while (t < end) {
      const int next = t + UNIT, next_page = next < end ? table[next / p.page_size] : 0;
      if (page >= 0 && page < p.num_pages) {
        const long long in_page = static_cast<long long>(t % p.page_size) * p.d;
        acc.tile(p, static_cast<const T*>(p.k) + page * p.k_page + h * p.k_head + in_page,
                 static_cast<const T*>(p.v) + page * p.v_page + h * p.v_head + in_page, t, limit, mask);
      } else if (lane == 0) {
        atomicCAS(p.status, kStatusOk, kStatusPageRange);
      }
      t = next, page = next_page;
    }
    acc.join(buf, ml);

    const bool whole = a == 0 && e == n_units;
    const long long slot = static_cast<long long>(blockIdx.x) * 2 + (a == 0 ? 1 : 0);
    T* out = static_cast<T*>(p.out) + (static_cast<long long>(query) * p.hkv + h) * p.group * p.d;
    for (int x = threadIdx.x; x < A::RT * (DP / 4); x += blockDim.x) {
      const int row = x / (DP / 4), dim = x % (DP / 4) * 4;
      if (row0 + row >= p.group || dim >= p.d) continue;
      float l = 0.f, m = -INFINITY;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < A::WARPS; ++w) {
        l += ml[(A::WARPS + w) * A::RT + row];
        m = fmaxf(m, ml[w * A::RT + row]);
        const float4 y = *reinterpret_cast<const float4*>(buf + (w * A::RT + row) * A::ROW + dim);
        s.x += y.x, s.y += y.y, s.z += y.z, s.w += y.w;
      }
      if (whole) {
        pa_store(out + (row0 + row) * p.d + dim, s, l);
      } else {
        *reinterpret_cast<float4*>(p.part_o + (slot * A::RT + row) * DP + dim) = s;
        if (dim == 0) p.part_ml[slot * A::RT + row] = make_float2(m, l);
      }
    }
    if (threadIdx.x == 0 && a > 0 && e == n_units) {
      const long long start = base + static_cast<long long>(seg) * n_units;
      p.shared_seg[blockIdx.x] = make_int4(static_cast<int>(((start + 1) * blocks - 1) / units), query, h, row0);
    }
    u += e - a;
    __syncthreads();  // buf is free for the next segment
  }
}

// Joins a segment that several blocks of the first kernel share.  Block (row, last block of the segment); warp w adds every
// eighth part, then the warps' sums are added.
template <typename T, int DP, bool WIDE, bool MASK>
__global__ void __launch_bounds__(256) paged_attention_join_kernel(const PagedAttnParams p) {
  using A = PagedAttn<T, DP, WIDE, MASK>;
  constexpr int V = DP / 128 > 0 ? DP / 128 : 1;  // float4s of a lane
  constexpr int LANES = DP / 4 < 32 ? DP / 4 : 32;
  __shared__ float4 sums[8][DP / 4];
  __shared__ float red[8];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 seg = p.shared_seg[blockIdx.y];
  const int row = blockIdx.x;
  if (seg.x < 0 || seg.w + row >= p.group) return;
  const int parts = blockIdx.y - seg.x + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const auto slot = [&](int i) { return (static_cast<long long>(seg.x + i) * 2 + (i == 0 ? 1 : 0)) * A::RT + row; };
  float m = -INFINITY;
  for (int i = threadIdx.x; i < parts; i += 256) m = fmaxf(m, p.part_ml[slot(i)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w]);
  __syncthreads();
  float l = 0.f;
  float4 o[V];
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = warp; i < parts; i += 8) {
    const float2 x = p.part_ml[slot(i)];
    const float w = A::weight(x.x, m);
    l += x.y * w;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int dim = (j * 32 + lane) * 4;
      if (lane < LANES && dim < p.d) {
        const float4 y = *reinterpret_cast<const float4*>(p.part_o + slot(i) * DP + dim);
        o[j].x += y.x * w, o[j].y += y.y * w, o[j].z += y.z * w, o[j].w += y.w * w;
      }
    }
  }
  if (lane == 0) red[warp] = l;
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (lane < LANES) sums[warp][j * 32 + lane] = o[j];
  __syncthreads();
  const int dim = threadIdx.x * 4;
  if (dim >= p.d) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  l = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const float4 y = sums[w][threadIdx.x];
    s.x += y.x, s.y += y.y, s.z += y.z, s.w += y.w;
    l += red[w];
  }
  T* out = static_cast<T*>(p.out) + ((static_cast<long long>(seg.y) * p.hkv + seg.z) * p.group + seg.w + row) * p.d;
  pa_store(out + dim, s, l);
}

// What the caller's workspace has to hold for one block of the grid, in bytes.
constexpr long long part_bytes(int rt, int dp) { return 2ll * rt * (dp * 4 + 8) + 16; }

template <typename T, int DP, bool WIDE, bool MASK>
struct PagedAttnLaunch {
  using A = PagedAttn<T, DP, WIDE, MASK>;
  // Blocks that one SM holds at once; negative: an error.
  static int resident() {
    auto kernel = paged_attention_kernel<T, DP, WIDE, MASK>;
    if (A::kSmem > 48 * 1024 &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(A::kSmem)) != cudaSuccess)
      return -2;
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, 128, A::kSmem) != cudaSuccess || n < 1) return -2;
    return n;
  }
  static int launch(PagedAttnParams& p, int grid, void* ws, long long ws_bytes, cudaStream_t st) {
    if (grid <= 0 || ws_bytes < grid * part_bytes(A::RT, DP)) return -1;
    char* w = static_cast<char*>(ws);
    p.part_o = reinterpret_cast<float*>(w);
    p.part_ml = reinterpret_cast<float2*>(w + static_cast<long long>(grid) * 2 * A::RT * DP * 4);
    p.shared_seg = reinterpret_cast<int4*>(w + static_cast<long long>(grid) * 2 * A::RT * (DP * 4 + 8));
    p.row_tiles = (p.group + A::RT - 1) / A::RT;
    paged_attention_kernel<T, DP, WIDE, MASK><<<grid, 128, A::kSmem, st>>>(p);
    if (cudaGetLastError() != cudaSuccess) return -2;
    if (grid == 1) return 0;  // nothing is shared
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.group < A::RT ? p.group : A::RT, grid);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_attention_join_kernel<T, DP, WIDE, MASK>, p) == cudaSuccess ? 0 : -2;
  }
};

// Calls f with the PagedAttnLaunch of these types and sizes.
template <typename T, int DP, typename F>
int paged_attention_dp(bool wide, bool mask, F f) {
  if (mask) return wide ? f(PagedAttnLaunch<T, DP, true, true>()) : f(PagedAttnLaunch<T, DP, false, true>());
  return wide ? f(PagedAttnLaunch<T, DP, true, false>()) : f(PagedAttnLaunch<T, DP, false, false>());
}
template <typename T, typename F>
int paged_attention_type(int d, bool wide, bool mask, F f) {
  if (d <= 64) return paged_attention_dp<T, 64>(wide, mask, f);
  if (d <= 128) return paged_attention_dp<T, 128>(wide, mask, f);
  return paged_attention_dp<T, 256>(wide, mask, f);
}
template <typename F>
int paged_attention_dispatch(int dtype, int d, int group, bool mask, F f) {
  const bool wide = group > 8;
  if (dtype == 0) return paged_attention_type<float>(d, wide, mask, f);
  if (dtype == 1) return paged_attention_type<__half>(d, wide, mask, f);
  if (dtype == 2) return paged_attention_type<__nv_bfloat16>(d, wide, mask, f);
  return -1;
}

}  // namespace oslo

extern "C" {

// Everything a call needs, eight bytes each.  Strides in elements.
struct OsloPagedAttentionArgs {
  long long q, k_pages, v_pages, table, lens, mask, out, workspace, status, stream;  // addresses; mask may be 0
  long long q_b, q_s, q_h, k_page, k_head, v_page, v_head, table_row, mask_b, mask_s;
  long long b, s, hkv, group, d, page_size, max_pages, num_pages, mask_len, dtype, grid, workspace_bytes;
  double scale;
};

// Blocks of the first kernel that one SM of the current device holds (negative: an error).
int oslo_paged_attention_resident_parts(int dtype, int d, int group, int mask) {
  using namespace oslo;
  return paged_attention_dispatch(dtype, d, group, mask != 0, [](auto l) { return decltype(l)::resident(); });
}
// Workspace of one block of the grid.
long long oslo_paged_attention_block_bytes(int d, int group) {
  return oslo::part_bytes(group > 8 ? 16 : 8, d <= 64 ? 64 : d <= 128 ? 128 : 256);
}

int oslo_paged_attention(const OsloPagedAttentionArgs* a) {
  using namespace oslo;
  if (a->b <= 0 || a->s <= 0) return 0;
  if (a->hkv <= 0 || a->group <= 0 || a->d <= 0 || a->d > 256 || a->d % 8 || a->page_size <= 0 || a->page_size % 16) return -1;
  if (a->b * a->s > 0x3fffffff || a->max_pages * a->page_size > 0x3fffffff) return -1;
  PagedAttnParams p{};
  p.q = reinterpret_cast<const void*>(a->q), p.k = reinterpret_cast<const void*>(a->k_pages), p.v = reinterpret_cast<const void*>(a->v_pages);
  p.mask = reinterpret_cast<const float*>(a->mask), p.out = reinterpret_cast<void*>(a->out);
  p.table = reinterpret_cast<const int*>(a->table), p.lens = reinterpret_cast<const int*>(a->lens);
  p.status = reinterpret_cast<int*>(a->status);
  p.q_sb = a->q_b, p.q_ss = a->q_s, p.q_sh = a->q_h, p.k_page = a->k_page, p.k_head = a->k_head, p.v_page = a->v_page;
  p.v_head = a->v_head, p.table_stride = a->table_row, p.m_sb = a->mask_b, p.m_ss = a->mask_s;
  p.b = a->b, p.s = a->s, p.hkv = a->hkv, p.group = a->group, p.d = a->d, p.page_size = a->page_size, p.max_pages = a->max_pages;
  p.num_pages = a->num_pages, p.mask_len = a->mask_len, p.scale = static_cast<float>(a->scale);
  return paged_attention_dispatch(a->dtype, a->d, a->group, a->mask != 0, [&](auto l) {
    return decltype(l)::launch(p, static_cast<int>(a->grid), reinterpret_cast<void*>(a->workspace), a->workspace_bytes,
                               reinterpret_cast<cudaStream_t>(a->stream));
  });
}
}
