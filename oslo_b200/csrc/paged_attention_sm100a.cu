// Attention of the newest tokens over a paged key / value cache.
//
//   o = softmax(scale * q K^T + mask) V   over the tokens of the sequence's pages that the query sees; a query that sees none
//   gives zeros.
//
// Every key and value is used by `group` query heads only, so HBM bounds it: 4 * head_dim bytes a token and key head against
// 4 * group * head_dim operations.  A block of four warps takes one (query token, key head); each warp walks 16-token tiles
// (8 for fp32) with its own running maximum, sum and output, and the four are joined at the end.
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
  int b, s, hkv, group, d, page_size, max_pages, num_pages, mask_len, row_tiles;
  float scale;
};

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

OSLO_DEVINL float pa_out(float x, float) { return x; }
OSLO_DEVINL __half pa_out(float x, __half) { return __float2half_rn(x); }
OSLO_DEVINL __nv_bfloat16 pa_out(float x, __nv_bfloat16) { return __float2bfloat16_rn(x); }

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

template <typename T, int DP, bool WIDE, bool MASK>
__global__ void __launch_bounds__(128) paged_attention_kernel(const PagedAttnParams p) {
  using A = PagedAttn<T, DP, WIDE, MASK>;
  extern __shared__ float4 smem4[];
  float* buf = reinterpret_cast<float*>(smem4);
  float* ml = buf + A::WARPS * A::RT * A::ROW;
  int seg = blockIdx.x;
  const int row0 = (seg % p.row_tiles) * A::RT;
  seg /= p.row_tiles;
  const int h = seg % p.hkv;
  const int query = seg / p.hkv, b = query / p.s, i = query % p.s;
  int limit = p.lens[b] - p.s + 1 + i;
  const int cap = MASK ? min(p.mask_len, p.max_pages * p.page_size) : p.max_pages * p.page_size;
  if (limit > cap) {
    limit = cap;
    if (threadIdx.x == 0) atomicCAS(p.status, kStatusOk, kStatusPageRange);
  }
  A a;
  a.load_q(p, static_cast<const T*>(p.q) + b * p.q_sb + i * p.q_ss + static_cast<long long>(h) * p.group * p.q_sh, row0);
  a.clear();
  const float* mask = MASK ? p.mask + b * p.m_sb + i * p.m_ss : nullptr;
  for (int t = (threadIdx.x >> 5) * A::TT; t < limit; t += A::WARPS * A::TT) {
    const int page = p.table[b * p.table_stride + t / p.page_size];
    const bool ok = page >= 0 && page < p.num_pages;
    if (!ok && (threadIdx.x & 31) == 0) atomicCAS(p.status, kStatusOk, kStatusPageRange);
    if (!ok) continue;
    const long long in_page = static_cast<long long>(t % p.page_size) * p.d;
    a.tile(p, static_cast<const T*>(p.k) + page * p.k_page + h * p.k_head + in_page,
           static_cast<const T*>(p.v) + page * p.v_page + h * p.v_head + in_page, t, limit, mask);
  }
  a.join(buf, ml);
  T* out = static_cast<T*>(p.out) + (static_cast<long long>(query) * p.hkv + h) * p.group * p.d;
  for (int x = threadIdx.x; x < A::RT * (DP / 4); x += blockDim.x) {
    const int row = x / (DP / 4), dim = x % (DP / 4) * 4;
    if (row0 + row >= p.group || dim >= p.d) continue;
    float l = 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < A::WARPS; ++w) {
      l += ml[(A::WARPS + w) * A::RT + row];
      const float4 y = *reinterpret_cast<const float4*>(buf + (w * A::RT + row) * A::ROW + dim);
      s.x += y.x, s.y += y.y, s.z += y.z, s.w += y.w;
    }
    const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
    T* dst = out + (row0 + row) * p.d + dim;
    dst[0] = pa_out(s.x * inv, T()), dst[1] = pa_out(s.y * inv, T()), dst[2] = pa_out(s.z * inv, T()), dst[3] = pa_out(s.w * inv, T());
  }
}

template <typename T, int DP, bool WIDE, bool MASK>
int paged_attention_launch(PagedAttnParams& p, cudaStream_t st) {
  using A = PagedAttn<T, DP, WIDE, MASK>;
  p.row_tiles = (p.group + A::RT - 1) / A::RT;
  const long long grid = static_cast<long long>(p.b) * p.s * p.hkv * p.row_tiles;
  if (grid > 0x7fffffffll) return -1;
  auto kernel = paged_attention_kernel<T, DP, WIDE, MASK>;
  if (A::kSmem > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(A::kSmem)) != cudaSuccess)
    return -2;
  kernel<<<static_cast<unsigned>(grid), 128, A::kSmem, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

template <typename T, int DP>
int paged_attention_dp(PagedAttnParams& p, cudaStream_t st) {
  const bool wide = p.group > 8;
  if (p.mask) return wide ? paged_attention_launch<T, DP, true, true>(p, st) : paged_attention_launch<T, DP, false, true>(p, st);
  return wide ? paged_attention_launch<T, DP, true, false>(p, st) : paged_attention_launch<T, DP, false, false>(p, st);
}

template <typename T>
int paged_attention_type(PagedAttnParams& p, cudaStream_t st) {
  if (p.d <= 64) return paged_attention_dp<T, 64>(p, st);
  if (p.d <= 128) return paged_attention_dp<T, 128>(p, st);
  return paged_attention_dp<T, 256>(p, st);
}

}  // namespace oslo

// strides (elements): batch, token, head of q; page, head of the two pools; rows of the table; batch, token of the mask.
extern "C" int oslo_paged_attention(const void* q, const void* k_pages, const void* v_pages, const int* table, const int* lens,
                                    const float* mask, void* out, const long long* strides, int b, int s, int hkv, int group, int d,
                                    int page_size, int max_pages, int num_pages, int mask_len, float scale, int dtype, int* status,
                                    void* stream) {
  using namespace oslo;
  if (b <= 0 || s <= 0) return 0;
  if (hkv <= 0 || group <= 0 || d <= 0 || d > 256 || d % 8 || page_size <= 0 || page_size % 16) return -1;
  PagedAttnParams p{};
  p.q = q, p.k = k_pages, p.v = v_pages, p.mask = mask, p.out = out, p.table = table, p.lens = lens, p.status = status;
  p.q_sb = strides[0], p.q_ss = strides[1], p.q_sh = strides[2];
  p.k_page = strides[3], p.k_head = strides[4], p.v_page = strides[5], p.v_head = strides[6], p.table_stride = strides[7];
  p.m_sb = strides[8], p.m_ss = strides[9];
  p.b = b, p.s = s, p.hkv = hkv, p.group = group, p.d = d, p.page_size = page_size, p.max_pages = max_pages, p.num_pages = num_pages;
  p.mask_len = mask_len, p.scale = scale;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == 0) return paged_attention_type<float>(p, st);
  if (dtype == 1) return paged_attention_type<__half>(p, st);
  if (dtype == 2) return paged_attention_type<__nv_bfloat16>(p, st);
  return -1;
}
