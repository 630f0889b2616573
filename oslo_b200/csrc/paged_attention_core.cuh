// Attention of the newest tokens over a paged key / value cache.
//
//   o = softmax(scale * q K^T + mask) V   over the tokens of the sequence's pages that the query sees; a query that sees none
//   gives zeros.
//
// Every key and value is used by `group` query heads (times the new tokens) only, so HBM bounds it: 4 * head_dim bytes a token and
// key head against 4 * group * head_dim operations.  Measured: 64 sequences of up to 6000 tokens, 32 key heads of 128, 5.48 GB in
// 907 us (94% of the copy bandwidth); one sequence of 131071 tokens, 8 key heads, 100 us (83%: SMs are served unevenly, the
// last block ends 7 us after the mean, and the joining launch follows).
//
// Work is cut into units of 64 tokens (32 for fp32) of one (sequence, key head, block of query rows), a "segment" being all
// units of one such triple.  As many blocks as the GPU holds at once take equal, contiguous ranges of units, found on the
// device from the lengths: one long sequence occupies every SM, a ragged batch leaves none idle, and the host needs to know
// no length.  Inside a block each of four warps walks every fourth 16-token tile (8 for fp32) with its own running maximum,
// sum and output; the four are joined when the segment or the range ends.  Segments that several blocks share are joined by a
// second kernel, launched programmatically so that its start overlaps the first one's end; the parts are added in block order,
// so results do not depend on timing.
//
// Each warp has a ring of tiles in shared memory, filled by 16-byte asynchronous copies that run ahead of the products; rows
// that the query does not see are filled with zeros and never read, so they may hold anything.  The products are mma.sync with
// the operands read 16 bytes at a time, without a transpose, because the order of the summed index is free as long as both
// operands share it:
//   scores   lane (r, q) = (lane / 4, lane % 4) holds 16 contiguous bytes of key r; Q is loaded with the same pattern.
//   output   the accumulator columns of the scores (tokens 2q, 2q + 1) are the A operand's summed index, so lane (r, q) loads
//            the values of exactly those tokens, 16 bytes at head dim r * E of each 8 E wide block.
// (Rows of the ring are 16 bytes longer than a head, which keeps the value loads free of bank conflicts.)  tcgen05 would
// multiply 128 rows where there are 1 to 16: the tensor cores are not what bounds this.
// The weights enter the second product as the sum of two 16-bit numbers (high part and remainder): 16 bits of a weight in bf16, 22
// in fp16.  In bf16 that is hidden by the result's own rounding: of 64 x 6000 tokens' results 24 in 10000 are the neighbour of the
// nearest bf16 number, 7 in 10000 with 32-bit weights; a third part would cost half the product again.  fp16 ends at 2^-24, so its
// weights and their sum carry a factor of 2^15, which the last division takes out: a token that weighs 2^-25 of the heaviest keeps
// 14 bits, and no weight loses more than 2^-22 of itself or 2^-40 of the heaviest.
// An infinite value times such a pair would be NaN, and so would a value that is not finite times the weight zero of a row that does
// not see it: blocks whose sums are not finite walk over their tokens once more, with care (see CAREFUL).
#pragma once
#include "common.cuh"

#include <atomic>
#include <type_traits>

namespace oslo {

struct PagedAttnParams {
  const void* q;
  const void* k;
  const void* v;
  const float* mask;  // additive, [b, s, mask_len] by strides; mask_len < 0: none
  void* out;          // [b, s, hq, d] contiguous
  const int* table;
  const int* lens;
  int* status;
  long long q_sb, q_ss, q_sh, k_page, k_head, v_page, v_head, table_stride, m_sb, m_ss;
  float* part_o;   // [grid, 2, rows of a block, DP] unnormalised outputs of shared segments: 0 = begun by an earlier block, 1 = begun here
  float2* part_ml;  // [grid, 2, rows of a block] their maxima and sums
  int4* shared_seg;  // [grid] of the segment begun earlier that ends here: (first block, query, key head, first row); x < 0: none
  int b, s, hkv, group, d, page_size, max_pages, num_pages, mask_len;
  int queries, rows, row_tiles;  // groups of query rows of a sequence; rows of a group and key head, and how many blocks' worth
  float scale;
};

// Rows of a segment.  The query tokens of a sequence that share a mask form one group: its row r is query head r % group of token
// first + r / group, so one pass over the keys serves several proposed tokens.  Tokens with masks of their own are groups.
struct Segment {
  int b, h, first, row0, rows;  // sequence, key head, first query token of the group, first row, rows in this block
  int length;                   // tokens that query token i of the sequence sees: length + i
  OSLO_DEVINL Segment(const PagedAttnParams& p, int query, int head, int row, int most) {
    b = query / p.queries, h = head, first = query - b * p.queries, row0 = row, rows = min(most, p.rows - row);
    length = 0;
  }
  OSLO_DEVINL int token(const PagedAttnParams& p, int r) const { return first + (row0 + r) / p.group; }
  OSLO_DEVINL int q_head(const PagedAttnParams& p, int r) const { return h * p.group + (row0 + r) % p.group; }
  OSLO_DEVINL long long q_at(const PagedAttnParams& p, int r) const { return b * p.q_sb + token(p, r) * p.q_ss + q_head(p, r) * p.q_sh; }
  OSLO_DEVINL long long out_at(const PagedAttnParams& p, int r) const {
    return ((static_cast<long long>(b) * p.s + token(p, r)) * p.hkv * p.group + q_head(p, r)) * p.d;
  }
};

constexpr float kLog2e = 1.4426950408889634f;

OSLO_DEVINL uint4 ldg16(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
// 16 bytes into shared memory, asynchronously; zeros where `valid` is false (nothing is read then)
OSLO_DEVINL void copy16(void* dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
OSLO_DEVINL void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
OSLO_DEVINL void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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
  static constexpr float WEIGHT = 1.f;  // of the heaviest token
  static OSLO_DEVINL void run(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static OSLO_DEVINL uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(r);
  }
  // all bits of those of the two that are infinite or not a number
  static OSLO_DEVINL uint32_t wild(uint32_t r) { return ((r & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((r & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u); }
  static OSLO_DEVINL float low(uint32_t r) { return __uint_as_float(r << 16); }
  static OSLO_DEVINL float high(uint32_t r) { return __uint_as_float(r & 0xffff0000u); }
};
template <>
struct Mma16<__half> {
  static constexpr float WEIGHT = 32768.f;
  static OSLO_DEVINL void run(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static OSLO_DEVINL uint32_t pack(float lo, float hi) {
    const __half2 r = __floats2half2_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(r);
  }
  static OSLO_DEVINL uint32_t wild(uint32_t r) { return ((r & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((r & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u); }
  static OSLO_DEVINL float low(uint32_t r) { return __low2float(reinterpret_cast<const __half2&>(r)); }
  static OSLO_DEVINL float high(uint32_t r) { return __high2float(reinterpret_cast<const __half2&>(r)); }
};
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

// Scores and weights of one mask mode.  With a mask the scores stay in natural units: a mask of the type's lowest value times
// log2(e) would leave its range.
template <bool MASK>
struct AttnMath {
  static OSLO_DEVINL float score(const PagedAttnParams& p, float s, float add) {
    return MASK ? fmaf(s, p.scale, add) : s * (p.scale * kLog2e);
  }
  // exp(x - m); m = -inf: nothing was seen yet
  static OSLO_DEVINL float weight(float x, float m) {
    const float mm = m == -INFINITY ? 0.f : m;
    return ex2(MASK ? (x - mm) * kLog2e : x - mm);
  }
};

// What a warp keeps of a segment and does with a tile.  T: element type; DP: head_dim rounded up to 64, 128 or 256; WIDE: 9 to
// 16 query heads per block instead of up to 8.  This one: 16-bit types on the tensor cores.
template <typename T, int DP, bool WIDE, bool MASK>
struct AttnWarp {
  using Math = AttnMath<MASK>;
  static constexpr int E = 8;   // elements of one load
  static constexpr int TT = 16;  // tokens of one tile
  static constexpr int NT = TT / 8;
  static constexpr int KC = DP / (4 * E);   // loads per key and lane
  static constexpr int VC = DP / (8 * E);   // loads per value and lane
  static constexpr int VT = TT / 4;         // value tokens of a lane
  static constexpr int RT = WIDE ? 16 : 8;  // query rows
  static constexpr int ROW = DP + 4;        // padded row of the joining buffer
  static constexpr int WARPS = 4;
  static constexpr int PITCH = DP + E;  // elements between two rows of a tile in the ring
  // Blocks an SM should hold; the ring's size is chosen for it.  128 dims: two blocks with three tiles a warp (one sequence of
  // 131071 tokens 100 us, ragged batch 30 us) against three blocks with two (105 and 32 us) and one with four (120 and 42 us).
  // 64 dims: three blocks with three tiles (64 x 4000 tokens, 12 heads: 116 us) against four (124 us) and two with five (137 us).
  static constexpr int BLOCKS = DP == 64 ? 3 : DP == 128 ? 2 : 1;
  static constexpr int SCRATCH = 0;  // floats of shared memory of the block, beside the rings

  uint4 q0[KC], q1[WIDE ? KC : 1];
  float o[VC][E][4];  // rows r and r + 8; with up to 8 rows the second pair holds what the remainders of the weights add
  float m0, m1, l0, l1;
  int end0, end1, least, most;  // tokens that rows r and r + 8 see; of the warp's rows, the least and the most

  OSLO_DEVINL void load_q(const PagedAttnParams& p, const Segment& seg, float*) {
    const int r = (threadIdx.x & 31) >> 2, quad = threadIdx.x & 3;
    const T* q = static_cast<const T*>(p.q);
    const long long a0 = r < seg.rows ? seg.q_at(p, r) : 0, a1 = WIDE && r + 8 < seg.rows ? seg.q_at(p, r + 8) : 0;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int dim = c * 4 * E + quad * E;
      q0[c] = r < seg.rows && dim < p.d ? ldg16(q + a0 + dim) : make_uint4(0, 0, 0, 0);
      if constexpr (WIDE) q1[c] = r + 8 < seg.rows && dim < p.d ? ldg16(q + a1 + dim) : make_uint4(0, 0, 0, 0);
    }
    end0 = seg.length + seg.token(p, min(r, seg.rows - 1)), end1 = seg.length + seg.token(p, min(r + 8, seg.rows - 1));
    least = seg.length + seg.token(p, 0), most = seg.length + seg.token(p, seg.rows - 1);
  }
  OSLO_DEVINL void clear() {
    m0 = m1 = -INFINITY;
    l0 = l1 = 0.f;
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[j][e][x] = 0.f;
  }

  // Block j of the values of this lane's tokens; zeros for those that are masked or, where `end` is given, at or past it.
  template <bool END>
  static OSLO_DEVINL void load_v(uint4 (&vr)[VT], const T* ring, int j, const bool (&seen)[NT][2], int end) {
    const int lane = threadIdx.x & 31, r = lane >> 2, quad = lane & 3;
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      vr[t] = *reinterpret_cast<const uint4*>(ring + TT * PITCH + ((t >> 1) * 8 + quad * 2 + (t & 1)) * PITCH + j * 8 * E + r * E);
      if constexpr (MASK || END) {  // a token that is not seen may hold anything: its values do not enter the product
        if (!seen[t >> 1][t & 1] || (END && (t >> 1) * 8 + quad * 2 + (t & 1) >= end)) vr[t] = make_uint4(0, 0, 0, 0);
      }
    }
  }
  // 16-bit B operands of column e from the values of the lane's four tokens
  static OSLO_DEVINL void columns(const uint4 (&vr)[VT], int e, uint32_t& b0, uint32_t& b1) {
    const uint32_t sel = e & 1 ? 0x7632 : 0x5410;
    b0 = __byte_perm(reinterpret_cast<const uint32_t*>(&vr[0])[e / 2], reinterpret_cast<const uint32_t*>(&vr[1])[e / 2], sel);
    b1 = __byte_perm(reinterpret_cast<const uint32_t*>(&vr[2])[e / 2], reinterpret_cast<const uint32_t*>(&vr[3])[e / 2], sel);
  }

  // One tile of the ring: its TT tokens start at `token`; tokens at or past `limit` are not seen.
  // CAREFUL: values may be infinite or not a number, see below.
  template <bool CAREFUL>
  OSLO_DEVINL void tile(const PagedAttnParams& p, const T* ring, int token, int limit, const float* mask, float*) {
    const int lane = threadIdx.x & 31, r = lane >> 2, quad = lane & 3;
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
    float sc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
      float odd[4] = {0.f, 0.f, 0.f, 0.f};  // two chains of products, each half as long
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint4 qa = q0[c], qb = WIDE ? q1[WIDE ? c : 0] : make_uint4(0, 0, 0, 0);
        const uint4 kr = *reinterpret_cast<const uint4*>(ring + (n * 8 + r) * PITCH + c * 4 * E + quad * E);
        Mma16<T>::run(sc[n], qa.x, qb.x, qa.y, qb.y, kr.x, kr.y);
        Mma16<T>::run(odd, qa.z, qb.z, qa.w, qb.w, kr.z, kr.w);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) sc[n][x] += odd[x];
    }
    float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int t = token + n * 8 + quad * 2 + x;
        sc[n][x] = seen[n][x] && t < end0 ? Math::score(p, sc[n][x], add[n][x]) : -INFINITY;
        t0 = fmaxf(t0, sc[n][x]);
        if constexpr (WIDE) {
          sc[n][2 + x] = seen[n][x] && t < end1 ? Math::score(p, sc[n][2 + x], add[n][x]) : -INFINITY;
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
      const float f0 = Math::weight(m0, n0), f1 = WIDE ? Math::weight(m1, n1) : 0.f;
      m0 = n0, m1 = n1;
      l0 *= f0, l1 *= f1;
#pragma unroll
      for (int j = 0; j < VC; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          o[j][e][0] *= f0, o[j][e][1] *= f0;
          o[j][e][2] *= WIDE ? f1 : f0, o[j][e][3] *= WIDE ? f1 : f0;
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        sc[n][x] = Math::weight(sc[n][x], m0) * Mma16<T>::WEIGHT;
        l0 += sc[n][x];
        if constexpr (WIDE) {
          sc[n][2 + x] = Math::weight(sc[n][2 + x], m1) * Mma16<T>::WEIGHT;
          l1 += sc[n][2 + x];
        }
      }
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
    if constexpr (!WIDE) hi[1] = lo[0], hi[3] = lo[2];  // the remainders take the empty rows
    if constexpr (!CAREFUL) {
#pragma unroll
      for (int j = 0; j < VC; ++j) {
        uint4 vr[VT];
        load_v<false>(vr, ring, j, seen, 0);
#pragma unroll
        for (int part = 0; part < (WIDE ? 2 : 1); ++part)  // all high parts, then all remainders: neighbours do not wait for each other
#pragma unroll
          for (int e = 0; e < E; ++e) {
            uint32_t b0, b1;
            columns(vr, e, b0, b1);
            const uint32_t(&a)[4] = part ? lo : hi;
            Mma16<T>::run(o[j][e], a[0], a[1], a[2], a[3], b0, b1);
          }
      }
    } else {
      // An infinite value (or one that is not a number) times a weight in two parts, or times the weight zero of a row that does not
      // see it, would be NaN.  So each query token gets a product of its own, over the tokens that it sees, and in it such values
      // are left out of the parts' product and get another one, with 1 for every weight above zero.
      uint32_t one[4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          one[2 * n + x] = x == 0 || WIDE ? Mma16<T>::pack(sc[n][2 * x] > 0.f ? 1.f : 0.f, sc[n][2 * x + 1] > 0.f ? 1.f : 0.f) : 0u;
#pragma unroll 1
      for (int end = min(token + TT, limit) <= least ? most : least; end <= most; ++end) {
        const bool mine0 = min(token + TT, limit) <= least || end0 == end, mine1 = min(token + TT, limit) <= least || end1 == end;
#pragma unroll
        for (int j = 0; j < VC; ++j) {
          uint4 vr[VT], inf[VT];
          load_v<true>(vr, ring, j, seen, end - token);
#pragma unroll
          for (int t = 0; t < VT; ++t) {
            inf[t].x = vr[t].x & Mma16<T>::wild(vr[t].x), inf[t].y = vr[t].y & Mma16<T>::wild(vr[t].y);
            inf[t].z = vr[t].z & Mma16<T>::wild(vr[t].z), inf[t].w = vr[t].w & Mma16<T>::wild(vr[t].w);
            vr[t].x ^= inf[t].x, vr[t].y ^= inf[t].y, vr[t].z ^= inf[t].z, vr[t].w ^= inf[t].w;
          }
#pragma unroll
          for (int e = 0; e < E; ++e) {
            uint32_t b0, b1;
            columns(vr, e, b0, b1);
            float c[4] = {o[j][e][0], o[j][e][1], o[j][e][2], o[j][e][3]}, w[4] = {0.f, 0.f, 0.f, 0.f};
            Mma16<T>::run(c, hi[0], hi[1], hi[2], hi[3], b0, b1);
            if constexpr (WIDE) Mma16<T>::run(c, lo[0], lo[1], lo[2], lo[3], b0, b1);
            columns(inf, e, b0, b1);
            Mma16<T>::run(w, one[0], one[1], one[2], one[3], b0, b1);
            if (mine0) o[j][e][0] = c[0] + w[0], o[j][e][1] = c[1] + w[1];
            if (WIDE ? mine1 : mine0) o[j][e][2] = WIDE ? c[2] + w[2] : c[2], o[j][e][3] = WIDE ? c[3] + w[3] : c[3];
          }
        }
      }
    }
  }

  OSLO_DEVINL void join(T* ring, float* ml) {
    float* buf = reinterpret_cast<float*>(ring);
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
    const float f0 = Math::weight(m0, top0), f1 = WIDE ? Math::weight(m1, top1) : 0.f;
    if (quad == 0) {
      ml[WARPS * RT + warp * RT + r] = l0 * f0;
      if constexpr (WIDE) ml[WARPS * RT + warp * RT + 8 + r] = l1 * f1;
    }
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int x = 0; x < (WIDE ? 4 : 2); ++x) {
        float* dst = buf + (r + (x >> 1) * 8) * ROW + j * 8 * E + (quad * 2 + (x & 1)) * E;
        const float f = x >> 1 ? f1 : f0;
        const auto sum = [&](int e) { return (WIDE ? o[j][e][x] : o[j][e][x] + o[j][e][(x + 2) & 3]) * f; };
#pragma unroll
        for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(dst + e) = make_float4(sum(e), sum(e + 1), sum(e + 2), sum(e + 3));
      }
    __syncthreads();
  }

  // Without a join: the warp has rows of its own, whose sums go to `buf` as they are.
  OSLO_DEVINL void leave(float* buf, float* ml) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, quad = lane & 3;
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    if (quad == 0) {
      ml[warp * RT + r] = m0, ml[WARPS * RT + warp * RT + r] = l0;
      if constexpr (WIDE) ml[warp * RT + 8 + r] = m1, ml[WARPS * RT + warp * RT + 8 + r] = l1;
    }
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int x = 0; x < (WIDE ? 4 : 2); ++x) {
        float* dst = buf + (r + (x >> 1) * 8) * ROW + j * 8 * E + (quad * 2 + (x & 1)) * E;
#pragma unroll
        for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(dst + e) = make_float4(o[j][e][x], o[j][e + 1][x], o[j][e + 2][x], o[j][e + 3][x]);
      }
  }
};

// 32-bit inputs, on the FMA units: tensor cores would round them to 10 bits, and splitting each into three products was both
// less exact (2e-6 against 7e-7 for 32-bit sums at 256 dims) and slower.  Lane (r, q) multiplies its quarter of key r with every
// query row; a reduce-scatter leaves a quarter of the rows' scores with each of the four lanes.  For the output a lane owns four
// dims (eight of 256) and walks over the tile's tokens; the weights come from shared memory.
template <int DP, bool WIDE, bool MASK>
struct AttnWarp<float, DP, WIDE, MASK> {
  using Math = AttnMath<MASK>;
  static constexpr int E = 4;
  static constexpr int TT = 8;
  static constexpr int RT = WIDE ? 16 : 8;
  static constexpr int OWN = RT / 4;  // rows whose scores a lane holds
  static constexpr int ROW = DP + 4;
  static constexpr int WARPS = 4;
  static constexpr int PITCH = DP + 16;  // eight lanes of a key load then touch all banks
  static constexpr int BLOCKS = DP == 64 ? 3 : DP == 128 ? 2 : 1;
  static constexpr int KC = DP / 16;              // loads per key and lane
  static constexpr int VC = DP < 128 ? 1 : DP / 128;  // loads per value and lane
  static constexpr int HALVES = DP == 64 ? 2 : 1;  // 16 lanes cover 64 dims: the two halves of the warp take alternate tokens
  static constexpr int WEIGHTS = RT * TT + RT;     // of a warp: weights [RT][TT], then factors [RT]
  static constexpr int SCRATCH = RT * DP + WARPS * WEIGHTS;  // the block's queries, then each warp's weights

  float4 o[RT][VC];
  float m[OWN], l[OWN];
  int end[OWN];  // tokens that the lane's rows see
  int rows, first, group, least;  // row g sees least + (first + g) / group tokens

  static OSLO_DEVINL int own_row(int i) {
    const int quad = threadIdx.x & 3;
    return (quad & 1) * (RT / 2) + (quad >> 1) * (RT / 4) + i;
  }
  OSLO_DEVINL void load_q(const PagedAttnParams& p, const Segment& seg, float* scratch) {
    rows = seg.rows;
    for (int x = threadIdx.x; x < rows * (DP / 4); x += 32 * WARPS) {
      const int row = x / (DP / 4), dim = x % (DP / 4) * 4;
      reinterpret_cast<uint4*>(scratch)[x] = dim < p.d ? ldg16(static_cast<const float*>(p.q) + seg.q_at(p, row) + dim) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < OWN; ++i) end[i] = seg.length + seg.token(p, min(own_row(i), rows - 1));
    first = seg.row0 % p.group, group = p.group, least = seg.length + seg.token(p, 0);
    __syncthreads();
  }
  OSLO_DEVINL void clear() {
#pragma unroll
    for (int i = 0; i < OWN; ++i) m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int g = 0; g < RT; ++g)
#pragma unroll
      for (int j = 0; j < VC; ++j) o[g][j] = make_float4(0.f, 0.f, 0.f, 0.f);
  }

  template <bool CAREFUL>
  OSLO_DEVINL void tile(const PagedAttnParams& p, const float* ring, int token, int limit, const float* mask, float* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, quad = lane & 3;
    float* const weights = scratch + RT * DP + warp * WEIGHTS;
    float* const factors = weights + RT * TT;
    bool seen = token + r < limit;
    float add = 0.f;
    if constexpr (MASK) {
      if (seen) add = mask[token + r];
      seen = seen && add != -INFINITY;
    }
    const unsigned visible = __ballot_sync(0xffffffffu, seen);  // token t: bit 4 t
    float part[RT];
#pragma unroll
    for (int g = 0; g < RT; ++g) part[g] = 0.f;
#pragma unroll
    for (int c0 = 0; c0 < KC; c0 += 4) {
      float4 k[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) k[c] = *reinterpret_cast<const float4*>(ring + r * PITCH + (c0 + c) * 16 + quad * 4);
#pragma unroll
      for (int g = 0; g < RT; ++g) {
        if (g >= rows) break;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float4 q = *reinterpret_cast<const float4*>(scratch + g * DP + (c0 + c) * 16 + quad * 4);
          part[g] = fmaf(q.x, k[c].x, fmaf(q.y, k[c].y, fmaf(q.z, k[c].z, fmaf(q.w, k[c].w, part[g]))));
        }
      }
    }
    // of each pair of lanes one goes on with the first half of the rows, the other with the second
#pragma unroll
    for (int i = 0; i < RT / 2; ++i) {
      const bool up = quad & 1;
      const float keep = up ? part[i + RT / 2] : part[i], give = up ? part[i] : part[i + RT / 2];
      part[i] = keep + __shfl_xor_sync(0xffffffffu, give, 1);
    }
#pragma unroll
    for (int i = 0; i < RT / 4; ++i) {
      const bool up = quad & 2;
      const float keep = up ? part[i + RT / 4] : part[i], give = up ? part[i] : part[i + RT / 4];
      part[i] = keep + __shfl_xor_sync(0xffffffffu, give, 2);
    }
    float top[OWN];
    bool higher = false;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      part[i] = seen && token + r < end[i] ? Math::score(p, part[i], add) : -INFINITY;
      top[i] = part[i];
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], x));
      higher = higher || top[i] > m[i];
    }
    const bool rescale = __any_sync(0xffffffffu, higher);
    if (rescale) {
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const float n = fmaxf(m[i], top[i]), f = Math::weight(m[i], n);
        m[i] = n, l[i] *= f;
        if (r == 0) factors[own_row(i)] = f;
      }
    }
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const float w = Math::weight(part[i], m[i]);
      l[i] += w;
      // tokens of one half of the warp lie side by side
      weights[own_row(i) * TT + (HALVES == 2 ? (r & 1) * 4 + (r >> 1) : r)] = w;
    }
    __syncwarp();
    if (rescale) {
#pragma unroll
      for (int g = 0; g < RT; ++g) {
        if (g >= rows) break;
        const float f = factors[g];
#pragma unroll
        for (int j = 0; j < VC; ++j) o[g][j].x *= f, o[g][j].y *= f, o[g][j].z *= f, o[g][j].w *= f;
      }
    }
    constexpr int N = TT / HALVES;  // tokens of a lane
    const int half = HALVES == 2 ? lane >> 4 : 0, column = (HALVES == 2 ? lane & 15 : lane) * 4;
    const bool mixed = min(token + TT, limit) > least;
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int t0 = 0; t0 < N; t0 += 4) {
        float4 v[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int at = HALVES == 2 ? 2 * (t0 + t) + half : t0 + t;
          v[t] = *reinterpret_cast<const float4*>(ring + TT * PITCH + at * PITCH + j * 128 + column);
          if constexpr (MASK) {  // a masked token may hold anything: its values do not enter the product
            if (!((visible >> (4 * at)) & 1)) v[t] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
        }
        if (mixed) {  // tokens that some rows do not see have weight zero for them, which is enough where the values are finite
          bool wild = false;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t most_bits = 0x7f800000u;
            wild = wild || (__float_as_uint(v[t].x) & most_bits) == most_bits || (__float_as_uint(v[t].y) & most_bits) == most_bits ||
                   (__float_as_uint(v[t].z) & most_bits) == most_bits || (__float_as_uint(v[t].w) & most_bits) == most_bits;
          }
          if (__any_sync(0xffffffffu, wild)) {
#pragma unroll
            for (int g = 0; g < RT; ++g) {
              if (g >= rows) break;
              const int sees = least + (first + g) / group - token;
#pragma unroll
              for (int t = 3; t >= 0; --t) {  // the order of the sums below
                if ((HALVES == 2 ? 2 * (t0 + t) + half : t0 + t) >= sees) continue;
                const float w = weights[g * TT + half * 4 + t0 + t];
                float4& y = o[g][j];
                y.x = fmaf(w, v[t].x, y.x), y.y = fmaf(w, v[t].y, y.y), y.z = fmaf(w, v[t].z, y.z), y.w = fmaf(w, v[t].w, y.w);
              }
            }
            continue;
          }
        }
#pragma unroll
        for (int g = 0; g < RT; ++g) {
          if (g >= rows) break;
          const float4 w = *reinterpret_cast<const float4*>(weights + g * TT + half * 4 + t0);
          float4& y = o[g][j];
          y.x = fmaf(w.x, v[0].x, fmaf(w.y, v[1].x, fmaf(w.z, v[2].x, fmaf(w.w, v[3].x, y.x))));
          y.y = fmaf(w.x, v[0].y, fmaf(w.y, v[1].y, fmaf(w.z, v[2].y, fmaf(w.w, v[3].y, y.y))));
          y.z = fmaf(w.x, v[0].z, fmaf(w.y, v[1].z, fmaf(w.z, v[2].z, fmaf(w.w, v[3].z, y.z))));
          y.w = fmaf(w.x, v[0].w, fmaf(w.y, v[1].w, fmaf(w.z, v[2].w, fmaf(w.w, v[3].w, y.w))));
        }
      }
  }

  OSLO_DEVINL void join(float* buf, float* ml) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
      if (r == 0) ml[warp * RT + own_row(i)] = m[i];
    }
    __syncthreads();
    const auto factor = [&](int g) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, ml[w * RT + g]);
      return Math::weight(ml[warp * RT + g], top);
    };
#pragma unroll
    for (int i = 0; i < OWN; ++i)
      if (r == 0) ml[WARPS * RT + warp * RT + own_row(i)] = l[i] * factor(own_row(i));
#pragma unroll
    for (int g = 0; g < RT; ++g) {
      if (g >= rows) break;
      const float f = factor(g);
#pragma unroll
      for (int j = 0; j < VC; ++j) {
        float4 y = o[g][j];
        if constexpr (HALVES == 2) {
          y.x += __shfl_xor_sync(0xffffffffu, y.x, 16), y.y += __shfl_xor_sync(0xffffffffu, y.y, 16);
          y.z += __shfl_xor_sync(0xffffffffu, y.z, 16), y.w += __shfl_xor_sync(0xffffffffu, y.w, 16);
        }
        if (HALVES == 1 || lane < 16)
          *reinterpret_cast<float4*>(buf + g * ROW + j * 128 + lane * 4) = make_float4(y.x * f, y.y * f, y.z * f, y.w * f);
      }
    }
    __syncthreads();
  }
};

// The block's side of it: rings of tiles in shared memory, and the walk over a segment's tokens.  The four warps share out the
// tokens, or (SPLIT, where there are many query rows) each takes 16 rows and all read every warp's tiles: a key is then read once
// for 64 rows.
template <typename T, int DP, bool WIDE, bool MASK, bool SPLIT>
struct PagedAttn : AttnWarp<T, DP, WIDE, MASK> {
  using W = AttnWarp<T, DP, WIDE, MASK>;
  using W::BLOCKS, W::E, W::PITCH, W::ROW, W::RT, W::SCRATCH, W::TT, W::WARPS;
  static constexpr int TILE = TT * PITCH * 2;  // keys, then values
  static constexpr int STAGES = DP == 64 || (DP == 128 && sizeof(T) == 2) ? 3 : 2;
  static constexpr size_t kRing = sizeof(T) * TILE * STAGES;  // of one warp; the joining buffer takes its place at the end
  static constexpr int ROWS = SPLIT ? WARPS * RT : RT;  // query rows of the block
  // Starting a segment costs a block about as long as two units: each segment has that many units without tokens at its front.
  // (Ragged batch of 32, 8 key heads: 35 us without, 30 us with them; 32 x 500 tokens, 32 key heads: 36 and 28 us.)  A unit of
  // 64 rows takes longer.
  static constexpr int SEGMENT_UNITS = SPLIT ? 1 : 2;
  static constexpr int MIN_UNITS = SPLIT ? 3 : 4;  // a range of work has at least so many
  static constexpr size_t kSmem = kRing * WARPS + sizeof(float) * (2 * WARPS * RT + SCRATCH + WARPS);
  static_assert(kRing >= sizeof(float) * RT * ROW, "a warp's part of the joining buffer fits its ring");
  static_assert((kSmem + 1024) * BLOCKS <= 228 * 1024, "shared memory of the blocks of an SM");

  static OSLO_DEVINL float weight(float x, float m) { return W::Math::weight(x, m); }

  // Starts the copy of one tile, `rows` of whose tokens are seen, into the ring.
  static OSLO_DEVINL void fill(const PagedAttnParams& p, T* ring, const T* k, const T* v, int rows) {
    constexpr int CHUNKS = DP / E;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const T* src = half ? v : k;
      T* dst = ring + half * TT * PITCH;
#pragma unroll
      for (int i = 0; i < TT * CHUNKS / 32; ++i) {
        const int row = (i * 32 + lane) / CHUNKS, c = (i * 32 + lane) % CHUNKS;
        const bool valid = row < rows && c * E < p.d;
        copy16(dst + row * PITCH + c * E, valid ? src + row * p.d + c * E : src, valid);
      }
    }
  }

  // Where the block's sum of a row is put for the other blocks of a cluster.
  static OSLO_DEVINL size_t place(int row, int dim) { return kRing * (row / RT) + sizeof(float) * (row % RT * ROW + dim); }
  // Row maxima of the four warps, then their row sums.
  static OSLO_DEVINL float* ml_of(char* smem) { return reinterpret_cast<float*>(smem + kRing * WARPS); }

  // The warps' sums over tokens [begin, end) of a segment.
  template <bool CAREFUL>
  OSLO_DEVINL void pass(const PagedAttnParams& p, char* smem, const Segment& seg, int limit, int begin, int end) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = seg.h;
    const float* mask = MASK ? p.mask + seg.b * p.m_sb + seg.first * p.m_ss : nullptr;
    const int* table = p.table + seg.b * p.table_stride;
    T* ring = reinterpret_cast<T*>(smem + kRing * warp);
    const T* k = static_cast<const T*>(p.k) + h * p.k_head;
    const T* v = static_cast<const T*>(p.v) + h * p.v_head;
    constexpr int STEP = WARPS * TT;
    int ahead = begin + warp * TT;  // the next tile to copy, and its page
    int page = ahead < end ? table[ahead / p.page_size] : 0;
    unsigned missing = 0;  // bit i: the tile in slot i of the ring has no page
    volatile unsigned* const all_missing = reinterpret_cast<unsigned*>(ml_of(smem) + 2 * WARPS * RT + SCRATCH);
    const auto advance = [&](int slot) {
      if (ahead < end) {
        const bool ok = page >= 0 && page < p.num_pages;
        const long long in_page = static_cast<long long>(ahead % p.page_size) * p.d;
        fill(p, ring + slot * TILE, ok ? k + page * p.k_page + in_page : k, ok ? v + page * p.v_page + in_page : v, ok ? limit - ahead : 0);
        missing = (missing & ~(1u << slot)) | (ok ? 0u : 1u << slot);
        if (!ok && lane == 0) atomicCAS(p.status, kStatusOk, kStatusPageRange);
        ahead += STEP;
        if (ahead < end) page = table[ahead / p.page_size];
      }
      copy_commit();
    };
    int t = ahead;
#pragma unroll
    for (int x = 0; x < STAGES; ++x) advance(x);
    float* const scratch = ml_of(smem) + 2 * WARPS * RT;
    if constexpr (SPLIT) {
      Segment mine = seg;
      mine.row0 += warp * RT, mine.rows = min(RT, seg.rows - warp * RT);
      const bool active = mine.rows > 0;  // warps without rows still copy
      if (active) this->load_q(p, mine, scratch);
      this->clear();
      t = begin;
      for (int slot = 0; t < end; t += STEP) {
        if (lane == 0) all_missing[warp] = missing;
        copy_wait<STAGES - 1>();
        __syncthreads();
        if (active) {
#pragma unroll 1
          for (int w = 0; w < WARPS; ++w)
            if (t + w * TT < end)
              this->template tile<CAREFUL>(p, reinterpret_cast<const T*>(smem + kRing * w) + slot * TILE, t + w * TT,
                                           (all_missing[w] >> slot) & 1 ? 0 : limit, mask, scratch);
        }
        __syncthreads();
        advance(slot);
        slot = slot + 1 == STAGES ? 0 : slot + 1;
      }
    } else {
      this->load_q(p, seg, scratch);
      this->clear();
      for (int slot = 0; t < end; t += STEP) {
        copy_wait<STAGES - 1>();
        __syncwarp();
        this->template tile<CAREFUL>(p, ring + slot * TILE, t, (missing >> slot) & 1 ? 0 : limit, mask, scratch);
        __syncwarp();
        advance(slot);
        slot = slot + 1 == STAGES ? 0 : slot + 1;
      }
    }
    copy_wait<0>();
    __syncwarp();
  }
  // Attends over tokens [begin, end) of a segment with all warps of the block; every thread may then read row sums, maxima and outputs.
  template <bool CAREFUL>
  OSLO_DEVINL void walk(const PagedAttnParams& p, char* smem, Segment& seg, int limit, int begin, int end) {
    T* ring = reinterpret_cast<T*>(smem + kRing * (threadIdx.x >> 5));
    seg.length = p.lens[seg.b] - p.s + 1;
    this->template pass<CAREFUL>(p, smem, seg, limit, begin, end);
    if constexpr (SPLIT) {
      this->leave(reinterpret_cast<float*>(ring), ml_of(smem));
      __syncthreads();
    } else {
      this->join(ring, ml_of(smem));  // the warps' outputs, scaled to one maximum
    }
  }
};

// The tokens that a group's last query token sees, as far as the table (and the mask) reach.
template <bool MASK>
OSLO_DEVINL int query_limit(const PagedAttnParams& p, int query, bool report) {
  const int b = query / p.queries;
  const long long limit = static_cast<long long>(p.lens[b]) + (query - b * p.queries) - (p.queries - 1);
  const int cap = MASK ? min(p.mask_len, p.max_pages * p.page_size) : p.max_pages * p.page_size;
  if (limit > cap && report) atomicCAS(p.status, kStatusOk, kStatusPageRange);
  return static_cast<int>(min(max(limit, 0ll), static_cast<long long>(cap)));
}

// Sum of the four warps' outputs at (row, dim) after join(), and the row's total.
template <typename A>
OSLO_DEVINL float4 block_sum(const char* smem, int row, int dim, float& l, float& m) {
  const float* ml = A::ml_of(const_cast<char*>(smem));
  if constexpr (A::ROWS > A::RT) {
    const int w = row / A::RT, r = row % A::RT;
    l = ml[(A::WARPS + w) * A::RT + r], m = ml[w * A::RT + r];
    return *reinterpret_cast<const float4*>(smem + A::kRing * w + sizeof(float) * (r * A::ROW + dim));
  }
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  l = 0.f, m = -INFINITY;
#pragma unroll
  for (int w = 0; w < A::WARPS; ++w) {
    l += ml[(A::WARPS + w) * A::RT + row];
    m = fmaxf(m, ml[w * A::RT + row]);
    const float4 y = *reinterpret_cast<const float4*>(smem + A::kRing * w + sizeof(float) * (row * A::ROW + dim));
    s.x += y.x, s.y += y.y, s.z += y.z, s.w += y.w;
  }
  return s;
}

// Where a block's sums of a segment go.
struct Finish {
  float2* total;   // with it: to shared memory for the cluster, maxima and sums to total[row]
  long long slot;  // else, where not negative: to this slot of the parts
};

// Puts the block's sums where they go; whether one of this thread's is infinite or not a number.
template <typename A, typename T, int DP>
OSLO_DEVINL bool finish(const PagedAttnParams& p, char* smem, const Segment& seg, const Finish& to) {
  const int quads = p.d / 4;
  float wild = 0.f;  // 0, or NaN
  for (int x = threadIdx.x; x < seg.rows * quads; x += 128) {
    const int row = x / quads, dim = (x - row * quads) * 4;
    float l, m;
    const float4 s = block_sum<A>(smem, row, dim, l, m);
    wild = fmaf(s.x, 0.f, fmaf(s.y, 0.f, fmaf(s.z, 0.f, fmaf(s.w, 0.f, wild))));
    if (to.total != nullptr) {  // in place of the first warp's output, or where its warp left it
      *reinterpret_cast<float4*>(smem + A::place(row, dim)) = s;
      if (dim == 0) to.total[row] = make_float2(m, l);
    } else if (to.slot >= 0) {
      *reinterpret_cast<float4*>(p.part_o + (to.slot * A::ROWS + row) * DP + dim) = s;
      if (dim == 0) p.part_ml[to.slot * A::ROWS + row] = make_float2(m, l);
    } else {
      pa_store(static_cast<T*>(p.out) + seg.out_at(p, row) + dim, s, l);
    }
  }
  return wild != 0.f;
}

// Units of a segment: those that starting it costs, then its tokens.
template <typename A>
OSLO_DEVINL int segment_units(int limit) {
  constexpr int UNIT = A::WARPS * A::TT;
  return A::SEGMENT_UNITS + max(1, (limit + UNIT - 1) / UNIT);
}

// A block's range of units.
struct Range {
  long long u, u_end, base, units, blocks;  // base: first unit of the query that u is in; units: of the whole grid
  int query;
};

// Attends over the segments of a range; whether one of the thread's sums is infinite or not a number.
template <typename A, typename T, int DP, bool MASK, bool CAREFUL>
OSLO_DEVINL bool attend_range(const PagedAttnParams& p, char* smem, const Range& range) {
  constexpr int UNIT = A::WARPS * A::TT;
  const int heads = p.hkv * p.row_tiles;
  long long u = range.u, base = range.base;
  int query = range.query;
  int limit = query_limit<MASK>(p, query, threadIdx.x == 0);
  int n_units = segment_units<A>(limit);
  bool wild = false;

  while (u < range.u_end) {
    if (u >= base + static_cast<long long>(n_units) * heads) {
      base += static_cast<long long>(n_units) * heads;
      ++query;
      limit = query_limit<MASK>(p, query, threadIdx.x == 0);
      n_units = segment_units<A>(limit);
    }
    const int seg = static_cast<int>((u - base) / n_units);
    // [a, e) of the segment's units; a range that begins in the units without tokens begins with the segment, and one that ends
    // there leaves the segment to the next block
    const int a0 = static_cast<int>((u - base) - static_cast<long long>(seg) * n_units), a = a0 <= A::SEGMENT_UNITS ? 0 : a0;
    const int e = static_cast<int>(min(static_cast<long long>(n_units), a0 + (range.u_end - u)));
    if (e <= A::SEGMENT_UNITS) break;
    const int h = seg / p.row_tiles, row0 = (seg - h * p.row_tiles) * A::ROWS;

    Segment rows(p, query, h, row0, A::ROWS);
    {
      A acc;
      acc.template walk<CAREFUL>(p, smem, rows, limit, max(0, a - A::SEGMENT_UNITS) * UNIT, min(limit, (e - A::SEGMENT_UNITS) * UNIT));
    }
    const bool whole = a == 0 && e == n_units;
    wild |= finish<A, T, DP>(p, smem, rows, Finish{nullptr, whole ? -1 : static_cast<long long>(blockIdx.x) * 2 + (a == 0 ? 1 : 0)});
    if (threadIdx.x == 0 && a > 0 && e == n_units) {
      const long long start = base + static_cast<long long>(seg) * n_units;
      p.shared_seg[blockIdx.x] = make_int4(static_cast<int>(((start + A::SEGMENT_UNITS + 1) * range.blocks - 1) / range.units), query, h, row0);
    }
    u += e - a0;
    __syncthreads();  // the rings are free for the next segment
  }
  return wild;
}
// The range once more, with care for infinite values.  A function of its own at the kernel's end, so that the ordinary walk gets its
// registers as if this one were not there: in one loop with it 64 bytes and more went to memory, and a ragged batch of 32 took 33 us
// instead of 30.
template <typename A, typename T, int DP, bool MASK>
__device__ __noinline__ void attend_range_again(const PagedAttnParams& p, char* smem, Range range) {
  attend_range<A, T, DP, MASK, true>(p, smem, range);
}

template <typename T, int DP, bool WIDE, bool MASK, bool SPLIT>
__global__ void __launch_bounds__(128, PagedAttn<T, DP, WIDE, MASK, SPLIT>::BLOCKS) paged_attention_kernel(const __grid_constant__ PagedAttnParams p) {
  using A = PagedAttn<T, DP, WIDE, MASK, SPLIT>;
  constexpr int UNIT = A::WARPS * A::TT;
  extern __shared__ float4 smem4[];
  __shared__ long long scan[A::WARPS + 2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // This block's range of units: an exclusive prefix sum of the queries' units over the block's threads, each of which owns a
  // contiguous run of queries.  A query without tokens is one unit, so that its zeros are written.
  const int queries = p.b * p.queries, run = (queries + 127) / 128;
  const int first = min(queries, static_cast<int>(threadIdx.x) * run), last = min(queries, first + run);
  long long mine = 0;
  for (int i = first; i < last; ++i) mine += segment_units<A>(query_limit<MASK>(p, i, false));
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
  const long long blocks = min(static_cast<long long>(gridDim.x), max(1ll, units / A::MIN_UNITS));
  if (threadIdx.x == 0) p.shared_seg[blockIdx.x] = make_int4(-1, 0, 0, 0);
  if (blockIdx.x >= blocks) return;
  long long u = units * blockIdx.x / blocks;
  const long long u_end = units * (blockIdx.x + 1) / blocks;
  const long long at = u / heads;
  __syncthreads();
  if (mine > 0 && at >= before && at < before + mine) {
    int i = first;
    long long n;
    while (at >= before + (n = segment_units<A>(query_limit<MASK>(p, i, false)))) before += n, ++i;
    scan[0] = i;
    scan[1] = before;
  }
  __syncthreads();
  const Range range{u, u_end, scan[1] * heads, units, blocks, static_cast<int>(scan[0])};
  char* smem = reinterpret_cast<char*>(smem4);
  const bool wild = attend_range<A, T, DP, MASK, false>(p, smem, range);
  if constexpr (sizeof(T) == 2) {
    if (__syncthreads_or(wild)) attend_range_again<A, T, DP, MASK>(p, smem, range);
  }
}

OSLO_DEVINL void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
OSLO_DEVINL uint32_t peer_smem(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
OSLO_DEVINL float4 peer_load4(uint32_t addr) {
  float4 r;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w) : "r"(addr) : "memory");
  return r;
}
OSLO_DEVINL float2 peer_load2(uint32_t addr) {
  float2 r;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(r.x), "=f"(r.y) : "r"(addr) : "memory");
  return r;
}

OSLO_DEVINL void peer_store(uint32_t addr, int x) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(x) : "memory"); }

// A cluster's segment: each block takes an equal part of its tokens, and the parts are joined through distributed shared memory.
// Sets `wild` of all its blocks where a sum is infinite or not a number.
template <typename A, typename T, int DP, bool MASK, bool CAREFUL>
OSLO_DEVINL void attend_cluster(const PagedAttnParams& p, int cluster, char* smem, float2* total, int* wild) {
  constexpr int UNIT = A::WARPS * A::TT;
  const int rank = blockIdx.x % cluster, seg = blockIdx.x / cluster;
  const int heads = p.hkv * p.row_tiles, query = seg / heads, rest = seg - query * heads;
  const int h = rest / p.row_tiles, row0 = (rest - h * p.row_tiles) * A::ROWS;
  const int limit = query_limit<MASK>(p, query, threadIdx.x == 0);
  const int units = (limit + UNIT - 1) / UNIT;
  Segment part(p, query, h, row0, A::ROWS);
  {
    A acc;
    acc.template walk<CAREFUL>(p, smem, part, limit, units * rank / cluster * UNIT, min(limit, units * (rank + 1) / cluster * UNIT));
  }
  const bool mine = finish<A, T, DP>(p, smem, part, Finish{cluster == 1 ? nullptr : total, -1});
  if (cluster == 1) {
    if (!CAREFUL && mine) *wild = 1;
    return;
  }
  cluster_barrier();
  T* out = static_cast<T*>(p.out);
  const int rows = part.rows, quads = p.d / 4;
  float sums = 0.f;  // 0, or NaN
  for (int x = rank * 128 + threadIdx.x; x < rows * quads; x += cluster * 128) {
    const int row = x / quads, dim = (x - row * quads) * 4;
    const uint32_t at = smem_u32(smem) + static_cast<uint32_t>(A::place(row, dim)), at_total = smem_u32(total + row);
    float2 t[8];
    float4 y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < cluster) t[i] = peer_load2(peer_smem(at_total, i)), y[i] = peer_load4(peer_smem(at, i));
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < cluster) m = fmaxf(m, t[i].x);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < cluster) {
        const float w = A::weight(t[i].x, m);
        l += t[i].y * w;
        s.x += y[i].x * w, s.y += y[i].y * w, s.z += y[i].z * w, s.w += y[i].w * w;
      }
    pa_store(out + part.out_at(p, row) + dim, s, l);
    sums = fmaf(s.x, 0.f, fmaf(s.y, 0.f, fmaf(s.z, 0.f, fmaf(s.w, 0.f, sums))));
  }
  if (!CAREFUL && sizeof(T) == 2 && sums != 0.f)
    for (int i = 0; i < cluster; ++i) peer_store(peer_smem(smem_u32(wild), i), 1);
  cluster_barrier();  // a block's shared memory stays until all have read it
}
template <typename A, typename T, int DP, bool MASK>
__device__ __noinline__ void attend_cluster_again(const PagedAttnParams& p, int cluster, char* smem, float2* total) {
  attend_cluster<A, T, DP, MASK, true>(p, cluster, smem, total, nullptr);
}

// The same attention in one launch, for sequences that cannot be long: a cluster of up to eight blocks takes one segment.
template <typename T, int DP, bool WIDE, bool MASK, bool SPLIT>
__global__ void __launch_bounds__(128, PagedAttn<T, DP, WIDE, MASK, SPLIT>::BLOCKS) paged_attention_cluster_kernel(const __grid_constant__ PagedAttnParams p, int cluster) {
  using A = PagedAttn<T, DP, WIDE, MASK, SPLIT>;
  extern __shared__ float4 smem4[];
  __shared__ float2 total[A::ROWS];
  __shared__ int wild;
  if (threadIdx.x == 0) wild = 0;  // every walk has a barrier before its sums are there
  attend_cluster<A, T, DP, MASK, false>(p, cluster, reinterpret_cast<char*>(smem4), total, &wild);
  if constexpr (sizeof(T) == 2) {
    if (cluster == 1) __syncthreads();
    if (*static_cast<volatile int*>(&wild)) attend_cluster_again<A, T, DP, MASK>(p, cluster, reinterpret_cast<char*>(smem4), total);
  }
}

// Joins a segment that several blocks of the first kernel share.  Block (a few rows, last block of the segment); of a row's W warps
// each adds every W-th part with a running maximum, then the warps' sums are added.
template <int ROWS>
struct JoinShape {  // rows of a block, warps of a row
  static constexpr int R = ROWS == 64 ? 8 : 2, W = ROWS == 64 ? 2 : 8;
};

template <typename T, int DP, bool WIDE, bool MASK, bool SPLIT>
__global__ void __launch_bounds__(512) paged_attention_join_kernel(const PagedAttnParams p) {
  using A = PagedAttn<T, DP, WIDE, MASK, SPLIT>;
  constexpr int kJoinRows = JoinShape<A::ROWS>::R, kJoinWarps = JoinShape<A::ROWS>::W;
  constexpr int V = DP / 128 > 0 ? DP / 128 : 1;  // float4s of a lane
  constexpr int LANES = DP / 4 < 32 ? DP / 4 : 32;
  __shared__ float4 sums[kJoinRows][kJoinWarps][DP / 4];
  __shared__ float tops[kJoinRows][kJoinWarps], totals[kJoinRows][kJoinWarps];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 seg = p.shared_seg[blockIdx.y];
  if (seg.x < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, line = warp / kJoinWarps, piece = warp % kJoinWarps;
  const int row = blockIdx.x * kJoinRows + line;
  const Segment rows(p, seg.y, seg.z, seg.w, A::ROWS);
  const bool used = row < rows.rows;
  const int parts = used ? blockIdx.y - seg.x + 1 : 0;
  float m = -INFINITY, l = 0.f;
  float4 o[V];
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = piece; i < parts; i += kJoinWarps) {
    const long long slot = (static_cast<long long>(seg.x + i) * 2 + (i == 0 ? 1 : 0)) * A::ROWS + row;
    const float2 x = p.part_ml[slot];
    const float top = fmaxf(m, x.x), f = A::weight(m, top), w = A::weight(x.x, top);
    m = top;
    l = l * f + x.y * w;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int dim = (j * 32 + lane) * 4;
      if (lane < LANES && dim < p.d) {
        const float4 y = *reinterpret_cast<const float4*>(p.part_o + slot * DP + dim);
        o[j].x = o[j].x * f + y.x * w, o[j].y = o[j].y * f + y.y * w, o[j].z = o[j].z * f + y.z * w, o[j].w = o[j].w * f + y.w * w;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (lane < LANES) sums[line][piece][j * 32 + lane] = o[j];
  if (lane == 0) tops[line][piece] = m, totals[line][piece] = l;
  __syncthreads();
  if (!used || piece != 0) return;
  float w[kJoinWarps];
  m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < kJoinWarps; ++i) m = fmaxf(m, tops[line][i]);
#pragma unroll
  for (int i = 0; i < kJoinWarps; ++i) w[i] = A::weight(tops[line][i], m), l += totals[line][i] * w[i];
  T* out = static_cast<T*>(p.out) + rows.out_at(p, row);
  for (int x = lane; x * 4 < p.d; x += 32) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kJoinWarps; ++i) {
      const float4 y = sums[line][i][x];
      s.x += y.x * w[i], s.y += y.y * w[i], s.z += y.z * w[i], s.w += y.w * w[i];
    }
    pa_store(out + x * 4, s, l);
  }
}

// How a call is launched.  cluster > 0: one launch of clusters; else `grid` blocks and the join, with a workspace of `bytes`.
struct PagedAttnPlan {
  int cluster, grid, resident;
  long long bytes;
};
// Tokens that a block of the one-launch form takes at most (8 sequences of up to 4000 tokens: 20 us with 512, 26 us with 1024).
constexpr int kClusterTokens = 512;

template <typename T, int DP, bool WIDE, bool MASK, bool SPLIT>
struct PagedAttnLaunch {
  using A = PagedAttn<T, DP, WIDE, MASK, SPLIT>;
  // Blocks that the current device holds at once; negative: an error.  The first call on a device sets the kernels up.
  static int resident() {
    static std::atomic<int> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return -2;
    if (dev < 64 && known[dev].load(std::memory_order_acquire) > 0) return known[dev].load(std::memory_order_acquire);
    auto kernel = paged_attention_kernel<T, DP, WIDE, MASK, SPLIT>;
    const int smem = static_cast<int>(A::kSmem);
    int n = 0, sms = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
        cudaFuncSetAttribute(paged_attention_cluster_kernel<T, DP, WIDE, MASK, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, 128, A::kSmem) != cudaSuccess || n < 1 ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return -2;
    if (dev < 64) known[dev].store(n * sms, std::memory_order_release);
    return n * sms;
  }
  // Where the table keeps sequences short and the GPU holds all of it at once, a cluster of blocks takes each segment and one
  // launch does it (200 tokens, 16 heads: 5.5 us, against 8.4 us for two launches; 128 x 1000 tokens, where it would take
  // three rounds of blocks: 118 us, against 88 us).  Else equal ranges of the work go to as many blocks as the device holds, or
  // as the longest possible sequences have units for.
  static PagedAttnPlan plan(const PagedAttnParams& p) {
    PagedAttnPlan x{8, 0, resident(), 0};
    if (x.resident < 0) return x;
    const int most = MASK ? min(p.mask_len, p.max_pages * p.page_size) : p.max_pages * p.page_size;
    const long long segments = static_cast<long long>(p.b) * p.queries * p.hkv * p.row_tiles;
    while (x.cluster > 1 && (segments * x.cluster > x.resident || x.cluster * 32 > most)) x.cluster /= 2;
    if (segments <= x.resident && most <= static_cast<long long>(kClusterTokens) * x.cluster) return x;
    x.cluster = 0;
    const long long units = segments * ((most + A::WARPS * A::TT - 1) / (A::WARPS * A::TT));
    x.grid = static_cast<int>(units < 1 ? 1 : units < x.resident ? units : x.resident);
    x.bytes = x.grid * (2ll * A::ROWS * (DP * 4 + 8) + 16);
    return x;
  }
  static int launch(PagedAttnParams& p, const PagedAttnPlan& plan, void* ws, cudaStream_t st) {
    if (plan.cluster > 0) {
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(static_cast<unsigned>(p.b) * p.queries * p.hkv * p.row_tiles * plan.cluster);
      cfg.blockDim = dim3(128);
      cfg.dynamicSmemBytes = A::kSmem;
      cfg.stream = st;
      cudaLaunchAttribute attr{};
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = plan.cluster, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = plan.cluster > 1 ? 1 : 0;
      return cudaLaunchKernelEx(&cfg, paged_attention_cluster_kernel<T, DP, WIDE, MASK, SPLIT>, p, plan.cluster) == cudaSuccess ? 0 : -2;
    }
    char* w = static_cast<char*>(ws);
    if (w == nullptr) return -1;
    p.part_o = reinterpret_cast<float*>(w);
    p.part_ml = reinterpret_cast<float2*>(w + static_cast<long long>(plan.grid) * 2 * A::ROWS * DP * 4);
    p.shared_seg = reinterpret_cast<int4*>(w + static_cast<long long>(plan.grid) * 2 * A::ROWS * (DP * 4 + 8));
    paged_attention_kernel<T, DP, WIDE, MASK, SPLIT><<<plan.grid, 128, A::kSmem, st>>>(p);
    if (cudaGetLastError() != cudaSuccess) return -2;
    if (plan.grid == 1) return 0;  // nothing is shared
    cudaLaunchConfig_t cfg{};
    using J = JoinShape<A::ROWS>;
    cfg.gridDim = dim3(((p.rows < A::ROWS ? p.rows : A::ROWS) + J::R - 1) / J::R, plan.grid);
    cfg.blockDim = dim3(32 * J::R * J::W);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_attention_join_kernel<T, DP, WIDE, MASK, SPLIT>, p) == cudaSuccess ? 0 : -2;
  }
};

// How a call's query rows are dealt to blocks: up to 8 a block, up to 16, or 16 to each of the four warps.  64 rows read a key once
// instead of four times but cut the work into fewer pieces, so they pay where `groups` (sequences x key heads) are many: 49 x 12
// groups of 96 rows 127 us in blocks of 16 rows and 103 us in blocks of 64, 8 x 8 groups of 64 rows 47 and 40 us, one group of 64
// rows 25 and 36 us.  32-bit rows of 256 dims do not fit the registers twice: 24 rows took 1297 us in blocks of 16, 671 us of 8.
enum : int { kRows8 = 8, kRows16 = 16, kRows64 = 64 };
inline int paged_attention_rows(int dtype, int d, long long rows, long long groups) {
  if (rows <= 8 || (dtype == 0 && d > 128)) return kRows8;
  return rows <= 32 || dtype == 0 || groups * ((rows + 63) / 64) < 64 ? kRows16 : kRows64;
}

// Plans the call, and launches it where `ws` says so: what a type's translation unit offers.
template <typename L>
int paged_attention_do(PagedAttnParams& p, PagedAttnPlan& plan, bool run, void* ws, cudaStream_t st) {
  plan = L::plan(p);
  if (plan.resident < 0) return plan.resident;
  return run ? L::launch(p, plan, ws, st) : 0;
}
template <typename T, int DP, bool MASK>
int paged_attention_mask(PagedAttnParams& p, int block_rows, PagedAttnPlan& plan, bool run, void* ws, cudaStream_t st) {
  if (block_rows == kRows8) return paged_attention_do<PagedAttnLaunch<T, DP, false, MASK, false>>(p, plan, run, ws, st);
  if constexpr (sizeof(T) == 2) {
    if (block_rows == kRows64) return paged_attention_do<PagedAttnLaunch<T, DP, true, MASK, true>>(p, plan, run, ws, st);
  }
  if constexpr (sizeof(T) == 2 || DP < 256) {
    if (block_rows == kRows16) return paged_attention_do<PagedAttnLaunch<T, DP, true, MASK, false>>(p, plan, run, ws, st);
  }
  return -1;
}
template <typename T, int DP>
int paged_attention_dp(PagedAttnParams& p, int block_rows, PagedAttnPlan& plan, bool run, void* ws, cudaStream_t st) {
  return p.mask_len >= 0 ? paged_attention_mask<T, DP, true>(p, block_rows, plan, run, ws, st) : paged_attention_mask<T, DP, false>(p, block_rows, plan, run, ws, st);
}
template <typename T>
int paged_attention_type(PagedAttnParams& p, int block_rows, PagedAttnPlan& plan, bool run, void* ws, cudaStream_t st) {
  if (p.d <= 64) return paged_attention_dp<T, 64>(p, block_rows, plan, run, ws, st);
  if (p.d <= 128) return paged_attention_dp<T, 128>(p, block_rows, plan, run, ws, st);
  return paged_attention_dp<T, 256>(p, block_rows, plan, run, ws, st);
}

int paged_attention_f32(PagedAttnParams& p, int block_rows, PagedAttnPlan& plan, bool run, void* ws, cudaStream_t st);
int paged_attention_f16(PagedAttnParams& p, int block_rows, PagedAttnPlan& plan, bool run, void* ws, cudaStream_t st);
int paged_attention_bf16(PagedAttnParams& p, int block_rows, PagedAttnPlan& plan, bool run, void* ws, cudaStream_t st);

}  // namespace oslo
