// Penalties for repeated tokens, biases and a grammar mask on next-token logits, one pass over the vocabulary.
//
//   x = x > 0 ? x / r : x * r            where the token occurs in the row's history (prompt or generated)
//   x = x - presence * [c > 0] - frequency * c        c = occurrences among the generated tokens
//   x = x + bias;   x = -inf where the token is not allowed
//
// Every logit is read once and written once.  A block owns a slice of one row's vocabulary and counts the history's tokens
// of that slice in shared memory (integer atomics: their order does not matter), while its first logits are already on their
// way; then it streams the slice, 16 bytes a thread.  Counters have 16 bits for histories of less than 32768 tokens: a group of
// eight 16-bit logits then meets one 16-byte load of counters, most of them zero.  Plain streaming runs at 85 % of the copy
// bandwidth (192 x 250112 bf16: 35 us); with a history of 4095 tokens, a bias and a mask the same logits take 58 us, bound by
// issue and latency: the history is read by each of a row's 16 slices, the bias comes from L2 (as many bytes as the logits twice
// over), and every element's mask is two instructions.  Adding a cluster's tokens to each other's counters through distributed
// shared memory, so that a row reads its history once, was slower (105 us): frequent tokens serialise the remote atomics.
#include "common.cuh"
#include "step_args.h"

#include <type_traits>

namespace oslo {

struct LogitsParams {
  const void* x;
  void* y;
  const void* tokens;      // [rows, history], int64 or int32; null: no history
  const int* token_lens;   // null: the whole history
  const int* prompt_lens;  // null: 0
  const float* rep;        // per row, or null: the scalar
  const float* pres;
  const float* freq;
  const float* bias;
  const int* allowed;
  long long x_stride, y_stride, tok_stride, bias_stride, allowed_stride;
  float rep_s, pres_s, freq_s;
  int rows, vocab, history, tok64, slice, slices;  // tokens of a slice, slices of a row
};

constexpr int kLogitsThreads = 256;
template <typename T>
constexpr int kLogitsAhead = sizeof(T) / 2 * 2;  // 16-byte groups of a thread in flight: sixteen logits
constexpr int kLogitsCounters = 32 * 1024;  // bytes of counters of a block
constexpr int kLogitsLeast = 2048;          // tokens of a slice at least

// A token's counter: the top bit says that the prompt holds it, the others how often it was generated.
template <typename C>
struct Counter {
  static constexpr unsigned kPrompt = 1u << (8 * sizeof(C) - 1);
};

OSLO_DEVINL float lg_f(float x) { return x; }
OSLO_DEVINL float lg_f(__half x) { return __half2float(x); }
OSLO_DEVINL float lg_f(__nv_bfloat16 x) { return __bfloat162float(x); }
OSLO_DEVINL void lg_st(float& p, float x) { p = x; }
OSLO_DEVINL void lg_st(__half& p, float x) { p = __float2half_rn(x); }
OSLO_DEVINL void lg_st(__nv_bfloat16& p, float x) { p = __float2bfloat16_rn(x); }

template <typename C>
struct LogitsRow {
  float rep, inv, pres, freq;
  // x / r is x times the reciprocal, both rounded to 32 bits: off by 2^-23 of the quotient at most, where a division is by 2^-24
  // (192 x 250112 bf16 with every option: 58 us, with a division 70 us under a branch and 74 us
  // without).  No branches here: some lane of a warp has a seen token nearly always.
  OSLO_DEVINL float operator()(float f, unsigned seen) const {
    const unsigned c = seen & ~Counter<C>::kPrompt;
    const float r = f * (f > 0.f ? inv : rep);
    f = seen ? r : f;
    return c ? f - pres - freq * static_cast<float>(c) : f;
  }
};

// Room for a slice's counters and for their shift to a 16-byte boundary, by up to seven of them.
template <typename C>
__host__ __device__ constexpr int counter_bytes(int slice) { return (slice + 8) * static_cast<int>(sizeof(C)); }

// Adds the history's tokens in [v0, v0 + n) to their counters.
template <typename I, typename C>
OSLO_DEVINL void count_tokens(const I* tokens, int len, int prompt, int v0, int n, C* seen) {
  for (int i0 = threadIdx.x; i0 < len; i0 += kLogitsThreads * 8) {
    I id[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) id[j] = i0 + j * kLogitsThreads < len ? __ldg(tokens + i0 + j * kLogitsThreads) : static_cast<I>(-1);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned at = static_cast<unsigned>(id[j]) - v0;
      if (at < static_cast<unsigned>(n) && (sizeof(I) == 4 || static_cast<unsigned>(static_cast<unsigned long long>(id[j]) >> 32) == 0)) {
        // two 16-bit counters share a word; a count below 32768 never carries into its neighbour or its own top bit
        const uint32_t addr = smem_u32(seen + at), sh = (addr & 3) * 8;
        if (i0 + j * kLogitsThreads < prompt) asm volatile("red.shared::cta.or.b32 [%0], %1;" ::"r"(addr & ~3u), "r"(Counter<C>::kPrompt << sh) : "memory");
        else asm volatile("red.shared::cta.add.u32 [%0], %1;" ::"r"(addr & ~3u), "r"(1u << sh) : "memory");
      }
    }
  }
}

// C: counter type, uint16_t for histories of less than 32768 tokens, uint32_t for longer ones, void without a history
template <typename T, typename C, bool BIAS, bool ALLOWED>
__global__ void __launch_bounds__(kLogitsThreads, 5) process_logits_kernel(const LogitsParams p) {
  constexpr bool HISTORY = sizeof(C) > 1;
  constexpr int E = 16 / sizeof(T), AHEAD = kLogitsAhead<T>;
  extern __shared__ uint4 counters4[];
  C* const counters = reinterpret_cast<C*>(counters4);
  const int row = blockIdx.x / p.slices, v0 = (blockIdx.x - row * p.slices) * p.slice;
  const int n = min(p.slice, p.vocab - v0);
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride + v0;
  T* y = static_cast<T*>(p.y) + row * p.y_stride + v0;
  // elements before the first 16-byte boundary of the slice; the counters are shifted so that a group's are aligned too
  const int to_edge = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T));
  const int head = min(to_edge, n);
  C* const seen = counters + ((E - to_edge) & (E - 1));
  const bool aligned = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  const int groups = aligned ? (n - head) / E : 0;
  // the first logits are on their way while the history is counted
  uint4 ahead[AHEAD];
  const auto fetch = [&](int g0) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (g0 + j * kLogitsThreads < groups)
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(ahead[j].x), "=r"(ahead[j].y), "=r"(ahead[j].z), "=r"(ahead[j].w) : "l"(x + head + (g0 + j * kLogitsThreads) * E));
  };
  fetch(threadIdx.x);
  LogitsRow<C> pen{p.rep_s, 1.f, p.pres_s, p.freq_s};
  if constexpr (HISTORY) {
    for (int i = threadIdx.x; i < counter_bytes<C>(p.slice) / 16; i += kLogitsThreads) counters4[i] = make_uint4(0, 0, 0, 0);
    if (p.rep) pen.rep = p.rep[row];
    if (p.pres) pen.pres = p.pres[row];
    if (p.freq) pen.freq = p.freq[row];
    pen.inv = __fdiv_rn(1.f, pen.rep);
    const int len = p.token_lens ? min(max(p.token_lens[row], 0), p.history) : p.history;
    const int prompt = p.prompt_lens ? p.prompt_lens[row] : 0;
    __syncthreads();
    if (p.tok64) count_tokens(static_cast<const long long*>(p.tokens) + row * p.tok_stride, len, prompt, v0, n, seen);
    else count_tokens(static_cast<const int*>(p.tokens) + row * p.tok_stride, len, prompt, v0, n, seen);
    __syncthreads();
  }
  const float* bias = p.bias ? p.bias + row * p.bias_stride + v0 : nullptr;
  const int* allowed = p.allowed ? p.allowed + row * p.allowed_stride : nullptr;
  const auto one = [&](int i) {
    float f = lg_f(x[i]);
    if constexpr (HISTORY) f = pen(f, seen[i]);
    if (BIAS) f += bias[i];
    if (ALLOWED && !((allowed[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1)) f = -INFINITY;
    lg_st(y[i], f);
  };
  if (!aligned) {
    for (int i = threadIdx.x; i < n; i += kLogitsThreads) one(i);  // rows of input and output that no 16-byte access serves
    return;
  }
  const int tail = head + groups * E;
  if (threadIdx.x < head) one(threadIdx.x);
  if (threadIdx.x < n - tail) one(tail + threadIdx.x);
  const bool bias16 = BIAS && (reinterpret_cast<uintptr_t>(bias + head) & 15) == 0;
  for (int g0 = threadIdx.x; g0 < groups; g0 += AHEAD * kLogitsThreads) {
    // all operands of the groups in flight are requested before the first is used
    float4 b[AHEAD][E / 4];
    unsigned lo[AHEAD], hi[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int g = g0 + j * kLogitsThreads, i = head + g * E, at = v0 + i;
      if (g >= groups) break;
      if constexpr (BIAS) {
#pragma unroll
        for (int e = 0; e < E; e += 4)
          b[j][e / 4] = bias16 ? __ldg(reinterpret_cast<const float4*>(bias + i + e))
                               : make_float4(__ldg(bias + i + e), __ldg(bias + i + e + 1), __ldg(bias + i + e + 2), __ldg(bias + i + e + 3));
      }
      if constexpr (ALLOWED) {
        lo[j] = __ldg(allowed + (at >> 5));
        hi[j] = (at & 31) + E > 32 ? __ldg(allowed + (at >> 5) + 1) : 0u;  // the last group ends inside the last word
      }
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int g = g0 + j * kLogitsThreads, i = head + g * E;
      if (g >= groups) break;
      union {
        uint4 u;
        T t[E];
      } in, out;
      in.u = ahead[j];
      float f[E];
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = lg_f(in.t[e]);
      if constexpr (HISTORY) {
        constexpr int W = E * sizeof(C) / 4;  // words of the group's counters
        unsigned w[W];
        if constexpr (W == 2) {
          *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(seen + i);
        } else {
#pragma unroll
          for (int k = 0; k < W; k += 4) *reinterpret_cast<uint4*>(w + k) = *reinterpret_cast<const uint4*>(seen + i + k * (4 / sizeof(C)));
        }
        unsigned any = 0;
#pragma unroll
        for (int k = 0; k < W; ++k) any |= w[k];
        if (any) {
#pragma unroll
          for (int e = 0; e < E; ++e)
            f[e] = pen(f[e], sizeof(C) == 4 ? w[e * sizeof(C) / 4] : (w[e * sizeof(C) / 4] >> (e % (4 / sizeof(C)) * 16)) & 0xffffu);
        }
      }
      if constexpr (BIAS) {
#pragma unroll
        for (int e = 0; e < E; e += 4) f[e] += b[j][e / 4].x, f[e + 1] += b[j][e / 4].y, f[e + 2] += b[j][e / 4].z, f[e + 3] += b[j][e / 4].w;
      }
      if constexpr (ALLOWED) {
        const unsigned bits = __funnelshift_r(lo[j], hi[j], (v0 + i) & 31);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (!((bits >> e) & 1)) f[e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) lg_st(out.t[e], f[e]);
      *reinterpret_cast<uint4*>(y + i) = out.u;
    }
    fetch(g0 + AHEAD * kLogitsThreads);
  }
}

template <typename T>
int process_logits_launch(LogitsParams& p, cudaStream_t st) {
  const bool small = p.history < 32768;
  // Four blocks an SM (148 of them) when the work is small, else slices as large as the counters' room: every slice reads its
  // row's history again.  One row of 50304: 4.6 us with 8192-token slices, 3.1 us with 2048; 128 rows of 32000 with histories of
  // 8000: 15.9 us in 444 blocks, 23.3 us in 1776.
  const int most = kLogitsCounters / (small ? 2 : 4);
  const long long fair = static_cast<long long>(p.rows) * p.vocab / 592;
  const int want = static_cast<int>(fair < kLogitsLeast ? kLogitsLeast : fair > most ? most : fair);
  p.slices = (p.vocab + want - 1) / want;
  p.slice = ((p.vocab + p.slices - 1) / p.slices + 31) / 32 * 32;
  p.slices = (p.vocab + p.slice - 1) / p.slice;
  const long long grid = static_cast<long long>(p.rows) * p.slices;
  if (grid > 0x7fffffffll) return -1;
  const unsigned blocks = static_cast<unsigned>(grid);
  const auto go = [&](auto bias, auto allowed) {
    constexpr bool B = decltype(bias)::value, A = decltype(allowed)::value;
    if (!p.tokens) process_logits_kernel<T, char, B, A><<<blocks, kLogitsThreads, 0, st>>>(p);
    else if (small) process_logits_kernel<T, uint16_t, B, A><<<blocks, kLogitsThreads, counter_bytes<uint16_t>(p.slice), st>>>(p);
    else process_logits_kernel<T, uint32_t, B, A><<<blocks, kLogitsThreads, counter_bytes<uint32_t>(p.slice), st>>>(p);
  };
  if (p.bias && p.allowed) go(std::true_type(), std::true_type());
  else if (p.bias) go(std::true_type(), std::false_type());
  else if (p.allowed) go(std::false_type(), std::true_type());
  else go(std::false_type(), std::false_type());
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace oslo

extern "C" int oslo_process_logits(const OsloProcessLogitsArgs* a) {
  using namespace oslo;
  if (a->rows <= 0 || a->vocab <= 0) return 0;
  if (a->vocab > 0x3fffffff || a->history > 0x3fffffff || a->rows > 0x7fffffff) return -1;
  LogitsParams p{};
  p.x = reinterpret_cast<const void*>(a->x), p.y = reinterpret_cast<void*>(a->y);
  p.tokens = a->history > 0 ? reinterpret_cast<const void*>(a->tokens) : nullptr;
  p.token_lens = reinterpret_cast<const int*>(a->token_lens), p.prompt_lens = reinterpret_cast<const int*>(a->prompt_lens);
  p.rep = reinterpret_cast<const float*>(a->rep), p.pres = reinterpret_cast<const float*>(a->pres);
  p.freq = reinterpret_cast<const float*>(a->freq), p.bias = reinterpret_cast<const float*>(a->bias);
  p.allowed = reinterpret_cast<const int*>(a->allowed);
  p.x_stride = a->x_stride, p.y_stride = a->y_stride, p.tok_stride = a->tok_stride, p.bias_stride = a->bias_stride;
  p.allowed_stride = a->allowed_stride, p.rep_s = static_cast<float>(a->rep_s), p.pres_s = static_cast<float>(a->pres_s);
  p.freq_s = static_cast<float>(a->freq_s), p.rows = a->rows, p.vocab = a->vocab, p.history = a->history, p.tok64 = a->tok64;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a->stream);
  if (a->dtype == 0) return process_logits_launch<float>(p, st);
  if (a->dtype == 1) return process_logits_launch<__half>(p, st);
  if (a->dtype == 2) return process_logits_launch<__nv_bfloat16>(p, st);
  return -1;
}
