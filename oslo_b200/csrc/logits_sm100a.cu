// Penalties for repeated tokens, biases and a grammar mask on next-token logits, one pass over the vocabulary.
//
//   x = x > 0 ? x / r : x * r            where the token occurs in the row's history (prompt or generated)
//   x = x - presence * [c > 0] - frequency * c        c = occurrences among the generated tokens
//   x = x + bias;   x = -inf where the token is not allowed
//
// HBM bounds it: every logit is read once and written once.  A block owns a slice of one row's vocabulary, with one 32-bit
// counter of the history per token in shared memory (bit 31: seen in the prompt; the rest: generated so often; both are
// updated by integer atomics, whose order does not matter).  The blocks of a cluster own neighbouring slices: each reads
// one part of the history and adds every token to the counter of the block that owns it, through distributed shared memory, so
// a row of up to 65536 tokens reads its history once.  Slices of at most 8192 tokens (32 KB) let an SM hold six blocks, whose
// counting and streaming phases overlap.
#include "common.cuh"

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
  int rows, vocab, history, tok64, slice, slices;  // slices a row, a multiple of the cluster's size
};

constexpr int kLogitsSlice = 8192;
constexpr int kLogitsThreads = 256;
constexpr unsigned kSeenInPrompt = 0x80000000u;

OSLO_DEVINL float lg_f(float x) { return x; }
OSLO_DEVINL float lg_f(__half x) { return __half2float(x); }
OSLO_DEVINL float lg_f(__nv_bfloat16 x) { return __bfloat162float(x); }
OSLO_DEVINL void lg_st(float& p, float x) { p = x; }
OSLO_DEVINL void lg_st(__half& p, float x) { p = __float2half_rn(x); }
OSLO_DEVINL void lg_st(__nv_bfloat16& p, float x) { p = __float2bfloat16_rn(x); }

OSLO_DEVINL void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// shared-memory address of the same variable in another block of the cluster
OSLO_DEVINL uint32_t peer_smem(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

struct LogitsRow {
  float rep, pres, freq;
  OSLO_DEVINL float operator()(float f, unsigned seen) const {
    if (seen == 0) return f;
    f = f > 0.f ? __fdiv_rn(f, rep) : f * rep;
    const unsigned c = seen & ~kSeenInPrompt;
    return c ? f - pres - freq * static_cast<float>(c) : f;
  }
};

template <typename T, bool HISTORY>
__global__ void __launch_bounds__(kLogitsThreads) process_logits_kernel(const LogitsParams p, int cluster) {
  constexpr int E = 16 / sizeof(T);
  extern __shared__ uint4 seen4[];
  unsigned* const counters = reinterpret_cast<unsigned*>(seen4);
  const int row = blockIdx.x / p.slices, part = blockIdx.x % p.slices;
  const int v0 = min(part * p.slice, p.vocab), n = min(p.slice, p.vocab - v0);
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride + v0;
  T* y = static_cast<T*>(p.y) + row * p.y_stride + v0;
  // elements before the first 16-byte boundary of the slice; the counters are shifted so that a group's are aligned too
  const int to_edge = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T));
  const int head = min(to_edge, n), shift = (4 - (to_edge & 3)) & 3;
  if constexpr (HISTORY) {
    for (int i = threadIdx.x; i < (p.slice + 3) / 4 + 1; i += kLogitsThreads) seen4[i] = make_uint4(0, 0, 0, 0);
    if (cluster > 1) cluster_barrier();
    else __syncthreads();
    const int len = p.token_lens ? min(max(p.token_lens[row], 0), p.history) : p.history;
    const int prompt = p.prompt_lens ? p.prompt_lens[row] : 0;
    const int rank = part % cluster, c0 = (part - rank) * p.slice;  // the cluster's first token
    const long long range = min(static_cast<long long>(p.slice) * cluster, static_cast<long long>(p.vocab) - c0);
    const uint32_t mine = smem_u32(counters);
    for (int i = rank * kLogitsThreads + threadIdx.x; i < len; i += cluster * kLogitsThreads) {
      const long long at = row * p.tok_stride + i;
      const long long id = (p.tok64 ? static_cast<const long long*>(p.tokens)[at] : static_cast<const int*>(p.tokens)[at]) - c0;
      if (id < 0 || id >= range) continue;
      const int owner = static_cast<int>(id) / p.slice;
      // the owner shifts its counters by its own slice's distance to a 16-byte boundary
      const T* ox = static_cast<const T*>(p.x) + row * p.x_stride + (c0 + owner * p.slice);
      const int edge = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(ox) & 15)) & 15) / static_cast<int>(sizeof(T));
      const uint32_t local = mine + 4 * (static_cast<int>(id) - owner * p.slice + ((4 - (edge & 3)) & 3));
      const uint32_t addr = cluster > 1 ? peer_smem(local, owner) : local;
      if (i < prompt) asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(addr), "r"(kSeenInPrompt) : "memory");
      else asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(addr), "r"(1u) : "memory");
    }
    if (cluster > 1) cluster_barrier();
    else __syncthreads();
  }
  if (n <= 0) return;
  const unsigned* seen = counters + shift;
  LogitsRow pen{p.rep_s, p.pres_s, p.freq_s};
  if constexpr (HISTORY) {
    if (p.rep) pen.rep = p.rep[row];
    if (p.pres) pen.pres = p.pres[row];
    if (p.freq) pen.freq = p.freq[row];
  }
  const float* bias = p.bias ? p.bias + row * p.bias_stride + v0 : nullptr;
  const int* allowed = p.allowed ? p.allowed + row * p.allowed_stride : nullptr;
  const auto one = [&](int i) {
    float f = lg_f(x[i]);
    if constexpr (HISTORY) f = pen(f, seen[i]);
    if (bias) f += bias[i];
    if (allowed && !((allowed[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1)) f = -INFINITY;
    lg_st(y[i], f);
  };
  if ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15) {
    for (int i = threadIdx.x; i < n; i += kLogitsThreads) one(i);  // rows of input and output that no 16-byte access serves
    return;
  }
  const int groups = (n - head) / E, tail = head + groups * E;
  if (threadIdx.x < head) one(threadIdx.x);
  if (threadIdx.x < n - tail) one(tail + threadIdx.x);
  const bool bias16 = bias && (reinterpret_cast<uintptr_t>(bias + head) & 15) == 0;
#pragma unroll 2
  for (int g = threadIdx.x; g < groups; g += kLogitsThreads) {
    const int i = head + g * E;
    union {
      uint4 u;
      T t[E];
    } in, out;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(in.u.x), "=r"(in.u.y), "=r"(in.u.z), "=r"(in.u.w) : "l"(x + i));
    float f[E];
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = lg_f(in.t[e]);
    if constexpr (HISTORY) {
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        const uint4 s = *reinterpret_cast<const uint4*>(seen + i + e);
        if (s.x | s.y | s.z | s.w) f[e] = pen(f[e], s.x), f[e + 1] = pen(f[e + 1], s.y), f[e + 2] = pen(f[e + 2], s.z), f[e + 3] = pen(f[e + 3], s.w);
      }
    }
    if (bias) {
      if (bias16) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
          const float4 b = *reinterpret_cast<const float4*>(bias + i + e);
          f[e] += b.x, f[e + 1] += b.y, f[e + 2] += b.z, f[e + 3] += b.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] += bias[i + e];
      }
    }
    if (allowed) {
      const int at = v0 + i, w = at >> 5, sh = at & 31;
      const unsigned lo = allowed[w], hi = sh + E > 32 ? allowed[w + 1] : 0u;  // the last group ends inside the last word
      const unsigned bits = __funnelshift_r(lo, hi, sh);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (!((bits >> e) & 1)) f[e] = -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) lg_st(out.t[e], f[e]);
    *reinterpret_cast<uint4*>(y + i) = out.u;
  }
}

template <typename T>
int process_logits_launch(LogitsParams& p, cudaStream_t st) {
  int cluster = 1;
  if (p.tokens) {
    while (cluster < 8 && cluster * 2048 < p.vocab) cluster *= 2;  // eight blocks read the history from 16384 tokens on
  }
  const int spans = (p.vocab + cluster * kLogitsSlice - 1) / (cluster * kLogitsSlice);  // clusters a row
  p.slices = spans * cluster;
  p.slice = ((p.vocab + p.slices - 1) / p.slices + 31) / 32 * 32;
  const long long grid = static_cast<long long>(p.rows) * p.slices;
  if (grid > 0x7fffffffll) return -1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kLogitsThreads);
  cfg.dynamicSmemBytes = p.tokens ? (p.slice + 8) * sizeof(unsigned) : 0;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  const cudaError_t rc = p.tokens ? cudaLaunchKernelEx(&cfg, process_logits_kernel<T, true>, p, cluster)
                                  : cudaLaunchKernelEx(&cfg, process_logits_kernel<T, false>, p, cluster);
  return rc == cudaSuccess ? 0 : -2;
}

}  // namespace oslo

// Everything a call needs, eight bytes each.  Strides in elements.
struct OsloProcessLogitsArgs {
  long long x, y, tokens, token_lens, prompt_lens, rep, pres, freq, bias, allowed, stream;  // addresses; from tokens on they may be 0
  long long x_stride, y_stride, tok_stride, bias_stride, allowed_stride, rows, vocab, history, tok64, dtype;
  double rep_s, pres_s, freq_s;
};

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
