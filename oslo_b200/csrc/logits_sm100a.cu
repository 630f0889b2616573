// Penalties for repeated tokens, biases and a grammar mask on next-token logits, one pass over the vocabulary.
//
//   x = x > 0 ? x / r : x * r            where the token occurs in the row's history (prompt or generated)
//   x = x - presence * [c > 0] - frequency * c        c = occurrences among the generated tokens
//   x = x + bias;   x = -inf where the token is not allowed
//
// A block owns a slice of one row's vocabulary and counts the history's tokens of that slice in shared memory (integer adds:
// the result does not depend on their order).
#include "common.cuh"

namespace oslo {

struct LogitsParams {
  const void* x;
  void* y;
  const void* tokens;        // [rows, history], int64 or int32
  const int* token_lens;     // null: the whole history
  const int* prompt_lens;    // null: 0
  const float* rep;          // per row, or null: the scalar
  const float* pres;
  const float* freq;
  const float* bias;
  const int* allowed;
  long long x_stride, y_stride, tok_stride, bias_stride, allowed_stride;
  float rep_s, pres_s, freq_s;
  int rows, vocab, history, tok64;
};

constexpr int kLogitsSlice = 8192;
constexpr unsigned kSeenInPrompt = 0x80000000u;

OSLO_DEVINL float lg_f(float x) { return x; }
OSLO_DEVINL float lg_f(__half x) { return __half2float(x); }
OSLO_DEVINL float lg_f(__nv_bfloat16 x) { return __bfloat162float(x); }
OSLO_DEVINL void lg_st(float* p, float x) { *p = x; }
OSLO_DEVINL void lg_st(__half* p, float x) { *p = __float2half_rn(x); }
OSLO_DEVINL void lg_st(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

template <typename T>
__global__ void __launch_bounds__(512) process_logits_kernel(const LogitsParams p, int slices) {
  __shared__ unsigned seen[kLogitsSlice];
  const int row = blockIdx.x / slices, v0 = (blockIdx.x % slices) * kLogitsSlice;
  const int n = min(kLogitsSlice, p.vocab - v0);
  if (p.history > 0) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) seen[i] = 0;
    __syncthreads();
    const int len = p.token_lens ? min(max(p.token_lens[row], 0), p.history) : p.history;
    const int prompt = p.prompt_lens ? p.prompt_lens[row] : 0;
    for (int i = threadIdx.x; i < len; i += blockDim.x) {
      const long long at = row * p.tok_stride + i;
      const long long id = (p.tok64 ? static_cast<const long long*>(p.tokens)[at] : static_cast<const int*>(p.tokens)[at]) - v0;
      if (id >= 0 && id < n) {
        if (i < prompt) atomicOr(&seen[id], kSeenInPrompt);
        else atomicAdd(&seen[id], 1u);
      }
    }
    __syncthreads();
  }
  const float rep = p.rep ? p.rep[row] : p.rep_s, pres = p.pres ? p.pres[row] : p.pres_s, freq = p.freq ? p.freq[row] : p.freq_s;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride + v0;
  T* y = static_cast<T*>(p.y) + row * p.y_stride + v0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    float f = lg_f(x[i]);
    const unsigned s = p.history > 0 ? seen[i] : 0u;
    if (s) {
      const unsigned c = s & ~kSeenInPrompt;
      f = f > 0.f ? __fdiv_rn(f, rep) : f * rep;
      if (c) f = f - pres - freq * static_cast<float>(c);
    }
    if (p.bias) f += p.bias[row * p.bias_stride + v0 + i];
    if (p.allowed && !((p.allowed[row * p.allowed_stride + ((v0 + i) >> 5)] >> ((v0 + i) & 31)) & 1)) f = -INFINITY;
    lg_st(y + i, f);
  }
}

}  // namespace oslo

extern "C" int oslo_process_logits(const void* x, void* y, const void* tokens, const int* token_lens, const int* prompt_lens,
                                   const float* rep, const float* pres, const float* freq, const float* bias, const int* allowed,
                                   long long x_stride, long long y_stride, long long tok_stride, long long bias_stride,
                                   long long allowed_stride, float rep_s, float pres_s, float freq_s, int rows, int vocab, int history,
                                   int tok64, int dtype, void* stream) {
  using namespace oslo;
  if (rows <= 0 || vocab <= 0) return 0;
  const LogitsParams p{x, y, tokens, token_lens, prompt_lens, rep, pres, freq, bias, allowed, x_stride, y_stride, tok_stride,
                       bias_stride, allowed_stride, rep_s, pres_s, freq_s, rows, vocab, tokens ? history : 0, tok64};
  const int slices = (vocab + kLogitsSlice - 1) / kLogitsSlice;
  const long long grid = static_cast<long long>(rows) * slices;
  if (grid > 0x7fffffffll) return -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == 0) process_logits_kernel<float><<<static_cast<unsigned>(grid), 512, 0, st>>>(p, slices);
  else if (dtype == 1) process_logits_kernel<__half><<<static_cast<unsigned>(grid), 512, 0, st>>>(p, slices);
  else if (dtype == 2) process_logits_kernel<__nv_bfloat16><<<static_cast<unsigned>(grid), 512, 0, st>>>(p, slices);
  else return -1;
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
