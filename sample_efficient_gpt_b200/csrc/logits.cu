// Logits on their way to the sampler: penalties for repeated tokens, sparse biases, a bit mask of allowed tokens.  Per row:
//   seen tokens (prompt and answer):  x = x > 0 ? x / repetition : x * repetition
//   tokens of the answer:             x -= frequency * count + presence
//   x += bias[i] for every i with ids[i] = v (added in the order of the list);  x = -inf where the mask's bit v is 0.
//
// Bound by bytes: one read and one write of the logits.  A CTA takes kPer * threads neighbouring entries of a row, with their
// loads in flight while it counts the row's history that falls into its range in shared memory (integer atomics: the order
// does not matter).  Bit 31 of a count says that the prompt has the token, bit 30 that a bias waits for it: such entries are
// left to the threads that hold the biases, so that no second array is needed and the call may work in place.
#include "common.cuh"
#include "paged.h"

namespace seg {

namespace {

constexpr uint32_t kPrompt = 1u << 31, kBiased = 1u << 30, kCount = kBiased - 1;

struct RowScale {
  float rep, pres, freq;
};

__device__ __forceinline__ float penalise(float x, uint32_t seen, const RowScale& s) {
  if ((seen & (kPrompt | kCount)) != 0) x = x > 0.f ? x / s.rep : x * s.rep;
  const uint32_t n = seen & kCount;
  if (n != 0) x = x - s.freq * (float)n - s.pres;
  return x;
}

template <typename T, int kThreads, int kPer, bool kCounts>
__global__ void __launch_bounds__(kThreads) process_logits_kernel(const LogitsParams p) {
  constexpr int kRange = kThreads * kPer;
  extern __shared__ uint32_t seen[];
  __shared__ int dup;
  const int b = blockIdx.y, v0 = blockIdx.x * kRange, n = min(kRange, p.V - v0), tid = threadIdx.x;
  const T* x = static_cast<const T*>(p.x) + b * p.x_row + v0;
  T* y = static_cast<T*>(p.y) + b * p.y_row + v0;
  float f[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) f[i] = i * kThreads + tid < n ? to_f<T>(x[i * kThreads + tid]) : 0.f;
  const int* words = nullptr;
  if (p.mask != nullptr) {
    const int r = p.mask_rows[b];
    if (r >= p.n_masks && tid == 0) atomicCAS(p.status, 0, kStatusLogitsMask);
    if (r >= 0 && r < p.n_masks) words = p.mask + r * p.mask_row;
  }
  RowScale s{1.f, 0.f, 0.f};
  if (kCounts) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) seen[i * kThreads + tid] = 0u;
    if (tid == 0) dup = 0;
    if (p.repetition != nullptr) s.rep = p.repetition[b];
    if (p.presence != nullptr) s.pres = p.presence[b];
    if (p.frequency != nullptr) s.freq = p.frequency[b];
    __syncthreads();
    if (p.tokens != nullptr) {
      int len = p.token_lens[b];
      if (len < 0 || len > p.tokens_width) {
        if (tid == 0) atomicCAS(p.status, 0, kStatusLogitsLength);
        len = len < 0 ? 0 : p.tokens_width;
      }
      const int prompt = p.prompt_lens != nullptr ? p.prompt_lens[b] : 0;
      for (int i = tid; i < len; i += kThreads) {
        const int64_t tok = p.tokens64 ? static_cast<const int64_t*>(p.tokens)[b * p.tokens_row + i] : static_cast<const int*>(p.tokens)[b * p.tokens_row + i];
        const int64_t v = tok - v0;
        if (v < 0 || v >= n) continue;
        if (i < prompt) atomicOr(&seen[v], kPrompt);
        else atomicAdd(&seen[v], 1u);
      }
    }
    for (int i = tid; i < p.K; i += kThreads) {
      const int64_t v = (int64_t)p.bias_ids[(int64_t)b * p.K + i] - v0;
      if (v >= 0 && v < n && (atomicOr(&seen[v], kBiased) & kBiased) != 0) dup = 1;
    }
    __syncthreads();
  }
  const auto allowed = [&](int v) { return words == nullptr || ((words[(v0 + v) >> 5] >> ((v0 + v) & 31)) & 1) != 0; };
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int v = i * kThreads + tid;
    if (v >= n) continue;
    const uint32_t c = kCounts ? seen[v] : 0u;
    if (c & kBiased) continue;
    const float r = c != 0 ? penalise(f[i], c, s) : f[i];
    y[v] = from_f<T>(allowed(v) ? r : -INFINITY);
  }
  if (kCounts && p.K > 0) {
    const int* ids = p.bias_ids + (int64_t)b * p.K;
    const float* bias = p.bias + (int64_t)b * p.K;
    for (int i = tid; i < p.K; i += kThreads) {
      const int64_t v = (int64_t)ids[i] - v0;
      if (v < 0 || v >= n) continue;
      float r = penalise(to_f<T>(x[v]), seen[v], s) + bias[i];
      if (dup) {  // an id given more than once: the first entry's thread adds them all
        bool first = true;
        for (int j = 0; j < i && first; ++j) first = ids[j] != ids[i];
        if (!first) continue;
        for (int j = i + 1; j < p.K; ++j)
          if (ids[j] == ids[i]) r += bias[j];
      }
      y[v] = from_f<T>(allowed((int)v) ? r : -INFINITY);
    }
  }
}

template <typename T, int kThreads, int kPer>
int launch(const LogitsParams& p, cudaStream_t st) {
  constexpr int kRange = kThreads * kPer;
  const dim3 grid((p.V + kRange - 1) / kRange, p.B);
  if (p.tokens != nullptr || p.K > 0) process_logits_kernel<T, kThreads, kPer, true><<<grid, kThreads, kRange * 4, st>>>(p);
  else process_logits_kernel<T, kThreads, kPer, false><<<grid, kThreads, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace

int process_logits(const LogitsParams& p, cudaStream_t st) {
  if (p.B == 0 || p.V == 0) return 0;
  if (p.B > 65535) return -10;
  return p.bf16 ? launch<__nv_bfloat16, 512, 16>(p, st) : launch<float, 512, 16>(p, st);
}

}  // namespace seg
