// Logits on their way to the sampler: penalties for repeated tokens, sparse biases, a bit mask of allowed tokens.  Per row:
//   seen tokens (prompt and answer):  x = x > 0 ? x / repetition : x * repetition
//   tokens of the answer:             x -= frequency * count + presence
//   x += bias[i] for every i with ids[i] = v (added in the order of the list);  x = -inf where the mask's bit v is 0.
//
// Bound by bytes: one read and one write of the logits.  A CTA takes a range of neighbouring entries of a row, 16 bytes a
// thread and access, with their loads in flight while it counts the part of the row's history that falls into its range in
// shared memory (integer atomics: the order does not matter).  Every CTA of a row reads the whole history, out of L2; four
// loads a thread are in flight, otherwise their latency bounds the kernel.  Bit 31 of a count says that the prompt has the
// token, bit 30 that a bias waits for it, bit 29 that more than one does: entries with a bias are left to the threads that hold
// the biases, so that no second array is needed and the call may work in place.
// Measured: 512 rows of 100003 fp32, 8192 tokens each, 111 us (418 MB, 3.8 TB/s): 73 as a copy, 88 with biases alone; the
// counting and the penalties 14, the mask 13.  64 rows of 49152 bf16: 11 us, one row 4.9: one chain of loads after the other.
#include <type_traits>

#include "paged_common.cuh"

namespace seg {

namespace {

constexpr uint32_t kPrompt = 1u << 31, kBiased = 1u << 30, kTwice = 1u << 29, kCount = kTwice - 1;
constexpr int kThreads = 512;
constexpr int kBatch = 4;                     // history loads of a thread in flight

struct RowScale {
  float rep, inv, pres, freq;  // inv = 1 / rep: x * inv is within one and a half roundings of x / rep, at a twentieth of its instructions
};

__device__ __forceinline__ float penalise(float x, uint32_t seen, const RowScale& s) {
  if ((seen & (kPrompt | kCount)) != 0) x *= x > 0.f ? s.inv : s.rep;
  const uint32_t n = seen & kCount;
  if (n != 0) x = x - s.freq * (float)n - s.pres;
  return x;
}

// VEC neighbouring entries in one access: 16 bytes, or one entry where the rows of input and output are aligned differently.
template <typename T, int VEC> struct Pack;
template <> struct Pack<float, 4> {
  float4 v;
  __device__ void get(float* f) const { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
  __device__ void set(const float* f) { v = make_float4(f[0], f[1], f[2], f[3]); }
};
template <> struct Pack<__nv_bfloat16, 8> {
  uint4 v;
  __device__ void get(float* f) const { unpack8(load16(&v), f); }
  __device__ void set(const float* f) { store16(&v, pack8(f)); }
};
template <typename T> struct Pack<T, 1> {
  T v;
  __device__ void get(float* f) const { f[0] = to_f<T>(v); }
  __device__ void set(const float* f) { v = from_f<T>(f[0]); }
};

template <typename Tok>
__device__ __forceinline__ void count_history(const Tok* tokens, int len, int prompt, int lo, int n, int base, uint32_t* seen) {
  for (int i0 = threadIdx.x; i0 < len; i0 += kBatch * kThreads) {
    Tok tok[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) tok[j] = i0 + j * kThreads < len ? tokens[i0 + j * kThreads] : (Tok)-1;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if ((std::make_unsigned_t<Tok>)(tok[j] - (Tok)lo) >= (std::make_unsigned_t<Tok>)n) continue;
      uint32_t* at = &seen[(int)tok[j] - base];
      if (i0 + j * kThreads < prompt) atomicOr(at, kPrompt);
      else atomicAdd(at, 1u);
    }
  }
}

// kEntries: entries of a thread, 16 or 32.
template <typename T, int VEC, bool kCounts, int kEntries>
__global__ void __launch_bounds__(kThreads, kEntries == 32 ? 2 : 3) process_logits_kernel(const LogitsParams p) {
  constexpr int kVecs = kEntries / VEC, kRange = kThreads * kEntries;
  extern __shared__ uint4 seen4[];  // [kRange + VEC] counts
  uint32_t* seen = reinterpret_cast<uint32_t*>(seen4);
  const int b = blockIdx.y, tid = threadIdx.x;
  const T* x = static_cast<const T*>(p.x) + b * p.x_row;
  T* y = static_cast<T*>(p.y) + b * p.y_row;
  // The vectors of a row start at its first aligned entry; the entries before it belong to the first CTA.  base: the entry
  // that the first count stands for.
  const int head = VEC == 1 ? 0 : (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T);
  const int first = head + blockIdx.x * kRange, base = first - VEC;
  const int lo = blockIdx.x == 0 ? 0 : first, hi = min(p.V, first + kRange);
  if (lo >= hi) return;
  // What does not depend on anything is asked for first: the row's scalars, its logits, the thread's bias.
  int mask_row = -1, len = 0, prompt = 0;
  if (p.mask != nullptr) mask_row = p.mask_rows[b];
  RowScale s{1.f, 1.f, 0.f, 0.f};
  const int* ids = p.bias_ids + (int64_t)b * p.K;
  const float* bias = p.bias + (int64_t)b * p.K;
  int my_id = -1;
  float my_bias = 0.f, my_x = 0.f;
  if (kCounts) {
    if (p.tokens != nullptr) {
      len = p.token_lens[b];
      if (p.prompt_lens != nullptr) prompt = p.prompt_lens[b];
    }
    if (p.repetition != nullptr) s.rep = p.repetition[b];
    if (p.presence != nullptr) s.pres = p.presence[b];
    if (p.frequency != nullptr) s.freq = p.frequency[b];
    if (tid < p.K) {
      my_id = ids[tid];
      my_bias = bias[tid];
    }
  }
  Pack<T, VEC> in[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int v = first + (i * kThreads + tid) * VEC;
    if (v + VEC <= hi) in[i] = *reinterpret_cast<const Pack<T, VEC>*>(x + v);
  }
  const int* words = nullptr;
  if (mask_row >= p.n_masks && tid == 0 && p.mask != nullptr) atomicCAS(p.status, 0, kStatusLogitsMask);
  if (mask_row >= 0 && mask_row < p.n_masks) words = p.mask + mask_row * p.mask_row;
  if (kCounts) {
    for (int i = tid; i < (kRange + VEC + 3) / 4; i += kThreads) seen4[i] = make_uint4(0, 0, 0, 0);
    if (len < 0 || len > p.tokens_width) {
      if (tid == 0) atomicCAS(p.status, 0, kStatusLogitsLength);
      len = len < 0 ? 0 : p.tokens_width;
    }
    s.inv = 1.f / s.rep;
    if (my_id >= lo && my_id < hi) my_x = to_f<T>(x[my_id]);
    __syncthreads();
    if (p.tokens64) count_history(static_cast<const int64_t*>(p.tokens) + b * p.tokens_row, len, prompt, lo, hi - lo, base, seen);
    else count_history(static_cast<const int*>(p.tokens) + b * p.tokens_row, len, prompt, lo, hi - lo, base, seen);
    for (int i = tid; i < p.K; i += kThreads) {
      const int v = i == tid ? my_id : ids[i];
      if (v >= lo && v < hi && (atomicOr(&seen[v - base], kBiased) & kBiased) != 0) atomicOr(&seen[v - base], kTwice);
    }
    __syncthreads();
  }
  // bit j: entry v + j is allowed
  const auto allowed = [&](int v) -> uint32_t {
    if (words == nullptr) return ~0u;
    const int w = v >> 5;
    const uint32_t a = words[w];
    if (VEC == 1 || (v & 31) + VEC <= 32) return a >> (v & 31);
    return __funnelshift_r(a, (w + 1) * 32 < p.V ? (uint32_t)words[w + 1] : 0u, v & 31);
  };
  const auto entry = [&](int v) {  // one entry by itself
    const uint32_t c = kCounts ? seen[v - base] : 0u;
    if (c & kBiased) return;
    const float f = to_f<T>(x[v]);
    y[v] = from_f<T>(allowed(v) & 1 ? (c != 0 ? penalise(f, c, s) : f) : -INFINITY);
  };
  if (VEC > 1 && blockIdx.x == 0 && tid < min(head, p.V)) entry(tid);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int v = first + (i * kThreads + tid) * VEC;
    if (v + VEC > hi) {  // the row's end
      for (int j = v; j < hi; ++j) entry(j);
      continue;
    }
    float f[VEC];
    in[i].get(f);
    uint32_t c[VEC], any = 0;
    if (kCounts) {
      if constexpr (VEC > 1) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) *reinterpret_cast<uint4*>(c + j) = seen4[(v - base + j) / 4];
      } else {
        c[0] = seen[v - base];
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) any |= c[j];
    }
    if (any != 0) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (c[j] != 0) f[j] = penalise(f[j], c[j], s);
    }
    const uint32_t ok = allowed(v);
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (((ok >> j) & 1) == 0) f[j] = -INFINITY;
    if (any & kBiased) {  // those with a bias are not written here
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if ((c[j] & kBiased) == 0) y[v + j] = from_f<T>(f[j]);
    } else {
      Pack<T, VEC> out;
      out.set(f);
      *reinterpret_cast<Pack<T, VEC>*>(y + v) = out;
    }
  }
  if (kCounts && p.K > 0) {
    for (int i = tid; i < p.K; i += kThreads) {
      const int v = i == tid ? my_id : ids[i];
      if (v < lo || v >= hi) continue;
      const uint32_t c = seen[v - base];
      float r = penalise(i == tid ? my_x : to_f<T>(x[v]), c, s) + (i == tid ? my_bias : bias[i]);
      if (c & kTwice) {  // the first entry's thread adds them all
        bool mine = true;
#pragma unroll 8
        for (int j = 0; j < i; ++j) mine &= ids[j] != v;
        if (!mine) continue;
#pragma unroll 8
        for (int j = i + 1; j < p.K; ++j)
          if (ids[j] == v) r += bias[j];
      }
      y[v] = from_f<T>(allowed(v) & 1 ? r : -INFINITY);
    }
  }
}

template <typename T, int VEC, int kEntries>
int launch(const LogitsParams& p, cudaStream_t st) {
  constexpr int kRange = kThreads * kEntries, kSmem = (kRange + VEC + 3) / 4 * 16;
  const dim3 grid((p.V + kRange - 1) / kRange, p.B);
  if (p.tokens != nullptr || p.K > 0) {
    if (kSmem > 48 * 1024) {
      static bool configured[64] = {};
      int dev = 0;
      if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -2;
      if (!configured[dev]) {
        if (cudaFuncSetAttribute(process_logits_kernel<T, VEC, true, kEntries>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess) return -2;
        configured[dev] = true;
      }
    }
    process_logits_kernel<T, VEC, true, kEntries><<<grid, kThreads, kSmem, st>>>(p);
  } else {
    process_logits_kernel<T, VEC, false, kEntries><<<grid, kThreads, 0, st>>>(p);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace

int process_logits(const LogitsParams& p, cudaStream_t st) {
  if (p.B == 0 || p.V == 0) return 0;
  if (p.B > 65535) return -10;
  const int size = p.bf16 ? 2 : 4;
  // 16-byte accesses need every row of the output at the input's distance from a 16-byte boundary.  64 rows of 49152 bf16: 11.1 us,
  // one entry at a time 15.0; 512 rows of 100003 fp32: 111 and 146.
  const bool aligned = ((reinterpret_cast<uintptr_t>(p.x) - reinterpret_cast<uintptr_t>(p.y)) & 15) == 0 && (p.B == 1 || ((p.x_row - p.y_row) * size & 15) == 0);
  if (!p.bf16) return aligned ? launch<float, 4, 16>(p, st) : launch<float, 1, 16>(p, st);
  if (!aligned) return launch<__nv_bfloat16, 1, 16>(p, st);
  // bf16, more CTAs than run at once: twice the entries (as many bytes in flight as fp32 has), so that fewer CTAs read a row's history.  16
  // against 32 entries a thread, rows of 49152, us: 11.2 / 14.4 for 72 rows (432 CTAs), 14.3 / 13.7 for 96 (576), 52.9 / 48.3 for 512; 512 rows
  // of 100003: 96.4 / 84.2.  For fp32 111.9 / 110.2, and one row 5.1 / 6.5.
  const bool many = (int64_t)((p.V + kThreads * 16 - 1) / (kThreads * 16)) * p.B > 148 * 3;
  return many ? launch<__nv_bfloat16, 8, 32>(p, st) : launch<__nv_bfloat16, 8, 16>(p, st);
}

}  // namespace seg
