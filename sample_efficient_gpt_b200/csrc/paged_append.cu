// The packed qkv projection of new tokens -> queries for the attention, and keys and values in the pages of a cache.
//
//   r = R(pos) x (split-half rotation, fp32), q = qgain * r / rms(r), k = r / rms(r) (rms over the head, eps 1e-6; both
//   unnormalised without QK-norm), v = s c (a1 v + a2 v1), c = rsqrt(a1^2 + a2^2 + 1e-8)
// Same formulas as qkv_post.cu; the results of token t of sequence b go to slot p % P of page table[b][p / P], where
// p = lens[b] + (t - cu[b]), and the rotation is that of position p + pos_base[b].
//
// Bound by bytes: every element of the projection is read once and written once, about six operations each.  A CTA takes a
// few whole tokens (kItems * 256 work items, an item being 16 elements of one head: 8 rotary pairs, two 16-byte loads), one
// thread per token finds its sequence and page while the loads of all its items are already in flight; hd / 16 neighbouring
// lanes share a head and sum its squares with shuffles.
#include "common.cuh"
#include "paged.h"

namespace seg {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;  // tokens of a CTA
constexpr float kQkEps = 1e-6f;
constexpr float kMixEps = 1e-8f;

template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
  const unsigned lane = threadIdx.x & 31u;
  const unsigned mask = ((1u << LPH) - 1u) << (lane & ~(unsigned)(LPH - 1));  // lanes of other heads may be in another branch
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
  return v;
}

// Where a token's rows go: page < 0 = nowhere (behind the last sequence, or an error that the status word tells).
struct TokenPlace {
  int page, slot, pos;
};

__device__ __forceinline__ TokenPlace find_place(const PagedAppendParams& p, int t) {
  TokenPlace w{-1, 0, 0};
  int b = t, first = t;
  if (p.cu != nullptr) {
    int lo = 0, hi = p.B;  // last b with cu[b] <= t: empty sequences before t's own are passed over
    if (t < p.cu[0] || t >= p.cu[p.B]) return w;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.cu[mid] <= t) lo = mid; else hi = mid;
    }
    b = lo;
    first = p.cu[b];
  }
  const int64_t at = (int64_t)p.lens[b] + (t - first);
  const int64_t pos = at + (p.pos_base != nullptr ? p.pos_base[b] : 0);
  if (p.lens[b] < 0 || at >= (int64_t)p.table_width * p.pool.P || pos < 0 || pos >= p.rope_rows) {
    atomicCAS(p.status, 0, kStatusAppendTable);
    return w;
  }
  const int i = p.pool.shift >= 0 ? (int)(at >> p.pool.shift) : (int)at / p.pool.P;
  const int page = p.table[b * p.table_stride + i];
  if ((unsigned)page >= (unsigned)p.pool.n_pages) {
    atomicCAS(p.status, 0, kStatusAppendPage);
    return w;
  }
  w.page = page;
  w.slot = (int)at - i * p.pool.P;
  w.pos = (int)pos;
  return w;
}

// Loads of one item, issued before anything is known about where the token goes.
struct Item {
  bf16x8 x1, x2, u1, u2;
};

template <int HD, int kItems>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const PagedAppendParams p, int tokens_per_cta) {
  constexpr int HALF = HD / 2, LPH = HD / 16;
  __shared__ TokenPlace place[kMaxTokens];
  const int nslots = p.H + 2 * p.Hkv, nrot = p.H + p.Hkv;
  const int t0 = blockIdx.x * tokens_per_cta;
  const int n_tok = min(tokens_per_cta, p.T - t0);
  const int n_items = n_tok * nslots * LPH;
  const __nv_bfloat16* qkv = static_cast<const __nv_bfloat16*>(p.qkv);
  const __nv_bfloat16* v1 = static_cast<const __nv_bfloat16*>(p.v1);
  const float a1 = *p.alpha1, a2 = *p.alpha2, vs = *p.vscale, qg = *p.qgain;
  const float c = vs * rsqrtf(a1 * a1 + a2 * a2 + kMixEps);
  for (int base = 0; base < n_items; base += kItems * kThreads) {
    Item it[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int item = base + i * kThreads + threadIdx.x;
      if (item < n_items) {
        const int sub = item % LPH, rest = item / LPH, tok = rest / nslots, slot = rest - tok * nslots;
        const __nv_bfloat16* src = qkv + (int64_t)(t0 + tok) * p.qkv_stride + slot * HD + sub * 8;
        it[i].x1 = *reinterpret_cast<const bf16x8*>(src);
        it[i].x2 = *reinterpret_cast<const bf16x8*>(src + HALF);
        if (slot >= nrot && v1 != nullptr) {
          const __nv_bfloat16* u = v1 + ((int64_t)(t0 + tok) * p.Hkv + (slot - nrot)) * HD + sub * 8;
          it[i].u1 = *reinterpret_cast<const bf16x8*>(u);
          it[i].u2 = *reinterpret_cast<const bf16x8*>(u + HALF);
        }
      }
    }
    if (base == 0) {
      if ((int)threadIdx.x < n_tok) place[threadIdx.x] = find_place(p, t0 + threadIdx.x);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int item = base + i * kThreads + threadIdx.x;
      if (item >= n_items) continue;  // the LPH lanes of a head leave together: n_items is a multiple of LPH
      const int sub = item % LPH, rest = item / LPH, tok = rest / nslots, slot = rest - tok * nslots;
      const int64_t t = t0 + tok;
      const TokenPlace w = place[tok];
      float x1[8], x2[8];
      unpack8(it[i].x1, x1);
      unpack8(it[i].x2, x2);
      if (w.page < 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x1[j] = x2[j] = 0.f;
      } else if (slot < nrot) {
        float cs[8], sn[8];
        load8<float>(p.cos + (int64_t)w.pos * HALF + sub * 8, cs);
        load8<float>(p.sin + (int64_t)w.pos * HALF + sub * 8, sn);
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float r1 = x1[j] * cs[j] - x2[j] * sn[j], r2 = x1[j] * sn[j] + x2[j] * cs[j];
          x1[j] = r1;
          x2[j] = r2;
          ss += r1 * r1 + r2 * r2;
        }
        if (p.qknorm) {
          ss = head_sum<LPH>(ss);
          const float mul = rsqrtf(ss / HD + kQkEps) * (slot < p.H ? qg : 1.f);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            x1[j] *= mul;
            x2[j] *= mul;
          }
        }
      } else {
        float u1[8], u2[8];
        if (v1 != nullptr) {
          unpack8(it[i].u1, u1);
          unpack8(it[i].u2, u2);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x1[j] = c * (a1 * x1[j] + a2 * (v1 != nullptr ? u1[j] : x1[j]));
          x2[j] = c * (a1 * x2[j] + a2 * (v1 != nullptr ? u2[j] : x2[j]));
        }
      }
      const bf16x8 y1 = pack8(x1), y2 = pack8(x2);
      if (slot < p.H) {
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.q) + (t * p.H + slot) * HD + sub * 8;
        *reinterpret_cast<bf16x8*>(dst) = y1;
        *reinterpret_cast<bf16x8*>(dst + HALF) = y2;
        continue;
      }
      const bool is_k = slot < nrot;
      const int h = slot - (is_k ? p.H : nrot);
      if (w.page >= 0) {
        __nv_bfloat16* dst =
            is_k ? static_cast<__nv_bfloat16*>(p.pool.k) + w.page * p.pool.k_page + w.slot * p.pool.k_slot + h * p.pool.k_head
                 : static_cast<__nv_bfloat16*>(p.pool.v) + w.page * p.pool.v_page + w.slot * p.pool.v_slot + h * p.pool.v_head;
        *reinterpret_cast<bf16x8*>(dst + sub * 8) = y1;
        *reinterpret_cast<bf16x8*>(dst + HALF + sub * 8) = y2;
      }
      void* out = is_k ? p.k_out : p.v_out;
      if (out != nullptr) {
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(out) + (t * p.Hkv + h) * HD + sub * 8;
        *reinterpret_cast<bf16x8*>(dst) = y1;
        *reinterpret_cast<bf16x8*>(dst + HALF) = y2;
      }
    }
  }
}

template <int HD>
int launch(const PagedAppendParams& p, cudaStream_t st) {
  const int per_token = (p.H + 2 * p.Hkv) * (HD / 16);
  // Few tokens: a token per CTA and an item per thread, so that the call lasts as long as one chain of dependent loads.
  // Many: four items per thread keep enough loads in flight to saturate the memory.
  if ((int64_t)p.T * per_token <= 148 * 2 * kThreads) {
    paged_append_kernel<HD, 1><<<p.T, kThreads, 0, st>>>(p, 1);
  } else {
    int n = 4 * kThreads / per_token;
    n = n < 1 ? 1 : n > kMaxTokens ? kMaxTokens : n;
    paged_append_kernel<HD, 4><<<(p.T + n - 1) / n, kThreads, 0, st>>>(p, n);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace

int paged_append(const PagedAppendParams& p, cudaStream_t st) {
  if (p.T == 0) return 0;
  switch (p.hd) {
    case 32: return launch<32>(p, st);
    case 64: return launch<64>(p, st);
    case 128: return launch<128>(p, st);
  }
  return -10;
}

}  // namespace seg
