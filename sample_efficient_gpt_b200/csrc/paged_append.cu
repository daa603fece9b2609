// The packed qkv projection of new tokens -> queries for the attention, and keys and values in the pages of a cache.
//
//   r = R(pos) x (split-half rotation, fp32), q = qgain * r / rms(r), k = r / rms(r) (rms over the head, eps 1e-6; both
//   unnormalised without QK-norm), v = s c (a1 v + a2 v1), c = rsqrt(a1^2 + a2^2 + 1e-8)
// Same formulas as qkv_post.cu; the results of token t of sequence b go to slot p % P of page table[b][p / P], where
// p = lens[b] + (t - cu[b]), and the rotation is that of position p + pos_base[b].
//
// Bound by bytes: every element of the projection is read once and written once, about six operations each.  A work item is 16
// elements of one head (8 rotary pairs: two 16-byte accesses); hd / 16 neighbouring lanes share a head and sum its squares with
// shuffles.  Few tokens: a CTA per token and an item per thread, so that the call lasts as long as one chain of dependent
// loads (length -> page -> rotation).  Many: that chain, longer by the search for the token's sequence, would stand in front
// of every CTA's work, so a producer warp runs it ahead and brings each group of tokens - projection rows, first values,
// rotation rows - into a ring in shared memory with bulk copies, from which eight warps compute and store.
// Measured: one token 2.6 us; 8191 tokens of 32 + 16 heads of 128 with the first values 42 us (222 MB, 5.3 TB/s), 32768 tokens of
// 18 + 12 heads of 64 59 us (279 MB, 4.7 TB/s; the stores of 16 bytes a lane take most of 0.6 of the issue slots).  Results put back into
// the ring and sent away as bulk copies: 57 us, but 44 where a token's heads lie apart, and later for few tokens.
#include "paged_common.cuh"
#include "sm100.cuh"

namespace seg {

using namespace sm100;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
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

// An item's 16 elements -> the finished query, key or value elements.  u1, u2: the first block's values (or nullptr).
template <int HD>
__device__ __forceinline__ void finish(const PagedAppendParams& p, int slot, const float* cs, const float* sn, const void* u1, const void* u2, float c,
                                       float a1, float a2, float qg, float* x1, float* x2) {
  if (slot < p.H + p.Hkv) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float r1 = x1[j] * cs[j] - x2[j] * sn[j], r2 = x1[j] * sn[j] + x2[j] * cs[j];
      x1[j] = r1;
      x2[j] = r2;
      ss += r1 * r1 + r2 * r2;
    }
    if (p.qknorm) {
      ss = head_sum<HD / 16>(ss);
      const float mul = rsqrtf(ss / HD + kQkEps) * (slot < p.H ? qg : 1.f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x1[j] *= mul;
        x2[j] *= mul;
      }
    }
  } else {
    float w1[8], w2[8];
    if (u1 != nullptr) {
      unpack8(load16(u1), w1);
      unpack8(load16(u2), w2);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x1[j] = c * (a1 * x1[j] + a2 * (u1 != nullptr ? w1[j] : x1[j]));
      x2[j] = c * (a1 * x2[j] + a2 * (u1 != nullptr ? w2[j] : x2[j]));
    }
  }
}

// Stores an item where it belongs; tokens without a place give zeros and leave the cache alone.
template <int HD>
__device__ __forceinline__ void store_item(const PagedAppendParams& p, int64_t t, const TokenPlace& w, int slot, int sub, const float* x1, const float* x2) {
  constexpr int HALF = HD / 2;
  const bf16x8 y1 = pack8(x1), y2 = pack8(x2);
  if (slot < p.H) {
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.q) + (t * p.H + slot) * HD + sub * 8;
    store16(dst, y1);
    store16(dst + HALF, y2);
    return;
  }
  const bool is_k = slot < p.H + p.Hkv;
  const int h = slot - (is_k ? p.H : p.H + p.Hkv);
  if (w.page >= 0) {
    __nv_bfloat16* dst = is_k ? static_cast<__nv_bfloat16*>(p.pool.k) + w.page * p.pool.k_page + w.slot * p.pool.k_slot + h * p.pool.k_head
                              : static_cast<__nv_bfloat16*>(p.pool.v) + w.page * p.pool.v_page + w.slot * p.pool.v_slot + h * p.pool.v_head;
    store16(dst + sub * 8, y1);
    store16(dst + HALF + sub * 8, y2);
  }
  void* out = is_k ? p.k_out : p.v_out;
  if (out != nullptr) {
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(out) + (t * p.Hkv + h) * HD + sub * 8;
    store16(dst, y1);
    store16(dst + HALF, y2);
  }
}

// ---------------------------------------------------------------------------------------------- a CTA per token
template <int HD>
__global__ void __launch_bounds__(kThreads) paged_append_few_kernel(const PagedAppendParams p) {
  constexpr int HALF = HD / 2, LPH = HD / 16;
  __shared__ TokenPlace place;
  const int64_t t = blockIdx.x;
  const int nslots = p.H + 2 * p.Hkv, nrot = p.H + p.Hkv, n_items = nslots * LPH;
  const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(p.qkv) + t * p.qkv_stride;
  for (int base = 0; base < n_items; base += kThreads) {
    const int item = base + threadIdx.x, sub = item % LPH, slot = item / LPH;
    const bool live = item < n_items;
    bf16x8 x[2], u[2];
    if (live) {  // on their way before anything is known about where the token goes
      x[0] = load16(row + slot * HD + sub * 8);
      x[1] = load16(row + slot * HD + HALF + sub * 8);
      if (slot >= nrot && p.v1 != nullptr) {
        const __nv_bfloat16* v1 = static_cast<const __nv_bfloat16*>(p.v1) + (t * p.Hkv + (slot - nrot)) * HD + sub * 8;
        u[0] = load16(v1);
        u[1] = load16(v1 + HALF);
      }
    }
    const float a1 = *p.alpha1, a2 = *p.alpha2, qg = *p.qgain, c = *p.vscale * rsqrtf(a1 * a1 + a2 * a2 + kMixEps);
    if (base == 0) {
      if (threadIdx.x == 0) place = find_place(p, (int)t);
      __syncthreads();
    }
    if (!live) continue;  // the LPH lanes of a head leave together: n_items is a multiple of LPH
    const TokenPlace w = place;
    float x1[8] = {}, x2[8] = {};
    if (w.page >= 0) {
      unpack8(x[0], x1);
      unpack8(x[1], x2);
      const int64_t rot = (int64_t)w.pos * HALF + sub * 8;
      float cs[8], sn[8];
      load8<float>(p.cos + rot, cs);
      load8<float>(p.sin + rot, sn);
      finish<HD>(p, slot, cs, sn, p.v1 != nullptr ? &u[0] : nullptr, &u[1], c, a1, a2, qg, x1, x2);
    }
    store_item<HD>(p, t, w, slot, sub, x1, x2);
  }
}

// ---------------------------------------------------------------------------------------------- a ring of token groups
constexpr int kRing = 4;              // stages at most
constexpr int kMaxTokens = 16;        // tokens of a group at most
constexpr int kSmemCta = 110 * 1024;  // two CTAs share an SM

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// A stage: for each token its projection row, its v1 row, its cos and sin rows (token_bytes in all).  tokens: 1, 2, 4, 8 or 16;
// eight warps share them, each walks over the heads of one token (or of a part of it) with the rotation in registers.
template <int HD>
__global__ void __launch_bounds__(kThreads + 32) paged_append_ring_kernel(const PagedAppendParams p, int tokens, int ring, int token_bytes) {
  constexpr int HALF = HD / 2, LPH = HD / 16, kHeads = 32 / LPH;  // heads that a warp covers at once
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ TokenPlace place[kRing][kMaxTokens];
  __shared__ uint64_t full[kRing], empty[kRing];
  __shared__ int abort_flag;
  const int nslots = p.H + 2 * p.Hkv, nrot = p.H + p.Hkv;
  const int row_bytes = nslots * HD * 2, v1_bytes = p.v1 != nullptr ? p.Hkv * HD * 2 : 0;
  const int n_groups = (p.T + tokens - 1) / tokens, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AbortState ab{&abort_flag, p.status};
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < ring; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), kWarps);
    }
    fence_barrier_init();
  }
  __syncthreads();
  if (warp == kWarps) {
    // a lane per token: finds its place and fetches its rows
    int st = 0, ph = 0;
    for (int g = blockIdx.x; g < n_groups; g += gridDim.x) {
      const int t = g * tokens + lane;
      const bool live = lane < tokens && t < p.T;
      TokenPlace w{-1, 0, 0};
      if (live) w = find_place(p, t);
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&empty[st]), ph ^ 1, ab, 81))) break;
      if (live) place[st][lane] = w;
      const int n = __popc(__ballot_sync(0xffffffffu, live && w.page >= 0));
      __syncwarp();  // the places of all lanes are written before lane 0 arrives
      const uint32_t bar = smem_u32(&full[st]);
      if (lane == 0) mbar_expect_tx(bar, n * (row_bytes + v1_bytes + HD * 4));
      __syncwarp();
      if (live && w.page >= 0) {
        const uint32_t dst = smem_u32(smem) + (st * tokens + lane) * token_bytes;
        bulk_load(dst, static_cast<const __nv_bfloat16*>(p.qkv) + (int64_t)t * p.qkv_stride, row_bytes, bar);
        if (v1_bytes != 0) bulk_load(dst + row_bytes, static_cast<const __nv_bfloat16*>(p.v1) + (int64_t)t * p.Hkv * HD, v1_bytes, bar);
        bulk_load(dst + row_bytes + v1_bytes, p.cos + (int64_t)w.pos * HALF, HD * 2, bar);
        bulk_load(dst + row_bytes + v1_bytes + HD * 2, p.sin + (int64_t)w.pos * HALF, HD * 2, bar);
      }
      if (++st == ring) st = 0, ph ^= 1;
    }
  } else {
    const float a1 = *p.alpha1, a2 = *p.alpha2, qg = *p.qgain, c = *p.vscale * rsqrtf(a1 * a1 + a2 * a2 + kMixEps);
    const int sub = lane % LPH, head = lane / LPH;
    const int share = tokens < kWarps ? kWarps / tokens : 1;  // warps per token
    int st = 0, ph = 0;
    for (int g = blockIdx.x; g < n_groups; g += gridDim.x) {
      const int t0 = g * tokens;
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&full[st]), ph, ab, 82))) break;
      for (int tok = warp / share; tok < tokens && t0 + tok < p.T; tok += kWarps / share) {
        const TokenPlace w = place[st][tok];
        const uint8_t* src = smem + (st * tokens + tok) * token_bytes;
        const float* rot = reinterpret_cast<const float*>(src + row_bytes + v1_bytes) + sub * 8;
        float cs[8], sn[8];
        if (w.page >= 0) {
          load8<float>(rot, cs);
          load8<float>(rot + HALF, sn);
        }
#pragma unroll 2
        for (int slot = warp % share * kHeads + head; slot < nslots; slot += share * kHeads) {  // the LPH lanes of a head stay together
          float x1[8] = {}, x2[8] = {};
          if (w.page >= 0) {
            unpack8(load16(src + (slot * HD + sub * 8) * 2), x1);
            unpack8(load16(src + (slot * HD + HALF + sub * 8) * 2), x2);
            const uint8_t* u = src + row_bytes + ((slot - nrot) * HD + sub * 8) * 2;
            finish<HD>(p, slot, cs, sn, v1_bytes != 0 ? u : nullptr, u + HD, c, a1, a2, qg, x1, x2);
          }
          store_item<HD>(p, t0 + tok, w, slot, sub, x1, x2);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&empty[st]));
      if (++st == ring) st = 0, ph ^= 1;
    }
  }
  if (*static_cast<volatile int*>(&abort_flag) != 0) {
    for (int i = 0; i < 2000; ++i) __nanosleep(100);  // copies in flight land before the CTA's memory is given away
  }
}

template <int HD>
int launch(const PagedAppendParams& p, cudaStream_t st) {
  const int nslots = p.H + 2 * p.Hkv, per_token = nslots * (HD / 16);
  const int token_bytes = nslots * HD * 2 + (p.v1 != nullptr ? p.Hkv * HD * 2 : 0) + HD * 4;
  int tokens = kMaxTokens;
  while (tokens > 0 && 2 * tokens * token_bytes > kSmemCta) tokens /= 2;
  // Up to four CTAs' items per SM.  A CTA per token against the ring, us: 18 + 12 heads of 64 3.2 / 6.1 for 256 tokens, 5.6 / 6.4 for
  // 1024, 9.1 / 7.5 for 2048, 140.9 / 59.5 for 32768; 32 + 16 heads of 128 5.6 / 5.9 for 256, 6.3 / 6.5 for 512, 9.9 / 9.1 for 1024.
  if ((int64_t)p.T * per_token <= 148 * 4 * kThreads || tokens == 0) {
    paged_append_few_kernel<HD><<<p.T, kThreads, 0, st>>>(p);
  } else {
    int ring = kSmemCta / (tokens * token_bytes);
    if (ring > kRing) ring = kRing;
    static bool configured[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -2;
    if (!configured[dev]) {
      if (cudaFuncSetAttribute(paged_append_ring_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemCta) != cudaSuccess) return -2;
      configured[dev] = true;
    }
    const int groups = (p.T + tokens - 1) / tokens;
    paged_append_ring_kernel<HD><<<groups < 148 * 2 ? groups : 148 * 2, kThreads + 32, ring * tokens * token_bytes, st>>>(p, tokens, ring, token_bytes);
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
