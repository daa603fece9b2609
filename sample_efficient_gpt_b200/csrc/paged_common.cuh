// What the kernels of the paged attention share: the plan of a call, the checked reads of lengths and group borders, and the
// dealing of key tiles to CTAs.
#pragma once
#include "common.cuh"
#include "paged.h"

namespace seg {

// Which kernel walks over the prefixes: 16 rows at a time next to the sequences' own pages (paged_attn.cu), or one of the two
// tcgen05 forms (paged_prefix.cu): 256 rows of one group per CTA, or 128 rows with the keys dealt to the two halves of a CTA.
enum PrefixForm { kPrefixSmall = 0, kPrefixRows = 1, kPrefixKeys = 2 };

struct Plan {            // sizes that host and device derive alike
  int gqa, RT;           // query heads per kv head; 16-row tiles of a sequence's item row
  int rows_s, items_s;   // rows of a part of an own-pages item; number of such items
  int form;              // PrefixForm
  int rows_p, items_p;   // rows of a prefix item; upper bound on their number
  int parts_p, part_rows_p;  // parts that a CTA leaves of a prefix item, rows of each
  int ctas;              // of the kernel over own pages (and prefixes in the small form)
  int ctas_p;            // of the kernel over prefixes
};

// Every (item, CTA) pair with work gets the part number item + CTA: both only grow along the row of tiles, so the numbers are
// distinct, and consecutive for the parts of one item.
struct Work {
  float* acc_s;    // [items_s + ctas, rows_s, HD]
  float2* ml_s;    // [items_s + ctas, rows_s]
  float* acc_p;    // [(items_p + ctas_p) * parts_p, part_rows_p, HD]
  float2* ml_p;
  int2* meta;      // [items_s + items_p] first part and number of parts of every item that has tiles
};

__device__ __forceinline__ float exp2_(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ int clamp_len(int n, int width, int P, int* status) {
  const int64_t cap = (int64_t)width * P;
  if (n >= 0 && n <= cap) return n;
  atomicCAS(status, 0, kStatusAttnLength);
  return n < 0 ? 0 : (int)cap;
}
struct Group {
  int r0, r1, len;
};
__device__ __forceinline__ Group load_group(const PagedAttnParams& p, int g) {
  Group w;
  w.r0 = p.groups != nullptr ? p.groups[g] : 0;
  w.r1 = p.groups != nullptr ? p.groups[g + 1] : p.B;
  if (w.r0 < 0 || w.r1 < w.r0 || w.r1 > p.B) {
    atomicCAS(p.status, 0, kStatusAttnGroups);
    w.r0 = w.r1 = 0;
  }
  w.len = w.r1 > w.r0 ? clamp_len(p.plens[g], p.ptable_width, p.pool.P, p.status) : 0;
  return w;
}
__device__ __forceinline__ int row_tiles(const Group& g, const Plan& n) { return ((g.r1 - g.r0) * n.gqa + n.rows_p - 1) / n.rows_p; }
// First item of a group's prefix: leaves room for the row tiles of the groups before it, whatever their sizes.
__device__ __forceinline__ int first_item(const Plan& n, const PagedAttnParams& p, int g, int r0) {
  return n.items_s + p.Hkv * (r0 * n.gqa / n.rows_p + g);
}

// sum[i + 1] = tiles of the first i + 1 lists; all kThreads threads take part, warp_tot has a word per warp
template <int kThreads, typename F>
__device__ void scan_tiles(int* sum, int n, F tiles, int* warp_tot) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int carry = 0;
  if (threadIdx.x == 0) sum[0] = 0;
  for (int base = 0; base < n; base += kThreads) {
    const int i = base + threadIdx.x;
    int v = i < n ? tiles(i) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) warp_tot[warp] = v;
    __syncthreads();
    int add = carry;
    for (int w = 0; w < warp; ++w) add += warp_tot[w];
    if (i < n) sum[i + 1] = v + add;
    for (int w = 0; w < kWarps; ++w) carry += warp_tot[w];
    __syncthreads();
  }
}
// last i with sum[i] <= t (t < sum[n]); empty lists are passed over
__device__ __forceinline__ int find_list(const int* sum, int n, int t) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sum[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

// The part of item [first tile, first tile + n_tiles) of `total` tiles dealt to `ctas` CTAs: first part number and number of parts.
__device__ __forceinline__ int2 item_parts(int item, int64_t first_tile, int n_tiles, int64_t ctas, int64_t total) {
  const int a = (int)(((first_tile + 1) * ctas - 1) / total), b = (int)(((first_tile + n_tiles) * ctas - 1) / total);
  return make_int2(item + a, b - a + 1);
}

constexpr int kMaxLists = 8192;  // sequences + groups of a call (their cumulative tile counts live in shared memory)

// ---- paged_prefix.cu: whether the pool can be read in the tcgen05 forms, and their launch
bool paged_prefix_usable(const PagedAttnParams& p);
int paged_prefix(const PagedAttnParams& p, const Plan& n, const Work& ws, cudaStream_t st);

}  // namespace seg
