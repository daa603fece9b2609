// What the paged kernels share: 16-byte accesses; of the attention the plan of a call, the checked reads of lengths and group borders, and the
// dealing of key tiles to CTAs.
#pragma once
#include <cuda.h>

#include "common.cuh"
#include "paged.h"

namespace seg {

// Eight bf16 in one 16-byte access.  (The compiler splits the copy of a structure of bf16 pairs into 4-byte accesses.)
__device__ __forceinline__ bf16x8 load16(const void* p) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  bf16x8 r;
  r.v[0] = *reinterpret_cast<const __nv_bfloat162*>(&v.x);
  r.v[1] = *reinterpret_cast<const __nv_bfloat162*>(&v.y);
  r.v[2] = *reinterpret_cast<const __nv_bfloat162*>(&v.z);
  r.v[3] = *reinterpret_cast<const __nv_bfloat162*>(&v.w);
  return r;
}
__device__ __forceinline__ void store16(void* p, const bf16x8& r) {
  uint4 v;
  v.x = *reinterpret_cast<const uint32_t*>(&r.v[0]);
  v.y = *reinterpret_cast<const uint32_t*>(&r.v[1]);
  v.z = *reinterpret_cast<const uint32_t*>(&r.v[2]);
  v.w = *reinterpret_cast<const uint32_t*>(&r.v[3]);
  *reinterpret_cast<uint4*>(p) = v;
}

// Which kernel walks over the prefixes: 16 rows at a time next to the sequences' own pages (paged_attn.cu), or one of the two
// tcgen05 forms (paged_prefix.cu): 256 rows of one group per CTA, or 128 rows with the keys dealt to the two halves of a CTA.
enum PrefixForm { kPrefixSmall = 0, kPrefixRows = 1, kPrefixKeys = 2 };

struct Plan {            // sizes that host and device derive alike
  int gqa, RT;           // query heads per kv head; 16-row tiles of a sequence's item row
  int rows_s, items_s;   // rows of a part of an own-pages item; number of such items
  int rows_q;            // query rows that a warp keeps of an item: 8, or 16 where some item has more
  int form;              // PrefixForm
  int rows_p, items_p;   // rows of a prefix item; upper bound on their number
  int parts_p, part_rows_p;  // parts that a CTA leaves of a prefix item, rows of each
  int ctas, workers;     // of the kernel over own pages (and prefixes in the small form); its warps
  int ctas_p;            // workers of the kernel over prefixes: warps, or CTAs in the tcgen05 forms
};

// Every (item, worker) pair with work gets the part number item + worker: both only grow along the row of tiles, so the numbers are
// distinct, and consecutive for the parts of one item.  The small form's prefix items have 1 to 16 rows; there the part of worker w
// starts at row `rows of the items before + 16 w`, distinct for the same reason, so that many small groups take no more than their rows.
struct Work {
  float* acc_s;    // [items_s + workers, rows_s, HD]
  float2* ml_s;    // [items_s + workers, rows_s]
  float* acc_p;    // [(items_p + ctas_p) * parts_p, part_rows_p, HD]; small form: [B H + 16 workers, HD]
  float2* ml_p;
  int2* meta;      // [items_s + items_p + 1] first part (small form's prefix items: first worker) and number of parts of every item that
                   // has tiles; x of the last: group_rows are out of order (written where there are any)
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
  bool bad;  // borders out of order
};
__device__ __forceinline__ Group load_group(const PagedAttnParams& p, int g) {
  Group w;
  w.r0 = p.groups != nullptr ? p.groups[g] : 0;
  w.r1 = p.groups != nullptr ? p.groups[g + 1] : p.B;
  w.bad = w.r0 < 0 || w.r1 < w.r0 || w.r1 > p.B;
  if (w.bad) {
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

// sum[i + 1] = tiles of the first i + 1 lists; all kThreads threads take part, warp_tot has a word per warp.  A thread adds up
// neighbouring lists, whose loads do not wait for one another.
template <int kThreads, typename F>
__device__ void scan_tiles(int* sum, int n, F tiles, int* warp_tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (n + kThreads - 1) / kThreads, first = min((int)threadIdx.x * per, n), last = min(first + per, n);
  int mine = 0;
#pragma unroll 4
  for (int i = first; i < last; ++i) {
    const int v = tiles(i);
    sum[i + 1] = v;
    mine += v;
  }
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (lane == 31) warp_tot[warp] = upto;
  if (threadIdx.x == 0) sum[0] = 0;
  __syncthreads();
  int at = upto - mine;
  for (int w = 0; w < warp; ++w) at += warp_tot[w];
  for (int i = first; i < last; ++i) {
    at += sum[i + 1];
    sum[i + 1] = at;
  }
  __syncthreads();
}
// sum of the groups' tiles (`tiles` of a group's length, for each of its row tiles); false: borders out of order somewhere, and no
// prefix counts - groups that overlap could hold more rows than the call, beyond every bound that the host has checked.
template <int kThreads, typename F>
__device__ bool scan_groups(int* sum, const PagedAttnParams& p, const Plan& n, const Work& ws, F tiles, int* warp_tot) {
  bool bad = false;
  scan_tiles<kThreads>(sum, p.G, [&](int g) {
    const Group w = load_group(p, g);
    bad |= w.bad;
    return tiles(w.len) * row_tiles(w, n);
  }, warp_tot);
  if (p.groups == nullptr) return true;
  bad = __syncthreads_or(bad) != 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) ws.meta[n.items_s + n.items_p] = make_int2(bad, 0);
  return !bad;
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

// The parts of item [first tile, first tile + n_tiles) of `total` tiles dealt to `ctas` workers: first number, and how many.
__device__ __forceinline__ int2 item_parts(int item, int64_t first_tile, int n_tiles, int64_t ctas, int64_t total) {
  const int a = (int)(((first_tile + 1) * ctas - 1) / total), b = (int)(((first_tile + n_tiles) * ctas - 1) / total);
  return make_int2(item + a, b - a + 1);
}

constexpr int kMaxLists = 8192;  // sequences + groups of a call (their cumulative tile counts live in shared memory)

// ---- reading a pool with TMA
// Tokens of a box: the largest power of two that divides the page (so that a box never leaves its page), at most `most`.
inline int pool_box(int P, int most) {
  const int box = P & -P;
  return box < most ? box : most;
}
// 5-D bf16 map over a pool [pages, P, Hkv, hd] with any strides: (up to 64 dims, token, block of 64 dims, head, page).  A box is `box`
// tokens with all their dims, swizzled over rows of 128 (hd 32: 64) bytes; at head_dim 128 the blocks of 64 dims follow each other
// in shared memory for 8 tokens at a time (box 8), so that a box of few tokens still is one copy: 2 KB, and half as many of
// them.  96 sequences on 7 prefixes of 4001 tokens in pages of 24, 8 heads of 128: 55 us with a copy per block, 47 us in pages of 64.
// A box of page n_pages lies outside and reads as zeros.
inline int make_pool_map(CUtensorMap* map, void* base, const PagedAttnParams& p, int64_t page, int64_t slot, int64_t head, int box) {
  typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static EncodeFn fn = nullptr;
  if (fn == nullptr) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &res) != cudaSuccess || res != cudaDriverEntryPointSuccess) return -1;
    fn = reinterpret_cast<EncodeFn>(ptr);
  }
  // a dimension of one element may have any stride in the framework; the map wants a multiple of 16 bytes
  const cuuint32_t row = (cuuint32_t)(p.hd < 64 ? p.hd : 64), blocks = (cuuint32_t)(p.hd / row);
  const cuuint64_t dims[5] = {row, (cuuint64_t)p.pool.P, blocks, (cuuint64_t)p.Hkv, (cuuint64_t)p.pool.n_pages};
  const cuuint64_t strides[4] = {(cuuint64_t)(p.pool.P == 1 ? p.hd : slot) * 2, row * 2, (cuuint64_t)(p.Hkv == 1 ? p.hd : head) * 2,
                                 (cuuint64_t)(p.pool.n_pages == 1 ? p.hd : page) * 2};
  const cuuint32_t boxes[5] = {row, (cuuint32_t)box, blocks, 1, 1}, ones[5] = {1, 1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, base, dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            p.hd < 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -1;
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int slot, int head, int page) {
  asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %3, %5, %6}], [%2];" ::"r"(dst), "l"(map),
               "r"(bar), "r"(0), "r"(slot), "r"(head), "r"(page)
               : "memory");
}

// ---- paged_prefix.cu: whether the pool can be read in the tcgen05 forms, and their launch
bool paged_prefix_usable(const PagedAttnParams& p);
int paged_prefix(const PagedAttnParams& p, const Plan& n, const Work& ws, cudaStream_t st);

}  // namespace seg
