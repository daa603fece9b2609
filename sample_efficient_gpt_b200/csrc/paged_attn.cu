// One-token attention over a paged key/value cache, with a prefix that the sequences of a group share.
//
//   s_n = scale * q . k_n over the tokens n of the row's group prefix and of its own pages;  m = max s, l = sum exp(s_n - m),
//   o = sum exp(s_n - m) v_n / l,  lse = m + log l;   a row that sees no token: o = 0, lse = -inf.
//
// Work items: (sequence, kv head, 16 of its query heads) over the sequence's own pages, and (group, kv head, 16 of the group's
// rows x query heads) over the group's prefix, which is therefore read once per 16 rows and not once per sequence (groups
// with many rows have a kernel of their own, paged_prefix.cu).  Items are cut into steps of 32 keys; the
// steps of all items in one row are dealt to the warps of one resident wave in equal, contiguous ranges, so that ragged lengths
// and single long sequences fill the machine alike.  A range that does not hold an item alone leaves (m, l, unnormalised o) in
// fp32, and a second kernel joins the parts of every row in a fixed order (no atomics: the result does not depend on timing).
//
// A warp works alone: its own ring of asynchronous copies (TMA boxes that never leave a page; 16-byte copies by all lanes where
// the page size is no multiple of 8) runs ahead over the borders of items, and no barrier is crossed after the plan.  Scores and
// the weighted sum are m16n8k16 tensor core products with the query heads as (padded) rows; the bound is the bytes of the cache, so what counts is few instructions a byte.  The
// exponentials are taken relative to a reference that is only moved when a score exceeds it by more than 2^8, which a vote
// finds without reducing the maximum over lanes; weights are then at most 256, harmless for bf16 operands and fp32 sums.
// Keys behind the length are masked by index and their values set to zero: what lies in those slots does not count.
// Measured: 64 sequences of up to 8192 tokens, 6 kv heads of 64: 403 MB in 73 us, join included (5.5 TB/s); one sequence of 700
// tokens 7.8 us, the latency of two launches and of length -> page -> keys -> parts.
#include <algorithm>

#include "paged_common.cuh"
#include "sm100.cuh"

namespace seg {

using namespace sm100;

namespace {

constexpr int kWarps = 2;               // small CTAs: one or two fit next to a CTA of the prefix kernel
constexpr int kJoinWarps = 4;
constexpr int kRows = 16;               // query rows per item
// What an item costs next to its steps (queries, first maximum, outputs), in steps.  64 ragged sequences of up to 8192 tokens:
// 79.6 us at 0, 73.2 at 1, 72.9 at 2; 1000 sequences of up to 64: 40.3, 37.0, 37.0.
constexpr int kItemCost = 1;
constexpr int kThreads = kWarps * 32;

template <int HD> struct Cfg {
  static constexpr int kKeys = 32;                         // keys per warp and step
  static constexpr int kStages = HD == 32 ? 4 : 2;
  static constexpr int kChunks = HD / 8;                   // 16-byte chunks of a row
  static constexpr int kMat = kKeys * HD * 2;              // K or V of one step
  static constexpr int kStageBytes = 2 * kMat;
  static constexpr int kRing = kStages * kStageBytes;      // per warp
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {  // d = a b
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Weight of a part (m, l) under the common maximum mm.  A part without a finite score has m = -inf and l = 0, unless NaN scores
// made l NaN: then the row becomes NaN, as the formula says.
__device__ __forceinline__ float part_weight(float m, float l, float mm) { return m == -INFINITY ? l : exp2_(m - mm); }
__device__ __forceinline__ float row_lse(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f; }
// Byte offset of 16-byte chunk c of row r in a step's K or V: eight rows at a time, of them blocks of 64 dims (hd 32: 32), chunks of
// neighbouring rows permuted (the pattern that TMA writes) so that the eight rows of an ldmatrix phase fall on different banks.
template <int HD> __device__ __forceinline__ uint32_t swz(int r, int c) {
  if (HD == 32) return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  return (r >> 3) * (HD * 16) + (c >> 3) * 1024 + (r & 7) * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// Addresses of one walk's keys: a list of pages and the kv head inside them.
struct KeyWalk {
  const int* pages;
  const __nv_bfloat16 *k, *v;  // pools at the item's kv head
  int kvh, len;
};

__device__ __forceinline__ int64_t checked_page(const PagedAttnParams& p, const int* pages, int j) {
  const int page = __ldg(pages + j);
  if ((unsigned)page < (unsigned)p.pool.n_pages) return page;
  atomicCAS(p.status, 0, kStatusAttnPage);
  return -1;
}

// An item, and the unit of it that a cursor stands at: kItemCost units for the item itself, then one per step.
struct Cursor {
  bool own;
  int list, i, items;        // sequence or group; item of it; number of its items
  int item;                  // number of the item
  int kvh, h0, rows, row0;   // query rows r = 0 .. rows-1: sequence row0 + (h0 + r) / gqa, head kvh * gqa + (h0 + r) % gqa
  int unit, units;
  KeyWalk w;
};

struct Lists {  // cumulative units per item of the sequences, and units per kv head of the groups
  const int *sum_s, *sum_p;
  int n_groups;
};

// Rows of the prefix items before the one that starts at row h0 of a group's `all` rows of head kvh (small form).
__device__ __forceinline__ int64_t prefix_row(const PagedAttnParams& p, int r0, int all, int kvh, int h0) {
  return (int64_t)r0 * p.H + (int64_t)kvh * all + h0;
}

template <int HD>
__device__ __forceinline__ int units_of(int len) { return len > 0 ? (len + Cfg<HD>::kKeys - 1) / Cfg<HD>::kKeys + kItemCost : 0; }

template <int HD>
__device__ __forceinline__ void set_list(const PagedAttnParams& p, const Plan& n, Cursor& c) {
  if (c.own) {
    c.row0 = c.list;
    c.items = p.Hkv * n.RT;
    c.item = c.list * c.items;
    c.w.len = clamp_len(p.lens[c.list], p.table_width, p.pool.P, p.status);
    c.w.pages = p.table + c.list * p.table_stride;
  } else {
    const Group g = load_group(p, c.list);
    c.row0 = g.r0;
    c.items = p.Hkv * row_tiles(g, n);
    c.item = first_item(n, p, c.list, g.r0);
    c.w.len = g.len;
    c.w.pages = p.ptable + c.list * p.ptable_stride;
    c.rows = (g.r1 - g.r0) * n.gqa;
  }
  c.units = units_of<HD>(c.w.len);
}
// Item i of the cursor's list; `all`: the rows of the list (a sequence's heads of a kv head, a group's rows).
__device__ __forceinline__ void set_item(const PagedAttnParams& p, const Plan& n, Cursor& c, int i, int all) {
  const int tiles = (all + kRows - 1) / kRows;
  c.item += i - c.i;
  c.i = i;
  c.kvh = i / tiles;
  c.h0 = (i - c.kvh * tiles) * kRows;
  c.rows = min(kRows, all - c.h0);
  c.w.kvh = c.kvh;
  c.w.k = static_cast<const __nv_bfloat16*>(p.pool.k) + c.kvh * p.pool.k_head;
  c.w.v = static_cast<const __nv_bfloat16*>(p.pool.v) + c.kvh * p.pool.v_head;
}

// The item of unit t, and the unit's place in it.
template <int HD>
__device__ __forceinline__ Cursor cursor_at(const PagedAttnParams& p, const Plan& n, const Lists& L, int64_t units_s, int64_t t, int& all) {
  Cursor c;
  c.own = t < units_s;
  const int per = c.own ? p.Hkv * n.RT : p.Hkv;
  const int64_t u = c.own ? t : t - units_s;
  const int* sum = c.own ? L.sum_s : L.sum_p;
  c.list = find_list(sum, c.own ? p.B : L.n_groups, (int)(u / per));
  set_list<HD>(p, n, c);
  all = c.own ? n.gqa : c.rows;
  const int local = (int)(u - (int64_t)sum[c.list] * per), i = local / c.units;
  c.unit = local - i * c.units;
  c.i = 0;
  set_item(p, n, c, i, all);
  return c;
}

// To the next item; there is one.
template <int HD>
__device__ __forceinline__ void next_item(const PagedAttnParams& p, const Plan& n, const Lists& L, Cursor& c, int& all) {
  c.unit = 0;
  int i = c.i + 1;
  if (i == c.items) {
    const int* sum = c.own ? L.sum_s : L.sum_p;
    const int last = c.own ? p.B : L.n_groups;
    do ++c.list;
    while (c.list < last && sum[c.list + 1] == sum[c.list]);
    if (c.list == last) {  // from the sequences to the groups
      c.own = false;
      c.list = 0;
      while (L.sum_p[c.list + 1] == L.sum_p[c.list]) ++c.list;
    }
    set_list<HD>(p, n, c);
    all = c.own ? n.gqa : c.rows;
    i = c.i = 0;
  }
  set_item(p, n, c, i, all);
}

// Where a warp's ring lies, and the queries beside it.
struct Ring {
  uint32_t base;  // shared memory of the stages
  uint32_t full;  // mbarriers of the stages (TMA)
  uint32_t q;     // query rows of the items that the loads have begun: kStages buffers of q_rows rows
  int q_rows;
};
constexpr int kQPad = 16;  // bytes behind a query row, so that the rows of an ldmatrix phase fall on different banks

// Brings the query rows of cursor c into buffer `at` (cp.async; the caller commits).
template <int HD>
__device__ __forceinline__ void load_queries(const PagedAttnParams& p, const Plan& n, const Cursor& c, const Ring& ring, int at) {
  constexpr int kChunks = Cfg<HD>::kChunks;
  const uint32_t dst = ring.q + at % Cfg<HD>::kStages * ring.q_rows * (HD * 2 + kQPad);
  for (int i = threadIdx.x & 31; i < ring.q_rows * kChunks; i += 32) {
    const int r = i / kChunks, ch = i % kChunks, x = c.h0 + r;
    const bool live = r < c.rows;
    const int q = live ? x / n.gqa : 0, h = live ? x - q * n.gqa : 0;
    copy16(dst + r * (HD * 2 + kQPad) + ch * 16, static_cast<const __nv_bfloat16*>(p.q) + (int64_t)(c.row0 + q) * p.q_row + (c.kvh * n.gqa + h) * p.q_head + ch * 8, live);
  }
}

template <int HD, bool kTma>
__device__ __forceinline__ void load_step(const PagedAttnParams& p, const CUtensorMap* map_k, const CUtensorMap* map_v, int box, const KeyWalk& w, int key0,
                                          const Ring& ring, int it) {
  using C = Cfg<HD>;
  const int lane = threadIdx.x & 31;
  const int st = it % C::kStages;
  const uint32_t stage = ring.base + st * C::kStageBytes;
  if constexpr (kTma) {
    // a lane per box: K or V, tokens
    const uint32_t bar = ring.full + st * 8;
    if (lane == 0) mbar_expect_tx(bar, C::kStageBytes);
    __syncwarp();
    if (lane < 2 * (C::kKeys / box)) {
      const int kv = lane & 1, b = lane >> 1, key = key0 + b * box;
      int page = p.pool.n_pages, slot = 0;  // outside the pool: zeros
      if (key < w.len) {
        const int j = p.pool.shift >= 0 ? key >> p.pool.shift : key / p.pool.P;
        const int64_t found = checked_page(p, w.pages, j);
        if (found >= 0) {
          page = (int)found;
          slot = key - j * p.pool.P;
        }
      }
      load_box(stage + kv * C::kMat + b * box * HD * 2, kv ? map_v : map_k, bar, slot, w.kvh, page);
    }
  } else {
    constexpr int kRowsPer = 32 / C::kChunks;  // rows that the warp covers at once
#pragma unroll
    for (int i = 0; i < C::kKeys / kRowsPer; ++i) {
      const int r = i * kRowsPer + lane / C::kChunks, c = lane % C::kChunks, key = key0 + r;
      int64_t page = -1;
      int slot = 0;
      if (key < w.len) {
        const int j = key / p.pool.P;
        page = checked_page(p, w.pages, j);
        slot = key - j * p.pool.P;
      }
      const bool live = page >= 0;
      if (!live) page = slot = 0;
      copy16(stage + swz<HD>(r, c), w.k + page * p.pool.k_page + slot * p.pool.k_slot + c * 8, live);
      copy16(stage + C::kMat + swz<HD>(r, c), w.v + page * p.pool.v_page + slot * p.pool.v_slot + c * 8, live);
    }
  }
}

// One step: the keys [key0, key0 + left) of a list in stage st.  kHalf: at most eight of the item's sixteen rows exist; the
// products' upper rows are zero and their softmax is left out.
template <int HD, bool kTma, bool kHalf>
__device__ __forceinline__ void attend(const PagedAttnParams& p, int left, const uint32_t (*qf)[4], const Ring& ring, int st, float (*o)[4], float* m, float* l) {
  using C = Cfg<HD>;
  constexpr int kN = C::kKeys / 8;      // 8-key columns of the score tile
  constexpr int kE = kHalf ? 2 : 4;     // scores of a lane per column tile that count
  const int lane = threadIdx.x & 31;
  {
    const uint32_t sk = ring.base + st * C::kStageBytes, sv = sk + C::kMat;
    float sc[kN][4];
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) {
#pragma unroll
      for (int n = 0; n < kN; n += 2) {
        uint32_t b[4];
        ldsm4(b, sk + swz<HD>(n * 8 + (lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)));
        if (kk == 0) {
          mma_first(sc[n], qf[kk], b[0], b[1]);
          mma_first(sc[n + 1], qf[kk], b[2], b[3]);
        } else {
          mma(sc[n], qf[kk], b[0], b[1]);
          mma(sc[n + 1], qf[kk], b[2], b[3]);
        }
      }
    }
    // relative to the reference; scaled before the mask and the maximum, for the scale may be zero or negative
    const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < kE; ++e) sc[n][e] = fmaf(sc[n][e], p.scale_log2, -ref[e >> 1]);
    if (left < C::kKeys) {
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int e = 0; e < kE; ++e)
          if (n * 8 + (lane & 3) * 2 + (e & 1) >= left) sc[n][e] = -INFINITY;
      if (kTma) {  // a box may bring slots behind the length: their values must not meet the weights of zero
        for (int i = left * C::kChunks + lane; i < C::kKeys * C::kChunks; i += 32)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sv + swz<HD>(i / C::kChunks, i % C::kChunks)), "r"(0) : "memory");
        fence_proxy_async();
        __syncwarp();
      }
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < kE; e += 2) mx[e >> 1] = max3(mx[e >> 1], sc[n][e], sc[n][e + 1]);
    bool low = mx[0] > 8.f || (m[0] == -INFINITY && mx[0] > -INFINITY);
    if (!kHalf) low = low || mx[1] > 8.f || (m[1] == -INFINITY && mx[1] > -INFINITY);
    if (__any_sync(0xffffffffu, low)) {  // move the references to the maxima (always in an item's first step, rarely after it)
#pragma unroll
      for (int h = 0; h < (kHalf ? 1 : 2); ++h) {
        float t = mx[h];
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
        const float m_new = fmaxf(m[h], ref[h] + t);
        if (m_new == -INFINITY) continue;
        const float a = m[h] == -INFINITY ? 1.f : exp2_(m[h] - m_new);
        l[h] *= a;
#pragma unroll
        for (int d = 0; d < HD / 8; ++d) {
          o[d][2 * h] *= a;
          o[d][2 * h + 1] *= a;
        }
        // In this order no score ends above zero.  (One above 1e8 may have come here by its own rounding, 2^-24 of it, with the reference
        // left where it was.)
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          sc[n][2 * h] = __fadd_rn(__fadd_rn(sc[n][2 * h], ref[h]), -m_new);
          sc[n][2 * h + 1] = __fadd_rn(__fadd_rn(sc[n][2 * h + 1], ref[h]), -m_new);
        }
        m[h] = m_new;
      }
    }
    uint32_t pf[kN / 2][4];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (kHalf && h == 1) {
          pf[n / 2][(n & 1) * 2 + 1] = 0u;
          continue;
        }
        const float e0 = exp2_(sc[n][2 * h]), e1 = exp2_(sc[n][2 * h + 1]);
        l[h] += e0 + e1;
        pf[n / 2][(n & 1) * 2 + h] = pack_bf16(e0, e1);  // weights rounded to bf16 (at most 2^-8 relative), as operands of the tensor core
      }
    }
#pragma unroll
    for (int kk = 0; kk < kN / 2; ++kk) {
#pragma unroll
      for (int dd = 0; dd < HD / 16; ++dd) {
        uint32_t b[4];
        ldsm4t(b, sv + swz<HD>(kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, dd * 2 + (lane >> 4)));
        mma(o[2 * dd], pf[kk], b[0], b[1]);
        mma(o[2 * dd + 1], pf[kk], b[2], b[3]);
      }
    }
  }
}

// hd 64: at most 128 registers, so that CTAs fit next to one of the prefix kernel's
template <int HD, bool kTma>
__global__ void __launch_bounds__(kThreads, HD == 128 ? 4 : 8)
paged_attn_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PagedAttnParams p, const Plan n, const Work ws,
                  const int box) {
  using C = Cfg<HD>;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int warp_tot[kWarps];
  __shared__ uint64_t full[kWarps][C::kStages];
  __shared__ int abort_flag;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AbortState ab{&abort_flag, p.status};
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kWarps * C::kStages; ++i) mbar_init(smem_u32(&full[0][0] + i), 1);
    fence_barrier_init();
  }
  const int q_bytes = C::kStages * n.rows_q * (HD * 2 + kQPad);  // per warp
  const Ring ring{smem_u32(smem + warp * C::kRing), smem_u32(full[warp]), smem_u32(smem + kWarps * C::kRing + warp * q_bytes), n.rows_q};
  int* sum_s = reinterpret_cast<int*>(smem + kWarps * (C::kRing + q_bytes));
  int* sum_p = sum_s + p.B + 1;
  scan_tiles<kThreads>(sum_s, p.B, [&](int b) { return units_of<HD>(clamp_len(p.lens[b], p.table_width, p.pool.P, p.status)); }, warp_tot);
  Lists L{sum_s, sum_p, n.form == kPrefixSmall ? p.G : 0};
  if (L.n_groups > 0 && !scan_groups<kThreads>(sum_p, p, n, ws, [](int len) { return units_of<HD>(len); }, warp_tot)) L.n_groups = 0;
  const int64_t units_s = (int64_t)sum_s[p.B] * p.Hkv * n.RT, total = units_s + (L.n_groups > 0 ? (int64_t)sum_p[L.n_groups] * p.Hkv : 0);
  // every worker has a unit, so the parts of an item have consecutive numbers.  (At least two or four for each: 700 tokens of one
  // sequence take 9.1 and 11.4 us instead of 7.9.)
  const int64_t workers = min((int64_t)gridDim.x * kWarps, total);
  const int64_t worker = (int64_t)warp * gridDim.x + blockIdx.x;  // few workers: on SMs of their own
  const int64_t t0 = worker < workers ? total * worker / workers : 0;
  const int share = worker < workers ? (int)(total * (worker + 1) / workers - t0) : 0;  // all units of a call fit into 31 bits
  int t = 0;  // units of the share behind this worker
  if (t < share) {
    int all, all_ahead;
    Cursor c = cursor_at<HD>(p, n, L, units_s, t0, all);
    // The loads run ahead: their cursor, the unit that it stands at, items and steps that it has begun.
    Cursor ahead = c;
    all_ahead = all;
    int t_ahead = 0, items_ahead = 0, it_ahead = 0;
    load_queries<HD>(p, n, ahead, ring, 0);
    if (kTma) copy_commit();
    const auto load_next = [&]() {
      // over the units that are no steps
      while (t_ahead < share && (ahead.unit < kItemCost || ahead.unit == ahead.units)) {
        if (ahead.unit == ahead.units) {
          next_item<HD>(p, n, L, ahead, all_ahead);
          load_queries<HD>(p, n, ahead, ring, ++items_ahead);
          if (kTma) copy_commit();
        }
        const int skip = min(share - t_ahead, max(0, kItemCost - ahead.unit));
        ahead.unit += skip;
        t_ahead += skip;
      }
      if (t_ahead < share) {
        load_step<HD, kTma>(p, &map_k, &map_v, box, ahead.w, (ahead.unit - kItemCost) * C::kKeys, ring, it_ahead++);
        ++ahead.unit;
        ++t_ahead;
      }
      if (!kTma) copy_commit();  // one group a call, with or without a step: the waits count them
    };
    bool ok = true;
    int it = 0, items = 0;
#pragma unroll
    for (int s = 0; s < C::kStages - 1; ++s) load_next();
    while (t < share && ok) {
      const int units = min(share - t, c.units - c.unit);
      const int step0 = max(0, c.unit - kItemCost), steps = max(0, c.unit + units - kItemCost) - step0;
      if (c.unit == 0 && lane == 0) ws.meta[c.item] = item_parts(c.own ? c.item : 0, t0 + t, c.units, workers, total);
      float o[HD / 8][4] = {};
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      uint32_t qf[HD / 16][4];
      const bool half = c.rows <= 8;
      for (int s = 0; s < steps; ++s, ++it) {
        const int st = it % C::kStages;
        if constexpr (kTma) {
          ok = __all_sync(0xffffffffu, mbar_wait(ring.full + st * 8, (it / C::kStages) & 1, ab, 59));
          if (!ok) break;
        } else {
          copy_wait<C::kStages - 2>();
          __syncwarp();
        }
        if (s == 0) {  // queries: the A operand (rows 8 to 15 only where there are any)
          if (kTma) {
            copy_wait<0>();
            __syncwarp();
          }
          const uint32_t src = ring.q + items % C::kStages * ring.q_rows * (HD * 2 + kQPad);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            // matrices: rows 0-7 and 8-15 of the first eight columns, then of the second
            const int r = (lane & 7) + (half ? 0 : ((lane >> 3) & 1) * 8);
            ldsm4(qf[kk], src + r * (HD * 2 + kQPad) + (kk * 2 + (lane >> 4)) * 16);
            if (half) qf[kk][1] = qf[kk][3] = 0u;
          }
          __syncwarp();
        }
        load_next();
        const int left = c.w.len - (step0 + s) * C::kKeys;
        if (half) attend<HD, kTma, true>(p, left, qf, ring, st, o, m, l);
        else attend<HD, kTma, false>(p, left, qf, ring, st, o, m, l);
        __syncwarp();
      }
      // ---- the row's result, or the part of it
      const bool whole = c.own && p.G == 0 && units == c.units;
      const int64_t part = c.own ? (c.item + worker) * n.rows_s : prefix_row(p, c.row0, all, c.kvh, c.h0) + worker * kRows;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = (lane >> 2) + 8 * h, x = c.h0 + r, col = (lane & 3) * 2;
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if (r >= c.rows) continue;
        if (whole) {
          const int64_t out = (int64_t)(c.row0 + x / n.gqa) * p.H + c.kvh * n.gqa + x % n.gqa;
          const float inv = l[h] == 0.f ? 0.f : 1.f / l[h];
          __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.o) + out * HD + col;
#pragma unroll
          for (int d = 0; d < HD / 8; ++d) *reinterpret_cast<uint32_t*>(dst + d * 8) = pack_bf16(o[d][2 * h] * inv, o[d][2 * h + 1] * inv);
          if (col == 0) p.lse[out] = row_lse(m[h], l[h]);
        } else {
          if (steps > 0) {
            float* dst = (c.own ? ws.acc_s : ws.acc_p) + (part + r) * HD + col;
#pragma unroll
            for (int d = 0; d < HD / 8; ++d) *reinterpret_cast<float2*>(dst + d * 8) = make_float2(o[d][2 * h], o[d][2 * h + 1]);
          }
          if (col == 0) (c.own ? ws.ml_s : ws.ml_p)[part + r] = make_float2(m[h], l[h]);
        }
      }
      t += units;
      if (t < share) {
        next_item<HD>(p, n, L, c, all);
        ++items;
      }
    }
    copy_wait<0>();
  }
  // The prefix kernel before this one let it start early.  It must have ended when this one ends, for the join waits for this
  // one alone: the last CTA waits for it, and the others make room for those that do not fit beside it yet.
  if (blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (*static_cast<volatile int*>(&abort_flag) != 0) {
    for (int i = 0; i < 2000; ++i) __nanosleep(100);  // copies in flight land before the CTA's memory is given away
  }
}

// Joins the parts of one (row, head) - the prefix's, then the sequence's own, in order - with kSplit warps: 1, or 4 where few
// rows with many parts each would leave the machine empty.  A lane reads one part's (m, l) and the warp's common maximum turns
// them into weights; the sums over o then have no dependent loads.
template <int HD, int kSplit>
__global__ void __launch_bounds__(kJoinWarps * 32, 8) paged_attn_join_kernel(const PagedAttnParams p, const Plan n, const Work ws) {
  constexpr int kPer = HD / 32;  // columns of a lane
  constexpr int kAtOnce = 8;     // parts in flight
  __shared__ float acc_w[kJoinWarps][HD];
  __shared__ float2 ml_w[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bh = kSplit == 1 ? blockIdx.x * kJoinWarps + warp : blockIdx.x;
  if (bh >= p.B * p.H) return;  // kSplit 1 only: no barrier follows
  const int b = bh / p.H, h = bh - b * p.H;
  const int kvh = h / n.gqa, hl = h - kvh * n.gqa;
  // The chain of dependent loads is the cost of this kernel: lengths and group (the call's inputs: before the wait), then both
  // items' entries, then the parts.
  Group gr{0, 0, 0};
  int g = 0;
  if (p.G > 0) {
    if (p.groups != nullptr) {
      int hi = p.G;
      while (hi - g > 1) {
        const int mid = (g + hi) >> 1;
        if (p.groups[mid] <= b) g = mid; else hi = mid;
      }
    }
    gr = load_group(p, g);
  }
  const int len = clamp_len(p.lens[b], p.table_width, p.pool.P, p.status);
  bool shared = gr.len > 0 && b >= gr.r0 && b < gr.r1;
  const int x = shared ? (b - gr.r0) * n.gqa + hl : 0, row_p = x % n.rows_p;
  const int item_p = shared ? first_item(n, p, g, gr.r0) + kvh * row_tiles(gr, n) + x / n.rows_p : 0;
  const int64_t pre_row = row_p + (n.form == kPrefixSmall ? prefix_row(p, gr.r0, (gr.r1 - gr.r0) * n.gqa, kvh, x - row_p) : 0);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (p.groups != nullptr && ws.meta[n.items_s + n.items_p].x != 0) shared = false;  // borders out of order: no prefixes
  int2 pre = make_int2(0, 0), own = make_int2(0, 0);
  if (shared) pre = ws.meta[item_p];
  if (len > 0) own = ws.meta[(b * p.Hkv + kvh) * n.RT + hl / kRows];
  if (p.G == 0 && own.y == 1) return;  // written by the worker that held the whole item (the same for all warps of the row)
  // a wait that gave up leaves items without their entries
  if (pre.x < 0 || pre.y < 0 || (int64_t)pre.x + pre.y > (n.form == kPrefixSmall ? 0 : (int64_t)n.items_p) + n.ctas_p) pre = make_int2(0, 0);
  if (own.x < 0 || own.y < 0 || (int64_t)own.x + own.y > (int64_t)n.items_s + n.workers) own = make_int2(0, 0);
  pre.x *= n.parts_p;
  pre.y *= n.parts_p;
  const int total = pre.y + own.y;
  const auto place = [&](int i) {
    return i < pre.y ? (int64_t)(pre.x + i) * n.part_rows_p + pre_row : (int64_t)(own.x + i - pre.y) * n.rows_s + hl % kRows;
  };
  float m = -INFINITY, l = 0.f, acc[kPer] = {};
  const int first = kSplit == 1 ? 0 : total * warp / kSplit, last = kSplit == 1 ? total : total * (warp + 1) / kSplit;
  for (int i0 = first; i0 < last; i0 += 32) {
    const int count = min(32, last - i0), i = i0 + lane;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < count) ml = (i < pre.y ? ws.ml_p : ws.ml_s)[place(i)];
    float w = 0.f;
    for (int j0 = 0; j0 < count; j0 += kAtOnce) {
      float part[kAtOnce][kPer];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int j = min(j0 + k, count - 1);
        const float* src = (i0 + j < pre.y ? ws.acc_p : ws.acc_s) + place(i0 + j) * HD + lane * kPer;
#pragma unroll
        for (int c = 0; c < kPer; ++c) part[k][c] = src[c];
      }
      if (j0 == 0) {  // after the loads of the first parts
        const float m_new = fmaxf(m, warp_max(ml.x)), old = part_weight(m, l, m_new);
        w = part_weight(ml.x, ml.y, m_new);
        l = l * old + warp_sum(w * ml.y);
        if (ml.x == -INFINITY && ml.y == 0.f) w = -0.f;  // may not have been written
#pragma unroll
        for (int c = 0; c < kPer; ++c) acc[c] *= old;
        m = m_new;
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        // left out by the sign, not by being zero: a weight that underflowed still meets what is no number among its part's values
        const float wj = j0 + k < count ? __shfl_sync(0xffffffffu, w, j0 + k) : -0.f;
#pragma unroll
        for (int c = 0; c < kPer; ++c) acc[c] += __float_as_uint(wj) != 0x80000000u ? wj * part[k][c] : 0.f;
      }
    }
  }
  if constexpr (kSplit > 1) {
#pragma unroll
    for (int c = 0; c < kPer; ++c) acc_w[warp][lane * kPer + c] = acc[c];
    if (lane == 0) ml_w[warp] = make_float2(m, l);
    __syncthreads();
    if (warp != 0) return;
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int v = 0; v < kJoinWarps; ++v) mm = fmaxf(mm, ml_w[v].x);
#pragma unroll
    for (int c = 0; c < kPer; ++c) acc[c] = 0.f;
#pragma unroll
    for (int v = 0; v < kJoinWarps; ++v) {
      const float a = part_weight(ml_w[v].x, ml_w[v].y, mm);
      ll += a * ml_w[v].y;
#pragma unroll
      for (int c = 0; c < kPer; ++c) acc[c] += a * acc_w[v][lane * kPer + c];
    }
    m = mm;
    l = ll;
  }
  const int64_t at = (int64_t)b * p.H + h;
  __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.o) + at * HD + lane * kPer;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int c = 0; c < kPer; ++c) dst[c] = __float2bfloat16_rn(acc[c] * inv);
  if (lane == 0) p.lse[at] = row_lse(m, l);
}

template <int HD> int smem_bytes(const PagedAttnParams& p, const Plan& n) {
  return kWarps * (Cfg<HD>::kRing + Cfg<HD>::kStages * n.rows_q * (HD * 2 + kQPad)) + (p.B + p.G + 2) * (int)sizeof(int);
}

// The tcgen05 forms walk over the prefixes where the small form would read them more than once (more than 16 rows of a kv head
// in the average group) and would read this many elements of keys in all (tiles of 16 rows x kv heads x tokens that the tables
// hold x dims).  They start about 10 us later, for their tensor memory, deeper pipeline and larger join, and then pass 128 or 256
// rows at a time.  Small form against them, us, by millions of elements, prefix alone:
//   6: 21.8 / 29.7 (128 rows x 12 heads, 1024 tokens)   12: 20.9 / 20.4 (126 x 6, 4096)   16: 25.2 / 27.4 (32 x 8, hd 128, 8000)
//   18: 28.6 / 30.7 (768 x 6, 1024)   24: 32.5 / 32.0 (128 x 12, 4096)   31: 41.7 / 31.7 (128 x 8, hd 128, 4001)
//   60: 48.4 / 29.2 (66 x 6, 32768)
constexpr int64_t kDenseElements = 20 << 20;

PrefixForm prefix_form(const PagedAttnParams& p) {
  const int64_t gqa = p.H / p.Hkv, rows = p.G > 0 ? p.B * gqa / p.G : 0;  // of an average group
  if (rows <= kRows || !paged_prefix_usable(p)) return kPrefixSmall;
  const int64_t tiles = (rows + kRows - 1) / kRows * p.G;
  if ((double)tiles * p.Hkv * p.hd * p.ptable_width * p.pool.P < kDenseElements) return kPrefixSmall;
  // their parts have room for 256 rows of every group and kv head: with many groups of few rows the small form's take less
  if ((double)p.Hkv * (p.B * gqa / 128 + p.G + 1) * 256 * p.hd * 4 > 1 << 30) return kPrefixSmall;
  // 32768 tokens, 6 kv heads, 256 rows at a time against 128: 35.1 / 39.2 us for 129 rows, 43.3 / 45.1 for 255, 54.6 / 54.5 for
  // 384, 74.3 / 87.1 for 768; up to 128 rows the second half of a CTA has work in the latter form alone: 34.8 / 30.5.
  return p.hd == 64 && rows > 128 ? kPrefixRows : kPrefixKeys;
}

Plan make_plan(const PagedAttnParams& p) {
  Plan n;
  n.gqa = p.H / p.Hkv;
  n.RT = (n.gqa + kRows - 1) / kRows;
  n.rows_s = n.gqa < kRows ? n.gqa : kRows;
  n.items_s = p.B * p.Hkv * n.RT;
  n.form = prefix_form(p);
  n.rows_q = n.gqa <= 8 && (p.G == 0 || n.form != kPrefixSmall) ? 8 : kRows;
  n.rows_p = n.form == kPrefixSmall ? kRows : n.form == kPrefixRows ? 256 : 128;
  n.parts_p = n.form == kPrefixKeys ? 2 : 1;
  n.part_rows_p = n.rows_p;
  n.items_p = p.G > 0 ? p.Hkv * (int)((int64_t)p.B * n.gqa / n.rows_p + p.G + 1) : 0;
  // one resident wave, but no more CTAs than there can be tiles
  const int64_t P = p.pool.P, keys = p.hd == 128 ? Cfg<128>::kKeys : Cfg<64>::kKeys;
  int64_t steps = (int64_t)n.items_s * ((p.table_width * P + keys - 1) / keys + kItemCost), tiles_p = 0;
  if (n.form == kPrefixSmall) steps += (int64_t)n.items_p * ((p.ptable_width * P + keys - 1) / keys + kItemCost);
  else tiles_p = (int64_t)n.items_p * ((p.ptable_width * P + 63) / 64);
  const int smem = (p.hd == 128 ? smem_bytes<128>(p, n) : p.hd == 64 ? smem_bytes<64>(p, n) : smem_bytes<32>(p, n)) + 2048;
  const int per_sm = std::max(1, std::min(228 * 1024 / smem, p.hd == 128 ? 4 : 8));
  n.ctas = (int)(steps < 148 * per_sm ? (steps < 1 ? 1 : steps) : 148 * per_sm);  // worker w sits in CTA w % ctas
  n.workers = n.ctas * kWarps;
  n.ctas_p = n.form == kPrefixSmall ? n.workers : (int)(tiles_p < 148 ? tiles_p : 148);
  return n;
}

int64_t round_up(int64_t n) { return (n + 255) / 256 * 256; }
int64_t own_part_rows(const Plan& n) { return ((int64_t)n.items_s + n.workers) * n.rows_s; }
int64_t prefix_part_rows(const PagedAttnParams& p, const Plan& n) {
  if (p.G == 0) return 0;
  if (n.form == kPrefixSmall) return (int64_t)p.B * p.H + (int64_t)n.workers * kRows;
  return ((int64_t)n.items_p + n.ctas_p) * n.parts_p * n.part_rows_p;
}

template <int HD, bool kTma>
int launch(const PagedAttnParams& p, const Plan& n, const Work& ws, cudaStream_t st) {
  const int box = pool_box(p.pool.P, HD == 128 ? 8 : Cfg<HD>::kKeys);
  CUtensorMap mk = {}, mv = {};
  if (kTma && (make_pool_map(&mk, p.pool.k, p, p.pool.k_page, p.pool.k_slot, p.pool.k_head, box) != 0 ||
               make_pool_map(&mv, p.pool.v, p, p.pool.v_page, p.pool.v_slot, p.pool.v_head, box) != 0))
    return -5;
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -2;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(paged_attn_kernel<HD, kTma>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWarps * (Cfg<HD>::kRing + Cfg<HD>::kStages * kRows * (HD * 2 + kQPad)) + (kMaxLists + 2) * 4) != cudaSuccess) return -2;
    if (cudaFuncSetAttribute(paged_attn_kernel<HD, kTma>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess) return -2;
    configured[dev] = true;
  }
  // The kernels after the first may be brought in while the one before still runs: the walk over own pages needs nothing of the
  // prefix kernel and shares the SMs with it (one is bound by bytes, the other by arithmetic); the join waits in
  // griddepcontrol.wait.
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.stream = st;
  cfg.blockDim = dim3(kThreads);
  if (n.form != kPrefixSmall) {
    const int rc = paged_prefix(p, n, ws, st);
    if (rc != 0) return rc;
    cfg.numAttrs = 1;
  }
  cfg.gridDim = dim3(n.ctas);
  cfg.dynamicSmemBytes = smem_bytes<HD>(p, n);
  if (cudaLaunchKernelEx(&cfg, paged_attn_kernel<HD, kTma>, mk, mv, p, n, ws, box) != cudaSuccess) return -3;
  cfg.numAttrs = 1;
  cfg.dynamicSmemBytes = 0;
  // Four warps a row against one, us: 9.1 / 9.8 for 18 rows, 13.2 / 15.5 for 96, 51.8 / 57.0 and 73.1 / 72.3 for 1152; 20.6 / 18.5
  // for 2304, 120.4 / 112.2 for 4608.
  const bool few = p.B * p.H <= 148 * 8;
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.gridDim = dim3(few ? p.B * p.H : (p.B * p.H + kJoinWarps - 1) / kJoinWarps);
  return cudaLaunchKernelEx(&cfg, few ? paged_attn_join_kernel<HD, kJoinWarps> : paged_attn_join_kernel<HD, 1>, p, n, ws) == cudaSuccess ? 0 : -3;
}

}  // namespace

int64_t paged_attn_workspace(const PagedAttnParams& p) {
  if (p.hd != 32 && p.hd != 64 && p.hd != 128) return -1;
  if (p.B + p.G > kMaxLists) return -1;
  const Plan n = make_plan(p);
  const int64_t ss = own_part_rows(n), sp = prefix_part_rows(p, n);
  return round_up(ss * p.hd * 4) + round_up(ss * 8) + round_up(sp * p.hd * 4) + round_up(sp * 8) + round_up(((int64_t)n.items_s + n.items_p + 1) * 8);
}

int paged_attn(const PagedAttnParams& p, void* workspace, cudaStream_t st) {
  if (p.B == 0) return 0;
  if (p.H < 1 || p.Hkv < 1 || p.H % p.Hkv != 0 || p.H > 65535 || p.B + p.G > kMaxLists) return -10;
  const Plan n = make_plan(p);
  const int64_t ss = own_part_rows(n), sp = prefix_part_rows(p, n);
  uint8_t* at = static_cast<uint8_t*>(workspace);
  Work ws;
  ws.acc_s = reinterpret_cast<float*>(at);
  at += round_up(ss * p.hd * 4);
  ws.ml_s = reinterpret_cast<float2*>(at);
  at += round_up(ss * 8);
  ws.acc_p = reinterpret_cast<float*>(at);
  at += round_up(sp * p.hd * 4);
  ws.ml_p = reinterpret_cast<float2*>(at);
  at += round_up(sp * 8);
  ws.meta = reinterpret_cast<int2*>(at);
  // Whole 8-row groups of the swizzle pattern.  64 ragged sequences of up to 8192 tokens: 73 us, with cp.async 109.
  const bool tma = pool_box(p.pool.P, 8) == 8;
  switch (p.hd) {
    case 32: return tma ? launch<32, true>(p, n, ws, st) : launch<32, false>(p, n, ws, st);
    case 64: return tma ? launch<64, true>(p, n, ws, st) : launch<64, false>(p, n, ws, st);
    case 128: return tma ? launch<128, true>(p, n, ws, st) : launch<128, false>(p, n, ws, st);
  }
  return -10;
}

}  // namespace seg
