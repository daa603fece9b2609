// The prefix part of the paged attention for groups with many rows, on tcgen05 tensor cores (head_dim 64 and 128, bf16).
//
// For every (group, kv head) the rows are the group's sequences x query heads of the kv head; all of them see the same keys, so
// this is a plain (unmasked) attention with few "queries" and a long walk: S = Q K^T, P = exp2(scale S - m), O += P V, with the
// keys and values gathered page by page.  Its results are parts (m, l, unnormalised O) that the join kernel of paged_attn.cu
// merges with the sequences' own tokens.
//
// Work: items of 256 rows (two tiles of 128 that share every key tile; kRows form) or of 128 rows whose key tiles are dealt to
// the CTA's two halves alternately (kKeys form: fewer rows, or head_dim 128, where two query tiles would not fit into shared
// memory).  The key tiles (128 keys; 64 in the kKeys form, which is bound by the latency of its loads and wants more of them in
// flight) of all items in one row are dealt to one CTA per SM in equal, contiguous ranges.
//
// Roles of a CTA (384 threads): warps 0 and 3 load K and V, every lane one box of a page (1 to 16 boxes of 8 to 128 keys a
// tile) into rings of tiles; keys behind the length come as zeros or are masked, their values are set to zero before the products see
// them; warps 1 and 2 issue the products of half 0 / 1; warps 4-7 and 8-11 are the softmax of half 0 / 1, a row per thread.
//
// Bound: one exp2 per score, 16 a cycle and SM on the special-function unit: 2048 cycles for 256 x 128 scores against 1024 of
// the tensor core at head_dim 64.  A quarter of the exponentials therefore runs as a polynomial on the FMA pipe, and the
// softmax keeps the maximum off its critical path: the exponentials use the reference of the tiles before, and only when a
// new score exceeds it by more than 2^8 (rare after the first tile) is the row's sum rescaled and the tile repeated from tensor
// memory.  Scores pass through the registers 32 columns at a time, the next load in flight; P goes back to tensor memory, from
// where the second product reads it (through shared memory, each warp's fence between its stores and the tensor core's reads
// cost 290 cycles a tile).  Registers and, at head_dim 64, shared memory leave room on the SM for CTAs of the kernel over own pages.
// Measured: 256 sequences x 18 heads on 32768 tokens (6 kv heads of 64) 75 us with the join, of them about 20 before the first and
// after the last tile; a 256 x 128 tile takes 2200 cycles, in which both halves do their softmax at the same time and then wait
// for the products together (1075 cycles of the tensor core).  Four softmax warps a scheduler, 64-key tiles in two buffers and halves that take
// turns were slower.
#include <cuda.h>

#include <type_traits>

#include "paged_common.cuh"
#include "sm100.cuh"

namespace seg {

using namespace sm100;

namespace {

constexpr int kThreads = 384;
// Scale and reference are applied in one fused operation, which leaves the rounding of the product they stand for: up to 2^-24 of the
// score, in the exponent.  Beyond this score (log2 units) a warp rounds product and difference one after the other and takes the
// rounded products' maximum as reference, so that the best key lies at exactly zero.  (In all tiles: 256 sequences on 32768 tokens take
// 118 us instead of 113.)
constexpr float kApart = 16777216.f;
constexpr int kBlock = 128 * 128;  // bytes of 128 rows of 64 bf16: the unit of the query tiles

template <int HD, bool kSplit> struct Lay {
  static constexpr int kKeys = kSplit ? 64 : 128;              // keys per tile
  static constexpr int kDepth = 3;                             // places of a ring
  static constexpr int kRings = kSplit ? 2 : 1;                // rings: one for both halves, or one each
  static constexpr int kSlots = kDepth * kRings;
  static constexpr int kGroup = HD / 64 * 1024;                // bytes of 8 keys: blocks of 64 dims behind each other
  static constexpr int kTile = kKeys / 8 * kGroup;
  static constexpr int kQTile = HD / 64 * kBlock;
  static constexpr int kPCols = 2 * kKeys + 2 * HD;            // tensor memory: first column of P (bf16, two keys a column)
  static_assert(kPCols + kKeys <= 512, "tensor memory");
  static constexpr int kK = (kSplit ? 1 : 2) * kQTile, kV = kK + kSlots * kTile, kBars = kV + kSlots * kTile, kSum = kBars + 512;
};

// 32 lanes x 16 consecutive 32-bit columns
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15])
      : "memory");
}

// 2^x for a pair on the FMA and integer pipes: x = n + f with n the nearest integer (rounding by a large constant), |f| <= 1/2, a
// polynomial of degree 4 for 2^f (minimax of the relative error, 2.6e-6; a weight is rounded to bf16 anyway), n added to the
// exponent.  x <= 100; below -126 the result is 2^-126 instead of 0, and so it is for NaN, which the caller keeps in the row's maximum.
// One pair of four takes it: none 79.3 us, one 77.2, two 85.2 (768 rows on 32768 tokens, 6 kv heads).
__device__ __forceinline__ void exp2_pair(uint64_t x, float& p0, float& p1) {
  float x0, x1;
  unpack2(x, x0, x1);
  const uint64_t xc = pack2(fmaxf(x0, -126.f), fmaxf(x1, -126.f)), magic = pack2(12582912.f, 12582912.f);  // 1.5 * 2^23
  const uint64_t t = add2(xc, magic), f = sub2(xc, sub2(t, magic));
  uint64_t q = fma2(pack2(0.009570102207362652f, 0.009570102207362652f), f, pack2(0.05591785907745361f, 0.05591785907745361f));
  q = fma2(q, f, pack2(0.240247443318367f, 0.240247443318367f));
  q = fma2(q, f, pack2(0.6931217908859253f, 0.6931217908859253f));
  q = fma2(q, f, pack2(0.9999992847442627f, 0.9999992847442627f));
  uint32_t t0, t1, q0, q1;
  unpack2(t, t0, t1);
  unpack2(q, q0, q1);
  p0 = __uint_as_float(q0 + (t0 << 23));
  p1 = __uint_as_float(q1 + (t1 << 23));
}

struct Seg {
  int item, kvh, rows, row0, x0;  // rows r = x0 .. x0 + rows - 1 of the group: sequence row0 + r / gqa, head kvh * gqa + r % gqa
  int len, tile0, n_tiles, steps;
  const int* pages;
};

template <int kTileKeys>
__device__ __forceinline__ Seg find_seg(const PagedAttnParams& p, const Plan& n, const int* sum, int64_t t, int64_t t_end) {
  Seg s;
  const int g = find_list(sum, p.G, (int)(t / p.Hkv));
  const Group gr = load_group(p, g);
  s.n_tiles = (gr.len + kTileKeys - 1) / kTileKeys;
  const int local = (int)(t - (int64_t)sum[g] * p.Hkv), i = local / s.n_tiles, rt = row_tiles(gr, n);
  s.tile0 = local - i * s.n_tiles;
  s.kvh = i / rt;
  s.x0 = (i - s.kvh * rt) * n.rows_p;
  s.item = first_item(n, p, g, gr.r0) + i;
  s.row0 = gr.r0;
  s.rows = min(n.rows_p, (gr.r1 - gr.r0) * n.gqa - s.x0);
  s.len = gr.len;
  s.steps = (int)min(t_end - t, (int64_t)(s.n_tiles - s.tile0));
  s.pages = p.ptable + g * p.ptable_stride;
  return s;
}

template <int HD, bool kSplit>
__global__ void __maxnreg__(128)  // of 384 threads: leaves 16384 registers for a CTA of the kernel over own pages
paged_prefix_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PagedAttnParams p, const Plan n, const Work ws,
                    const int box) {
  using L = Lay<HD, kSplit>;
  constexpr int kTileKeys = L::kKeys;
  extern __shared__ __align__(1024) uint8_t smem[];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled tiles need a 1024-byte aligned base
    if (threadIdx.x == 0) atomicCAS(p.status, 0, 60);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t *q_full = bars, *s_full = bars + 2, *s_empty = bars + 4, *p_full = bars + 6, *pv_full = bars + 8, *tail = bars + 10, *q_free = bars + 11,
           *k_full = bars + 12, *k_empty = k_full + L::kSlots, *v_full = k_empty + L::kSlots, *v_empty = v_full + L::kSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_empty + L::kSlots);
  volatile int* cta_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* warp_tot = reinterpret_cast<int*>(tmem_slot + 2);
  static_assert((12 + 4 * L::kSlots) * 8 + 8 + kThreads / 32 * 4 <= 512, "the barriers must fit into their region");
  int* sum = reinterpret_cast<int*>(smem + L::kSum);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AbortState ab{cta_abort, p.status};

  if (threadIdx.x == 0) {
    *cta_abort = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&q_full[i]), 4);
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&s_empty[i]), 4);
      mbar_init(smem_u32(&p_full[i]), 4);
      mbar_init(smem_u32(&pv_full[i]), 1);
    }
    for (int i = 0; i < L::kSlots; ++i) {
      mbar_init(smem_u32(&k_full[i]), 1);
      mbar_init(smem_u32(&v_full[i]), 1);
      mbar_init(smem_u32(&k_empty[i]), kSplit ? 1 : 2);  // released by the products of every half that reads the tile
      mbar_init(smem_u32(&v_empty[i]), kSplit ? 1 : 2);
    }
    mbar_init(smem_u32(tail), 1);
    mbar_init(smem_u32(q_free), 5);  // the second half's softmax warps and its issuer
    fence_barrier_init();
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  if (warp == 0) {
    __syncwarp();
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  const bool in_order = scan_groups<kThreads>(sum, p, n, ws, [](int len) { return (len + kTileKeys - 1) / kTileKeys; }, warp_tot);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // scores of half 0 / 1, outputs of half 0 / 1, P of half 0 / 1
  const int64_t total = in_order ? (int64_t)sum[p.G] * p.Hkv : 0;
  // One prefix: a number of CTAs that gives each a part of one item only, where that leaves at most a sixteenth of them idle (a
  // second part costs a CTA about 5 us: queries, first maximum, outputs; 256 sequences on 32768 tokens: 74 us, otherwise 78).
  int64_t ctas = min((int64_t)gridDim.x, total);
  if (p.G == 1 && total > 0) {
    const int64_t items = (int64_t)p.Hkv * row_tiles(load_group(p, 0), n), even = ctas / items * items;
    if (even * 16 >= ctas * 15) ctas = even;
  }
  const int64_t t_begin = blockIdx.x < ctas ? total * blockIdx.x / ctas : 0, t_end = blockIdx.x < ctas ? total * (blockIdx.x + 1) / ctas : 0;

  if (warp == 0 || warp == 3) {
    // ------------------------------------------------------------------------------------------------ loads: K (warp 0), V (warp 3)
    const bool is_v = warp == 3;
    uint64_t *full = is_v ? v_full : k_full, *empty = is_v ? v_empty : k_empty;
    const CUtensorMap* map = is_v ? &map_v : &map_k;
    int used[2] = {0, 0}, tails = 0;  // tiles so far of each ring
    bool ok = true;
    const bool mine = lane * box < kTileKeys;
    for (int64_t t = t_begin; t < t_end && ok;) {
      const Seg s = find_seg<kTileKeys>(p, n, sum, t, t_end);
      const auto lookup = [&](int j) {  // the page of this lane's box of tile j, one tile ahead and unchecked
        const int key = (s.tile0 + j) * kTileKeys + lane * box;
        return mine && j < s.steps && key < s.len ? s.pages[p.pool.shift >= 0 ? key >> p.pool.shift : key / p.pool.P] : -1;
      };
      int found = lookup(0);
      for (int j = 0; j < s.steps && ok; ++j) {
        const int ring = kSplit ? j & 1 : 0, c = ring ? used[1]++ : used[0]++, st = ring * L::kDepth + c % L::kDepth, ph = (c / L::kDepth) & 1;
        const int first = (s.tile0 + j) * kTileKeys, key = first + lane * box;
        int page = p.pool.n_pages, slot = 0;  // a box outside the pool reads as zeros
        if (mine && key < s.len) {
          if ((unsigned)found < (unsigned)p.pool.n_pages) {
            page = found;
            slot = p.pool.shift >= 0 ? key & (p.pool.P - 1) : key % p.pool.P;
          } else {
            atomicCAS(p.status, 0, kStatusAttnPage);
          }
        }
        found = lookup(j + 1);
        const bool mend = is_v && s.len < first + kTileKeys && s.len % box != 0;  // the last box brings slots behind the length
        const uint32_t dst = (is_v ? L::kV : L::kK) + st * L::kTile, bar = smem_u32(mend ? tail : &full[st]);
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&empty[st]), ph ^ 1, ab, 61 + is_v));
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(bar, L::kTile);
        __syncwarp();
        if (mine) load_box(smem_u32(smem) + dst + lane * box * (HD * 2), map, bar, slot, s.kvh, page);
        if (mend) {
          // values behind the length: zeros, so that no weight of zero meets what lies there
          ok = __all_sync(0xffffffffu, mbar_wait(bar, tails & 1, ab, 63));
          if (!ok) break;
          ++tails;
          for (int i = (s.len - first) * 8 + lane; i < kTileKeys * 8; i += 32) {  // key i / 8, 16 bytes of each block
#pragma unroll
            for (int b = 0; b < HD / 64; ++b) *reinterpret_cast<uint4*>(smem + dst + (i >> 6) * L::kGroup + b * 1024 + (i & 63) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&full[st]));
        }
      }
      t += s.steps;
    }
  } else if (warp <= 2) {
    // ------------------------------------------------------------------------------------------------ products of half x
    const int x = warp - 1;
    if (elect_one()) {
      constexpr uint32_t idesc_s = make_idesc_bf16(128, kTileKeys, false, false);  // Q (K-major) x K (K-major)
      constexpr uint32_t idesc_o = make_idesc_bf16(128, HD, false, true);          // P (K-major) x V (MN-major)
      const uint64_t d_q = make_smem_desc(smem_u32(smem) + (kSplit ? 0 : x * L::kQTile), 16, 1024);
      const uint32_t t_p = tmem + L::kPCols + x * (kTileKeys / 2);
      const uint32_t t_s = tmem + x * kTileKeys, t_o = tmem + 2 * kTileKeys + x * HD;
      int cx = 0, seg = 0;  // tiles of this half, segments
      bool ok = true;
      for (int64_t t = t_begin; t < t_end && ok; ++seg) {
        const Seg s = find_seg<kTileKeys>(p, n, sum, t, t_end);
        const int mine = kSplit ? (s.steps + 1 - x) / 2 : s.steps;
        ok = mbar_wait(smem_u32(&q_full[kSplit ? 0 : x]), seg & 1, ab, 64);  // in every segment, so that no phase is missed
        if (kSplit && x == 1 && ok) mbar_arrive(smem_u32(q_free));
        auto scores = [&](int i) {
          const int at = cx + i, st = (kSplit ? x * L::kDepth : 0) + at % L::kDepth, ph = (at / L::kDepth) & 1;
          if (!mbar_wait(smem_u32(&k_full[st]), ph, ab, 65)) return false;
          if (at > 0 && !mbar_wait(smem_u32(&s_empty[x]), (at - 1) & 1, ab, 66)) return false;
          const uint64_t d_k = make_smem_desc(smem_u32(smem + L::kK + st * L::kTile), 16, L::kGroup);
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < HD / 16; ++k) {
            const uint64_t oq = (uint64_t)(((k >> 2) * kBlock + (k & 3) * 32) >> 4), ok_ = (uint64_t)(((k >> 2) * 1024 + (k & 3) * 32) >> 4);
            umma_bf16(t_s, d_q + oq, d_k + ok_, idesc_s, k > 0);
          }
          umma_commit(smem_u32(&s_full[x]));
          umma_commit(smem_u32(&k_empty[st]));
          return true;
        };
        if (ok && mine > 0) ok = scores(0);
        for (int i = 0; i < mine && ok; ++i) {
          if (i + 1 < mine && !scores(i + 1)) { ok = false; break; }
          const int at = cx + i, st = (kSplit ? x * L::kDepth : 0) + at % L::kDepth, ph = (at / L::kDepth) & 1;
          if (!mbar_wait(smem_u32(&v_full[st]), ph, ab, 67) || !mbar_wait(smem_u32(&p_full[x]), at & 1, ab, 68)) { ok = false; break; }
          const uint64_t d_v = make_smem_desc(smem_u32(smem + L::kV + st * L::kTile), 1024, L::kGroup);
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < kTileKeys / 16; ++k)
            umma_bf16_ts(t_o, t_p + k * 8, d_v + (uint64_t)(2 * k * (L::kGroup >> 4)), idesc_o, i > 0 || k > 0);
          umma_commit(smem_u32(&pv_full[x]));
          umma_commit(smem_u32(&v_empty[st]));
        }
        cx += mine;
        t += s.steps;
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------------------------------------------------------ softmax of half x
    const int x = (warp >> 2) - 1, sub = warp & 3, r = sub * 32 + lane;  // r: row of the half's tile == TMEM lane
    const uint32_t lane_addr = (uint32_t)(sub * 32) << 16;
    const uint32_t t_s = tmem + x * kTileKeys + lane_addr, t_o = tmem + 2 * kTileKeys + x * HD + lane_addr;
    const uint32_t t_p = tmem + L::kPCols + x * (kTileKeys / 2) + lane_addr;
    const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2);
    int cx = 0, seg = 0;
    bool ok = true;
    // tensor memory is read by whole warps: when a wait gives up, all lanes leave together
    auto wait = [&](uint64_t* bar, int parity, int code) { return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, ab, code)) != 0; };
    for (int64_t t = t_begin; t < t_end && ok; ++seg) {
      const Seg s = find_seg<kTileKeys>(p, n, sum, t, t_end);
      const int mine = kSplit ? (s.steps + 1 - x) / 2 : s.steps;
      if (s.tile0 == 0 && threadIdx.x == 128) ws.meta[s.item] = item_parts(s.item - n.items_s, t, s.n_tiles, ctas, total);
      const int row = (kSplit ? 0 : x * 128) + r;
      // Queries of the segment.  The products of the segment before with the old ones are complete: this warp has seen its last
      // scores, and where both halves read one query tile the other half says so (its issuer too: it may have had no tile).
      if (kSplit && x == 0 && seg > 0) {
        ok = wait(q_free, (seg - 1) & 1, 73);
        if (!ok) break;
      }
      if (!kSplit || x == 0) {
        uint8_t* sQ = smem + (kSplit ? 0 : x * L::kQTile) + r * 128;
        const int q = s.x0 + row;
        const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.q) + (s.row0 + q / n.gqa) * p.q_row + (s.kvh * n.gqa + q % n.gqa) * p.q_head;
        const bool live = row < s.rows;
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
          const uint4 v = live ? *reinterpret_cast<const uint4*>(src + c * 8) : make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(sQ + (c >> 3) * kBlock + (((c & 7) ^ (r & 7)) << 4)) = v;
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&q_full[kSplit ? 0 : x]));
      } else {  // without a tile of its own in a segment this half would run ahead and count twice on q_free
        ok = wait(&q_full[0], seg & 1, 74);
        if (!ok) break;
      }
      float m = -INFINITY, l = 0.f;  // m: reference of the exponentials, the row's maximum up to 2^8
      bool apart = false;            // of a warp: a reference beyond kApart
      for (int i = 0; i < mine && ok; ++i) {
        const int at = cx + i, tile = s.tile0 + (kSplit ? 2 * i + x : i);
        const int left = s.len - tile * kTileKeys;  // keys of this tile that exist
        ok = wait(&s_full[x], at & 1, 69);
        if (!ok) break;
        tc_fence_after();
        // The scores of chunk c relative to the reference, and the row's running maximum of them, NaN where one of them is.  Careful
        // tiles: keys behind the length are masked; product and difference apart, and the maximum is that of the products.
        auto scaled = [&](auto careful, const uint32_t* w, int c, uint64_t neg2, uint64_t* y, float* mx) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint64_t w2 = pack2(w[2 * e], w[2 * e + 1]);
            y[e] = decltype(careful)::value ? mul2(w2, scale2) : fma2(w2, scale2, neg2);
            float a, b;
            unpack2(y[e], a, b);
            if (decltype(careful)::value) {
              if (c * 32 + 2 * e >= left) a = -INFINITY;
              if (c * 32 + 2 * e + 1 >= left) b = -INFINITY;
              y[e] = pack2(a, b);
            }
            mx[e & 3] = max3_nan(mx[e & 3], a, b);
            if (decltype(careful)::value) y[e] = add2(y[e], neg2);
          }
        };
        constexpr int kChunks = kTileKeys / 32;
        // kAgain: a reference beyond kApart, nothing of the tile has been kept
        enum { kGaveUp, kDone, kAgain };
        auto one_tile = [&](auto careful) -> int {
          constexpr bool kCareful = decltype(careful)::value;
          uint32_t v[2][32];
          uint64_t y[16];
          if (i == 0) {  // no reference yet: the tile's maximum
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            tmem_ld_32x32(t_s, v[0]);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
              tmem_ld_wait_regs(v[c & 1]);
              if (c + 1 < kChunks) tmem_ld_32x32(t_s + (c + 1) * 32, v[(c + 1) & 1]);
              scaled(careful, v[c & 1], c, 0ull, y, mx);
            }
            m = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3]));
            if (!kCareful && __any_sync(0xffffffffu, m > kApart || (m < -kApart && m > -INFINITY))) return kAgain;
          }
          for (int pass = 0;; ++pass) {  // a second pass where the reference was too low
            const float base = m == -INFINITY ? 0.f : m;
            const uint64_t neg2 = pack2(-base, -base);
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            uint64_t l2[2] = {0ull, 0ull};
            bool redo = false;
            tmem_ld_32x32(t_s, v[0]);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
              tmem_ld_wait_regs(v[c & 1]);
              if (c + 1 < kChunks) tmem_ld_32x32(t_s + (c + 1) * 32, v[(c + 1) & 1]);
              scaled(careful, v[c & 1], c, neg2, y, mx);
              if (c == kChunks - 1) {
                const float top = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3]));
                const float above = kCareful ? top - base : top, there = kCareful ? top : top + base;
                const bool low = above > 8.f || (m == -INFINITY && top > -INFINITY);
                redo = pass == 0 && __any_sync(0xffffffffu, low);
                if (redo) {
                  if (!kCareful && __any_sync(0xffffffffu, low && fabsf(there) > kApart)) {
                    tmem_st_wait();  // of the weights stored so far, before others take their place
                    return kAgain;
                  }
                  const float m_new = low ? there : m;
                  if (i > 0) {  // what was summed so far is rescaled
                    const float a = low && m != -INFINITY ? exp2_(m - m_new) : 1.f;
                    l *= a;
#pragma unroll
                    for (int o = 0; o < HD / 32; ++o) {
                      tmem_ld_32x32(t_o + o * 32, v[0]);
                      tmem_ld_wait_regs(v[0]);
#pragma unroll
                      for (int e = 0; e < 32; ++e) v[0][e] = __float_as_uint(__uint_as_float(v[0][e]) * a);
                      tmem_st_32x32(t_o + o * 32, v[0]);
                    }
                    tmem_st_wait();
                  }
                  m = m_new;
                  break;
                }
                if (above != above) l = above;  // a score of NaN or +inf makes the row NaN; its weight may not (exp2_pair)
                // the scores are in registers: the next product may overwrite them
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s_empty[x]));
              }
              uint32_t pk[16];
#pragma unroll
              for (int q4 = 0; q4 < 4; ++q4) {
                float e[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  if (k == 3 && !kCareful) {
                    exp2_pair(y[q4 * 4 + k], e[2 * k], e[2 * k + 1]);
                  } else {
                    float a, b;
                    unpack2(y[q4 * 4 + k], a, b);
                    e[2 * k] = exp2_(a);
                    e[2 * k + 1] = exp2_(b);
                  }
                  l2[k & 1] = add2(l2[k & 1], pack2(e[2 * k], e[2 * k + 1]));
                }
                const bf16x8 b8 = pack8(e);
#pragma unroll
                for (int k = 0; k < 4; ++k) pk[q4 * 4 + k] = *reinterpret_cast<const uint32_t*>(&b8.v[k]);
              }
              if (c == 0 && i > 0 && pass == 0) {  // P V of the tile before has read the P tile
                if (!wait(&pv_full[x], (at - 1) & 1, 71)) {
                  tmem_ld_wait();
                  return kGaveUp;
                }
                tc_fence_after();
              }
              tmem_st_32x16(t_p + c * 16, pk);
            }
            if (redo) continue;
            float a0, a1, a2, a3;
            unpack2(l2[0], a0, a1);
            unpack2(l2[1], a2, a3);
            const float add = (a0 + a1) + (a2 + a3);
            l += m == -INFINITY && add == add ? 0.f : add;  // only -inf scores so far: weights of zero (the polynomial's are 2^-126)
            return kDone;
          }
        };
        int done = kAgain;
        if (!apart && left >= kTileKeys) {
          done = one_tile(std::false_type{});
          apart = done == kAgain;
        }
        if (done == kAgain) done = one_tile(std::true_type{});
        ok = done == kDone;
        if (!ok) break;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_full[x]));
      }
      if (kSplit && x == 1) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(q_free));
      }
      // ---- the part of this segment
      const int64_t part = kSplit ? ((int64_t)(s.item - n.items_s) + blockIdx.x) * 2 + x : (int64_t)(s.item - n.items_s) + blockIdx.x;
      const int64_t out = part * n.part_rows_p + row;
      if (ok && row < s.rows) ws.ml_p[out] = make_float2(m, l);
      if (ok && mine > 0) {
        ok = wait(&pv_full[x], (cx + mine - 1) & 1, 72);
        tc_fence_after();
        if (ok) {
#pragma unroll
          for (int o = 0; o < HD / 32; ++o) {
            uint32_t f[32];
            tmem_ld_32x32(t_o + o * 32, f);
            tmem_ld_wait_regs(f);
            if (row < s.rows) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                reinterpret_cast<uint4*>(ws.acc_p + out * HD + o * 32)[e] = make_uint4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
            }
          }
        }
      }
      cx += mine;
      t += s.steps;
    }
  }

  if (*cta_abort != 0) {
    tmem_ld_wait();
    for (int i = 0; i < 2000; ++i) __nanosleep(100);  // copies in flight land before the CTA's memory is given away
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

template <int HD, bool kSplit>
int launch(const PagedAttnParams& p, const Plan& n, const Work& ws, cudaStream_t st) {
  using L = Lay<HD, kSplit>;
  const int box = pool_box(p.pool.P, HD == 128 ? 8 : L::kKeys);
  CUtensorMap mk, mv;
  if (make_pool_map(&mk, p.pool.k, p, p.pool.k_page, p.pool.k_slot, p.pool.k_head, box) != 0 ||
      make_pool_map(&mv, p.pool.v, p, p.pool.v_page, p.pool.v_slot, p.pool.v_head, box) != 0)
    return -5;
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -2;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(paged_prefix_kernel<HD, kSplit>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) return -2;
    // all of the SM's memory as shared memory: with the least that this kernel needs, no CTA of the next one would fit beside it
    if (cudaFuncSetAttribute(paged_prefix_kernel<HD, kSplit>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess) return -2;
    configured[dev] = true;
  }
  paged_prefix_kernel<HD, kSplit><<<n.ctas_p, kThreads, L::kSum + (p.G + 1) * 4, st>>>(mk, mv, p, n, ws, box);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace

bool paged_prefix_usable(const PagedAttnParams& p) {
  if (p.hd != 64 && p.hd != 128) return false;
  if (pool_box(p.pool.P, 8) < 8) return false;  // whole 8-row groups of the swizzle pattern
  const int smem = (p.hd == 128 ? Lay<128, true>::kSum : Lay<64, false>::kSum) + (p.G + 1) * 4;
  return smem <= 227 * 1024;
}

int paged_prefix(const PagedAttnParams& p, const Plan& n, const Work& ws, cudaStream_t st) {
  if (n.form == kPrefixRows) return p.hd == 64 ? launch<64, false>(p, n, ws, st) : -10;
  return p.hd == 64 ? launch<64, true>(p, n, ws, st) : p.hd == 128 ? launch<128, true>(p, n, ws, st) : -10;
}

}  // namespace seg
