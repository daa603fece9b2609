// Launchers of the paged serving kernels (raw pointers + stream; no framework types): appending to a paged key/value cache,
// one-token attention over it with a prefix shared by a group of sequences, and the processing of logits before sampling.
//
// A pool holds pages of P tokens; element (page, slot, kv head, dim) of the key pool is at
//   k + page * k_page + slot * k_slot + head * k_head + dim      (strides in elements, multiples of 8; dims contiguous),
// so pools ordered by token ([pages, P, Hkv, hd]) and by head ([pages, Hkv, P, hd]) are both read and written in place.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace seg {

struct PagedPool {
  void* k;
  void* v;
  int64_t k_page, k_slot, k_head;
  int64_t v_page, v_slot, v_head;
  int n_pages, P;
  int shift;  // log2(P), or -1 where P is no power of two
};

// Codes of the package's status word (0 = all well) that these kernels set when data on the device does not fit; the token is
// then left out (append) or read as zeros (attention), and no access leaves its buffer.
constexpr int kStatusAppendTable = 51;   // append: a position beyond the page table or the rotation table, or a negative length
constexpr int kStatusAppendPage = 52;    // append: a page number outside the pool
constexpr int kStatusAttnLength = 53;    // attention: a length that is negative or beyond its page table
constexpr int kStatusAttnPage = 54;      // attention: a page number outside the pool
constexpr int kStatusAttnGroups = 55;    // attention: group_rows not ascending within [0, B]
constexpr int kStatusLogitsLength = 56;  // logits: a history length that is negative or beyond the token matrix
constexpr int kStatusLogitsMask = 57;    // logits: a mask row beyond the mask

// ---- paged_append.cu
struct PagedAppendParams {
  const void* qkv;     // bf16 rows of (H + 2 Hkv) * hd, qkv_stride elements apart
  int64_t qkv_stride;
  const void* v1;      // bf16 [T, Hkv, hd] or nullptr
  const float* cos;    // [rope_rows, hd / 2]
  const float* sin;
  const float *qgain, *alpha1, *alpha2, *vscale;
  PagedPool pool;
  const int* table;    // [B, table_width], rows table_stride apart
  int64_t table_stride;
  int table_width;
  const int* lens;     // [B] tokens that the sequence's pages hold already
  const int* cu;       // [B + 1] first row of every sequence, or nullptr: row t belongs to sequence t
  const int* pos_base; // [B] added to the position for the rotation, or nullptr
  void* q;             // bf16 [T, H, hd]
  void* k_out;         // bf16 [T, Hkv, hd] or nullptr
  void* v_out;         // likewise
  int* status;
  int T, B, H, Hkv, hd, rope_rows;
  bool qknorm;
};
// 0, or a negative number when the sizes are not supported or the launch failed
int paged_append(const PagedAppendParams& p, cudaStream_t st);

// ---- paged_attn.cu
struct PagedAttnParams {
  const void* q;  // bf16, rows q_row and heads q_head elements apart
  int64_t q_row, q_head;
  PagedPool pool;
  const int* table;  // [B, table_width]
  int64_t table_stride;
  int table_width;
  const int* lens;    // [B]
  const int* ptable;  // [G, ptable_width] pages of the groups' prefixes, or nullptr (G = 0)
  int64_t ptable_stride;
  int ptable_width;
  const int* plens;   // [G]
  const int* groups;  // [G + 1] first row of every group, or nullptr: one group of all rows
  int B, H, Hkv, hd, G;
  float scale_log2;  // scale * log2(e)
  void* o;           // bf16 [B, H, hd]
  float* lse;        // [B, H]
  int* status;
};
// Bytes of scratch that a call needs (uninitialised; free to reuse in stream order after the call), or -1: sizes not supported.
int64_t paged_attn_workspace(const PagedAttnParams& p);
int paged_attn(const PagedAttnParams& p, void* workspace, cudaStream_t st);

// ---- logits.cu
struct LogitsParams {
  const void* x;  // [B, V], rows x_row elements apart
  void* y;        // likewise; may be x
  int64_t x_row, y_row;
  int B, V;
  bool bf16;           // bf16 or fp32 logits
  const void* tokens;  // [B, tokens_width] int32 or int64, rows tokens_row apart, or nullptr
  bool tokens64;
  int64_t tokens_row;
  int tokens_width;
  const int* prompt_lens;                          // [B] or nullptr (no token is the prompt's)
  const int* token_lens;                           // [B]
  const float *repetition, *presence, *frequency;  // [B] or nullptr
  const int* bias_ids;                             // [B, K], contiguous, or nullptr
  const float* bias;                               // [B, K]
  int K;
  const int* mask;  // [n_masks, (V + 31) / 32], rows mask_row apart, or nullptr
  int64_t mask_row;
  int n_masks;
  const int* mask_rows;  // [B]
  int* status;
};
int process_logits(const LogitsParams& p, cudaStream_t st);

}  // namespace seg
