// Python bindings of the paged serving kernels (paged_append.cu, paged_attn.cu, logits.cu).  Everything that can be known on
// the host is checked here; lengths, page numbers and group borders live on the device and are checked by the kernels.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>

#include "paged.h"

int* package_status_ptr(const c10::Device& dev);  // gemm_bindings.cpp
bool package_status_ready(const c10::Device& dev);

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// Straight from the allocator: the small calls are bound by the host.
Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, const c10::Device& dev) {
  return at::detail::empty_cuda(sizes, type, dev, std::nullopt);
}

// The status word.  Made by the package's first call on a device; inside a capture it would be the graph's memory, and every
// replay would clear it.
int* status_word(const c10::Device& dev) {
  if (!package_status_ready(dev)) {
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    TORCH_CHECK(cudaStreamIsCapturing(cur_stream(), &capture) == cudaSuccess && capture == cudaStreamCaptureStatusNone,
                "the first call on a device cannot be captured into a graph: run the step once before");
  }
  return package_status_ptr(dev);
}

void check_on(const Tensor& t, const c10::Device& dev, const char* name) {
  TORCH_CHECK(t.device() == dev, name, " must be on ", dev, ", got ", t.device());
}
// bf16 tensor whose rows of the last dimension are contiguous and start on 16-byte boundaries
void check_rows16(const Tensor& t, const c10::Device& dev, const char* name) {
  check_on(t, dev, name);
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be bfloat16, got ", t.scalar_type());
  if (t.numel() == 0) return;
  TORCH_CHECK(t.stride(-1) == 1 || t.size(-1) == 1, name, " must be contiguous in its last dimension");
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    TORCH_CHECK(t.size(i) == 1 || t.stride(i) % 8 == 0, name, ": strides must be multiples of 8 elements (16 bytes)");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name, " must start on a 16-byte boundary");
}
void check_contig(const Tensor& t, at::ScalarType type, int64_t n, const c10::Device& dev, const char* name) {
  check_on(t, dev, name);
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
  TORCH_CHECK(t.is_contiguous() && t.numel() == n, name, " must be contiguous with ", n, " elements, got ", t.sizes());
}
const float* scalar_ptr(const Tensor& t, const c10::Device& dev, const char* name) {
  check_contig(t, at::kFloat, 1, dev, name);
  return t.data_ptr<float>();
}
// [rows, width] int32, unit column stride
void check_table(const Tensor& t, int64_t rows, const c10::Device& dev, const char* name) {
  check_on(t, dev, name);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == rows && t.size(1) >= 1, name, " must be int32 [", rows, ", >= 1], got ",
              t.scalar_type(), " ", t.sizes());
  TORCH_CHECK((t.size(1) == 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)), name, " must have contiguous rows that do not overlap");
}

seg::PagedPool make_pool(const Tensor& k, const Tensor& v, int64_t Hkv, int64_t hd, const c10::Device& dev) {
  check_rows16(k, dev, "k_pages");
  check_rows16(v, dev, "v_pages");
  TORCH_CHECK(k.dim() == 4 && k.size(2) == Hkv && k.size(3) == hd, "k_pages must be [pages, page size, ", Hkv, ", ", hd, "], got ", k.sizes());
  TORCH_CHECK(v.sizes() == k.sizes(), "v_pages must have k_pages' shape ", k.sizes(), ", got ", v.sizes());
  TORCH_CHECK(k.size(0) >= 1 && k.size(0) <= INT32_MAX, "the pool must have between 1 and 2^31 - 1 pages");
  TORCH_CHECK(k.size(1) >= 1 && k.size(1) <= 65536, "the page size must be between 1 and 65536 tokens");
  for (const Tensor* t : {&k, &v})
    for (int i = 0; i < 3; ++i) TORCH_CHECK(t->size(i) == 1 || t->stride(i) >= hd, "the pool's pages, tokens and heads must not overlap");
  seg::PagedPool p;
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.k_page = k.stride(0); p.k_slot = k.stride(1); p.k_head = k.stride(2);
  p.v_page = v.stride(0); p.v_slot = v.stride(1); p.v_head = v.stride(2);
  p.n_pages = (int)k.size(0);
  p.P = (int)k.size(1);
  p.shift = -1;
  for (int s = 0; s < 17; ++s)
    if (p.P == 1 << s) p.shift = s;
  return p;
}

void check_heads(int64_t H, int64_t Hkv, int64_t hd) {
  TORCH_CHECK(Hkv >= 1 && H >= 1 && H % Hkv == 0, "query heads (", H, ") must be a multiple of key/value heads (", Hkv, ")");
  TORCH_CHECK(H <= 65535, "at most 65535 query heads");
  TORCH_CHECK(hd == 32 || hd == 64 || hd == 128, "head_dim must be 32, 64 or 128, got ", hd);
}

std::tuple<Tensor, OptTensor, OptTensor> paged_append(const Tensor& qkv, const OptTensor& v1, const Tensor& cos, const Tensor& sin, const Tensor& qgain,
                                                      const Tensor& a1, const Tensor& a2, const Tensor& vs, int64_t H, int64_t Hkv, int64_t hd, bool qknorm,
                                                      const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lens,
                                                      const OptTensor& cu, const OptTensor& pos_base, bool want_k, bool want_v) {
  TORCH_CHECK(qkv.is_cuda(), "qkv must be a CUDA tensor");
  const auto dev = qkv.device();
  check_heads(H, Hkv, hd);
  TORCH_CHECK(qkv.dim() == 2 && qkv.size(1) == (H + 2 * Hkv) * hd, "qkv must be [tokens, (H + 2 Hkv) * hd = ", (H + 2 * Hkv) * hd, "], got ", qkv.sizes());
  check_rows16(qkv, dev, "qkv");
  const int64_t T = qkv.size(0);
  TORCH_CHECK(T < (int64_t)1 << 30, "too many tokens");
  seg::PagedAppendParams p;
  p.pool = make_pool(k_pages, v_pages, Hkv, hd, dev);
  const int64_t B = lens.numel();
  check_contig(lens, at::kInt, B, dev, "seq_lens");
  TORCH_CHECK(lens.dim() == 1, "seq_lens must have one dimension");
  check_table(table, B, dev, "page_table");
  if (cu.has_value()) {
    check_contig(*cu, at::kInt, B + 1, dev, "cu_seqlens");
  } else {
    TORCH_CHECK(B == T, "without cu_seqlens every sequence brings one token: ", T, " tokens for ", B, " sequences");
  }
  if (pos_base.has_value()) check_contig(*pos_base, at::kInt, B, dev, "pos_base");
  TORCH_CHECK(cos.dim() == 2 && cos.size(1) == hd / 2, "cos must be [positions, ", hd / 2, "], got ", cos.sizes());
  check_contig(cos, at::kFloat, cos.numel(), dev, "cos");
  check_contig(sin, at::kFloat, cos.numel(), dev, "sin");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(cos.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(sin.data_ptr()) % 16 == 0,
              "the rotation tables must start on 16-byte boundaries");
  if (v1.has_value()) {
    check_contig(*v1, at::kBFloat16, T * Hkv * hd, dev, "v1");
    check_rows16(*v1, dev, "v1");
  }
  TORCH_CHECK(table.size(1) * k_pages.size(1) < (int64_t)1 << 30, "page tables may hold at most 2^30 tokens per sequence");
  c10::cuda::CUDAGuard guard(dev);
  p.qkv = qkv.data_ptr();
  p.qkv_stride = qkv.stride(0);
  p.v1 = v1.has_value() ? v1->data_ptr() : nullptr;
  p.cos = cos.data_ptr<float>();
  p.sin = sin.data_ptr<float>();
  p.qgain = scalar_ptr(qgain, dev, "qgain");
  p.alpha1 = scalar_ptr(a1, dev, "alpha1");
  p.alpha2 = scalar_ptr(a2, dev, "alpha2");
  p.vscale = scalar_ptr(vs, dev, "vscale");
  p.table = table.data_ptr<int>();
  p.table_stride = table.stride(0);
  p.table_width = (int)table.size(1);
  p.lens = lens.data_ptr<int>();
  p.cu = cu.has_value() ? cu->data_ptr<int>() : nullptr;
  p.pos_base = pos_base.has_value() ? pos_base->data_ptr<int>() : nullptr;
  p.status = status_word(dev);
  p.T = (int)T; p.B = (int)B; p.H = (int)H; p.Hkv = (int)Hkv; p.hd = (int)hd;
  p.rope_rows = (int)cos.size(0);
  p.qknorm = qknorm;
  Tensor q = new_tensor({T, H, hd}, at::kBFloat16, dev);
  OptTensor k, v;
  if (want_k) k = new_tensor({T, Hkv, hd}, at::kBFloat16, dev);
  if (want_v) v = new_tensor({T, Hkv, hd}, at::kBFloat16, dev);
  p.q = q.data_ptr();
  p.k_out = want_k ? k->data_ptr() : nullptr;
  p.v_out = want_v ? v->data_ptr() : nullptr;
  if (B == 0) {  // no sequence: every row lies behind the last one
    q.zero_();
    if (want_k) k->zero_();
    if (want_v) v->zero_();
    return {q, k, v};
  }
  const int rc = seg::paged_append(p, cur_stream());
  TORCH_CHECK(rc == 0, "paged_append failed with code ", rc);
  return {q, k, v};
}

std::tuple<Tensor, Tensor> paged_attention(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lens,
                                           const OptTensor& ptable, const OptTensor& plens, const OptTensor& groups, std::optional<double> scale) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  const auto dev = q.device();
  TORCH_CHECK(q.dim() == 3 && k_pages.dim() == 4, "q must be [B, H, hd] and the pools [pages, page size, Hkv, hd], got ", q.sizes(), " and ", k_pages.sizes());
  const int64_t B = q.size(0), H = q.size(1), hd = q.size(2), Hkv = k_pages.size(2);
  check_heads(H, Hkv, hd);
  check_rows16(q, dev, "q");
  seg::PagedAttnParams p;
  p.pool = make_pool(k_pages, v_pages, Hkv, hd, dev);
  check_contig(lens, at::kInt, B, dev, "seq_lens");
  check_table(table, B, dev, "page_table");
  TORCH_CHECK(ptable.has_value() == plens.has_value(), "prefix_table and prefix_lens come together");
  int64_t G = 0;
  if (ptable.has_value()) {
    G = plens->numel();
    check_contig(*plens, at::kInt, G, dev, "prefix_lens");
    check_table(*ptable, G, dev, "prefix_table");
    if (groups.has_value()) check_contig(*groups, at::kInt, G + 1, dev, "group_rows");
    else TORCH_CHECK(G == 1, "without group_rows there is one prefix for all rows, got ", G);
  } else {
    TORCH_CHECK(!groups.has_value(), "group_rows needs prefix_table and prefix_lens");
  }
  const double sc = scale.has_value() ? *scale : 1.0 / std::sqrt((double)hd);
  const float scale_log2 = (float)(sc * 1.4426950408889634);
  TORCH_CHECK(std::isfinite(scale_log2), "scale must be finite (in 32 bits), got ", sc);
  c10::cuda::CUDAGuard guard(dev);
  p.q = q.data_ptr();
  p.q_row = q.stride(0);
  p.q_head = q.stride(1);
  p.table = table.data_ptr<int>();
  p.table_stride = table.stride(0);
  p.table_width = (int)table.size(1);
  p.lens = lens.data_ptr<int>();
  p.ptable = G > 0 ? ptable->data_ptr<int>() : nullptr;
  p.ptable_stride = G > 0 ? ptable->stride(0) : 0;
  p.ptable_width = G > 0 ? (int)ptable->size(1) : 0;
  p.plens = G > 0 ? plens->data_ptr<int>() : nullptr;
  p.groups = groups.has_value() ? groups->data_ptr<int>() : nullptr;
  p.B = (int)B; p.H = (int)H; p.Hkv = (int)Hkv; p.hd = (int)hd; p.G = (int)G;
  p.scale_log2 = scale_log2;
  p.status = status_word(dev);
  // positions and tile numbers are 32-bit inside the kernels
  const int64_t longest = std::max<int64_t>(p.table_width, p.ptable_width) * p.pool.P;
  TORCH_CHECK(longest < (int64_t)1 << 30, "page tables may hold at most 2^30 tokens per sequence");
  TORCH_CHECK((longest / 32 + 2) * (B + G) * H < (int64_t)1 << 31, "batch x heads x page-table width is too large for one call");
  Tensor o = new_tensor({B, H, hd}, at::kBFloat16, dev);
  Tensor lse = new_tensor({B, H}, at::kFloat, dev);
  p.o = o.data_ptr();
  p.lse = lse.data_ptr<float>();
  const int64_t bytes = seg::paged_attn_workspace(p);
  TORCH_CHECK(bytes >= 0, "at most 8192 sequences and groups in one call, got ", B + G);
  Tensor ws = new_tensor({bytes}, at::kByte, dev);
  const int rc = seg::paged_attn(p, ws.data_ptr(), cur_stream());
  TORCH_CHECK(rc == 0, "paged_attention failed with code ", rc);
  return {o, lse};
}

const float* row_values(const OptTensor& t, int64_t B, const c10::Device& dev, const char* name) {
  if (!t.has_value()) return nullptr;
  check_contig(*t, at::kFloat, B, dev, name);
  return t->data_ptr<float>();
}

Tensor process_logits(const Tensor& logits, const OptTensor& tokens, const OptTensor& prompt_lens, const OptTensor& token_lens, const OptTensor& repetition,
                      const OptTensor& presence, const OptTensor& frequency, const OptTensor& bias_ids, const OptTensor& bias, const OptTensor& mask,
                      const OptTensor& mask_rows, const OptTensor& out) {
  TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
  const auto dev = logits.device();
  TORCH_CHECK(logits.dim() == 2 && (logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16),
              "logits must be float32 or bfloat16 [B, V], got ", logits.scalar_type(), " ", logits.sizes());
  const int64_t B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(B <= 65535 && V < (int64_t)1 << 30, "at most 65535 rows and 2^30 columns");
  TORCH_CHECK(V <= 1 || logits.stride(1) == 1, "logits must have unit column stride");
  seg::LogitsParams p{};
  p.B = (int)B;
  p.V = (int)V;
  p.bf16 = logits.scalar_type() == at::kBFloat16;
  TORCH_CHECK(tokens.has_value() == token_lens.has_value(), "tokens and token_lens come together");
  if (tokens.has_value()) {
    check_on(*tokens, dev, "tokens");
    TORCH_CHECK((tokens->scalar_type() == at::kInt || tokens->scalar_type() == at::kLong) && tokens->dim() == 2 && tokens->size(0) == B &&
                    tokens->size(1) < (int64_t)1 << 30,
                "tokens must be int32 or int64 [", B, ", L], got ", tokens->scalar_type(), " ", tokens->sizes());
    TORCH_CHECK(tokens->size(1) <= 1 || tokens->stride(1) == 1, "tokens must have unit column stride");
    check_contig(*token_lens, at::kInt, B, dev, "token_lens");
    p.tokens = tokens->data_ptr();
    p.tokens64 = tokens->scalar_type() == at::kLong;
    p.tokens_row = tokens->stride(0);
    p.tokens_width = (int)tokens->size(1);
    p.token_lens = token_lens->data_ptr<int>();
    if (prompt_lens.has_value()) {
      check_contig(*prompt_lens, at::kInt, B, dev, "prompt_lens");
      p.prompt_lens = prompt_lens->data_ptr<int>();
    }
  } else {
    TORCH_CHECK(!prompt_lens.has_value() && !repetition.has_value() && !presence.has_value() && !frequency.has_value(),
                "penalties need tokens and token_lens");
  }
  p.repetition = row_values(repetition, B, dev, "repetition");
  p.presence = row_values(presence, B, dev, "presence");
  p.frequency = row_values(frequency, B, dev, "frequency");
  TORCH_CHECK(bias_ids.has_value() == bias.has_value(), "bias_ids and bias_values come together");
  if (bias_ids.has_value()) {
    TORCH_CHECK(bias_ids->dim() == 2 && bias_ids->size(0) == B, "bias_ids must be [", B, ", K], got ", bias_ids->sizes());
    p.K = (int)bias_ids->size(1);
    check_contig(*bias_ids, at::kInt, B * p.K, dev, "bias_ids");
    check_contig(*bias, at::kFloat, B * p.K, dev, "bias_values");
    p.bias_ids = bias_ids->data_ptr<int>();
    p.bias = bias->data_ptr<float>();
  }
  TORCH_CHECK(mask.has_value() == mask_rows.has_value(), "mask and mask_rows come together");
  if (mask.has_value()) {
    check_on(*mask, dev, "mask");
    TORCH_CHECK(mask->scalar_type() == at::kInt && mask->dim() == 2 && mask->size(1) == (V + 31) / 32 && (mask->size(1) <= 1 || mask->stride(1) == 1),
                "mask must be int32 [rows, ", (V + 31) / 32, "] with unit column stride, got ", mask->scalar_type(), " ", mask->sizes());
    check_contig(*mask_rows, at::kInt, B, dev, "mask_rows");
    p.mask = mask->data_ptr<int>();
    p.mask_row = mask->stride(0);
    p.n_masks = (int)mask->size(0);
    p.mask_rows = mask_rows->data_ptr<int>();
  }
  c10::cuda::CUDAGuard guard(dev);
  Tensor y;
  if (out.has_value()) {
    y = *out;
    check_on(y, dev, "out");
    TORCH_CHECK(y.scalar_type() == logits.scalar_type() && y.sizes() == logits.sizes(), "out must have the logits' type and shape");
    TORCH_CHECK((V <= 1 || y.stride(1) == 1) && (B <= 1 || y.stride(0) >= V), "out must have unit column stride and rows that do not overlap");
    const bool same = y.data_ptr() == logits.data_ptr() && (B <= 1 || y.stride(0) == logits.stride(0));
    if (!same && logits.numel() > 0) {
      const auto lo = [](const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); };
      const auto hi = [&](const Tensor& t) { return lo(t) + ((B - 1) * t.stride(0) + V) * t.element_size(); };
      TORCH_CHECK(hi(y) <= lo(logits) || hi(logits) <= lo(y), "out must be the logits themselves or memory of its own");
    }
  } else {
    y = new_tensor({B, V}, logits.scalar_type(), dev);
  }
  p.x = logits.data_ptr();
  p.x_row = logits.stride(0);
  p.y = y.data_ptr();
  p.y_row = y.stride(0);
  p.status = status_word(dev);
  const int rc = seg::process_logits(p, cur_stream());
  TORCH_CHECK(rc == 0, "process_logits failed with code ", rc);
  return y;
}

}  // namespace

void register_paged(pybind11::module_& m) {
  m.def("paged_append", &paged_append);
  m.def("paged_attention", &paged_attention);
  m.def("process_logits", &process_logits);
}
