// The operators around the decode path on the host side: torch::Tensor arguments checked, unpacked and handed to the C ABI
// on the current HIP stream of the tensors' device.  Registered with the dispatcher as torch.ops.xllm_ops.*; the Python
// functions of the same names call the same code through step_ops_python.cpp.  The checks cost a microsecond here and five
// in Python.  A violated precondition is a ValueError or a TypeError; what the library itself refuses -- rows off the 16-byte
// boundary, sizes that it has no kernel for -- is a RuntimeError with its words.
#include <ATen/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include "../../../include/xllm_mi355.h"
#include "ops_api.h"

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

int code_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case torch::kBFloat16: return XLLM_MI355_BF16;
    case torch::kFloat16: return XLLM_MI355_FP16;
    case torch::kFloat32: return XLLM_MI355_FP32;
    default: TORCH_CHECK_TYPE(false, name, ": dtype ", t.scalar_type(), " is not supported"); return -1;
  }
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// The library refuses operands that overlap; `overlap` says so in the words of the call, whose other arguments were found
// good before.
void check_rc(int rc, const char* what, const char* overlap) {
  TORCH_CHECK_VALUE(rc != XLLM_MI355_EINVAL, overlap);
  TORCH_CHECK(rc == 0, what, " failed with code ", rc, ": ", xllm_mi355_error_string(rc));
}

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

// These calls record no graph.  Where one would be recorded, an operand that requires grad is refused, as by the out= forms of
// torch's own functions: its gradient would be lost without a word.
void check_no_graph(const char* what, std::initializer_list<const Tensor*> operands) {
  if (!c10::GradMode::is_enabled()) return;
  for (const Tensor* t : operands)
    TORCH_CHECK_VALUE(!t->defined() || !t->requires_grad(), what, " records no graph, but one of its operands requires grad: call "
                      "it under torch.no_grad(), or in the forward of a torch.autograd.Function");
}

// Autograd keeps what its backward passes read by version: a tensor written here counts as written in place, so that a backward
// pass over its former values fails instead of using the new ones.  (Tensors made in inference mode have no version.)
void mark_written(std::initializer_list<const Tensor*> results) {
  for (const Tensor* t : results)
    if (t->defined() && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

void check_device(const Tensor& first, std::initializer_list<const Tensor*> rest) {
  TORCH_CHECK_VALUE(first.is_cuda(), "this path runs on the GPU only: every tensor must be a device tensor");
  for (const Tensor* t : rest) {
    if (!t->defined()) continue;
    TORCH_CHECK_VALUE(t->is_cuda(), "this path runs on the GPU only: every tensor must be a device tensor");
    TORCH_CHECK_VALUE(t->device() == first.device(), "all tensors must live on the same device");
  }
}

void check_vector(const Tensor& t, torch::ScalarType type, int64_t n, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 1 && t.scalar_type() == type && t.is_contiguous() && (n < 0 || t.numel() == n), name,
              " must be a contiguous vector of ", type, n < 0 ? std::string() : " [" + std::to_string(n) + "]");
}

void check_table(const Tensor& t, int64_t rows, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.scalar_type() == torch::kInt32 && t.size(0) == rows && t.size(1) > 0 && t.stride(1) == 1 &&
                  (rows <= 1 || t.stride(0) >= t.size(1)),
              name, " must be int32 [", rows, ", W] with unit column stride");
}

// (a stride means nothing where there is one row only)
int64_t stride_or(const Tensor& t, int64_t dim, int64_t single) { return t.size(dim) > 1 ? t.stride(dim) : single; }

struct Heads {   // a [T, H, D] operand and where its result goes
  int64_t T, H, D;
  int64_t in[2], out[2];
};
Heads heads_of(const Tensor& x, const Tensor& out, const char* name) {
  TORCH_CHECK_VALUE(x.dim() == 3 && x.size(1) > 0 && x.size(2) > 0 && (x.size(0) == 0 || x.stride(2) == 1), name,
              " must be [tokens, heads, head_dim], contiguous in its last dim");
  TORCH_CHECK_VALUE(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type() && (x.size(0) == 0 || out.stride(2) == 1),
              "the result of ", name, " must have its shape and dtype, contiguous in its last dim");
  return Heads{x.size(0), x.size(1), x.size(2), {stride_or(x, 0, 0), stride_or(x, 1, 0)}, {stride_or(out, 0, 0), stride_or(out, 1, 0)}};
}

void check_rows(const Tensor& cos_sin, const Tensor& position_ids, int64_t tokens) {
  TORCH_CHECK_VALUE(position_ids.scalar_type() == torch::kInt64 && position_ids.is_contiguous() && position_ids.numel() == tokens,
              "position_ids must be contiguous int64 [tokens]");
  TORCH_CHECK_VALUE(cos_sin.dim() == 2 && cos_sin.is_contiguous() && cos_sin.size(0) > 0,
              "cos_sin_cache must be [max_position, rotary_dim], contiguous");
}

}  // namespace

namespace xllm::kernel::mi355 {

void build_step_tables(const Tensor& kv_lens, const Tensor& new_lens, const Tensor& block_table, const Tensor& free_pages,
                       int64_t block_size, int64_t max_new_tokens, const OptTensor& free_head, StepTables& out) {
  const int64_t B = kv_lens.numel(), T = max_new_tokens;
  check_device(kv_lens, {&new_lens, &block_table, &free_pages, &out.block_table, &out.seq_lens, &out.q_cu_seq_lens,
                         &out.position_ids, &out.slot_mapping, &out.new_page_indptr, &out.counters});
  if (given(free_head)) {
    check_device(kv_lens, {&*free_head});
    TORCH_CHECK_VALUE(free_head->scalar_type() == torch::kInt32 && free_head->numel() == 1, "free_head must be int32 [1]");
  }
  check_vector(kv_lens, torch::kInt32, -1, "kv_lens");
  check_vector(new_lens, torch::kInt32, B, "new_lens");
  check_vector(free_pages, torch::kInt32, -1, "free_pages");
  check_table(block_table, B, "block_table");
  TORCH_CHECK_VALUE(block_size > 0 && T >= 0, "block_size must be positive and max_new_tokens not negative");
  const c10::DeviceGuard guard(kv_lens.device());
  auto make = [&](Tensor& t, int64_t n, torch::ScalarType type, const char* name) {
    if (t.defined()) check_vector(t, type, n, name);
    else t = torch::empty({n}, kv_lens.options().dtype(type));
  };
  if (out.block_table.defined()) {
    check_table(out.block_table, B, "out.block_table");
    TORCH_CHECK_VALUE(out.block_table.size(1) == block_table.size(1), "out.block_table must have block_table's width");
  } else {
    out.block_table = torch::empty({B, block_table.size(1)}, block_table.options());
  }
  make(out.seq_lens, B, torch::kInt32, "out.seq_lens");
  make(out.q_cu_seq_lens, B + 1, torch::kInt32, "out.q_cu_seq_lens");
  make(out.position_ids, T, torch::kInt64, "out.position_ids");
  make(out.slot_mapping, T, torch::kInt32, "out.slot_mapping");
  make(out.new_page_indptr, B + 1, torch::kInt32, "out.new_page_indptr");
  make(out.counters, 3, torch::kInt32, "out.counters");
  constexpr const char* kOverlap = "an output of build_step_tables overlaps an input or another output (in place means "
                                   "block_table itself)";
  if (B == 0) {   // no requests: offsets and counters of an empty step
    if (given(free_head))
      for (const Tensor* t : {&out.q_cu_seq_lens, &out.new_page_indptr, &out.counters, &out.position_ids, &out.slot_mapping}) {
        const char *lo = static_cast<const char*>(t->data_ptr()), *head = static_cast<const char*>(free_head->data_ptr());
        TORCH_CHECK_VALUE(head < lo || head >= lo + t->nbytes(), kOverlap);
      }
    for (const Tensor* t : {&out.q_cu_seq_lens, &out.new_page_indptr, &out.counters, &out.position_ids}) t->zero_();
    out.slot_mapping.fill_(-1);
    if (given(free_head)) out.counters.slice(0, 1, 2).copy_(free_head->view({1}).clamp(0, free_pages.numel()));
    return;
  }
  const int64_t W = block_table.size(1);
  check_rc(xllm_mi355_build_step_tables(
               kv_lens.data_ptr<int32_t>(), new_lens.data_ptr<int32_t>(), block_table.data_ptr<int32_t>(),
               stride_or(block_table, 0, W), out.block_table.data_ptr<int32_t>(), stride_or(out.block_table, 0, W), W,
               free_pages.data_ptr<int32_t>(), free_pages.numel(), given(free_head) ? free_head->data_ptr<int32_t>() : nullptr,
               out.seq_lens.data_ptr<int32_t>(), out.q_cu_seq_lens.data_ptr<int32_t>(), out.position_ids.data_ptr<int64_t>(),
               out.slot_mapping.data_ptr<int32_t>(), out.new_page_indptr.data_ptr<int32_t>(), out.counters.data_ptr<int32_t>(),
               B, block_size, T, stream_of(kv_lens)),
           "xllm_mi355_build_step_tables", kOverlap);
  mark_written({&out.block_table, &out.seq_lens, &out.q_cu_seq_lens, &out.position_ids, &out.slot_mapping, &out.new_page_indptr,
                &out.counters});
}

StepTables step_tables_memory(const Tensor& kv_lens, int64_t max_new_tokens) {
  StepTables t;
  const int64_t B = kv_lens.numel();
  if (max_new_tokens < 0) return t;   // (refused by the call)
  const std::vector<Tensor> part = torch::empty({3 * B + 5 + max_new_tokens}, kv_lens.options().dtype(torch::kInt32))
                                       .unsafe_split_with_sizes({B, B + 1, B + 1, 3, max_new_tokens});
  t.seq_lens = part[0];
  t.q_cu_seq_lens = part[1];
  t.new_page_indptr = part[2];
  t.counters = part[3];
  t.slot_mapping = part[4];
  return t;
}

Tensor build_cos_sin_cache(const Tensor& inv_freq, const OptTensor& position_ids, int64_t num_positions,
                           int64_t first_position, double attention_factor, torch::ScalarType dtype, const OptTensor& out_rows) {
  const Tensor none;
  check_no_graph("build_cos_sin_cache", {&inv_freq, given(out_rows) ? &*out_rows : &none});
  check_device(inv_freq, {});
  check_vector(inv_freq, torch::kFloat64, -1, "inv_freq");
  TORCH_CHECK_VALUE(inv_freq.numel() > 0, "inv_freq is empty");
  int64_t rows = num_positions;
  if (given(position_ids)) {
    check_device(inv_freq, {&*position_ids});
    check_vector(*position_ids, torch::kInt64, -1, "position_ids");
    rows = position_ids->numel();
    TORCH_CHECK_VALUE(first_position == 0 && (num_positions == 0 || num_positions == rows),
                "give position_ids or a range of positions, not both");
  } else {
    TORCH_CHECK_VALUE(rows > 0 && first_position >= 0, "num_positions must be positive and first_position not negative");
  }
  const c10::DeviceGuard guard(inv_freq.device());
  Tensor out;
  if (given(out_rows)) {
    out = *out_rows;
    check_device(inv_freq, {&out});
    TORCH_CHECK_VALUE(out.dim() == 2 && out.size(0) == rows && out.size(1) == 2 * inv_freq.numel() && out.is_contiguous(),
                      "out must be contiguous [rows, rotary_dim]");
  } else {
    out = torch::empty({rows, 2 * inv_freq.numel()}, inv_freq.options().dtype(dtype));
  }
  check_rc(xllm_mi355_rope_cos_sin(inv_freq.data_ptr<double>(), given(position_ids) ? position_ids->data_ptr<int64_t>() : nullptr,
                                   first_position, rows, inv_freq.numel(), attention_factor, out.data_ptr(),
                                   code_of(out, "cos_sin rows"), stream_of(out)),
           "xllm_mi355_rope_cos_sin", "out overlaps an input");
  mark_written({&out});
  return out;
}

void rotary_embedding(const Tensor& position_ids, const Tensor& query, const OptTensor& key, const Tensor& cos_sin_cache,
                      bool interleave, int64_t rotary_offset, std::optional<int64_t> key_rotary_offset, bool inverse,
                      const OptTensor& out_query, const OptTensor& out_key) {
  const Tensor oq = given(out_query) ? *out_query : query;
  const Tensor k = given(key) ? *key : Tensor();
  const Tensor ok = given(out_key) ? *out_key : k;
  TORCH_CHECK_VALUE(k.defined() || !ok.defined(), "out_key without a key");
  check_no_graph("rotary_embedding", {&query, &k, &cos_sin_cache, &oq, &ok});
  check_device(query, {&position_ids, &cos_sin_cache, &oq, &k, &ok});
  const Heads hq = heads_of(query, oq, "query");
  check_rows(cos_sin_cache, position_ids, hq.T);
  Heads hk = {hq.T, 0, 0, {0, 0}, {0, 0}};
  if (k.defined()) {
    hk = heads_of(k, ok, "key");
    TORCH_CHECK_VALUE(hk.T == hq.T && k.scalar_type() == query.scalar_type(), "key must have query's tokens and dtype");
  }
  const int64_t R = cos_sin_cache.size(1), k_off = key_rotary_offset.value_or(rotary_offset);
  TORCH_CHECK_VALUE(R > 0 && R % 2 == 0, "the rotary dim must be even");
  TORCH_CHECK_VALUE(rotary_offset >= 0 && rotary_offset + R <= hq.D && (!k.defined() || (k_off >= 0 && k_off + R <= hk.D)),
                    "the rotated part must lie inside the head");
  const c10::DeviceGuard guard(query.device());
  check_rc(xllm_mi355_rotary_embedding(
               position_ids.data_ptr<int64_t>(), cos_sin_cache.data_ptr(), cos_sin_cache.size(0), query.data_ptr(),
               oq.data_ptr(), k.defined() ? k.data_ptr() : nullptr, ok.defined() ? ok.data_ptr() : nullptr, hq.T, hq.H, hk.H,
               hq.D, hk.D, rotary_offset, k.defined() ? k_off : 0, R,
               hq.in, hq.out, hk.in, hk.out, interleave ? 1 : 0, inverse ? 1 : 0, code_of(query, "query"),
               code_of(cos_sin_cache, "cos_sin_cache"), stream_of(query)),
           "xllm_mi355_rotary_embedding",
           "a result of rotary_embedding overlaps itself, the other one or an input (in place means the operand itself)");
  mark_written({&oq, &ok});
}

void mla_norm_rope_and_cache(const Tensor& q_pe, const Tensor& kv, const Tensor& kv_norm_weight, double eps,
                             const Tensor& cos_sin_cache, bool interleave, const Tensor& position_ids,
                             const OptTensor& k_cache, const OptTensor& slot_mapping, const OptTensor& out_q_pe,
                             const OptTensor& out_kv) {
  const Tensor oq = given(out_q_pe) ? *out_q_pe : q_pe;
  const Tensor cache = given(k_cache) ? *k_cache : Tensor(), slots = given(slot_mapping) ? *slot_mapping : Tensor();
  const Tensor okv = given(out_kv) ? *out_kv : Tensor();
  check_no_graph("mla_norm_rope_and_cache", {&q_pe, &kv, &kv_norm_weight, &cos_sin_cache, &cache, &oq, &okv});
  check_device(q_pe, {&kv, &kv_norm_weight, &cos_sin_cache, &position_ids, &cache, &slots, &oq, &okv});
  TORCH_CHECK_TYPE(q_pe.scalar_type() == torch::kBFloat16 || q_pe.scalar_type() == torch::kFloat16, "q_pe must be bfloat16 or float16");
  const Heads h = heads_of(q_pe, oq, "q_pe");
  const int64_t latent = kv_norm_weight.numel(), row = latent + h.D;
  auto rows_of = [&](const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == h.T && t.size(1) == row && (h.T == 0 || t.stride(1) == 1) &&
                    t.scalar_type() == q_pe.scalar_type() && (h.T <= 1 || t.stride(0) >= row),
                name, " must be [tokens, latent + rope dims] of q_pe's dtype with contiguous rows apart from each other");
    return stride_or(t, 0, row);
  };
  const int64_t kv_row = rows_of(kv, "kv"), out_row = okv.defined() ? rows_of(okv, "out_kv") : 0;
  TORCH_CHECK_VALUE(kv_norm_weight.scalar_type() == q_pe.scalar_type() && kv_norm_weight.is_contiguous(),
              "kv_norm_weight must be contiguous, of q_pe's dtype");
  check_rows(cos_sin_cache, position_ids, h.T);
  TORCH_CHECK_VALUE(cos_sin_cache.size(1) == h.D, "cos_sin_cache must have the rope dims");
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative");
  TORCH_CHECK_VALUE(cache.defined() == slots.defined(), "k_cache and slot_mapping come together");
  TORCH_CHECK_VALUE(cache.defined() || okv.defined(), "the latent rows need a place: k_cache or out_kv");
  if (cache.defined()) {
    TORCH_CHECK_VALUE(cache.dim() == 4 && cache.size(2) == 1 && cache.size(3) == row && cache.is_contiguous() &&
                    cache.scalar_type() == q_pe.scalar_type(),
                "k_cache must be contiguous [P, bs, 1, latent + rope dims] of q_pe's dtype");
    TORCH_CHECK_VALUE(cache.numel() > 0, "k_cache is empty");
    check_vector(slots, torch::kInt32, h.T, "slot_mapping");
  }
  const c10::DeviceGuard guard(q_pe.device());
  check_rc(xllm_mi355_mla_norm_rope_and_cache(
               q_pe.data_ptr(), oq.data_ptr(), kv.data_ptr(), okv.defined() ? okv.data_ptr() : nullptr,
               kv_norm_weight.data_ptr(), static_cast<float>(eps), cos_sin_cache.data_ptr(), cos_sin_cache.size(0),
               position_ids.data_ptr<int64_t>(), cache.defined() ? cache.data_ptr() : nullptr,
               slots.defined() ? slots.data_ptr<int32_t>() : nullptr, h.T, h.H, latent, h.D, h.in[0], h.in[1], h.out[0],
               h.out[1], kv_row, out_row, cache.defined() ? cache.size(1) : 0, cache.defined() ? cache.size(0) : 0,
               interleave ? 1 : 0, code_of(q_pe, "q_pe"), code_of(cos_sin_cache, "cos_sin_cache"), stream_of(q_pe)),
           "xllm_mi355_mla_norm_rope_and_cache",
           "a result of mla_norm_rope_and_cache overlaps itself, another one or an input (in place means the operand itself)");
  mark_written({&oq, &okv, &cache});
}

void batch_decode_diff(const Tensor& query, const Tensor& k_cache, const Tensor& v_cache, Tensor& output,
                       const Tensor& block_table, const Tensor& seq_lens, const Tensor& lambda, double scale,
                       const OptTensor& norm_weight, double eps, double out_scale, int64_t window_left) {
  const Tensor weight = given(norm_weight) ? *norm_weight : Tensor();
  check_no_graph("batch_decode_diff", {&query, &k_cache, &v_cache, &output, &lambda, &weight});
  check_device(query, {&k_cache, &v_cache, &output, &block_table, &seq_lens, &lambda, &weight});
  TORCH_CHECK_TYPE(query.scalar_type() == torch::kBFloat16 || query.scalar_type() == torch::kFloat16,
                   "query must be bfloat16 or float16");
  TORCH_CHECK_VALUE(query.dim() == 3 && query.size(1) > 0 && query.size(1) % 2 == 0 && query.stride(2) == 1 &&
                  query.stride(1) == query.size(2),
              "query must be [B, 2 H, D] with contiguous last two dims");
  const int64_t B = query.size(0), H = query.size(1) / 2, D = query.size(2), row = 2 * H * D;
  TORCH_CHECK_VALUE(output.dim() == 3 && output.size(0) == B && output.size(1) == H && output.size(2) == 2 * D &&
                  output.scalar_type() == query.scalar_type() && output.stride(2) == 1 &&
                  (H == 1 || output.stride(1) == 2 * D) && (B <= 1 || output.stride(0) >= row),
              "output must be [B, H, 2 D] of query's dtype with contiguous last two dims");
  TORCH_CHECK_VALUE(k_cache.dim() == 4 && k_cache.is_contiguous() && k_cache.size(2) % 2 == 0 && k_cache.size(3) == D &&
                  k_cache.numel() > 0 && k_cache.scalar_type() == query.scalar_type(),
              "k_cache must be contiguous [P, bs, 2 pairs, D] of query's dtype");
  const int64_t pairs = k_cache.size(2) / 2;
  TORCH_CHECK_VALUE(v_cache.dim() == 4 && v_cache.is_contiguous() && v_cache.size(0) == k_cache.size(0) &&
                  v_cache.size(1) == k_cache.size(1) && v_cache.size(2) == pairs && v_cache.size(3) == 2 * D &&
                  v_cache.scalar_type() == query.scalar_type(),
              "v_cache must be contiguous [P, bs, pairs, 2 D] of query's dtype");
  TORCH_CHECK_VALUE(H % pairs == 0, "the heads must be a multiple of the KV pairs");
  check_table(block_table, B, "block_table");
  check_vector(seq_lens, torch::kInt32, B, "seq_lens");
  TORCH_CHECK_VALUE(lambda.scalar_type() == torch::kFloat32, "lambda must be float32");
  int64_t lb = 0, lh = 0;
  if (lambda.numel() != 1) {
    const bool both = lambda.dim() == 2 && lambda.size(0) == B && lambda.size(1) == H;
    TORCH_CHECK_VALUE(both || (lambda.dim() == 1 && lambda.size(0) == H), "lambda must hold one value, or be [H] or [B, H]");
    lb = both ? lambda.stride(0) : 0;
    lh = lambda.stride(both ? 1 : 0);
  }
  TORCH_CHECK_VALUE(!weight.defined() || (weight.scalar_type() == query.scalar_type() && weight.numel() == 2 * D && weight.is_contiguous()),
              "norm_weight must be contiguous [2 D] of query's dtype");
  TORCH_CHECK_VALUE(static_cast<float>(scale) > 0 && eps >= 0, "scale must be positive (in 32 bits) and eps not negative");
  TORCH_CHECK_VALUE(H <= 65535, "at most 65535 differential heads");
  TORCH_CHECK_VALUE(B <= 1 || query.stride(0) >= row, "query: rows must not overlap");
  if (B == 0) return;
  const c10::DeviceGuard guard(query.device());
  const size_t bytes = xllm_mi355_paged_decode_diff_workspace_bytes(H, pairs, D);
  Tensor ws = torch::empty({static_cast<int64_t>(bytes)}, query.options().dtype(torch::kUInt8));
  check_rc(xllm_mi355_paged_decode_diff(
               query.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), output.data_ptr(), block_table.data_ptr<int32_t>(),
               stride_or(block_table, 0, block_table.size(1)), block_table.size(1), seq_lens.data_ptr<int32_t>(),
               lambda.data_ptr<float>(), lb, lh, weight.defined() ? weight.data_ptr() : nullptr, static_cast<float>(eps),
               static_cast<float>(out_scale), B, H, pairs, D, k_cache.size(1), k_cache.size(0), stride_or(query, 0, row),
               stride_or(output, 0, row), window_left, static_cast<float>(scale), ws.data_ptr(), bytes, code_of(query, "query"),
               stream_of(query)),
           "xllm_mi355_paged_decode_diff", "output overlaps an input");
  mark_written({&output});
}

}  // namespace xllm::kernel::mi355

namespace {

namespace k = xllm::kernel::mi355;

using Tables = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

Tables op_build_step_tables(Tensor kv_lens, Tensor new_lens, Tensor block_table, Tensor free_pages, int64_t block_size,
                            int64_t max_new_tokens, OptTensor free_head) {
  k::StepTables t = k::step_tables_memory(kv_lens, max_new_tokens);
  k::build_step_tables(kv_lens, new_lens, block_table, free_pages, block_size, max_new_tokens, free_head, t);
  return {t.block_table, t.seq_lens, t.q_cu_seq_lens, t.position_ids, t.slot_mapping, t.new_page_indptr, t.counters};
}

void op_build_step_tables_out(Tensor kv_lens, Tensor new_lens, Tensor block_table, Tensor free_pages, int64_t block_size,
                              int64_t max_new_tokens, OptTensor free_head, Tensor out_block_table, Tensor out_seq_lens,
                              Tensor out_q_cu_seq_lens, Tensor out_position_ids, Tensor out_slot_mapping,
                              Tensor out_new_page_indptr, Tensor out_counters) {
  k::StepTables t{out_block_table, out_seq_lens, out_q_cu_seq_lens, out_position_ids, out_slot_mapping, out_new_page_indptr,
                  out_counters};
  k::build_step_tables(kv_lens, new_lens, block_table, free_pages, block_size, max_new_tokens, free_head, t);
}

Tensor op_build_cos_sin_cache(Tensor inv_freq, OptTensor position_ids, int64_t num_positions, int64_t first_position,
                              double attention_factor, torch::ScalarType dtype, OptTensor out) {
  return k::build_cos_sin_cache(inv_freq, position_ids, num_positions, first_position, attention_factor, dtype, out);
}

void op_rotary_embedding(Tensor position_ids, Tensor query, OptTensor key, Tensor cos_sin_cache, bool interleave,
                         int64_t rotary_offset, std::optional<int64_t> key_rotary_offset, bool inverse, OptTensor out_query,
                         OptTensor out_key) {
  k::rotary_embedding(position_ids, query, key, cos_sin_cache, interleave, rotary_offset, key_rotary_offset, inverse,
                      out_query, out_key);
}

void op_mla_norm_rope_and_cache(Tensor q_pe, Tensor kv, Tensor kv_norm_weight, double eps, Tensor cos_sin_cache,
                                bool interleave, Tensor position_ids, OptTensor k_cache, OptTensor slot_mapping,
                                OptTensor out_q_pe, OptTensor out_kv) {
  k::mla_norm_rope_and_cache(q_pe, kv, kv_norm_weight, eps, cos_sin_cache, interleave, position_ids, k_cache, slot_mapping,
                             out_q_pe, out_kv);
}

Tensor op_batch_decode_diff(Tensor query, Tensor k_cache, Tensor v_cache, Tensor output, Tensor block_table, Tensor seq_lens,
                            Tensor lambda, double scale, OptTensor norm_weight, double eps, double out_scale,
                            int64_t window_left) {
  k::batch_decode_diff(query, k_cache, v_cache, output, block_table, seq_lens, lambda, scale, norm_weight, eps, out_scale,
                       window_left);
  return output;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(xllm_ops, m) {
  m.def("build_step_tables(Tensor kv_lens, Tensor new_lens, Tensor block_table, Tensor free_pages, int block_size, "
        "int max_new_tokens, Tensor? free_head=None) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("build_step_tables_out(Tensor kv_lens, Tensor new_lens, Tensor block_table, Tensor free_pages, int block_size, "
        "int max_new_tokens, Tensor? free_head, Tensor(a!) out_block_table, Tensor(b!) out_seq_lens, "
        "Tensor(c!) out_q_cu_seq_lens, Tensor(d!) out_position_ids, Tensor(e!) out_slot_mapping, "
        "Tensor(f!) out_new_page_indptr, Tensor(g!) out_counters) -> ()");
  m.def("build_cos_sin_cache(Tensor inv_freq, Tensor? position_ids, int num_positions, int first_position, "
        "float attention_factor, ScalarType dtype, Tensor(a!)? out=None) -> Tensor");
  m.def("rotary_embedding(Tensor position_ids, Tensor(a!) query, Tensor(b!)? key, Tensor cos_sin_cache, "
        "bool interleave=False, int rotary_offset=0, int? key_rotary_offset=None, bool inverse=False, "
        "Tensor(c!)? out_query=None, Tensor(d!)? out_key=None) -> ()");
  m.def("mla_norm_rope_and_cache(Tensor(a!) q_pe, Tensor kv, Tensor kv_norm_weight, float eps, Tensor cos_sin_cache, "
        "bool interleave, Tensor position_ids, Tensor(b!)? k_cache=None, Tensor? slot_mapping=None, "
        "Tensor(c!)? out_q_pe=None, Tensor(d!)? out_kv=None) -> ()");
  m.def("batch_decode_diff(Tensor query, Tensor k_cache, Tensor v_cache, Tensor(a!) output, Tensor block_table, "
        "Tensor seq_lens, Tensor lambda_, float scale, Tensor? norm_weight=None, float eps=1e-5, float out_scale=1.0, "
        "int window_left=-1) -> Tensor");
}

// (for every device, so that tensors of another one meet the checks above)
TORCH_LIBRARY_IMPL(xllm_ops, CompositeExplicitAutograd, m) {
  m.impl("build_step_tables", &op_build_step_tables);
  m.impl("build_step_tables_out", &op_build_step_tables_out);
  m.impl("build_cos_sin_cache", &op_build_cos_sin_cache);
  m.impl("rotary_embedding", &op_rotary_embedding);
  m.impl("mla_norm_rope_and_cache", &op_mla_norm_rope_and_cache);
  m.impl("batch_decode_diff", &op_batch_decode_diff);
}
