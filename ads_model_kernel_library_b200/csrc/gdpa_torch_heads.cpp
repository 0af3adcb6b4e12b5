// Torch operators on either side of the attention: norm and rotation of heads (with their gradient), the same with the append to the paged cache,
// the cache read back, drafts verified and taken out of the cache.  As gdpa_torch.cpp: checks, outputs and launch in C++, fake kernels
// in Python.
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>

#include "gdpa_torch.h"

using namespace gdpa_torch;

namespace {

struct EntryPoints {
  int (*rotary)(const GdpaRotaryParams*, gdpa_stream_t);
  int (*rotary_bwd)(const GdpaRotaryParams*, gdpa_stream_t);
  size_t (*rotary_workspace)(int32_t);
  int (*append)(const GdpaRotatedAppendParams*, gdpa_stream_t);
  int (*read)(const GdpaCacheReadParams*, gdpa_stream_t);
  size_t (*verify_workspace)(int32_t, int32_t, int32_t);
  int (*verify)(const GdpaVerifyParams*, gdpa_stream_t);
  size_t (*drop_workspace)(int32_t, int32_t);
  int (*drop)(const GdpaDropParams*, gdpa_stream_t);
} g_call{};

using OptionalTensor = std::optional<at::Tensor>;

gdpa_stream_t stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// ------------------------------------------------------------------------------------------ norm and rotation

void check_heads(const char* name, const at::Tensor& t) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, name, " must be bf16 or fp32, got ", t.scalar_type());
  check_rows(name, t);
  TORCH_CHECK_VALUE(t.size(1) >= 1, name, " must have at least one head");
  TORCH_CHECK_NOT_IMPLEMENTED(t.size(2) == 64 || t.size(2) == 128, "head_dim ", t.size(2), " is not supported (supported: 64, 128)");
  TORCH_CHECK_VALUE(t.size(0) < int64_t{1} << 30, name, " has too many tokens");
}

GdpaRotarySpec rotary_spec(const at::Tensor& like, const at::Tensor& inv_freq, double eps, bool norm, bool interleaved, at::IntArrayRef sections) {
  check_device("inv_freq", inv_freq, like);
  TORCH_CHECK_TYPE(inv_freq.scalar_type() == at::kFloat || inv_freq.scalar_type() == at::kDouble, "inv_freq must be fp32 or fp64, got ",
                   inv_freq.scalar_type());
  check_vector("inv_freq", inv_freq, like, -1);
  const int64_t pairs = inv_freq.numel();
  TORCH_CHECK_VALUE(2 * pairs <= like.size(2), "inv_freq: ", 2 * pairs, " values of a head cannot be rotated, it has ", like.size(2));
  TORCH_CHECK_NOT_IMPLEMENTED(pairs % 8 == 0, "inv_freq must have a multiple of 8 entries (16 rotated values), got ", pairs);
  TORCH_CHECK_VALUE(sections.empty() || (sections.size() >= 2 && sections.size() <= 4), "sections must be those of 2 to 4 axes, got ", sections);
  TORCH_CHECK_VALUE(!norm || (eps >= 0 && eps < 3e38), "eps must be a finite number that is not negative, got ", eps);
  GdpaRotarySpec r{};
  r.inv_freq = inv_freq.const_data_ptr();
  r.inv_freq_is_fp64 = inv_freq.scalar_type() == at::kDouble;
  r.pairs = static_cast<int32_t>(pairs);
  r.interleaved = interleaved;
  r.axes = sections.empty() ? 1 : static_cast<int32_t>(sections.size());
  int64_t end = 0;
  for (size_t i = 0; i < sections.size(); ++i) {
    TORCH_CHECK_VALUE(sections[i] >= 0 && sections[i] <= pairs, "sections must be numbers of pairs, got ", sections);
    end += sections[i];
    r.section_ends[i] = static_cast<int32_t>(end);
  }
  TORCH_CHECK_VALUE(sections.empty() || end == pairs, "sections must add up to the ", pairs, " entries of inv_freq, got ", sections);
  r.norm = norm;
  r.eps = static_cast<float>(eps);
  return r;
}

// Whether they are 64 bits wide; their stride between axes.
bool check_positions(const char* name, const at::Tensor& t, const at::Tensor& like, int64_t axes, int64_t tokens, int64_t& stride) {
  check_device(name, t, like);
  const bool wide = check_int(name, t);
  const bool fits = axes == 1 ? t.dim() == 1 && t.size(0) == tokens : t.dim() == 2 && t.size(0) == axes && t.size(1) == tokens;
  TORCH_CHECK_VALUE(fits, name, " must be ", axes == 1 ? "[tokens]" : "[axes, tokens]", " with ", axes, " axes and ", tokens, " tokens, got ", t.sizes());
  TORCH_CHECK_VALUE(tokens <= 1 || t.stride(-1) == 1, name, " must be contiguous over the tokens");
  stride = axes == 1 ? 0 : t.stride(0);
  return wide;
}

bool check_weight(const char* name, const OptionalTensor& t, const at::Tensor& like) {  // whether it is bf16
  if (!t.has_value() || !t->defined()) return false;
  TORCH_CHECK_TYPE(t->scalar_type() == at::kBFloat16 || t->scalar_type() == at::kFloat, name, " must be bf16 or fp32, got ", t->scalar_type());
  check_vector(name, *t, like, like.size(2));
  return t->scalar_type() == at::kBFloat16;
}
const void* data(const OptionalTensor& t) { return t.has_value() && t->defined() ? t->const_data_ptr() : nullptr; }

GdpaRotaryTensor rotary_tensor(const char* name, const char* positions_name, const char* weight_name, const at::Tensor& x, const at::Tensor& positions,
                               const OptionalTensor& weight, const GdpaRotarySpec& r, const at::Tensor& like) {
  check_cuda(name, x);
  check_device(name, x, like);
  check_heads(name, x);
  check_type(name, x, like.scalar_type());
  TORCH_CHECK_VALUE(x.size(2) == like.size(2), "query and key must have the same head_dim");
  GdpaRotaryTensor t{};
  t.x = x.const_data_ptr();
  strides(t.x_strides, x);
  t.weight_is_bf16 = check_weight(weight_name, weight, x);
  t.weight = data(weight);
  t.heads = static_cast<int32_t>(x.size(1));
  t.tokens = x.size(0);
  t.positions_are_int64 = check_positions(positions_name, positions, x, r.axes, x.size(0), t.position_stride);
  t.positions = positions.const_data_ptr();
  return t;
}

GdpaRotaryParams rotary_params(const at::Tensor& query, const at::Tensor& key, const at::Tensor& inv_freq, const at::Tensor& query_positions,
                               const at::Tensor& key_positions, const OptionalTensor& query_weight, const OptionalTensor& key_weight, double eps, bool norm,
                               bool interleaved, at::IntArrayRef sections) {
  check_cuda("query", query);
  check_heads("query", query);
  GdpaRotaryParams p{};
  p.struct_size = sizeof(p);
  p.is_fp32 = query.scalar_type() == at::kFloat;
  p.head_dim = static_cast<int32_t>(query.size(2));
  p.rotary = rotary_spec(query, inv_freq, eps, norm, interleaved, sections);
  p.query = rotary_tensor("query", "query_positions", "query_weight", query, query_positions, query_weight, p.rotary, query);
  p.key = rotary_tensor("key", "key_positions", "key_weight", key, key_positions, key_weight, p.rotary, query);
  return p;
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rotary(const at::Tensor& query, const at::Tensor& key, const at::Tensor& inv_freq, const at::Tensor& query_positions,
                                                  const at::Tensor& key_positions, const OptionalTensor& query_weight, const OptionalTensor& key_weight,
                                                  double eps, bool norm, bool interleaved, at::IntArrayRef sections) {
  GdpaRotaryParams p = rotary_params(query, key, inv_freq, query_positions, key_positions, query_weight, key_weight, eps, norm, interleaved, sections);
  const c10::cuda::CUDAGuard guard(query.device());
  at::Tensor q = empty(query.sizes(), query.scalar_type(), query), k = empty(key.sizes(), key.scalar_type(), key);
  p.query.y = q.mutable_data_ptr();
  p.key.y = k.mutable_data_ptr();
  check(g_call.rotary(&p, stream()), "gdpa_qk_norm_rotary");
  return {q, k};
}

// A gradient of a result as the kernel can read it: expanded ones and those of other strides or addresses are copied.
at::Tensor readable_grad(const char* name, const at::Tensor& g, const at::Tensor& x) {
  check_device(name, g, x);
  check_type(name, g, x.scalar_type());
  TORCH_CHECK_VALUE(g.dim() == 3 && g.sizes() == x.sizes(), name, " must have the shape of the result, got ", g.sizes());
  bool own = !misaligned(g, 2);
  for (int i = 0; i < 2; ++i) own &= g.numel() == 0 || g.size(i) <= 1 || g.stride(i) >= g.size(2);
  return own ? g : g.contiguous();
}

// Without the norm x is not read: the gradients of the results, once they are readable, stand in for it.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rotary_backward(
    const at::Tensor& query_grad, const at::Tensor& key_grad, const at::Tensor& query, const at::Tensor& key, const at::Tensor& inv_freq,
    const at::Tensor& query_positions, const at::Tensor& key_positions, const OptionalTensor& query_weight, const OptionalTensor& key_weight, double eps, bool norm,
    bool interleaved, at::IntArrayRef sections, bool weight_grads) {
  check_cuda("query", query);
  check_device("key", key, query);
  const c10::cuda::CUDAGuard guard(query.device());
  const at::Tensor gq = readable_grad("query_grad", query_grad, query), gk = readable_grad("key_grad", key_grad, key);
  GdpaRotaryParams p = rotary_params(norm ? query : gq, norm ? key : gk, inv_freq, query_positions, key_positions, query_weight, key_weight, eps, norm,
                                     interleaved, sections);
  auto take = [](const at::Tensor& g, GdpaRotaryTensor& t) {
    t.dy = g.const_data_ptr();
    strides(t.dy_strides, g);
  };
  take(gq, p.query);
  take(gk, p.key);
  at::Tensor dq = empty(query.sizes(), query.scalar_type(), query), dk = empty(key.sizes(), key.scalar_type(), key), workspace;
  p.query.y = dq.mutable_data_ptr();
  p.key.y = dk.mutable_data_ptr();
  auto weight_grad = [&](const OptionalTensor& w, GdpaRotaryTensor& t) {
    const bool wanted = weight_grads && norm && w.has_value() && w->defined();
    at::Tensor d = empty({wanted ? w->numel() : 0}, wanted ? w->scalar_type() : at::kFloat, query);
    if (wanted) t.dweight = d.mutable_data_ptr();
    return d;
  };
  at::Tensor dqw = weight_grad(query_weight, p.query), dkw = weight_grad(key_weight, p.key);
  if (p.query.dweight != nullptr || p.key.dweight != nullptr) {
    const size_t bytes = g_call.rotary_workspace(p.head_dim);
    workspace = empty({static_cast<int64_t>(bytes)}, at::kByte, query);
    p.workspace = workspace.mutable_data_ptr();
    p.workspace_bytes = static_cast<int64_t>(bytes);
  }
  check(g_call.rotary_bwd(&p, stream()), "gdpa_qk_norm_rotary_bwd");
  return {dq, dk, dqw, dkw};
}

bool wants(const OptionalTensor& t) { return t.has_value() && t->defined() && t->requires_grad(); }
bool has_tangent(const OptionalTensor& t) { return t.has_value() && t->defined() && t->_fw_grad(/*level=*/0).defined(); }

class QkNormRotary : public torch::autograd::Function<QkNormRotary> {
 public:
  static auto op() {
    static const auto handle = c10::Dispatcher::singleton().findSchemaOrThrow("gdpa::qk_norm_rotary", "").typed<decltype(qk_norm_rotary)>();
    return handle;
  }
  static auto backward_op() {
    static const auto handle =
        c10::Dispatcher::singleton().findSchemaOrThrow("gdpa::qk_norm_rotary_backward", "").typed<decltype(qk_norm_rotary_backward)>();
    return handle;
  }
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& query, const at::Tensor& key,
                                                const at::Tensor& inv_freq, const at::Tensor& query_positions, const at::Tensor& key_positions,
                                                const OptionalTensor& query_weight, const OptionalTensor& key_weight, double eps, bool norm,
                                                bool interleaved, std::vector<int64_t> sections) {
    const at::AutoDispatchBelowADInplaceOrView below;
    auto [q, k] = op().call(query, key, inv_freq, query_positions, key_positions, query_weight, key_weight, eps, norm, interleaved, sections);
    ctx->save_for_backward({norm ? query : at::Tensor(), norm ? key : at::Tensor(), inv_freq, query_positions, key_positions, query_weight.value_or(at::Tensor()),
                            key_weight.value_or(at::Tensor())});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["norm"] = norm;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["query_weight"] = norm && wants(query_weight);
    ctx->saved_data["key_weight"] = norm && wants(key_weight);
    return {q, k};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool norm = ctx->saved_data["norm"].toBool();
    const at::Tensor &qw = saved[5], &kw = saved[6];
    const bool of_qw = ctx->saved_data["query_weight"].toBool(), of_kw = ctx->saved_data["key_weight"].toBool();
    auto [dq, dk, dqw, dkw] = backward_op().call(
        grads[0], grads[1], norm ? saved[0] : grads[0], norm ? saved[1] : grads[1], saved[2], saved[3], saved[4], qw.defined() ? OptionalTensor(qw) : std::nullopt,
        kw.defined() ? OptionalTensor(kw) : std::nullopt, ctx->saved_data["eps"].toDouble(), norm, ctx->saved_data["interleaved"].toBool(),
        ctx->saved_data["sections"].toIntVector(), of_qw || of_kw);
    const at::Tensor none;
    return {dq, dk, none, none, none, of_qw ? dqw : none, of_kw ? dkw : none, none, none, none, none};
  }
};

std::tuple<at::Tensor, at::Tensor> qk_norm_rotary_autograd(const at::Tensor& query, const at::Tensor& key, const at::Tensor& inv_freq,
                                                           const at::Tensor& query_positions, const at::Tensor& key_positions,
                                                           const OptionalTensor& query_weight, const OptionalTensor& key_weight, double eps, bool norm,
                                                           bool interleaved, at::IntArrayRef sections) {
  // Below autograd a tangent would be lost without a word.
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(query) && !has_tangent(key) && !has_tangent(query_weight) && !has_tangent(key_weight) && !has_tangent(inv_freq),
                              "gdpa::qk_norm_rotary has no forward-mode derivative: its inputs cannot have tangents");
  if (at::GradMode::is_enabled()) {
    TORCH_CHECK(!inv_freq.requires_grad(), "inv_freq cannot be differentiated: detach it");
    if (wants(query) || wants(key) || wants(query_weight) || wants(key_weight)) {
      auto out = QkNormRotary::apply(query, key, inv_freq, query_positions, key_positions, query_weight, key_weight, eps, norm, interleaved,
                                     sections.vec());
      return {out[0], out[1]};
    }
  }
  const at::AutoDispatchBelowADInplaceOrView below;
  return QkNormRotary::op().call(query, key, inv_freq, query_positions, key_positions, query_weight, key_weight, eps, norm, interleaved, sections);
}

// ------------------------------------------------------------------------------------------ a serving step

at::Tensor append_rotated(const at::Tensor& query, const at::Tensor& key, const at::Tensor& value, const at::Tensor& k_cache, const at::Tensor& v_cache,
                          const at::Tensor& k_scales, const at::Tensor& v_scales, const at::Tensor& slot_mapping, const at::Tensor& query_offset,
                          const at::Tensor& seq_lens, const at::Tensor& inv_freq, const OptionalTensor& positions, const OptionalTensor& query_weight,
                          const OptionalTensor& key_weight, double eps, bool norm, bool interleaved, at::IntArrayRef sections) {
  check_cuda("query", query);
  check_heads("query", query);
  for (auto& [name, t] : {std::pair<const char*, const at::Tensor&>("key", key), {"value", value}}) {
    check_device(name, t, query);
    check_type(name, t, query.scalar_type());
    check_rows(name, t);
  }
  check_cache(k_cache, v_cache, k_scales, v_scales, query);
  TORCH_CHECK_VALUE(key.sizes() == value.sizes() && key.size(0) == query.size(0), "query, key and value must have the same tokens, key and value the same shape");
  TORCH_CHECK_VALUE(key.size(1) == k_cache.size(2) && key.size(2) == k_cache.size(3) && query.size(2) == key.size(2), "key and value must be [tokens, ",
                    k_cache.size(2), ", ", k_cache.size(3), "] for this cache, query the same head_dim, got ", key.sizes(), " and ", query.sizes());
  check_type("slot_mapping", slot_mapping, at::kLong);
  check_vector("slot_mapping", slot_mapping, query, query.size(0));
  const bool wide_lens = check_int("seq_lens", seq_lens), wide_offsets = check_int("query_offset", query_offset);
  check_vector("seq_lens", seq_lens, query, -1);
  TORCH_CHECK_VALUE(seq_lens.numel() < int64_t{1} << 31, "too many requests");
  check_vector("query_offset", query_offset, query, seq_lens.numel() + 1);
  GdpaRotatedAppendParams p{};
  p.struct_size = sizeof(p);
  p.rotary = rotary_spec(query, inv_freq, eps, norm, interleaved, sections);
  if (positions.has_value()) {
    p.positions_are_int64 = check_positions("positions", *positions, query, p.rotary.axes, query.size(0), p.position_stride);
    p.positions = positions->const_data_ptr();
  }
  p.query_weight_is_bf16 = check_weight("query_weight", query_weight, query);
  p.key_weight_is_bf16 = check_weight("key_weight", key_weight, query);
  p.query_weight = data(query_weight);
  p.key_weight = data(key_weight);
  const c10::cuda::CUDAGuard guard(query.device());
  at::Tensor out = empty(query.sizes(), query.scalar_type(), query);
  p.heads = static_cast<int32_t>(query.size(1));
  p.query = query.const_data_ptr();
  strides(p.query_strides, query);
  p.query_out = out.mutable_data_ptr();
  p.batch = static_cast<int32_t>(seq_lens.numel());
  p.q_offsets = query_offset.const_data_ptr();
  p.seq_lens = seq_lens.const_data_ptr();
  p.offsets_are_int64 = wide_offsets;
  p.lens_are_int64 = wide_lens;
  GdpaCacheAppendParams& c = p.cache;
  c.struct_size = sizeof(c);
  c.x_is_fp32 = query.scalar_type() == at::kFloat;
  c.key = key.const_data_ptr();
  c.value = value.const_data_ptr();
  strides(c.key_strides, key);
  strides(c.value_strides, value);
  c.k_cache = k_cache.mutable_data_ptr();
  c.v_cache = v_cache.mutable_data_ptr();
  strides(c.k_cache_strides, k_cache);
  strides(c.v_cache_strides, v_cache);
  c.k_scales = k_scales.mutable_data_ptr<float>();
  c.v_scales = v_scales.mutable_data_ptr<float>();
  c.slot_mapping = slot_mapping.const_data_ptr<int64_t>();
  c.tokens = query.size(0);
  c.num_blocks = k_cache.size(0);
  c.block_size = static_cast<int32_t>(k_cache.size(1));
  c.kv_heads = static_cast<int32_t>(k_cache.size(2));
  c.head_dim = static_cast<int32_t>(k_cache.size(3));
  check(g_call.append(&p, stream()), "gdpa_append_rotated_kv_cache_fp8");
  return out;
}

std::tuple<at::Tensor, at::Tensor> read_cache(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& k_scales, const at::Tensor& v_scales,
                                              const at::Tensor& block_tables, const at::Tensor& key_offset, int64_t total_tokens,
                                              const OptionalTensor& first_tokens, at::ScalarType dtype) {
  check_cuda("k_cache", k_cache);
  check_cache(k_cache, v_cache, k_scales, v_scales, k_cache);
  TORCH_CHECK_TYPE(dtype == at::kBFloat16 || dtype == at::kFloat, "dtype must be bf16 or fp32, got ", dtype);
  const bool wide = check_int("key_offset", key_offset);
  check_vector("key_offset", key_offset, k_cache, -1);
  TORCH_CHECK_VALUE(key_offset.numel() >= 1, "key_offset must have at least one entry");
  const int64_t batch = key_offset.numel() - 1, size = k_cache.size(1);
  TORCH_CHECK_VALUE(batch < int64_t{1} << 31, "too many requests");
  check_table(block_tables, k_cache, batch, size);
  TORCH_CHECK_VALUE(total_tokens >= 0 && total_tokens < int64_t{1} << 36, "total_tokens must not be negative, got ", total_tokens);
  GdpaCacheReadParams p{};
  p.struct_size = sizeof(p);
  if (first_tokens.has_value()) {
    p.first_is_int64 = check_int("first_tokens", *first_tokens);
    check_vector("first_tokens", *first_tokens, k_cache, batch);
    p.first = first_tokens->const_data_ptr();
  }
  const c10::cuda::CUDAGuard guard(k_cache.device());
  at::Tensor key = empty({total_tokens, k_cache.size(2), k_cache.size(3)}, dtype, k_cache), value = empty(key.sizes(), dtype, k_cache);
  p.out_is_fp32 = dtype == at::kFloat;
  p.k_cache = k_cache.const_data_ptr();
  p.v_cache = v_cache.const_data_ptr();
  strides(p.k_cache_strides, k_cache);
  strides(p.v_cache_strides, v_cache);
  p.k_scales = k_scales.const_data_ptr<float>();
  p.v_scales = v_scales.const_data_ptr<float>();
  p.block_tables = block_tables.const_data_ptr<int32_t>();
  p.table_stride = block_tables.stride(0);
  p.table_width = static_cast<int32_t>(block_tables.size(1));
  p.block_size = static_cast<int32_t>(size);
  p.num_blocks = k_cache.size(0);
  p.offsets = key_offset.const_data_ptr();
  p.offsets_are_int64 = wide;
  p.batch = static_cast<int32_t>(batch);
  p.kv_heads = static_cast<int32_t>(k_cache.size(2));
  p.head_dim = static_cast<int32_t>(k_cache.size(3));
  p.total = total_tokens;
  p.key = key.mutable_data_ptr();
  p.value = value.mutable_data_ptr();
  check(g_call.read(&p, stream()), "gdpa_read_kv_cache_fp8");
  return {key, value};
}

// ------------------------------------------------------------------------------------------ drafts

std::tuple<at::Tensor, at::Tensor, at::Tensor> verify_drafts(const at::Tensor& target_probs, const OptionalTensor& draft_probs, const at::Tensor& draft_tokens,
                                                             const at::Tensor& query_offset, const at::Tensor& draft_offset, const at::Tensor& accept_uniform,
                                                             const at::Tensor& sample_uniform, int64_t max_drafts) {
  check_cuda("target_probs", target_probs);
  GdpaVerifyParams p{};
  p.struct_size = sizeof(p);
  auto check_probs = [&](const char* name, const at::Tensor& t, int64_t vocab) {
    check_device(name, t, target_probs);
    TORCH_CHECK_VALUE(t.dim() == 2 && (vocab < 0 || t.size(1) == vocab), name, " must be [rows, vocabulary], got ", t.sizes());
    TORCH_CHECK_VALUE(t.numel() == 0 || t.size(1) == 1 || t.stride(1) == 1, name, " must have contiguous rows");
  };
  TORCH_CHECK_TYPE(target_probs.scalar_type() == at::kFloat || target_probs.scalar_type() == at::kBFloat16, "target_probs must be fp32 or bf16, got ",
                   target_probs.scalar_type());
  check_probs("target_probs", target_probs, -1);
  const int64_t vocab = target_probs.size(1), drafts = draft_tokens.numel(), batch = sample_uniform.numel();
  TORCH_CHECK_VALUE(vocab >= 1, "target_probs must have a vocabulary of at least one token");
  TORCH_CHECK_NOT_IMPLEMENTED(vocab <= int64_t{1} << 20, "a vocabulary of ", vocab, " tokens is not supported (2^20 at most)");
  if (draft_probs.has_value()) {
    check_type("draft_probs", *draft_probs, target_probs.scalar_type());
    check_probs("draft_probs", *draft_probs, vocab);
    TORCH_CHECK_VALUE(draft_probs->size(0) == drafts, "draft_probs must have a row for each of the ", drafts, " draft_tokens, got ", draft_probs->sizes());
  }
  p.tokens_are_int64 = check_int("draft_tokens", draft_tokens);
  check_vector("draft_tokens", draft_tokens, target_probs, -1);
  check_type("accept_uniform", accept_uniform, at::kFloat);
  check_vector("accept_uniform", accept_uniform, target_probs, drafts);
  check_type("sample_uniform", sample_uniform, at::kFloat);
  check_vector("sample_uniform", sample_uniform, target_probs, -1);
  p.offsets_are_int64 = check_int("query_offset", query_offset);
  check_vector("query_offset", query_offset, target_probs, batch + 1);
  check_type("draft_offset", draft_offset, query_offset.scalar_type());
  check_vector("draft_offset", draft_offset, target_probs, batch + 1);
  TORCH_CHECK_VALUE(max_drafts >= 0 && max_drafts <= int64_t{1} << 20, "max_drafts must be in [0, 2^20], got ", max_drafts);
  TORCH_CHECK_VALUE(batch <= int64_t{1} << 27, "too many requests");
  const c10::cuda::CUDAGuard guard(target_probs.device());
  at::Tensor tokens = empty({batch, max_drafts + 1}, draft_tokens.scalar_type(), target_probs), accepted = empty({batch}, at::kInt, target_probs),
             refused = empty({batch}, at::kInt, target_probs);
  p.is_bf16 = target_probs.scalar_type() == at::kBFloat16;
  p.target = target_probs.const_data_ptr();
  p.target_stride = target_probs.stride(0);
  if (draft_probs.has_value() && drafts > 0) {
    p.draft = draft_probs->const_data_ptr();
    p.draft_stride = draft_probs->stride(0);
  }
  p.rows = target_probs.size(0);
  p.drafts = drafts;
  p.vocab = static_cast<int32_t>(vocab);
  p.tokens = draft_tokens.const_data_ptr();
  p.row_offsets = query_offset.const_data_ptr();
  p.draft_offsets = draft_offset.const_data_ptr();
  p.batch = static_cast<int32_t>(batch);
  p.accept = accept_uniform.const_data_ptr<float>();
  p.sample = sample_uniform.const_data_ptr<float>();
  p.max_drafts = static_cast<int32_t>(max_drafts);
  p.out_tokens = tokens.mutable_data_ptr();
  p.accepted = accepted.mutable_data_ptr<int32_t>();
  p.refused = refused.mutable_data_ptr<int32_t>();
  const size_t bytes = g_call.verify_workspace(p.batch, p.vocab, p.is_bf16);
  at::Tensor workspace;
  if (bytes > 0) {
    workspace = empty({static_cast<int64_t>(bytes)}, at::kByte, target_probs);
    p.workspace = workspace.mutable_data_ptr();
    p.workspace_bytes = static_cast<int64_t>(bytes);
  }
  check(g_call.verify(&p, stream()), "gdpa_verify_draft_tokens");
  return {tokens, accepted, refused};
}

std::tuple<at::Tensor, at::Tensor> drop_tokens(const at::Tensor& block_tables, const at::Tensor& seq_lens, const at::Tensor& dropped,
                                               const at::Tensor& free_blocks, const at::Tensor& num_free, int64_t block_size) {
  check_cuda("seq_lens", seq_lens);
  const int64_t batch = seq_lens.numel();
  GdpaDropParams p{};
  p.struct_size = sizeof(p);
  p.lens_are_int64 = check_int("seq_lens", seq_lens);
  check_vector("seq_lens", seq_lens, seq_lens, -1);
  p.dropped_is_int64 = check_int("dropped", dropped);
  check_vector("dropped", dropped, seq_lens, batch);
  check_type("free_blocks", free_blocks, at::kInt);
  check_vector("free_blocks", free_blocks, seq_lens, -1);
  check_type("num_free", num_free, at::kInt);
  check_vector("num_free", num_free, seq_lens, 1);
  check_block_size(block_size);
  check_table(block_tables, seq_lens, batch, block_size);
  TORCH_CHECK_VALUE(batch < (int64_t{1} << 31) - 16, "too many requests");
  const c10::cuda::CUDAGuard guard(seq_lens.device());
  at::Tensor lens = empty({batch}, at::kInt, seq_lens), left = empty({1}, at::kInt, seq_lens);
  p.block_size = static_cast<int32_t>(block_size);
  p.block_tables = block_tables.const_data_ptr<int32_t>();
  p.table_stride = block_tables.stride(0);
  p.table_width = static_cast<int32_t>(block_tables.size(1));
  p.batch = static_cast<int32_t>(batch);
  p.seq_lens = seq_lens.const_data_ptr();
  p.dropped = dropped.const_data_ptr();
  p.free_blocks = free_blocks.mutable_data_ptr<int32_t>();
  p.free_capacity = free_blocks.numel();
  p.num_free = num_free.const_data_ptr<int32_t>();
  p.seq_lens_after = lens.mutable_data_ptr<int32_t>();
  p.num_free_after = left.mutable_data_ptr<int32_t>();
  const size_t bytes = g_call.drop_workspace(p.batch, p.table_width);
  at::Tensor workspace;
  if (bytes > 0) {
    workspace = empty({static_cast<int64_t>(bytes)}, at::kByte, seq_lens);
    p.workspace = workspace.mutable_data_ptr();
    p.workspace_bytes = static_cast<int64_t>(bytes);
  }
  check(g_call.drop(&p, stream()), "gdpa_drop_cached_tokens");
  return {lens, left};
}

}  // namespace

// The entry points of the kernel library, in the order of EntryPoints.
extern "C" __attribute__((visibility("default"))) void gdpa_torch_init_heads(void* const* f) {
  g_call.rotary = reinterpret_cast<decltype(g_call.rotary)>(f[0]);
  g_call.rotary_bwd = reinterpret_cast<decltype(g_call.rotary_bwd)>(f[1]);
  g_call.rotary_workspace = reinterpret_cast<decltype(g_call.rotary_workspace)>(f[2]);
  g_call.append = reinterpret_cast<decltype(g_call.append)>(f[3]);
  g_call.read = reinterpret_cast<decltype(g_call.read)>(f[4]);
  g_call.verify_workspace = reinterpret_cast<decltype(g_call.verify_workspace)>(f[5]);
  g_call.verify = reinterpret_cast<decltype(g_call.verify)>(f[6]);
  g_call.drop_workspace = reinterpret_cast<decltype(g_call.drop_workspace)>(f[7]);
  g_call.drop = reinterpret_cast<decltype(g_call.drop)>(f[8]);
}

TORCH_LIBRARY_FRAGMENT(gdpa, m) {
  m.def(
      "qk_norm_rotary(Tensor query, Tensor key, Tensor inv_freq, Tensor query_positions, Tensor key_positions, Tensor? query_weight, Tensor? key_weight, "
      "float eps, bool norm, bool interleaved, int[] sections) -> (Tensor, Tensor)",
      {at::Tag::pt2_compliant_tag});
  m.def(
      "qk_norm_rotary_backward(Tensor query_grad, Tensor key_grad, Tensor query, Tensor key, Tensor inv_freq, Tensor query_positions, "
      "Tensor key_positions, Tensor? query_weight, Tensor? key_weight, float eps, bool norm, bool interleaved, int[] sections, bool weight_grads) -> "
      "(Tensor, Tensor, Tensor, Tensor)",
      {at::Tag::pt2_compliant_tag});
  m.def(
      "append_rotated_kv_cache_fp8(Tensor query, Tensor key, Tensor value, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scales, "
      "Tensor(d!) v_scales, Tensor slot_mapping, Tensor query_offset, Tensor seq_lens, Tensor inv_freq, Tensor? positions, Tensor? query_weight, "
      "Tensor? key_weight, float eps, bool norm, bool interleaved, int[] sections) -> Tensor",
      {at::Tag::pt2_compliant_tag});
  m.def(
      "read_kv_cache_fp8(Tensor k_cache, Tensor v_cache, Tensor k_scales, Tensor v_scales, Tensor block_tables, Tensor key_offset, SymInt total_tokens, "
      "Tensor? first_tokens, ScalarType dtype) -> (Tensor, Tensor)",
      {at::Tag::pt2_compliant_tag});
  m.def(
      "verify_draft_tokens(Tensor target_probs, Tensor? draft_probs, Tensor draft_tokens, Tensor query_offset, Tensor draft_offset, "
      "Tensor accept_uniform, Tensor sample_uniform, SymInt max_drafts) -> (Tensor, Tensor, Tensor)",
      {at::Tag::pt2_compliant_tag});
  m.def(
      "drop_cached_tokens(Tensor block_tables, Tensor seq_lens, Tensor dropped, Tensor(a!) free_blocks, Tensor num_free, SymInt block_size) -> "
      "(Tensor, Tensor)",
      {at::Tag::pt2_compliant_tag});
}
TORCH_LIBRARY_IMPL(gdpa, CUDA, m) {
  m.impl("qk_norm_rotary", &qk_norm_rotary);
  m.impl("qk_norm_rotary_backward", &qk_norm_rotary_backward);
  m.impl("append_rotated_kv_cache_fp8", &append_rotated);
  m.impl("read_kv_cache_fp8", &read_cache);
  m.impl("verify_draft_tokens", &verify_drafts);
  m.impl("drop_cached_tokens", &drop_tokens);
}
TORCH_LIBRARY_IMPL(gdpa, Autograd, m) {
  m.impl("qk_norm_rotary", &qk_norm_rotary_autograd);
  // Differentiating their outputs raises.
  m.impl("qk_norm_rotary_backward", torch::autograd::autogradNotImplementedFallback());
  m.impl("append_rotated_kv_cache_fp8", torch::autograd::autogradNotImplementedFallback());
  m.impl("read_kv_cache_fp8", torch::autograd::autogradNotImplementedFallback());
  m.impl("verify_draft_tokens", torch::autograd::autogradNotImplementedFallback());
  m.impl("drop_cached_tokens", torch::autograd::autogradNotImplementedFallback());
}
