// The paged cache's torch operators: argument checks, outputs and the calls of the C ABI, in C++.
//
// A step of generation on a few requests is host time: through Python (two passes of the dispatcher, the checks and a ctypes structure)
// the three calls took 28, 29 and 46 us, their kernels 3 to 18.  The operators have no gradient and only a CUDA kernel; their fake
// kernels are registered in Python.  The C ABI stays free of torch types: its entry points are handed over by address
// (gdpa_torch_init), so that this library needs no particular copy of it.
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>

#include <atomic>

#include "gdpa_torch.h"

using namespace gdpa_torch;

namespace {

struct EntryPoints {
  int (*build_block_tables)(const GdpaBlockTableParams*, gdpa_stream_t);
  int (*append)(const GdpaCacheAppendParams*, gdpa_stream_t);
  size_t (*workspace_bytes)(int64_t, int32_t, int32_t, int32_t, int32_t);
  int (*attend)(const GdpaPagedParams*, gdpa_stream_t);
} g_call{};
constexpr int kMaxDevices = 64;
// The word of each device into which a kernel writes when a wait of it runs out, or null as long as nobody has asked for it.  Python has it: the
// call returns it and, where it is set, clears it and says what happened in `message`.
std::atomic<int32_t*> g_status[kMaxDevices];
using StatusLook = int32_t* (*)(int device, char* message, int size);
std::atomic<StatusLook> g_look{nullptr};
std::atomic<void*> g_timing[2];               // events around the attention's kernel, or null

// The status word for a call on `device`; an error if a wait of an earlier call's kernel ran out.  Here, not in Python, so that a traced call does it too.
int32_t* status_of(int device) {
  if (device < 0 || device >= kMaxDevices) return nullptr;
  int32_t* word = g_status[device].load();
  if (word != nullptr && *static_cast<volatile int32_t*>(word) == 0) return word;
  const StatusLook look = g_look.load();
  if (look == nullptr) return word;
  char message[512] = "";
  g_status[device].store(word = look(device, message, sizeof(message)));
  TORCH_CHECK(message[0] == '\0', message);
  return word;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> build_block_tables(const at::Tensor& block_tables, const at::Tensor& cached_lens,
                                                                              const at::Tensor& new_lens, const at::Tensor& free_blocks,
                                                                              const at::Tensor& num_free, int64_t block_size, int64_t total_new) {
  check_cuda("cached_lens", cached_lens);
  const int64_t batch = cached_lens.numel();
  const bool wide = check_int("cached_lens", cached_lens);
  check_vector("cached_lens", cached_lens, cached_lens, -1);
  check_type("new_lens", new_lens, cached_lens.scalar_type());
  check_vector("new_lens", new_lens, cached_lens, batch);
  check_type("free_blocks", free_blocks, at::kInt);
  check_vector("free_blocks", free_blocks, cached_lens, -1);
  check_type("num_free", num_free, at::kInt);
  check_vector("num_free", num_free, cached_lens, 1);
  check_block_size(block_size);
  check_table(block_tables, cached_lens, batch, block_size);
  TORCH_CHECK_VALUE(batch <= 1 || block_tables.stride(0) >= block_tables.size(1), "block_tables must have rows of its own: they are written to");
  TORCH_CHECK_VALUE(batch < int64_t{1} << 31, "too many requests");
  TORCH_CHECK_VALUE(total_new >= 0 && total_new < int64_t{1} << 31, "total_new must be in [0, 2^31), got ", total_new);
  const c10::cuda::CUDAGuard guard(cached_lens.device());
  at::Tensor slots = empty({total_new}, at::kLong, cached_lens), query_offset = empty({batch + 1}, at::kInt, cached_lens),
             seq_lens = empty({batch}, at::kInt, cached_lens), num_free_after = empty({1}, at::kInt, cached_lens);
  GdpaBlockTableParams p{};
  p.struct_size = sizeof(p);
  p.lens_are_int64 = wide;
  p.cached_lens = cached_lens.const_data_ptr();
  p.new_lens = new_lens.const_data_ptr();
  p.batch = static_cast<int32_t>(batch);
  p.block_size = static_cast<int32_t>(block_size);
  p.block_tables = block_tables.mutable_data_ptr<int32_t>();
  p.table_stride = block_tables.stride(0);
  p.table_width = static_cast<int32_t>(block_tables.size(1));
  p.free_blocks = free_blocks.const_data_ptr<int32_t>();
  p.free_capacity = free_blocks.numel();
  p.num_free = num_free.const_data_ptr<int32_t>();
  p.total_new = total_new;
  p.slots = slots.mutable_data_ptr<int64_t>();
  p.query_offset = query_offset.mutable_data_ptr<int32_t>();
  p.seq_lens = seq_lens.mutable_data_ptr<int32_t>();
  p.num_free_after = num_free_after.mutable_data_ptr<int32_t>();
  check(g_call.build_block_tables(&p, c10::cuda::getCurrentCUDAStream().stream()), "gdpa_build_block_tables");
  return {slots, query_offset, seq_lens, num_free_after};
}

void append_kv_cache_fp8(const at::Tensor& key, const at::Tensor& value, const at::Tensor& k_cache, const at::Tensor& v_cache,
                         const at::Tensor& k_scales, const at::Tensor& v_scales, const at::Tensor& slot_mapping) {
  check_cuda("key", key);
  check_cuda("value", value);
  TORCH_CHECK_TYPE(key.scalar_type() == at::kBFloat16 || key.scalar_type() == at::kFloat, "key must be bf16 or fp32, got ", key.scalar_type());
  check_type("value", value, key.scalar_type());
  check_rows("key", key);
  check_rows("value", value);
  check_cache(k_cache, v_cache, k_scales, v_scales, key);
  TORCH_CHECK_VALUE(key.sizes() == value.sizes() && key.device() == value.device(), "key and value must have the same shape and device");
  TORCH_CHECK_VALUE(key.size(1) == k_cache.size(2) && key.size(2) == k_cache.size(3), "key and value must be [tokens, ", k_cache.size(2), ", ",
                    k_cache.size(3), "] for this cache, got ", key.sizes());
  check_type("slot_mapping", slot_mapping, at::kLong);
  check_vector("slot_mapping", slot_mapping, key, key.size(0));
  const c10::cuda::CUDAGuard guard(key.device());
  GdpaCacheAppendParams p{};
  p.struct_size = sizeof(p);
  p.x_is_fp32 = key.scalar_type() == at::kFloat;
  p.key = key.const_data_ptr();
  p.value = value.const_data_ptr();
  strides(p.key_strides, key);
  strides(p.value_strides, value);
  p.k_cache = k_cache.mutable_data_ptr();
  p.v_cache = v_cache.mutable_data_ptr();
  strides(p.k_cache_strides, k_cache);
  strides(p.v_cache_strides, v_cache);
  p.k_scales = k_scales.mutable_data_ptr<float>();
  p.v_scales = v_scales.mutable_data_ptr<float>();
  p.slot_mapping = slot_mapping.const_data_ptr<int64_t>();
  p.tokens = key.size(0);
  p.num_blocks = k_cache.size(0);
  p.block_size = static_cast<int32_t>(k_cache.size(1));
  p.kv_heads = static_cast<int32_t>(k_cache.size(2));
  p.head_dim = static_cast<int32_t>(k_cache.size(3));
  check(g_call.append(&p, c10::cuda::getCurrentCUDAStream().stream()), "gdpa_append_kv_cache_fp8");
}

at::Tensor attend_paged_fp8(const at::Tensor& query, const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& k_scales,
                            const at::Tensor& v_scales, const at::Tensor& block_tables, const at::Tensor& query_offset, const at::Tensor& seq_lens,
                            int64_t max_seq_len_q, double qk_scale, int64_t activation, bool is_causal, int64_t window_size) {
  check_cuda("query", query);
  int32_t* const status = status_of(query.get_device());
  check_type("query", query, at::kBFloat16);
  check_rows("query", query);
  check_cache(k_cache, v_cache, k_scales, v_scales, query);
  const int64_t total_q = query.size(0), heads = query.size(1), kv_heads = k_cache.size(2), dim = k_cache.size(3), size = k_cache.size(1);
  TORCH_CHECK_VALUE(query.size(2) == dim, "query must have the cache's head_dim ", dim, ", got ", query.size(2));
  TORCH_CHECK_VALUE(heads >= 1 && heads % kv_heads == 0, "the number of query heads must be a multiple of the number of key/value heads");
  const bool wide_lens = check_int("seq_lens", seq_lens), wide_offsets = check_int("query_offset", query_offset);
  check_vector("seq_lens", seq_lens, query, -1);
  const int64_t batch = seq_lens.numel();
  check_vector("query_offset", query_offset, query, batch + 1);
  check_table(block_tables, query, batch, size);
  TORCH_CHECK_VALUE(max_seq_len_q >= 0 && max_seq_len_q < int64_t{1} << 31, "max_seq_len_q must not be negative");
  TORCH_CHECK_VALUE(batch < int64_t{1} << 31, "too many requests");
  TORCH_CHECK_VALUE(window_size >= -1 && window_size < int64_t{1} << 29, "window_size must be in [0, 2^29)");
  const c10::cuda::CUDAGuard guard(query.device());
  at::Tensor o = empty({total_q, heads, dim}, at::kBFloat16, query);
  if (total_q == 0 || batch == 0) return o;
  const size_t bytes = g_call.workspace_bytes(total_q, static_cast<int32_t>(heads), static_cast<int32_t>(kv_heads), static_cast<int32_t>(dim),
                                              static_cast<int32_t>(max_seq_len_q));
  const at::Tensor workspace = empty({static_cast<int64_t>(bytes)}, at::kByte, query);
  GdpaPagedParams p{};
  p.struct_size = sizeof(p);
  p.activation = static_cast<int32_t>(activation);
  p.q = query.const_data_ptr();
  p.o = o.mutable_data_ptr();
  strides(p.q_strides, query);
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
  p.q_offsets = query_offset.const_data_ptr();
  p.seq_lens = seq_lens.const_data_ptr();
  p.offsets_are_int64 = wide_offsets;
  p.lens_are_int64 = wide_lens;
  p.batch = static_cast<int32_t>(batch);
  p.heads = static_cast<int32_t>(heads);
  p.kv_heads = static_cast<int32_t>(kv_heads);
  p.head_dim = static_cast<int32_t>(dim);
  p.total_q = total_q;
  p.max_seq_len_q = static_cast<int32_t>(max_seq_len_q);
  p.qk_scale = static_cast<float>(qk_scale);
  p.causal = is_causal;
  p.window_plus_one = static_cast<int32_t>(window_size + 1);
  p.workspace = workspace.mutable_data_ptr();
  p.workspace_bytes = static_cast<int64_t>(bytes);
  p.status = status;
  p.timing_start_event = g_timing[0].load();
  p.timing_stop_event = g_timing[1].load();
  check(g_call.attend(&p, c10::cuda::getCurrentCUDAStream().stream()), "gdpa_fwd_paged_fp8");
  return o;
}

}  // namespace

// The entry points of the kernel library (in the order of EntryPoints), and its error texts.
extern "C" __attribute__((visibility("default"))) void gdpa_torch_init(void* tables, void* append, void* workspace, void* attend, void* error) {
  g_call.build_block_tables = reinterpret_cast<decltype(g_call.build_block_tables)>(tables);
  g_call.append = reinterpret_cast<decltype(g_call.append)>(append);
  g_call.workspace_bytes = reinterpret_cast<decltype(g_call.workspace_bytes)>(workspace);
  g_call.attend = reinterpret_cast<decltype(g_call.attend)>(attend);
  strerror_of = reinterpret_cast<const char* (*)(int)>(error);
}
// Who has the status words, and the events around the next calls' kernel (null: none).
extern "C" __attribute__((visibility("default"))) void gdpa_torch_set_status_look(void* look) {
  for (auto& word : g_status) word.store(nullptr);
  g_look.store(reinterpret_cast<StatusLook>(look));
}
extern "C" __attribute__((visibility("default"))) void gdpa_torch_set_timing(void* start, void* stop) {
  g_timing[0].store(start);
  g_timing[1].store(stop);
}

TORCH_LIBRARY_FRAGMENT(gdpa, m) {
  m.def(
      "build_block_tables(Tensor(a!) block_tables, Tensor cached_lens, Tensor new_lens, Tensor free_blocks, Tensor num_free, SymInt block_size, "
      "SymInt total_new) -> (Tensor, Tensor, Tensor, Tensor)",
      {at::Tag::pt2_compliant_tag});
  m.def(
      "append_kv_cache_fp8(Tensor key, Tensor value, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scales, Tensor(d!) v_scales, "
      "Tensor slot_mapping) -> ()",
      {at::Tag::pt2_compliant_tag});
  m.def(
      "generalized_dot_product_attention_paged_fp8(Tensor query, Tensor k_cache, Tensor v_cache, Tensor k_scales, Tensor v_scales, "
      "Tensor block_tables, Tensor query_offset, Tensor seq_lens, SymInt max_seq_len_q, float qk_scale, int activation, bool is_causal, "
      "SymInt window_size) -> Tensor",
      {at::Tag::pt2_compliant_tag});
}
TORCH_LIBRARY_IMPL(gdpa, CUDA, m) {
  m.impl("build_block_tables", &build_block_tables);
  m.impl("append_kv_cache_fp8", &append_kv_cache_fp8);
  m.impl("generalized_dot_product_attention_paged_fp8", &attend_paged_fp8);
}
// Differentiating an output raises.
TORCH_LIBRARY_IMPL(gdpa, Autograd, m) {
  m.impl("build_block_tables", torch::autograd::autogradNotImplementedFallback());
  m.impl("append_kv_cache_fp8", torch::autograd::autogradNotImplementedFallback());
  m.impl("generalized_dot_product_attention_paged_fp8", torch::autograd::autogradNotImplementedFallback());
}
