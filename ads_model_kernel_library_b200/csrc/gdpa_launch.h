// Internal interface between the C-ABI entry points (gdpa_api.cu) and the kernel translation
// units.  Plain structs only.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace gdpa {

// Internal copies of the public return codes (include/gdpa_b200.h).
constexpr int GDPA_ERR_UNSUPPORTED_DIM_ = 2;
constexpr int GDPA_ERR_UNSUPPORTED_ACT_ = 4;
constexpr int GDPA_ERR_LAUNCH_ = 6;

// The tensor map of one operand tensor: boxes of 128 rows x 128 bytes (128-byte swizzle).
constexpr int kTmapHeights = 1;
constexpr int kTmapRows[kTmapHeights] = {128};
struct TmapSet {
  CUtensorMap m[kTmapHeights];
};

// The maps of the fp32 dQ accumulator: boxes of 32 columns x 32, 16, 8, 4, 2, 1 rows, so that the reduce-add of a
// ragged tile covers exactly the rows of its sequence.
constexpr int kDqTmapHeights = 6;
struct DqTmapSet {
  CUtensorMap m[kDqTmapHeights];
};

// The map of the forward's output: boxes of 32 columns x 32 rows (64-byte swizzle), one warp's staging slab.  A slab with fewer than 32 rows of its sequence is stored from registers
// instead: further maps for smaller boxes, on top of the loaders' own, made the TMA unit refetch descriptors.
struct OutTmap {
  CUtensorMap m;
};

struct FwdArgs {
  __nv_bfloat16* o;
  const void* q_off;
  const void* kv_off;
  int off64;
  int heads;
  int max_q;
  int max_kv;
  float scale;
  const int* sched;
  int* status;
  // FP8 path: per-(128-token block, head) fp32 scales and per-sequence block offsets.
  const float* q_scales;
  const float* k_scales;
  const float* v_scales;
  const void* q_blk_off;
  const void* kv_blk_off;
  long long* trace;  // optional cycle-stamp buffer of CTA 0 (performance analysis); null in normal use
  float* lse;        // softmax: optional [heads, total_q] log-sum-exp output (base 2)
  long long total_q;
  int kv_heads;      // K / V heads; query head h reads K / V head h / kv_group
  int kv_group;      // heads / kv_heads
  const void* kv_index;  // optional: sequence -> entry of the KV offsets (shared KV sequences)
  int window;            // band |q - kv| <= window of sequence-local positions; -1 = none
  // norm pipeline: optional [total_q, heads, D] bf16 tensor added to O before it is stored, and optional
  // [total_q] fp32 array that receives the sum over heads and columns of the squares of what is stored
  const __nv_bfloat16* residual;
  float* row_sumsq;
  long long total_kv;    // rows of K / V (bounds the sequence ranges read from the offsets)
  int kv_batch;          // sequences the KV offsets describe (bounds kv_index entries)
};

struct NormArgs {
  const __nv_bfloat16* x;
  __nv_bfloat16* out;
  const float* weight;
  const float* bias;
  const __nv_bfloat16* residual;
  const float* row_sumsq;
  float* row_mean;
  float* row_rstd;
  long long rows;
  int n;
  float eps;
};

struct QuantArgs {
  const void* x;
  void* x8;
  float* scales;
  const void* offsets;
  void* block_offsets;
  int off64;
  int batch;
  int heads;
  int head_dim;
  long long max_blocks;  // rows of `scales`: at least total / 128 + batch
  long long total;       // rows of x
  int vec16;             // head_dim a multiple of 16 and x, x8 16-byte aligned: 16-element vector accesses
};

struct MxArgs {
  void* x;        // [total, H, D] bf16 or fp32: input of the quantiser, output of the de-quantiser
  void* x8;       // [total, H, D] e4m3
  uint8_t* sf;    // e8m0 scales in 512-byte atoms
  const void* offsets;
  void* block_offsets;
  int off64;
  int batch;
  int heads;
  int head_dim;
  int scale_axis;       // 0: scales along the head dim (Q, K); 1: along the tokens (V)
  long long sf_blocks;  // 128-row token blocks the scale tensor is laid out for (its head stride)
  long long max_blocks; // grid bound: at least total / 128 + batch
};

struct NormBwdArgs {
  const __nv_bfloat16* dy;
  const __nv_bfloat16* dy_add;
  const __nv_bfloat16* x;
  __nv_bfloat16* dx;
  const float* weight;
  const float* row_mean;
  const float* row_rstd;
  float* dweight;
  float* dbias;
  long long rows;
  int n;
};

struct FwdLaunch {
  TmapSet tm_q, tm_k, tm_v;
  OutTmap tm_o;
  FwdArgs args;
  int grid;
  cudaStream_t stream;
};

struct BwdArgs {
  __nv_bfloat16* dk;
  __nv_bfloat16* dv;
  float* dq_accum;
  const void* q_off;
  const void* kv_off;
  int off64;
  int heads;
  int max_q;
  int max_kv;
  float scale;
  const int* sched;
  int* status;
  long long* trace;  // optional cycle-stamp buffer of CTA 0; null in normal use
  const float* lse;    // softmax backward: [heads, total_q] log-sum-exp of the forward (base 2)
  const float* dpsum;  // softmax backward: [heads, total_q] rowsum(dO * O)
  long long total_q;
  int q_heads;         // query heads; `heads` above is the number of K / V heads (the work items' heads)
  int kv_group;        // q_heads / heads: a work item walks the Q tiles of every query head of its group
  int window;          // band |q - kv| <= window of sequence-local positions; -1 = none
  float* dk_acc;       // start / end offsets: fp32 accumulators the dK / dV tiles are added into (else null)
  float* dv_acc;
  long long total_kv;  // rows of K / V (bounds the sequence ranges read from the offsets)
};

struct BwdLaunch {
  TmapSet tm_q, tm_k, tm_v, tm_do;
  DqTmapSet tm_dq;
  BwdArgs args;
  int grid;
  cudaStream_t stream;
};

struct SchedArgs {
  const void* q_off;
  const void* kv_off;
  int off64;
  int batch;
  int heads;
  int max_q;
  int max_kv;
  int mode;
  int* sched;
  long long capacity_items;
  const void* kv_index;  // optional: sequence -> entry of the KV offsets
  int kv_batch;          // sequences the KV offsets describe (bounds kv_index entries)
};

struct BlockTableArgs {
  const void* cached_lens;
  const void* new_lens;
  int lens_are_int64;
  int batch;
  int* block_tables;
  long long table_stride;
  int table_width;
  int block_shift;  // block_size = 1 << block_shift
  const int* free_blocks;
  long long free_capacity;
  const int* num_free;
  long long total_new;
  long long* slots;
  int* query_offset;
  int* seq_lens;
  int* num_free_after;
};

struct CacheAppendArgs {
  const void* key;
  const void* value;
  long long key_strides[2];      // token, head; in elements
  long long value_strides[2];
  uint8_t* k_cache;
  uint8_t* v_cache;
  long long k_cache_strides[3];  // block, row, head; in elements
  long long v_cache_strides[3];
  float* k_scales;               // [blocks, heads]
  float* v_scales;
  const long long* slot_mapping;
  long long tokens;
  long long num_blocks;
  int block_shift;
  int heads;
};

struct PagedArgs {
  const __nv_bfloat16* q;
  long long q_strides[2];  // token, head; in elements
  __nv_bfloat16* o;        // [total_q, heads, head_dim]
  const float* k_scales;   // [blocks, kv_heads]
  const float* v_scales;
  const uint8_t* v_cache;  // as tm_v has it, for a NaN that has to be found again
  long long v_strides[3];  // block, row, head
  const int* block_tables;
  long long table_stride;
  int table_width;
  int num_blocks;
  int block_shift;
  const void* q_off;
  const void* seq_lens;
  int off64, lens64;
  int batch;
  int heads, kv_heads, group;  // group = heads / kv_heads
  int max_q;
  long long total_q;
  int act;                     // activation class
  float scale;
  int causal;
  int window;                  // -1 = none
  float* qa;                   // [kv_heads, total_q * group]: factor of a row's scores
  int* counters;               // one per CTA
  float* part_o;               // [2 per CTA][rows of a tile][head_dim]
  float* part_ml;              // [2 per CTA][2][rows of a tile]
  int* status;
};

struct PagedLaunch {
  CUtensorMap tm_q;        // over q8, [2 * kv_heads, total_q * group, head_dim]: a box is a row tile of one head, hi or lo
  CUtensorMap tm_k, tm_v;  // over [blocks, kv_heads, block_size, head_dim]: a box is one block of one head
  uint8_t* q8;
  PagedArgs args;
  int rows;                // rows of an item: 16, 64 or 256
  int grid;
  cudaStream_t stream;
};

// How heads are rotated: pair i < pairs turns by position[axis of i] * inv_freq[i]; `ends` are the axes' ends among the pairs.
constexpr int kMaxAxes = 4;
struct RotarySpec {
  const void* inv_freq;  // [pairs], radians a position
  int inv_freq_is_fp64;
  int pairs;             // a multiple of 8, at most head_dim / 2
  int interleaved;       // pairs (2 i, 2 i + 1), else (i, i + pairs)
  int axes;
  int ends[kMaxAxes];
  int norm;              // RMS norm of the head before it is rotated
  float eps;
};

struct RotaryTensor {
  const void* x;
  long long x_strides[2];  // token, head; in elements
  void* y;                 // contiguous: the output, or the gradient of x
  const void* dy;          // gradient of the output
  long long dy_strides[2];
  const void* weight;      // [head_dim], or null
  int weight_is_bf16;
  int heads;
  long long tokens;
  const void* positions;   // [axes, tokens]
  long long position_stride;
  int positions_are_int64;
  void* dweight;           // [head_dim] of the weight's type, or null
};

struct RotaryArgs {
  RotarySpec rotary;
  RotaryTensor t[2];  // queries, keys
  float* partial;     // backward: [grid][2][head_dim] sums of the weights' gradients, or null
  // How the work is dealt out: of queries, then of keys; or, where both have the same tokens and positions, of both at once.
  int paired;
  int item_tokens;        // tokens of an item
  int per[2], chunks[2];  // units (the heads that a warp has at once) of an item, items of a token (1: some tokens are an item)
  unsigned items[2];
};

struct RotatedAppendArgs {
  CacheAppendArgs cache;  // its key and value are the new ones
  RotaryArgs queries;     // t[0]: the queries; t[1] has no tokens, its weight is the keys'.  Positions null: they follow from the lengths
  const void* q_off;      // [batch + 1]
  const void* seq_lens;   // [batch]
  int off64, lens64;
  int batch;
  int kv_windows, kv_parts;  // the grid's first kv_windows * kv_parts CTAs are for keys and values
};

struct CacheReadArgs {
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  long long k_cache_strides[3];  // block, row, head; in elements
  long long v_cache_strides[3];
  const float* k_scales;
  const float* v_scales;
  const int* block_tables;
  long long table_stride;
  int table_width;
  int block_shift;
  long long num_blocks;
  const void* offsets;   // [batch + 1]
  const void* first;     // [batch], or null: zeros
  int off64, first64;
  int batch;
  int heads;
  long long total;
  void* key;
  void* value;
  int warp_tokens;  // rows of a warp, 32 at most
};

struct VerifyArgs {
  const void* target;      // [rows, vocab]
  const void* draft;       // [drafts, vocab], or null
  long long target_stride, draft_stride;
  long long rows, drafts;
  int vocab;
  const void* tokens;      // [drafts]
  int tokens64;
  const void* row_offsets;    // [batch + 1]
  const void* draft_offsets;  // [batch + 1]
  int off64;
  const float* accept;     // [drafts]
  const float* sample;     // [batch]
  int batch;
  int max_drafts;
  void* out_tokens;        // [batch, max_drafts + 1], as tokens
  int* accepted;
  int* refused;
  // many requests: what each draws from, and its stretches' sums, most_stretches for each
  void* draws;
  double* sums;
  int most_stretches;
};
struct VerifyWorkspace {
  long long sums, bytes;  // where the sums are; all of it, 0 for calls that need none
};

struct DropArgs {
  const int* block_tables;
  long long table_stride;
  int table_width;
  int block_shift;
  const void* seq_lens;
  const void* dropped;
  int lens64, dropped64;
  int batch;
  int* free_blocks;
  long long free_capacity;
  const int* num_free;
  int* seq_lens_after;
  int* num_free_after;
  int chunks;   // that a request's entries are taken in, chunk_entries each: drop_chunks, set by launch_drop
  int chunk_entries;
  int* counts;  // drop_workspace_ints
};

}  // namespace gdpa
struct GdpaFwdParams;
namespace gdpa {
// Host-side argument checks of the forward entry points (no CUDA call): the return code gdpa_fwd / gdpa_fwd_fp8 would
// give for these parameters before they launch anything (`needs_schedule`: a null schedule pointer is an error).
int fwd_check_params(const GdpaFwdParams* p, bool fp8, bool needs_schedule);

int launch_fwd_bf16(const FwdLaunch& l, int head_dim, int act_class);
int launch_fwd_softmax_bf16(const FwdLaunch& l, int head_dim);
int launch_fwd_fp8(const FwdLaunch& l, int head_dim, int act_class);
int launch_bwd_bf16(const BwdLaunch& l, int head_dim, int act_class);
int launch_dpsum(const __nv_bfloat16* d_o, const __nv_bfloat16* o, float* dpsum, long long total_q, int heads, int head_dim,
                 cudaStream_t stream);
int launch_dq_convert(const float* acc, __nv_bfloat16* dq, long long n, cudaStream_t stream);
int launch_layernorm_rows(const NormArgs& a, cudaStream_t stream);
int launch_rmsnorm_rows(const NormArgs& a, cudaStream_t stream);
int launch_quant_fp8(const QuantArgs& a, int in_is_fp32, cudaStream_t stream);
int launch_mxfp8(const MxArgs& a, int quantize, int x_is_fp32, cudaStream_t stream);
int launch_norm_rows_bwd(const NormBwdArgs& a, int mode, cudaStream_t stream);
int launch_build_schedule(const SchedArgs& a, cudaStream_t stream);
int launch_block_tables(const BlockTableArgs& a, int sm_count, cudaStream_t stream);
int launch_cache_append(const CacheAppendArgs& a, int head_dim, int is_fp32, int sm_count, cudaStream_t stream);
int launch_rotary(RotaryArgs& a, int head_dim, int is_fp32, int sm_count, cudaStream_t stream);
int launch_rotary_bwd(RotaryArgs& a, int head_dim, int is_fp32, int sm_count, cudaStream_t stream);  // kernels launched, or -(an error)
int rotary_bwd_ctas(int sm_count);  // CTAs that have a row of RotaryArgs::partial each
int launch_rotated_append(RotatedAppendArgs& a, int head_dim, int is_fp32, int sm_count, cudaStream_t stream);
int launch_cache_read(CacheReadArgs& a, int head_dim, int out_is_fp32, int sm_count, cudaStream_t stream);
VerifyWorkspace verify_workspace(long long batch, long long vocab, int is_bf16);
int launch_verify(VerifyArgs& a, int is_bf16, int sm_count, cudaStream_t stream);
int verify_most_vocab();
long long drop_workspace_ints(long long batch, int table_width);
int launch_drop(DropArgs& a, cudaStream_t stream);
int launch_paged(const PagedLaunch& l, int head_dim);
int launch_paged_rows(const PagedLaunch& l, int head_dim);  // of launch_paged, for row tiles of 256
int paged_ctas_per_sm(int rows, int head_dim);  // resident CTAs of the kernel for row tiles of `rows`: a launch has that many

}  // namespace gdpa
