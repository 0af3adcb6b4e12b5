"""GDPA operator package: drop-in for the reference's ``gdpa`` entry point."""
from .drafts import verify_draft_tokens  # noqa: F401
from .host_pipeline import forward_backward_host  # noqa: F401
from .math import Activation, activation_string_to_int, activation_to_int, int_to_activation  # noqa: F401
from .megakernel import gdpa_megakernel, layernorm_rows, rmsnorm_rows, tlx_gdpa_megakernel  # noqa: F401
from .mxfp8 import dequantize_mxfp8, generalized_dot_product_attention_mxfp8, quantize_varlen_mxfp8_sf_only  # noqa: F401
from .ops import (  # noqa: F401
    expect_contiguous,
    generalized_dot_product_attention,
    generalized_dot_product_attention_fp8,
    kernel_status,
    kernel_timing,
    quantize_fp8_blockwise,
    set_offset_validation,
)
from .paged import (  # noqa: F401
    PagedKVCache,
    append_kv_cache_fp8,
    append_rotated_kv_cache_fp8,
    build_block_tables,
    drop_cached_tokens,
    generalized_dot_product_attention_paged_fp8,
    read_kv_cache_fp8,
)
from .rotary import qk_norm_rotary  # noqa: F401
from .sharding import gather_rows, max_over_ranks, plan_token_balanced_shards, shard_inputs, shard_jagged  # noqa: F401
from .workloads import WORKLOADS, make_workload, useful_flops  # noqa: F401
