from dcp_amd.ops.fused_ops import (  # noqa: F401
    flash_attn_update_out_lse,
    fused_blockwise_sum,
    fused_copy_bf16,
    fused_copy_bf16_varlen,
    fused_copy_bf16_varlen_dkv,
    fused_copy_bf16_varlen_lse,
    fused_copy_fp16,
    fused_copy_fp16_varlen,
    fused_copy_fp16_varlen_dkv,
    fused_copy_fp16_varlen_lse,
    fused_copy_fp32,
    fused_copy_fp32_varlen,
    fused_copy_fp32_varlen_dkv,
    fused_copy_fp32_varlen_lse,
    warmup_triton_ops,
)
from dcp_amd.ops.paged_cache import PagedCacheTables, paged_cache_tables, paged_cache_write  # noqa: F401
