"""Flash-decode kernels: the names the reference exports for this path from
``python/triton_dist/kernels/nvidia/__init__.py:32-35``."""
from .flash_decode import (  # noqa: F401
    gqa_fwd_batch_decode,
    gqa_fwd_batch_decode_aot,
    gqa_fwd_batch_decode_intra_rank,
    gqa_fwd_batch_decode_intra_rank_aot,
    gqa_fwd_batch_decode_persistent,
    gqa_fwd_batch_decode_persistent_aot,
    kernel_inter_rank_gqa_fwd_batch_decode_combine_kv,
    inter_rank_combine,
    schedule_sequences,
    PreparedDecode,
    decode_plan,
    workspace_bytes,
    get_split_kv_algo_info,
    get_combine_kv_algo_info,
    get_triton_split_kv_algo_info,
    get_triton_combine_kv_algo_info,
)
from .kv_append import (  # noqa: F401
    apply_rotary_pos_emb,
    flash_attn_with_kvcache,
    paged_kv_append,
    rope_kv_append,
)
from .pages import (  # noqa: F401
    paged_kv_compact,
    paged_kv_copy,
    paged_kv_fork,
    paged_kv_free,
    paged_kv_reserve,
)
from .prefill import (  # noqa: F401
    gqa_fwd_batch_decode_shared_prefix,
    gqa_fwd_batch_prefill,
    prefill_workspace_bytes,
)

__all__ = [
    "gqa_fwd_batch_prefill",
    "gqa_fwd_batch_decode_shared_prefix",
    "prefill_workspace_bytes",
    "paged_kv_copy",
    "paged_kv_reserve",
    "paged_kv_fork",
    "paged_kv_free",
    "paged_kv_compact",
    "apply_rotary_pos_emb",
    "flash_attn_with_kvcache",
    "paged_kv_append",
    "rope_kv_append",
    "get_triton_combine_kv_algo_info",
    "get_triton_split_kv_algo_info",
    "get_combine_kv_algo_info",
    "get_split_kv_algo_info",
    "gqa_fwd_batch_decode_aot",
    "gqa_fwd_batch_decode_intra_rank_aot",
    "gqa_fwd_batch_decode_intra_rank",
    "gqa_fwd_batch_decode_persistent_aot",
    "gqa_fwd_batch_decode_persistent",
    "gqa_fwd_batch_decode",
    "kernel_inter_rank_gqa_fwd_batch_decode_combine_kv",
    "inter_rank_combine",
    "schedule_sequences",
    "PreparedDecode",
    "decode_plan",
    "workspace_bytes",
]
