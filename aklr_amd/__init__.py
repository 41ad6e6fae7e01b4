"""aklr_amd -- MI355X (gfx950) block-scaled FP8 / MXFP4 GEMM path, drop-in for AKLR's, with the FP8 key/value
cache, the rotary positions and the attention between its projections, and what differs from request to request in a
batch: adapters beside the projections, drafted tokens to verify, pages of the cache.

Ops keep the reference's signatures (aklr/ops/quant/api.py, aklr/ops/gemm/api.py,
aklr/plugins/sglang/models/deepseek_v2/api.py) and return their
outputs or a ``FallbackReason``. They run hand-written HIP kernels through the C ABI of
``include/aklr_amd.h`` (``libaklr_amd.so``, built in-tree by ``aklr_amd._build``).
"""
from .attention import tree_attention_fp8
from .dispatch import FallbackReason, KernelInfo
from .drafts import verify_drafts
from .gemm import gemm_a4w4_mxfp4, gemm_a8w8_blockwise_scaled, quant_gemm_a8w8_blockwise_scaled
from .kv_cache import kv_cache_read_fp8, kv_cache_write_fp8, new_kv_cache_fp8, rotary_kv_cache_write_fp8
from .kv_pages import kv_cache_compact_fp8, kv_cache_copy_pages_fp8, kv_cache_update_pages, new_kv_page_refs
from .lora import lora_project
from .moe import deepseek_v2_fp8_moe, moe_fp8_experts, moe_fp8_route
from .quant import dynamic_mxfp4_quant, per_group_quant_fp8, per_group_quant_mxfp8
from .rotary import rotary_embedding, rotary_frequencies, rotary_magnitude

__all__ = [
    "FallbackReason",
    "KernelInfo",
    "deepseek_v2_fp8_moe",
    "dynamic_mxfp4_quant",
    "gemm_a4w4_mxfp4",
    "gemm_a8w8_blockwise_scaled",
    "kv_cache_compact_fp8",
    "kv_cache_copy_pages_fp8",
    "kv_cache_read_fp8",
    "kv_cache_update_pages",
    "kv_cache_write_fp8",
    "lora_project",
    "moe_fp8_experts",
    "moe_fp8_route",
    "new_kv_cache_fp8",
    "new_kv_page_refs",
    "per_group_quant_fp8",
    "per_group_quant_mxfp8",
    "quant_gemm_a8w8_blockwise_scaled",
    "rotary_embedding",
    "rotary_frequencies",
    "rotary_kv_cache_write_fp8",
    "rotary_magnitude",
    "tree_attention_fp8",
    "verify_drafts",
]
