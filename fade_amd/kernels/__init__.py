"""Attention ops of the FADE hot path on MI355X kernels."""

from .drafts import DraftTree, VerifiedDrafts, draft_tree, verify_drafts
from .fused_int4_attn import check_fused_parity, fused_int4_sdpa, fused_int4_sdpa_with_fallback
from .int4_attention import check_parity, int4_sdpa
from .paged import PagedAttentionPlan, paged_append, paged_attention, paged_compact, paged_copy
from .prefill import TieredPrefillPlan, tiered_prefill_attention
from .tiered_attn import MiddleTier, TieredDecodePlan, tiered_decode_attention

__all__ = [
    "DraftTree",
    "MiddleTier",
    "PagedAttentionPlan",
    "TieredDecodePlan",
    "TieredPrefillPlan",
    "VerifiedDrafts",
    "check_fused_parity",
    "check_parity",
    "draft_tree",
    "fused_int4_sdpa",
    "fused_int4_sdpa_with_fallback",
    "int4_sdpa",
    "paged_append",
    "paged_attention",
    "paged_compact",
    "paged_copy",
    "tiered_decode_attention",
    "tiered_prefill_attention",
    "verify_drafts",
]
