"""Operator API backed by libpfa_hip.so (reference kernels/__init__.py)."""

from .paged_attn import (
    KVPages,
    evict_kv_tokens,
    new_kv_pages,
    paged_attention,
    paged_sparse_attention,
    read_kv_pages,
    select_kv_pages,
    select_kv_tokens,
    write_kv_pages,
)
from .rotary import RotaryPositions, apply_rotary, new_rotary_positions, rotary_frequencies
from .sparse_attn import (
    aspa_sparse_attention,
    build_packed_shortlist_candidates,
    build_shortlist_candidates,
    get_last_backend,
    get_last_backend_info,
)

__all__ = [
    "aspa_sparse_attention",
    "build_shortlist_candidates",
    "build_packed_shortlist_candidates",
    "get_last_backend",
    "get_last_backend_info",
    "KVPages",
    "new_kv_pages",
    "write_kv_pages",
    "read_kv_pages",
    "select_kv_pages",
    "paged_attention",
    "paged_sparse_attention",
    "select_kv_tokens",
    "evict_kv_tokens",
    "RotaryPositions",
    "new_rotary_positions",
    "rotary_frequencies",
    "apply_rotary",
]
