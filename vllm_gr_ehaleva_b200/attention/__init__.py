"""Attention-side pieces of the beam-consecutive decode: the paged KV cache
(block tables and slot maps, cache write, attention over blocks) and the suffix
KV gather."""
from .paged import extend_block_tables, paged_attention, store_kv
from .suffix_kv import build_suffix_metadata, extract_suffix_kv, gather_desc, suffix_records

__all__ = ["build_suffix_metadata", "extend_block_tables", "extract_suffix_kv", "gather_desc", "paged_attention",
           "store_kv", "suffix_records"]
