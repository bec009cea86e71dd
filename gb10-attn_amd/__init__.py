"""MI355X (gfx950) paged attention: drop-in for gb10-attn's decode v1/v2/v3
and WMMA-prefill launchers, plus the KV-cache write that fills the paged pool
(alone, or with the norm and rotation of the new heads) and the forking, freeing,
compacting and copying of its pages, and attention that reads a prefix shared by
several sequences once.

The C-ABI lives in include/pagedattn.h and libpagedattn.so (built from
csrc/ by build.py); this package is its torch-facing mirror.  Import name:
gb10_attn_amd (the directory is gb10-attn_amd; __graft_entry__.load_package()
registers it).
"""
from ._lib import EXPORTS, LIB_PATH, PaTensor, check, last_error, last_launch, lib  # noqa: F401
from .ops import (choose_num_splits, choose_num_splits_for, compact_pages, copy_pages,  # noqa: F401
                  fork_sequences, free_sequences, paged_attention,
                  paged_attention_prefill, paged_attention_prefill_varlen, paged_attention_prefill_wmma,
                  paged_attention_shared_prefix, paged_attention_v2,
                  paged_attention_v3, plan_partitions, qk_norm_rope_write_kv, torch_ops, view, workspace_size, write_kv,
                  write_kv_blocks)

__all__ = [
    "paged_attention", "paged_attention_v2", "paged_attention_v3", "choose_num_splits",
    "paged_attention_prefill", "paged_attention_prefill_wmma", "paged_attention_prefill_varlen",
    "choose_num_splits_for",
    "plan_partitions", "workspace_size", "view", "lib", "LIB_PATH", "EXPORTS", "write_kv",
    "write_kv_blocks", "torch_ops", "qk_norm_rope_write_kv", "copy_pages", "fork_sequences", "free_sequences",
    "compact_pages", "paged_attention_shared_prefix",
]
