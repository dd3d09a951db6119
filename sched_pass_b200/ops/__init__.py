"""Tensor-level entry points of the sm_100a kernels (see csrc/kernels)."""
from .kernels import (PREFILL_TILE_ROWS, KernelStatusError, Workspace, add_rmsnorm, argmax, attention_decode,
                      attention_decode_scored, attention_merge, attention_prefill, check_status, embedding, kv_evict,
                      linear, linear_add_rmsnorm, linear_qkv_rope, qk_norm_rope_kv_append, rope_kv_append, row_counters,
                      status_buffer, workspace)

__all__ = [
    "PREFILL_TILE_ROWS", "KernelStatusError", "Workspace", "add_rmsnorm", "argmax", "attention_decode",
    "attention_decode_scored", "attention_merge", "attention_prefill", "check_status", "embedding", "kv_evict",
    "linear", "linear_add_rmsnorm", "linear_qkv_rope", "qk_norm_rope_kv_append", "rope_kv_append", "row_counters",
    "status_buffer", "workspace",
]
