"""Arguments of the paged K/V cache operators (b2q_kv_append_dev,
b2q_kv_gather_dev, b2q_attn_paged_dev, b2q_attn_prompt_dev): the C structures
of include/b2q.h with their fields as plain arguments.  Pointers are device
addresses (torch tensors' data_ptr()); a structure does not keep the tensors
alive.  The calls are methods of engine.CudaEngine.
"""
from __future__ import annotations

import ctypes as C

from ._lib import B2QError, EINVAL, KvBatch, KvConfig, Prompt, Rope, lib


def kv_config(n_heads: int, n_kv_heads: int, head_dim: int, kv_type: int, page_tokens: int, n_pages: int,
              max_pages: int) -> KvConfig:
    """b2q_kv_config: heads, cache type (ggml.Q4_0) and the pool's pages."""
    return KvConfig(n_heads, n_kv_heads, head_dim, kv_type, page_tokens, n_pages, max_pages)


def kv_batch(n_seqs: int, n_tokens: int, max_new: int, q_start_ptr: int, kv_len_ptr: int,
             page_table_ptr: int) -> KvBatch:
    """b2q_kv_batch: the tokens of a call and where their sequences' pages are."""
    return KvBatch(n_seqs, n_tokens, max_new, q_start_ptr, kv_len_ptr, page_table_ptr)


def rope(rot_dim: int, n_pos: int, cos_ptr: int, sin_ptr: int) -> Rope:
    """b2q_rope: tables [n_pos][rot_dim / 2] of the rotation's cosines and sines."""
    return Rope(rot_dim, n_pos, cos_ptr, sin_ptr)


def prompt(n_heads: int, n_kv_heads: int, head_dim: int, type_: int, n_seqs: int, n_q: int, n_kv: int, max_new: int,
           q_start_ptr: int, kv_start_ptr: int) -> Prompt:
    """b2q_prompt: the packed sequences of b2q_attn_prompt_dev."""
    return Prompt(n_heads, n_kv_heads, head_dim, type_, n_seqs, n_q, n_kv, max_new, q_start_ptr, kv_start_ptr)


def page_bytes(cfg: KvConfig) -> int:
    """Bytes of one page of the pool (b2q_kv_page_bytes; no device needed)."""
    n = int(lib().b2q_kv_page_bytes(C.byref(cfg)))
    if n == 0:
        raise B2QError(EINVAL, lib().b2q_last_error().decode())
    return n
