"""Attention of several new tokens per sequence over a paged cache (no reference module).

The reference serves a paged cache one token per sequence
(decode_flash_attention_redundant_var_len_paged.py:228).  ``flash_attention_chunk_paged`` takes
any number of new tokens of each sequence in one call: a chunk of a prompt against what is
cached of it, the drafted tokens of a step under verification, decoding sequences beside a
prompt.  It runs the HIP kernel ``akt_chunk_paged_fwd`` (csrc/paged_chunk.hip) on the cache
layout and page table of the paged decode.
"""
from __future__ import annotations

from . import _ops


def flash_attention_chunk_paged(q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices,
                                kv_last_page_len, causal=True, softmax_scale=None,
                                return_lse=False):
    """Returns O: [total_q, Hq, D] (and lse [total_q, Hq] fp32 when return_lse).

    q: [total_q, Hq, D] fp16 or bf16 (the cache's type); q_indptr: int32 [B + 1], sequence b's
    n_b query tokens are rows q_indptr[b]:q_indptr[b+1].  The cache (pool [P, 2, Hkv, page, D]
    and its CSR page table) already holds the new tokens' K and V (append_paged_kv): sequence b
    has len_b tokens and its query i sits at position len_b - n_b + i.
    causal=True: a query sees the keys up to its own position; causal=False: all len_b keys.
    softmax_scale defaults to 1/sqrt(D).  Any page_size; D = 64, 128 or 256; up to 128 query
    heads per kv head.  Rows that see no key get zeros (lse -inf); rows of q that belong to no
    sequence are left unwritten.  Probabilities are rounded to q's type for the product with V and
    in the normaliser (sums are fp32), so a single token's output may be a little less exact than
    flash_attention_decode_paged's.  A call under graph capture takes a workspace of its own from
    the graph's memory pool, so captured calls may replay side by side.
    """
    return _ops.chunk_paged(q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices,
                            kv_last_page_len, causal=causal, softmax_scale=softmax_scale,
                            return_lse=return_lse)


__all__ = ["flash_attention_chunk_paged"]
