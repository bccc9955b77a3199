"""Attention that cached tokens draw, summed over calls (no reference module).

A token that later queries hardly attend to can leave the cache (eviction by accumulated
attention weight: ``kept_index.select_heaviest``, ``paged_kv.keep_tokens``) or be left out of a
sparse decode.  ``accumulate_attention_weights_paged`` adds the softmax weights of an attention call
to such sums, from the normalisers that the call returned; it runs the HIP kernel
``akt_attention_weights_paged`` (csrc/attention_weights.hip) and reads K only.
"""
from __future__ import annotations

from . import _native as N


def accumulate_attention_weights_paged(weights, q, q_indptr, lse, paged_kv_cache, kv_page_indptr,
                                       kv_page_indices, kv_last_page_len, rows=None, causal=True,
                                       softmax_scale=None, window=None) -> None:
    """Adds to weights[rows[b], h, j] the softmax weight that token j of sequence b draws in kv head h.

    weights: float32 [N, Hkv, L] (unit last stride, no two rows with memory in common), written in
    place; tokens from L on are left out.
    rows: int32 [B], each sequence's row of weights (default: its own number); no row twice, and a
    sequence whose row is not in [0, N) is left out.
    q [total_q, Hq, D] (fp16 or bf16, the cache's type), q_indptr, the cache and its page table,
    causal and softmax_scale are those of flash_attention_chunk_paged (or of a paged decode: one
    token per sequence), and lse float32 [total_q, Hq] what it returned; rows of q with lse -inf
    count nothing.  The weights of all tokens of a sequence that see j and all query heads of h
    are summed, or of its last `window` tokens only.  Sums are in 32 bits and in a fixed order.
    D = 64, 128 or 256.
    """
    N.torch_ext().attention_weights_paged(weights, q, q_indptr, lse, paged_kv_cache,
                                          kv_page_indptr, kv_page_indices, kv_last_page_len,
                                          rows=rows, causal=causal, softmax_scale=softmax_scale,
                                          window=window)


__all__ = ["accumulate_attention_weights_paged"]
