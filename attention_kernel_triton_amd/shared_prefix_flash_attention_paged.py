"""Attention of sequences that share prefixes over a paged cache (no reference module).

Samples of one prompt, branches of a search and requests behind one system prompt hold the same
pages (``PagedKVCache.fork``), and a decode or chunk call reads them once for every sequence.
``flash_attention_shared_prefix_paged`` reads a shared prefix once for all sequences of its group:
the group's rows go through the matrix pipe together, and each row's two parts, prefix and own
keys, are joined under one normaliser.  It runs ``akt_shared_prefix_paged_fwd``
(csrc/paged_chunk.hip, csrc/paged_shared.hip) on the cache layout and page tables of
``flash_attention_chunk_paged``.
"""
from __future__ import annotations

from . import _ops


def flash_attention_shared_prefix_paged(q, q_indptr, paged_kv_cache, kv_page_indptr,
                                        kv_page_indices, kv_last_page_len, group_indptr,
                                        prefix_page_indptr, prefix_page_indices,
                                        prefix_last_page_len, causal=True, softmax_scale=None,
                                        return_lse=False):
    """Returns O: [total_q, Hq, D] (and lse [total_q, Hq] fp32 when return_lse).

    group_indptr: int32 [groups + 1], group i is sequences group_indptr[i]:group_indptr[i + 1];
    sequences before the first group and behind the last have no prefix.  prefix_page_indptr
    [groups + 1], prefix_page_indices and prefix_last_page_len [groups] are the prefixes' page table
    (``PagedKVCache.page_table`` of the sequences that hold them, say).
    The other arguments are those of flash_attention_chunk_paged, kv_page_* holding a sequence's
    own pages only: its keys are its group's prefix, then its own tokens, the new ones among
    them.  Every new token sees the whole prefix; of its sequence's own tokens it sees those up to itself
    (causal=True) or all.  fp16 or bf16; any page_size; D = 64, 128 or 256; up to 128 query heads
    per kv head.  Rows that see no key get zeros (lse -inf); rows of q that belong to no sequence
    are left unwritten.  Probabilities are rounded to q's type, as there.  total_q * Hq must be below
    2^25; the stream's workspace holds 2 (4 D + 16) bytes for each query row and head, besides
    the parts of cut units (up to 139 MB).

    It pays where prefixes are read by sequences of few new tokens (us, this call / the chunk call over
    whole tables, the same inputs each time: 32 single tokens behind 4,096 28 / 84, 64 behind 20,001
    76 / 569, 1 to 6 drafts of 24 sequences in four groups 35 / 43).  Prompts read a prefix once for each
    256 rows either way (eight of 150 to 350 tokens behind 8,000 324 / 317), and a call of a few short
    sequences is bound by its second launch (two behind 40 tokens 12.9 / 11.4).
    """
    return _ops.shared_prefix_paged(q, q_indptr, paged_kv_cache, kv_page_indptr, kv_page_indices,
                                    kv_last_page_len, group_indptr, prefix_page_indptr,
                                    prefix_page_indices, prefix_last_page_len, causal=causal,
                                    softmax_scale=softmax_scale, return_lse=return_lse)


__all__ = ["flash_attention_shared_prefix_paged"]
