"""Device-side kept-token index selection.

The reference builds sparse index lists in its test harness with a Python loop
over (batch, head) (sparsetoken_decode_flash_attention_redundant.py:283-295,
sparsetoken_decode_flash_attention_redundant_var_len_paged.py:341-353):
keep = rand(n) < p; keep index 0 if nothing is kept; indices =
nonzero(keep) ascending, -1 padded to L_max; nnz = count.  ``select_kept``
produces the same int32 arrays in one kernel launch (csrc/kept_index.hip),
bit-exact with torch.nonzero.

``select_heaviest`` chooses instead by sums of attention weight
(attention_weights_paged.accumulate_attention_weights_paged); it has no reference counterpart
(csrc/kept_heaviest.hip).
"""
from __future__ import annotations

from . import _native as N
from . import _ops


def select_kept(l_max, mask=None, uniform=None, kept_ratio=None, row_len=None,
                ensure_nonempty=True):
    """Returns (sparse_ind int32 [..., l_max], sparse_nnz int32 [..., 1]).

    Pass either ``mask`` (bool/uint8 [..., N]) or ``uniform`` (float32 [..., N])
    with ``kept_ratio``.  ``row_len`` (int32, one per row) limits each row's
    candidates to its first row_len entries.
    """
    return _ops.kept_indices(l_max, mask=mask, uniform=uniform, kept_ratio=kept_ratio,
                             row_len=row_len, ensure_nonempty=ensure_nonempty)


def select_heaviest(weights, lengths, keep, first=0, recent=0, rows=None):
    """Returns (sparse_ind int32 [B, H, keep], sparse_nnz int32 [B, H, 1]): the tokens to keep.

    weights: float32 [N, H, L] (unit last stride); lengths: int32 [B], how many tokens each
    sequence has (at most L count); rows: int32 [B], the sequences' rows of weights (default: their
    own numbers).  Of a sequence's tokens each head keeps the first `first`, the last `recent` and
    the heaviest of the others, `keep` in all, or all where there are no more.  Indices ascend and
    are padded with -1; of equal sums the lower index is kept, and a NaN counts as the heaviest.
    The lists are what keep_tokens takes, and per query head (repeat_interleave over dim 1) what
    the sparse decodes take.
    """
    return N.torch_ext().kept_heaviest(weights, lengths, keep, first=first, recent=recent,
                                       rows=rows)
