"""Paged KV cache write side (no reference module).

The reference reads paged caches (pool [P, 2, Hkv, page, D], CSR page table
kv_page_indptr / kv_page_indices / kv_last_page_len) but only builds them by
hand in its tests (decode_flash_attention_redundant_var_len_paged.py:349-353,
sparsetoken_decode_flash_attention_redundant_var_len_paged.py:321-330).
This module fills them:

- ``append_paged_kv`` runs the HIP kernel ``akt_paged_kv_append``: each
  sequence's new K/V rows become its last logical positions under an
  already-updated page table.
- ``append_paged_kv_rotary`` does the same for k that still has to be rotated by
  its positions, and rotates q with it (``akt_paged_kv_append_rotary``).
- ``copy_pages`` copies pages within a pool (``akt_paged_copy``).
- ``keep_tokens`` moves the tokens that a selection keeps to the front of their sequences
  (``akt_paged_keep``).
- ``PagedKVCache`` owns a pool and a free list on the host, grows each
  sequence's page list as tokens are appended (prefill chunks or one token
  per decode step), and hands out the page table the decode entry points
  take.  Sequences may share pages (``fork``); a shared page that is about
  to be written is copied first.  Sequences that grow too long can be cut down to the
  tokens that draw attention (``evict``).  Page bookkeeping is host-side; only the copies,
  the selections and the attention run on the GPU.
"""
from __future__ import annotations

import torch

from . import _native as N
from . import _ops
from .attention_weights_paged import accumulate_attention_weights_paged
from .kept_index import select_heaviest


def append_paged_kv(k_new, v_new, append_indptr, paged_kv_cache, kv_page_indptr,
                    kv_page_indices, kv_last_page_len) -> None:
    """Scatter k_new / v_new [total_new, Hkv, D] into paged_kv_cache [P, 2, Hkv, page, D].

    Sequence b's rows append_indptr[b]:append_indptr[b+1] become its last
    positions under the page table (which must already count them).  fp16 or
    bf16, one type.  Runs asynchronously on the current stream.
    """
    N.torch_ext().append_paged_kv(k_new, v_new, append_indptr, paged_kv_cache, kv_page_indptr,
                                  kv_page_indices, kv_last_page_len)


def append_paged_kv_rotary(q, k_new, v_new, append_indptr, paged_kv_cache, kv_page_indptr,
                           kv_page_indices, kv_last_page_len, inv_freq, interleaved=False,
                           factor=1.0, position_offset=None):
    """append_paged_kv of k_new rotated by its positions; returns q rotated by the same ones.

    q [total_new, Hq, D] has a row for every row of k_new / v_new [total_new, Hkv, D].  A row's
    position is the one it takes in its sequence, plus position_offset[b] (int32 [B]) where given:
    the tokens that sequence b has lost (keep_tokens).  inv_freq (float64 [rotary_dim / 2]),
    interleaved and factor as in rotary.apply_rotary.  fp16 or bf16, one type.  Rows of q that
    belong to no sequence are left unwritten.
    """
    return N.torch_ext().append_paged_kv_rotary(q, k_new, v_new, append_indptr, paged_kv_cache,
                                                kv_page_indptr, kv_page_indices, kv_last_page_len,
                                                inv_freq, interleaved=interleaved, factor=factor,
                                                position_offset=position_offset)


def copy_pages(paged_kv_cache, src, dst, num_tokens=None) -> None:
    """Copy pages src[i] to dst[i] within paged_kv_cache, K and V of every head.

    src, dst (and num_tokens: the slots to copy of each, default all) are int32 device tensors
    [N].  The copies run at once: no page may be a destination twice, or a source and a
    destination.  Pairs that name a page outside the pool are skipped.
    """
    N.torch_ext().copy_pages(paged_kv_cache, src, dst, num_tokens=num_tokens)


def keep_tokens(paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len, sparse_ind,
                sparse_nnz, dst_page_indices=None, weights=None, rows=None) -> None:
    """Move kept tokens' K and V to the front of their sequences, in place, and their sums along.

    sparse_ind int32 [B, Hkv, keep], sparse_nnz int32 [B, Hkv(, 1)]: ascending token indices, as
    kept_index.select_heaviest returns them.  Slot j of a (sequence, kv head) takes token
    sparse_ind[b, h, j]; an entry that names a token before its own slot, or past the sequence's
    end, is skipped.  The table still describes the sequences before the call; afterwards head h of
    sequence b has sparse_nnz[b, h] tokens.
    dst_page_indices: int32, in the place of kv_page_indices for the slots written, where a page
    must not be (it is shared); the pages that differ must be in no sequence of the call.  No page
    may be written for two sequences, nor written for one and read for another.
    weights float32 [N, Hkv, L] and rows as in select_heaviest, no row twice: the kept tokens' sums
    move with them, and those behind become 0.
    """
    N.torch_ext().keep_tokens(paged_kv_cache, kv_page_indptr, kv_page_indices, kv_last_page_len,
                              sparse_ind, sparse_nnz, dst_page_indices=dst_page_indices,
                              weights=weights, rows=rows)


class PagedKVCache:
    """A page pool plus per-sequence page lists, in the reference's layout.

    >>> cache = PagedKVCache(num_pages=1024, num_kv_heads=8, page_size=16, head_dim=128)
    >>> cache.append([7, 9], k, v, [300, 12])       # prefill chunks
    >>> cache.append([7, 9], k1, v1, [1, 1])        # one decode step
    >>> indptr, indices, last = cache.page_table([7, 9])
    >>> cache.fork(7, 8)                            # 8 continues 7's tokens, sharing its pages
    >>> o = cache.extend([7, 8], q, k, v, [4, 1], inv_freq=inv_freq)  # rotate, append, attend
    >>> cache.evict([7], keep=256, first=4, recent=64)  # with weight_rows: drop what draws little

    With weight_rows, `weights` [weight_rows, Hkv, weight_len] keeps for as many sequences the
    attention that each token has drawn from the steps so far (extend), by which evict chooses.
    Tokens from position weight_len on have no sums: a sequence that outgrows them is still served,
    and can be evicted again once truncate has cut it to weight_len.

    A page table describes the cache as it is: append, extend, fork, truncate, evict,
    release and compact make the tables handed out before them stale.
    """

    def __init__(self, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int,
                 device="cuda", dtype=torch.float16, weight_rows: int = 0, weight_len: int = 0):
        if weight_rows > 0 and weight_len < 1:
            raise ValueError("weight_rows need a weight_len: the most tokens whose sums a row holds")
        self.page_size = page_size
        self.pool = torch.zeros((num_pages, 2, num_kv_heads, page_size, head_dim), dtype=dtype,
                                device=device)
        self._free = list(range(num_pages - 1, -1, -1))  # pop() hands out page 0 first
        self._pages: dict = {}
        self._len: dict = {}
        self._refs = [0] * num_pages  # sequences that hold each page
        self._dropped: dict = {}  # tokens that evict took from each sequence
        # Sums of attention weight; those behind a sequence's last token are 0.
        self.weights = None
        if weight_rows:
            self.weights = torch.zeros((weight_rows, num_kv_heads, weight_len),
                                       dtype=torch.float32, device=device)
        self._free_rows = list(range(weight_rows - 1, -1, -1))
        self._rows: dict = {}  # each sequence's row of the sums, once it has any

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def seq_len(self, seq_id) -> int:
        return self._len.get(seq_id, 0)

    def next_position(self, seq_id) -> int:
        """Position of the sequence's next token: its length and what evict took from it."""
        return self._len.get(seq_id, 0) + self._dropped.get(seq_id, 0)

    def _drop(self, pages) -> None:
        for page in pages:
            self._refs[page] -= 1
            if self._refs[page] == 0:
                self._free.append(page)

    def release(self, seq_id) -> None:
        """Drop a sequence; pages that no other sequence holds return to the free list."""
        self._drop(reversed(self._pages.pop(seq_id, [])))
        self._len.pop(seq_id, None)
        self._dropped.pop(seq_id, None)
        if seq_id in self._rows:
            self._free_rows.append(self._rows.pop(seq_id))

    def truncate(self, seq_id, length: int) -> None:
        """Forget a sequence's tokens from position `length` on (rejected drafts, say).

        Their own sums of attention weight are cleared; what their queries added to the sums of the
        tokens that stay remains there (extend(observe=0) adds nothing)."""
        if not 0 <= length <= self.seq_len(seq_id):
            raise ValueError(f"length {length} is not in [0, {self.seq_len(seq_id)}]")
        if seq_id not in self._pages:
            return
        keep = -(-length // self.page_size)
        pages = self._pages[seq_id]
        self._drop(reversed(pages[keep:]))
        del pages[keep:]
        if seq_id in self._rows and length < self._len[seq_id]:
            self.weights[self._rows[seq_id], :, length:self._len[seq_id]].zero_()
        if length == 0:
            self._dropped.pop(seq_id, None)  # positions begin anew
        self._len[seq_id] = length

    def fork(self, seq_id, new_id) -> None:
        """Start sequence new_id with seq_id's tokens.  No data moves: the two share pages until
        one of them writes into a shared one, which it then copies (append, extend)."""
        if seq_id not in self._pages:
            raise KeyError(f"no sequence {seq_id!r}")
        if new_id in self._pages:
            raise ValueError(f"sequence {new_id!r} exists")
        if seq_id in self._rows:
            row, n = self._take_row(), self._len[seq_id]
            self.weights[row].zero_()
            self.weights[row, :, :n] = self.weights[self._rows[seq_id], :, :n]
            self._rows[new_id] = row
        if seq_id in self._dropped:
            self._dropped[new_id] = self._dropped[seq_id]
        for page in self._pages[seq_id]:
            self._refs[page] += 1
        self._pages[new_id] = list(self._pages[seq_id])
        self._len[new_id] = self._len[seq_id]

    def compact(self) -> int:
        """Move the pages in use to the front of the pool, so that the free ones are its tail
        (pool[num_pages - free_pages:]).  Returns the number of pages moved."""
        used = self.pool.shape[0] - len(self._free)
        holes = sorted(p for p in self._free if p < used)
        moved = {p: q for p, q in zip((p for p in range(used, len(self._refs)) if self._refs[p]),
                                      holes)}
        if not moved:
            return 0
        t = torch.tensor([list(moved), list(moved.values())], dtype=torch.int32,
                         device=self.pool.device)
        copy_pages(self.pool, t[0], t[1])
        for src, dst in moved.items():
            self._refs[dst], self._refs[src] = self._refs[src], 0
        for pages in self._pages.values():
            pages[:] = [moved.get(p, p) for p in pages]
        self._free = list(range(self.pool.shape[0] - 1, used - 1, -1))
        return len(moved)

    def _grow(self, seq_ids, counts) -> None:
        """Room for counts[i] more tokens of seq_ids[i].  Last pages that tokens will go into are
        copied where they are shared.  Nothing changes if the pages do not suffice or the copy fails."""
        if len(counts) != len(seq_ids):
            raise ValueError("one count per sequence")
        if any(n < 0 for n in counts):
            raise ValueError("counts must be non-negative")
        growing = [(s, int(n)) for s, n in zip(seq_ids, counts) if n]
        if len({s for s, _ in growing}) != len(growing):
            raise ValueError("a sequence can take new tokens once in a call")
        need, plan, copies, left = 0, [], [], {}  # left: how often this call gives up a shared page
        for s, n in growing:
            pages, length = self._pages.get(s, ()), self._len.get(s, 0)
            more, fill = -(-(length + n) // self.page_size) - len(pages), length % self.page_size
            own = False  # whether the last page is replaced; the last holder keeps it
            if fill and self._refs[pages[-1]] - left.get(pages[-1], 0) > 1:
                left[pages[-1]] = left.get(pages[-1], 0) + 1
                copies.append((pages[-1], need, fill))
                own, more = True, more + 1
            plan.append((s, own, need, need + more, length + n))
            need += more
        if need > len(self._free):
            raise MemoryError(f"page pool exhausted: need {need} pages, {len(self._free)} free")
        taken = self._free[len(self._free) - need:][::-1]
        if copies:  # into free pages: until they are made, the sequences stay as they are
            t = torch.tensor([(src, taken[at], fill) for src, at, fill in copies],
                             dtype=torch.int32, device=self.pool.device).t().contiguous()
            copy_pages(self.pool, t[0], t[1], num_tokens=t[2])
        del self._free[len(self._free) - need:]
        for s in seq_ids:
            self._pages.setdefault(s, [])
            self._len.setdefault(s, 0)
        for s, own, i, j, length in plan:
            pages = self._pages[s]
            if own:
                self._refs[pages.pop()] -= 1
            for page in taken[i:j]:
                self._refs[page] = 1
                pages.append(page)
            self._len[s] = length

    def _ints(self, v):
        return torch.tensor(v, dtype=torch.int32, device=self.pool.device)

    def _table(self, held):
        """Page table of (pages, tokens) pairs."""
        indptr, indices, last = [0], [], []
        for pages, n in held:
            indices.extend(pages)
            indptr.append(len(indices))
            last.append(0 if n == 0 else (n - 1) % self.page_size + 1)
        return self._ints(indptr), self._ints(indices), self._ints(last)

    def page_table(self, seq_ids):
        """(kv_page_indptr, kv_page_indices, kv_last_page_len) int32 device tensors."""
        return self._table([(self._pages.get(s, []), self._len.get(s, 0)) for s in seq_ids])

    def _groups(self, seq_ids, counts):
        """Neighbours that share leading pages: [first, end, pages shared] of each group.

        A page counts as shared where it holds no new token of either.  A sequence joins the group before
        it unless that would save less than the group saves without it."""
        room = [max(self._len.get(s, 0) - int(n), 0) // self.page_size
                for s, n in zip(seq_ids, counts)]
        groups = []
        for i, s in enumerate(seq_ids):
            pages = self._pages.get(s, [])
            if groups and groups[-1][1] == i:
                a, end, held = groups[-1]
                other = self._pages.get(seq_ids[a], [])
                lo, hi = 0, min(held if end - a > 1 else room[a], room[i])
                if pages[:hi] == other[:hi]:
                    lo = hi
                while lo < hi:  # pages[:lo] are shared, pages[:hi + 1] are not
                    mid = (lo + hi + 1) // 2
                    if pages[lo:mid] == other[lo:mid]:
                        lo = mid
                    else:
                        hi = mid - 1
                if lo and lo * (end - a) >= held * (end - a - 1):
                    groups[-1] = [a, i + 1, lo]
                    continue
            groups.append([i, i + 1, 0])
        return groups

    def split_table(self, seq_ids, counts=None):
        """(kv_page_indptr, kv_page_indices, kv_last_page_len, group_indptr, prefix_page_indptr,
        prefix_page_indices, prefix_last_page_len) as flash_attention_shared_prefix_paged takes them.

        Neighbours in seq_ids that share leading pages form groups; the last counts[i] tokens of each
        sequence (default: one) are its queries and stay out of the prefixes."""
        counts = [1] * len(seq_ids) if counts is None else counts
        if len(counts) != len(seq_ids):
            raise ValueError("one count per sequence")
        if any(n < 0 for n in counts):
            raise ValueError("counts must be non-negative")
        return self._split(seq_ids, self._groups(seq_ids, counts))

    def _split(self, seq_ids, groups):
        group, prefixes, own = [0], [], []
        for a, end, held in groups:
            group.append(end)
            prefixes.append((self._pages.get(seq_ids[a], [])[:held], held * self.page_size))
            for s in seq_ids[a:end]:
                own.append((self._pages.get(s, [])[held:],
                            self._len.get(s, 0) - held * self.page_size))
        prefix = self._table(prefixes)
        return (*self._table(own), self._ints(group), *prefix)

    def _take_row(self) -> int:
        if not self._free_rows:
            raise MemoryError(f"all {self.weights.shape[0]} rows of weights are taken")
        return self._free_rows.pop()

    def _row_table(self, seq_ids):
        """The sequences' rows of the sums, int32; those that have none get one, all or none."""
        new = [s for s in dict.fromkeys(seq_ids) if s not in self._rows]
        if len(new) > len(self._free_rows):
            raise MemoryError(f"all {self.weights.shape[0]} rows of weights are taken")
        for s in new:
            row = self._take_row()
            self.weights[row].zero_()
            self._rows[s] = row
        return self._ints([self._rows[s] for s in seq_ids])

    def _indptr(self, counts):
        ap = [0]
        for n in counts:
            ap.append(ap[-1] + int(n))
        return self._ints(ap)

    def _restore(self, before) -> None:
        """Gives sequences back the lengths (None: no sequence) that they had."""
        for s, n in before.items():
            if n is None:
                self.release(s)
            else:
                self.truncate(s, n)

    def append(self, seq_ids, k_new, v_new, counts):
        """Append counts[i] rows of k_new / v_new [sum(counts), Hkv, D] to seq_ids[i].

        Returns the batch's page table after the append.  Rows past sum(counts) belong to no
        sequence.  A call that is refused leaves the sequences with the tokens they had.
        """
        total = sum(int(n) for n in counts)
        for name, x in (("k_new", k_new), ("v_new", v_new)):
            if x.shape[0] < total:
                raise ValueError(f"{name} has {x.shape[0]} rows, the counts make {total}")
        before = {s: self._len.get(s) for s in seq_ids}
        self._grow(seq_ids, counts)
        try:
            indptr, indices, last = self.page_table(seq_ids)
            append_paged_kv(k_new, v_new, self._indptr(counts), self.pool, indptr, indices, last)
        except BaseException:
            self._restore(before)
            raise
        return indptr, indices, last

    def extend(self, seq_ids, q, k_new, v_new, counts, inv_freq=None, interleaved=False,
               factor=1.0, causal=True, softmax_scale=None, return_lse=False,
               shared_prefix=False, observe=None):
        """One attention step: append counts[i] tokens to seq_ids[i] and attend with them.

        q [sum(counts), Hq, D], k_new and v_new [sum(counts), Hkv, D]; with inv_freq, q and k_new
        are rotated by the tokens' positions first (append_paged_kv_rotary).  Returns what
        flash_attention_chunk_paged returns for q over the grown cache.  A call that is refused
        leaves the sequences with the tokens they had.
        shared_prefix: leading pages that neighbours in seq_ids share (fork) are read once for all
        of them (flash_attention_shared_prefix_paged); where none do, the step is as without it.
        observe: where the cache keeps sums of attention weight, the last `observe` of each
        sequence's new tokens add theirs (default: all; 0: none), drafted tokens that truncate takes
        away again among them.  A whole prompt's cost is about half its attention again.
        The page tables are made on the host at each step, with shared_prefix two of them.
        """
        watch = self.weights is not None and observe != 0
        if observe is not None and observe < 0:
            raise ValueError("observe must be non-negative")
        total = sum(int(n) for n in counts)
        for name, x in (("q", q), ("k_new", k_new), ("v_new", v_new)):
            if x.shape[0] != total:
                raise ValueError(f"{name} has {x.shape[0]} rows, the counts make {total}")
        before, rows_before = {s: self._len.get(s) for s in seq_ids}, set(self._rows)
        self._grow(seq_ids, counts)
        try:
            if watch:  # a sequence without new tokens draws nothing and needs no row
                self._row_table([s for s, n in zip(seq_ids, counts) if n])
                rows = self._ints([self._rows.get(s, -1) for s in seq_ids])
            table = self.page_table(seq_ids)
            q_indptr = self._indptr(counts)
            if inv_freq is None:
                append_paged_kv(k_new, v_new, q_indptr, self.pool, *table)
            else:
                lost = [self._dropped.get(s, 0) for s in seq_ids]
                at = {"position_offset": self._ints(lost)} if any(lost) else {}
                q = append_paged_kv_rotary(q, k_new, v_new, q_indptr, self.pool, *table, inv_freq,
                                           interleaved=interleaved, factor=factor, **at)
            kw = dict(causal=causal, softmax_scale=softmax_scale, return_lse=return_lse or watch)
            # With no page in common the shared call would only add states and their join (us, 16
            # prompts of 300 tokens 119 against 43, 64 single tokens over 100 keys 20.9 against 19.5).
            groups = self._groups(seq_ids, counts) if shared_prefix else []
            if any(held for _, _, held in groups):
                own = self._split(seq_ids, groups)
                out = _ops.shared_prefix_paged(q, q_indptr, self.pool, *own, **kw)
            else:
                out = _ops.chunk_paged(q, q_indptr, self.pool, *table, **kw)
            if watch:
                accumulate_attention_weights_paged(self.weights, q, q_indptr, out[1], self.pool,
                                                   *table, rows=rows, causal=causal,
                                                   softmax_scale=softmax_scale, window=observe)
            return out if return_lse or not watch else out[0]
        except BaseException:
            for s in seq_ids:
                if s in self._rows and s not in rows_before:
                    self._free_rows.append(self._rows.pop(s))
            self._restore(before)
            raise

    def _eviction_steps(self, seqs, held):
        """The sequences that give up tokens in one call each, as slices of seqs: all at once where the
        free pages replace every shared page that is written, else one after another in an order in
        which they suffice (found a sequence at a time, not among all orders): a page's last holder
        keeps it, and what one gives up the next can take."""
        free = len(self._free)
        need = sum(self._refs[p] > 1 for s in seqs for p in self._pages[s][:held])
        if need <= free:
            return [slice(0, len(seqs))]
        refs = {p: self._refs[p] for s in seqs for p in self._pages[s]}
        steps, left = [], list(range(len(seqs)))
        while left:
            # Those that give up as many pages as they take first, then those that give up most, now or
            # with the sequences that share their pages behind.
            best = None
            for i in left:
                pages = self._pages[seqs[i]]
                take = sum(refs[p] > 1 for p in pages[:held])
                give = sum(refs[p] == 1 for p in pages[held:])
                rank = (give >= take, give, sum(1 / refs[p] for p in pages[held:]))
                if take <= free and (best is None or rank > best[0]):
                    best = rank, i, give - take
            if best is None:
                raise MemoryError(f"page pool exhausted: need {need} pages, {len(self._free)} free")
            _, i, more = best
            for j, p in enumerate(self._pages[seqs[i]]):
                if j >= held or refs[p] > 1:
                    refs[p] -= 1
            free += more
            left.remove(i)
            steps.append(slice(i, i + 1))
        return steps

    def _close_up(self, seqs, keep, ind, nnz, rows) -> int:
        """Cuts sequences down to the tokens listed; returns the tokens dropped."""
        held = -(-keep // self.page_size)
        shared = [(s, i) for s in seqs for i in range(held) if self._refs[self._pages[s][i]] > 1]
        fresh = dict(zip(shared, self._free[len(self._free) - len(shared):][::-1]))
        dst = None
        if fresh:
            dst = self._ints([fresh.get((s, i), p) for s in seqs
                              for i, p in enumerate(self._pages[s])])
        keep_tokens(self.pool, *self.page_table(seqs), ind, nnz, dst_page_indices=dst,
                    weights=self.weights, rows=rows)
        del self._free[len(self._free) - len(shared):]
        dropped = 0
        for s in seqs:
            pages = self._pages[s]
            self._drop(reversed(pages[held:]))
            for i in range(held):
                if (s, i) in fresh:
                    self._drop([pages[i]])
                    pages[i] = fresh[s, i]
                    self._refs[pages[i]] = 1
            del pages[held:]
            dropped += self._len[s] - keep
            self._dropped[s] = self._dropped.get(s, 0) + self._len[s] - keep
            self._len[s] = keep
        return dropped

    def evict(self, seq_ids, keep: int, first: int = 0, recent: int = 0) -> int:
        """Cut sequences of more than `keep` tokens down to so many; returns the tokens dropped.

        Each kv head keeps the first `first` tokens, the last `recent`, and of the others those that
        drew most attention (select_heaviest over the cache's sums), in their order; K, V and sums
        move to the front of the sequence's pages, and the pages behind return to the free list.
        New tokens keep counting positions from the tokens there were (next_position).  Shared pages are
        left to the other sequences: the kept tokens go into free ones.  Where these do not suffice for
        all sequences at once, the sequences are cut one after another, those first that give up most
        pages, and the last holder of a shared page keeps it.  A call that is refused changes nothing.
        """
        if self.weights is None:
            raise ValueError("the cache keeps no sums of attention weight (weight_rows)")
        if keep < 1 or first < 0 or recent < 0 or first + recent > keep:
            raise ValueError("keep must be positive and at least first + recent")
        seqs = [s for s in dict.fromkeys(seq_ids) if self.seq_len(s) > keep]
        if not seqs:
            return 0
        for s in seqs:
            if self._len[s] > self.weights.shape[2]:
                raise ValueError(f"sequence {s!r} has {self._len[s]} tokens, the sums hold "
                                 f"{self.weights.shape[2]}")
        held = -(-keep // self.page_size)  # pages of a sequence afterwards
        steps = self._eviction_steps(seqs, held)
        rows = self._row_table(seqs)
        lens = [self._len[s] for s in seqs]
        # (Rows as wide as the longest sequence: the kernel is chosen by their width, not the cache's.)
        ind, nnz = select_heaviest(self.weights[:, :, :max(lens)], self._ints(lens), keep,
                                   first=first, recent=recent, rows=rows)
        dropped = 0
        for at in steps:
            dropped += self._close_up(seqs[at], keep, ind[at], nnz[at], rows[at])
        return dropped


__all__ = ["append_paged_kv", "append_paged_kv_rotary", "copy_pages", "keep_tokens",
           "PagedKVCache"]
