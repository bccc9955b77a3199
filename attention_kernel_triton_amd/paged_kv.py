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
- ``PagedKVCache`` owns a pool and a free list on the host, grows each
  sequence's page list as tokens are appended (prefill chunks or one token
  per decode step), and hands out the page table the decode entry points
  take.  Sequences may share pages (``fork``); a shared page that is about
  to be written is copied first.  Page bookkeeping is host-side; only the copies
  and the attention run on the GPU.
"""
from __future__ import annotations

import torch

from . import _native as N
from . import _ops


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
                           factor=1.0):
    """append_paged_kv of k_new rotated by its positions; returns q rotated by the same ones.

    q [total_new, Hq, D] has a row for every row of k_new / v_new [total_new, Hkv, D].  A row's
    position is the one it takes in its sequence; inv_freq (float64 [rotary_dim / 2]),
    interleaved and factor as in rotary.apply_rotary.  fp16 or bf16, one type.  Rows of q that
    belong to no sequence are left unwritten.
    """
    return N.torch_ext().append_paged_kv_rotary(q, k_new, v_new, append_indptr, paged_kv_cache,
                                                kv_page_indptr, kv_page_indices, kv_last_page_len,
                                                inv_freq, interleaved=interleaved, factor=factor)


def copy_pages(paged_kv_cache, src, dst, num_tokens=None) -> None:
    """Copy pages src[i] to dst[i] within paged_kv_cache, K and V of every head.

    src, dst (and num_tokens: the slots to copy of each, default all) are int32 device tensors
    [N].  The copies run at once: no page may be a destination twice, or a source and a
    destination.  Pairs that name a page outside the pool are skipped.
    """
    N.torch_ext().copy_pages(paged_kv_cache, src, dst, num_tokens=num_tokens)


class PagedKVCache:
    """A page pool plus per-sequence page lists, in the reference's layout.

    >>> cache = PagedKVCache(num_pages=1024, num_kv_heads=8, page_size=16, head_dim=128)
    >>> cache.append([7, 9], k, v, [300, 12])       # prefill chunks
    >>> cache.append([7, 9], k1, v1, [1, 1])        # one decode step
    >>> indptr, indices, last = cache.page_table([7, 9])
    >>> cache.fork(7, 8)                            # 8 continues 7's tokens, sharing its pages
    >>> o = cache.extend([7, 8], q, k, v, [4, 1], inv_freq=inv_freq)  # rotate, append, attend

    A page table describes the cache as it is: append, extend, fork, truncate,
    release and compact make the tables handed out before them stale.
    """

    def __init__(self, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int,
                 device="cuda", dtype=torch.float16):
        self.page_size = page_size
        self.pool = torch.zeros((num_pages, 2, num_kv_heads, page_size, head_dim), dtype=dtype,
                                device=device)
        self._free = list(range(num_pages - 1, -1, -1))  # pop() hands out page 0 first
        self._pages: dict = {}
        self._len: dict = {}
        self._refs = [0] * num_pages  # sequences that hold each page

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def seq_len(self, seq_id) -> int:
        return self._len.get(seq_id, 0)

    def _drop(self, pages) -> None:
        for page in pages:
            self._refs[page] -= 1
            if self._refs[page] == 0:
                self._free.append(page)

    def release(self, seq_id) -> None:
        """Drop a sequence; pages that no other sequence holds return to the free list."""
        self._drop(reversed(self._pages.pop(seq_id, [])))
        self._len.pop(seq_id, None)

    def truncate(self, seq_id, length: int) -> None:
        """Forget a sequence's tokens from position `length` on (rejected drafts, say)."""
        if not 0 <= length <= self.seq_len(seq_id):
            raise ValueError(f"length {length} is not in [0, {self.seq_len(seq_id)}]")
        if seq_id not in self._pages:
            return
        keep = -(-length // self.page_size)
        pages = self._pages[seq_id]
        self._drop(reversed(pages[keep:]))
        del pages[keep:]
        self._len[seq_id] = length

    def fork(self, seq_id, new_id) -> None:
        """Start sequence new_id with seq_id's tokens.  No data moves: the two share pages until
        one of them writes into a shared one, which it then copies (append, extend)."""
        if seq_id not in self._pages:
            raise KeyError(f"no sequence {seq_id!r}")
        if new_id in self._pages:
            raise ValueError(f"sequence {new_id!r} exists")
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

    def page_table(self, seq_ids):
        """(kv_page_indptr, kv_page_indices, kv_last_page_len) int32 device tensors."""
        indptr, indices, last = [0], [], []
        for s in seq_ids:
            pages = self._pages.get(s, [])
            indices.extend(pages)
            indptr.append(len(indices))
            n = self._len.get(s, 0)
            last.append(0 if n == 0 else (n - 1) % self.page_size + 1)
        dev = self.pool.device
        mk = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        return mk(indptr), mk(indices), mk(last)

    def _indptr(self, counts):
        ap = [0]
        for n in counts:
            ap.append(ap[-1] + int(n))
        return torch.tensor(ap, dtype=torch.int32, device=self.pool.device)

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
               factor=1.0, causal=True, softmax_scale=None, return_lse=False):
        """One attention step: append counts[i] tokens to seq_ids[i] and attend with them.

        q [sum(counts), Hq, D], k_new and v_new [sum(counts), Hkv, D]; with inv_freq, q and k_new
        are rotated by the tokens' positions first (append_paged_kv_rotary).  Returns what
        flash_attention_chunk_paged returns for q over the grown cache.  A call that is refused
        leaves the sequences with the tokens they had.
        """
        total = sum(int(n) for n in counts)
        for name, x in (("q", q), ("k_new", k_new), ("v_new", v_new)):
            if x.shape[0] != total:
                raise ValueError(f"{name} has {x.shape[0]} rows, the counts make {total}")
        before = {s: self._len.get(s) for s in seq_ids}
        self._grow(seq_ids, counts)
        try:
            table = self.page_table(seq_ids)
            q_indptr = self._indptr(counts)
            if inv_freq is None:
                append_paged_kv(k_new, v_new, q_indptr, self.pool, *table)
            else:
                q = append_paged_kv_rotary(q, k_new, v_new, q_indptr, self.pool, *table, inv_freq,
                                           interleaved=interleaved, factor=factor)
            return _ops.chunk_paged(q, q_indptr, self.pool, *table, causal=causal,
                                    softmax_scale=softmax_scale, return_lse=return_lse)
        except BaseException:
            self._restore(before)
            raise


__all__ = ["append_paged_kv", "append_paged_kv_rotary", "copy_pages", "PagedKVCache"]
