"""Eviction and shared prefixes on the host: PagedKVCache's bookkeeping with the kernels' work done
on the CPU, and refusals that need no GPU."""
import ctypes as C

import pytest
import torch

from attention_kernel_triton_amd import _native as N
from attention_kernel_triton_amd import paged_kv
from attention_kernel_triton_amd.attention_weights_paged import accumulate_attention_weights_paged
from attention_kernel_triton_amd.kept_index import select_heaviest
from attention_kernel_triton_amd.paged_kv import PagedKVCache, append_paged_kv_rotary, keep_tokens
from attention_kernel_triton_amd.shared_prefix_flash_attention_paged import (
    flash_attention_shared_prefix_paged)
from oracle import serving


@pytest.fixture
def host(monkeypatch):
    def copy(pool, src, dst, num_tokens=None):
        pool.copy_(serving.copy_pages(pool, src.tolist(), dst.tolist(),
                                      None if num_tokens is None else num_tokens.tolist()))

    def append(k, v, ap, pool, indptr, indices, last):
        page = pool.shape[3]
        for b in range(len(last)):
            n = int(ap[b + 1] - ap[b])
            length = (int(indptr[b + 1] - indptr[b]) - 1) * page + int(last[b])
            for i in range(n):
                t = length - n + i
                pg = int(indices[int(indptr[b]) + t // page])
                pool[pg, 0, :, t % page] = k[int(ap[b]) + i]
                pool[pg, 1, :, t % page] = v[int(ap[b]) + i]

    def move(pool, indptr, indices, last, ind, nnz, dst_page_indices=None, weights=None, rows=None):
        p, w = serving.keep_tokens(pool, indptr, indices, last, ind, nnz, dst_page_indices, weights, rows)
        pool.copy_(p)
        weights.copy_(w)

    monkeypatch.setattr(paged_kv, "copy_pages", copy)
    monkeypatch.setattr(paged_kv, "append_paged_kv", append)
    monkeypatch.setattr(paged_kv, "keep_tokens", move)
    monkeypatch.setattr(paged_kv, "select_heaviest",
                        lambda w, n, keep, first=0, recent=0, rows=None:
                        serving.heaviest(w, n.tolist(), keep, first, recent, rows))


def rows_of(cache, s):
    """K of the sequence's tokens, by head: [Hkv, len, D]."""
    n = cache.seq_len(s)
    kv = cache.pool[torch.tensor(cache._pages[s], dtype=torch.long)]
    return kv.permute(1, 2, 0, 3, 4).reshape(2, kv.shape[2], -1, kv.shape[4])[:, :, :n]


def test_random_walk_with_evictions(host):
    """Every sequence holds the tokens that its own history of appends, cuts and evictions leaves,
    and its sums with them; pages and rows are counted."""
    g = torch.Generator().manual_seed(3)
    r = lambda n: int(torch.randint(0, n, (1,), generator=g))  # noqa: E731
    cache = PagedKVCache(70, 2, 4, 8, device="cpu", weight_rows=9, weight_len=64)
    hist, names = {}, iter(range(10 ** 6))  # [K and V, sums, tokens dropped]
    evicted = 0
    for _ in range(700):
        live = list(hist)
        op = r(12)
        if op < 5 or not live:
            seqs = [s for s in live if r(3) == 0 and cache.seq_len(s) < 50]
            if len(live) < 8:
                seqs.append(next(names))
            counts = [1 + r(7) for _ in seqs]
            k, v = (torch.randn(sum(counts), 2, 8, generator=g).half() for _ in range(2))
            try:
                cache.append(seqs, k, v, counts)
            except MemoryError:
                cache.release(live[0])
                del hist[live[0]]
                continue
            rows = cache._row_table(seqs)
            t = 0
            for s, n, row in zip(seqs, counts, rows.tolist()):
                new = torch.stack((k[t:t + n], v[t:t + n])).transpose(1, 2)
                old = hist.setdefault(s, [new[:, :, :0], torch.zeros(2, 0), 0])
                m = old[1].shape[1]
                draw = torch.rand(2, m + n, generator=g)  # what the step's queries draw
                cache.weights[row, :, :m + n] += draw
                hist[s] = [torch.cat((old[0], new), 2),
                           torch.cat((old[1], torch.zeros(2, n)), 1) + draw, old[2]]
                t += n
        elif op < 8:
            seqs = [s for s in live if r(2) == 0]
            keep = 3 + r(20)
            first, recent = r(2), r(3)
            free = (list(cache._free), {s: list(p) for s, p in cache._pages.items()})
            try:
                got = cache.evict(seqs, keep, first, recent)
            except MemoryError:
                assert free == (cache._free, cache._pages)
                continue
            want = 0
            for s in seqs:
                kv, w, lost = hist[s]
                n = w.shape[1]
                if n <= keep:
                    continue
                ind = serving.heaviest(w[None], [n], keep, first, recent)[0][0].long()
                hist[s] = [torch.stack([kv[:, h, ind[h]] for h in range(2)], 1),
                           torch.stack([w[h, ind[h]] for h in range(2)]), lost + n - keep]
                want += n - keep
            assert got == want
            evicted += got
        elif op == 8 and len(live) < 8:
            s, t = live[r(len(live))], next(names)
            cache.fork(s, t)
            hist[t] = list(hist[s])
        elif op == 9:
            s = live[r(len(live))]
            n = r(cache.seq_len(s) + 1)
            cache.truncate(s, n)
            hist[s] = [hist[s][0][:, :, :n], hist[s][1][:, :n], hist[s][2] if n else 0]
        elif op == 10:
            s = live[r(len(live))]
            cache.release(s)
            del hist[s]
        elif op == 11:
            cache.compact()
        for s, (kv, w, lost) in hist.items():
            assert cache.seq_len(s) == w.shape[1] and cache.next_position(s) == w.shape[1] + lost
            assert torch.equal(rows_of(cache, s), kv)
            if s in cache._rows:
                row = cache.weights[cache._rows[s]]
                assert torch.allclose(row[:, :w.shape[1]], w, atol=1e-5) and not row[:, w.shape[1]:].any()
        held = [p for s in hist for p in cache._pages[s]]
        assert sorted(set(held) | set(cache._free)) == list(range(70))
        assert all(cache._refs[p] == held.count(p) for p in range(70))
        assert len(cache._free_rows) + len(cache._rows) == 9
    assert evicted > 300


def test_evictions_that_are_refused_change_nothing(host):
    cache = PagedKVCache(6, 1, 4, 8, device="cpu", weight_rows=2, weight_len=20)
    z = lambda n: torch.randn(n, 1, 8).half()  # noqa: E731
    cache.append([0], z(20), z(20), [20])
    cache.fork(0, 1)
    state = lambda: (list(cache._free), {s: list(p) for s, p in cache._pages.items()},  # noqa: E731
                     dict(cache._len), list(cache._refs), dict(cache._rows), cache.pool.clone())
    before = state()
    with pytest.raises(MemoryError):
        cache.evict([0], 10)  # three shared pages to replace, one free
    with pytest.raises(ValueError):
        cache.evict([0], 0)
    with pytest.raises(ValueError):
        cache.evict([0], 5, first=3, recent=3)
    assert before[:5] == state()[:5] and torch.equal(before[5], cache.pool)
    assert cache.evict([0, 1], 20) == 0 and cache.evict([], 3) == 0 and cache.evict(["none"], 3) == 0
    cache.release(1)
    cache.append([0], z(1), z(1), [1])
    with pytest.raises(ValueError, match="sums hold"):
        cache.evict([0], 10)
    cache.truncate(0, 20)
    assert cache.evict([0, 0], 9, recent=9) == 11 and cache.seq_len(0) == 9
    assert cache.next_position(0) == 20 and cache.free_pages == 3
    plain = PagedKVCache(6, 1, 4, 8, device="cpu")
    with pytest.raises(ValueError, match="sums"):
        plain.evict([0], 3)
    cache.append([1], z(1), z(1), [1])
    cache._row_table([0, 1])
    with pytest.raises(MemoryError, match="rows"):
        cache._row_table([2])
    with pytest.raises(MemoryError, match="rows"):
        cache.fork(0, 5)
    assert 5 not in cache._pages


def test_groups_of_shared_pages(host):
    cache = PagedKVCache(80, 1, 4, 8, device="cpu")
    z = lambda n: torch.randn(n, 1, 8).half()  # noqa: E731
    cache.append(["a"], z(41), z(41), [41])
    for s in ("b", "c", "d"):
        cache.fork("a", s)
    cache.append(["a", "b", "c"], z(6), z(6), [2, 1, 3])
    cache.append(["x"], z(9), z(9), [9])
    cache.truncate("d", 7)
    cache.append(["d"], z(30), z(30), [30])  # shares one whole page
    own = lambda seqs, counts=None: [t.tolist() for t in cache.split_table(seqs, counts)]  # noqa: E731
    indptr, indices, last, group, pptr, pind, plast = own(["a", "b", "c", "x"])
    assert group == [0, 3, 4] and pptr == [0, 10, 10] and pind == cache._pages["a"][:10] and plast == [4, 0]
    assert indices == [p for s in "abc" for p in cache._pages[s][10:]] + cache._pages["x"]
    assert indptr == [0, 1, 2, 3, 6] and last == [3, 2, 4, 1]
    # One page in common would cost the group its other nine; alone with one it joins.
    assert own(["a", "b", "d"])[3] == [0, 2, 3] and own(["a", "d"])[3] == [0, 2]
    assert own(["a", "d"])[4] == [0, 1]
    # A sequence between breaks a group; pages with new tokens stay out.
    assert own(["a", "x", "b"])[3] == [0, 1, 2, 3]
    assert own(["a", "b"], [9, 2])[4] == [0, 8] and own(["a", "b"], [99, 1])[4] == [0, 0, 0]
    assert own([])[3] == [0] and own(["none", "a"])[3] == [0, 1, 2]


# --------------------------------------------------------------------------- refusals
def _i64(*v):
    return (C.c_int64 * len(v))(*v)


P16 = C.c_void_p(16)


def test_shared_prefix_refuses_before_any_launch():
    lib = N.load()
    size = lib.akt_shared_prefix_paged_workspace_size
    need = size(4, 4, 8, 2, 128, 16, 40, 1, 20)
    assert need > size(4, 4, 8, 2, 64, 16, 40, 1, 20) > 0
    for bad in ((0, 4, 8, 2, 128, 16, 40, 1, 20), (4, 4, 8, 3, 128, 16, 40, 1, 20),
                (4, 4, 8, 2, 96, 16, 40, 1, 20), (4, 4, 8, 2, 128, 16, 40, -1, 20),
                (4, 4, 8, 2, 128, 16, 40, 1, -1), (4, 4, 8, 2, 128, 0, 40, 1, 20)):
        assert size(*bad) == 0

    def call(B=4, T=4, Hq=8, Hkv=2, D=128, page=16, total=40, groups=1, prefix=20, P=60, scale=0.1,
             dtype=0, ws=P16, n=need, q=P16, group=P16, qs=(1024, 128, 1)):
        return lib.akt_shared_prefix_paged_fwd(
            q, P16, P16, P16, P16, P16, group, P16, P16, P16, P16, None, B, T, Hq, Hkv, D, page, total,
            groups, prefix, P, _i64(*qs), _i64(8192, 4096, 2048, 128, 1), scale, 1, dtype, ws, n, None)

    for rc, kw in ((1, {"dtype": 1}), (1, {"groups": -1}), (1, {"prefix": -1}), (1, {"Hkv": 3}),
                   (2, {"D": 96}), (1, {"page": 0}), (1, {"prefix": 1 << 29}), (1, {"group": None}),
                   (1, {"q": C.c_void_p(8)}), (1, {"qs": (1024, 128, 2)}), (3, {"n": need - 1}),
                   (3, {"ws": None}), (1, {"scale": float("nan")}), (1, {"T": 1 << 25}),
                   (2, {"Hq": 258})):
        assert call(**kw) == rc, (kw, lib.akt_last_error())
    assert call(B=0) == 0 and call(T=0) == 0


def test_attention_weights_refuse_before_any_launch():
    lib = N.load()
    size = lib.akt_attention_weights_paged_workspace_size
    need = size(4, 4, 8, 2, 128, 16, 40)
    assert need > N.WORKSPACE_ZERO_BYTES
    assert size(0, 4, 8, 2, 128, 16, 40) == size(4, 4, 8, 3, 128, 16, 40) == size(4, 4, 8, 2, 96, 16, 40) == 0

    def call(B=4, T=4, Hq=8, Hkv=2, D=128, page=16, total=40, P=60, rows=4, L=100, scale=0.1, dtype=0,
             window=1 << 40, q=P16, lse=P16, w=P16, which=P16, ks=(8192, 4096, 2048, 128, 1), ws=P16,
             n=need):
        return lib.akt_attention_weights_paged(
            q, P16, lse, P16, P16, P16, P16, w, which, B, T, Hq, Hkv, D, page, total, P, rows, L,
            _i64(1024, 128, 1), _i64(*ks), _i64(200, 100), scale, 1, window, dtype, ws, n, None)

    for rc, kw in ((1, {"dtype": 1}), (1, {"rows": -1}), (1, {"window": -1}), (1, {"Hkv": 3}),
                   (2, {"D": 192}), (1, {"page": 0}), (1, {"lse": None}), (1, {"w": None}),
                   (1, {"which": None, "rows": 3}), (1, {"q": C.c_void_p(8)}),
                   (1, {"ks": (8192, 4096, 2048, 128, 2)}), (1, {"ks": (8192, 4096, 2048, 100, 1)}),
                   (1, {"scale": float("inf")}), (1, {"w": C.c_void_p(18)}),
                   (1, {"total": 1 << 28}), (1, {"T": 1 << 29}), (3, {"n": need - 1}), (3, {"ws": None})):
        assert call(**kw) == rc, (kw, lib.akt_last_error())
    assert all(call(**kw) == 0 for kw in ({"B": 0}, {"T": 0}, {"rows": 0}, {"L": 0}, {"window": 0}))


def test_selections_and_moves_refuse_before_any_launch():
    lib = N.load()

    def select(B=2, H=2, rows=2, L=50, keep=10, first=2, recent=3, w=P16, n=P16, which=P16, ind=P16):
        return lib.akt_kept_index_heaviest(w, n, which, ind, P16, B, H, rows, L, _i64(100, 50), keep,
                                           first, recent, None)

    for kw in ({"keep": 4}, {"first": -1}, {"recent": 9}, {"L": 1 << 28}, {"w": None}, {"n": None},
               {"ind": None}, {"which": None, "rows": 1}, {"w": C.c_void_p(6)}, {"B": -1}):
        assert select(**kw) == 1, kw
    assert select(B=0) == 0 and select(H=0) == 0

    def move(B=2, H=2, D=64, page=16, total=8, P=9, keep=10, rows=2, L=50, w=P16, ind=P16, which=P16,
             ks=(4096, 2048, 1024, 64, 1)):
        return lib.akt_paged_keep(P16, P16, P16, P16, None, ind, P16, w, which, B, H, D, page, total, P,
                                  keep, rows, L, _i64(*ks), _i64(100, 50), None)

    for kw in ({"D": 68}, {"D": 2048}, {"page": 0}, {"keep": -1}, {"ind": None}, {"H": 0},
               {"ks": (4096, 2048, 1024, 64, 2)}, {"ks": (4096, 2048, 1024, 60, 1)},
               {"which": None, "rows": 1}, {"total": 1 << 28}, {"w": C.c_void_p(6)}):
        assert move(**kw) == 1, kw
    assert move(B=0) == 0 and move(total=0) == 0


def test_cpu_tensors_are_refused():
    q, pool = torch.zeros(1, 2, 64).half(), torch.zeros(2, 2, 1, 16, 64).half()
    i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    t = (i(0, 1), i(0), i(3))
    w = torch.zeros(1, 1, 20)
    with pytest.raises(ValueError):
        flash_attention_shared_prefix_paged(q, i(0, 1), pool, *t, i(0, 1), i(0, 1), i(1), i(2))
    with pytest.raises(ValueError):
        accumulate_attention_weights_paged(w, q, i(0, 1), torch.zeros(1, 2), pool, *t)
    with pytest.raises(ValueError):
        select_heaviest(w, i(3), 2)
    with pytest.raises(ValueError):
        keep_tokens(pool, *t, torch.zeros(1, 1, 2, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(ValueError):
        append_paged_kv_rotary(q, q, q, i(0, 1), pool, *t, torch.zeros(4, dtype=torch.float64),
                               position_offset=i(3))
