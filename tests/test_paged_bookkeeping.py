"""PagedKVCache's page bookkeeping on the host, and refusals that need no GPU."""
import ctypes as C

import pytest
import torch

from attention_kernel_triton_amd import _native as N
from attention_kernel_triton_amd import paged_kv
from attention_kernel_triton_amd.chunk_flash_attention_paged import flash_attention_chunk_paged
from attention_kernel_triton_amd.paged_kv import PagedKVCache
from attention_kernel_triton_amd.rotary import apply_rotary, rotary_frequencies


@pytest.fixture
def host(monkeypatch):
    """Page copies on the CPU, so that the bookkeeping runs without a GPU."""
    from oracle import serving

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

    monkeypatch.setattr(paged_kv, "copy_pages", copy)
    monkeypatch.setattr(paged_kv, "append_paged_kv", append)


def test_random_walk_keeps_every_history(host):
    """Appends, forks, truncations, releases and compactions in a random order: each
    sequence's cached rows stay its own, and every page is counted."""
    g = torch.Generator().manual_seed(7)
    r = lambda n: int(torch.randint(0, n, (1,), generator=g))  # noqa: E731
    cache = PagedKVCache(60, 1, 4, 8, device="cpu")
    hist, names = {}, iter(range(10 ** 6))
    for _ in range(600):
        live = list(hist)
        op = r(10)
        if op < 5 or not live:
            seqs = [s for s in live if r(3) == 0] + ([next(names)] if r(3) == 0 else [])
            counts = [r(7) for _ in seqs]
            k = torch.randn(sum(counts), 1, 8, generator=g).half()
            v = torch.randn(sum(counts), 1, 8, generator=g).half()
            try:
                cache.append(seqs, k, v, counts)
            except MemoryError:
                cache.release(live[0])
                del hist[live[0]]
                continue
            t = 0
            for s, n in zip(seqs, counts):
                old = hist.get(s, (k[:0], v[:0]))
                hist[s] = (torch.cat([old[0], k[t:t + n]]), torch.cat([old[1], v[t:t + n]]))
                t += n
        elif op == 5:
            cache.release(live[r(len(live))])
            hist = {s: h for s, h in hist.items() if s in cache._pages}
        elif op < 8:
            s, new = live[r(len(live))], next(names)
            cache.fork(s, new)
            hist[new] = hist[s]
        elif op == 8:
            s = live[r(len(live))]
            n = r(cache.seq_len(s) + 1)
            cache.truncate(s, n)
            hist[s] = tuple(x[:n] for x in hist[s])
        else:
            cache.compact()
            used = 60 - cache.free_pages
            assert {p for ps in cache._pages.values() for p in ps} == set(range(used))
        refs = [0] * 60
        for ps in cache._pages.values():
            for p in ps:
                refs[p] += 1
        assert refs == cache._refs
        assert sorted(cache._free) == [p for p in range(60) if refs[p] == 0]
        for s, (k, v) in hist.items():
            n = cache.seq_len(s)
            assert n == k.shape[0] and len(cache._pages[s]) == -(-n // 4)
            for t in range(n):
                pg = cache._pages[s][t // 4]
                assert torch.equal(cache.pool[pg, 0, :, t % 4], k[t])
                assert torch.equal(cache.pool[pg, 1, :, t % 4], v[t])


def test_bookkeeping_refusals(host):
    cache = PagedKVCache(4, 1, 4, 8, device="cpu")
    with pytest.raises(KeyError):
        cache.fork("none", "new")
    with pytest.raises(ValueError):
        cache.truncate("none", 1)
    cache.truncate("none", 0)
    z = torch.zeros(3, 1, 8).half()
    cache.append(["a"], z, z, [3])
    with pytest.raises(ValueError):
        cache.fork("a", "a")
    for n in (-1, 4):
        with pytest.raises(ValueError):
            cache.truncate("a", n)
    cache.release("b")  # unknown: nothing to release
    assert cache.free_pages == 3


def test_a_refused_extend_leaves_the_sequences_as_they_were(host):
    cache = PagedKVCache(8, 1, 4, 64, device="cpu")
    z = lambda n, d=64: torch.zeros(n, 1, d).half()  # noqa: E731
    cache.append(["a"], torch.ones(6, 1, 64).half(), torch.ones(6, 1, 64).half(), [6])
    cache.fork("a", "b")
    for q, k, v, counts in ((z(3), z(4), z(4), [3, 1]), (z(4), z(3), z(4), [3, 1]),
                            (z(4), z(4), z(5), [3, 1]), (z(5), z(5), z(5), [3, 1])):
        with pytest.raises(ValueError):  # rows that are not those of the counts
            cache.extend(["a", "c"], q, k, v, counts)
        assert cache.free_pages == 6 and cache.seq_len("a") == 6 and "c" not in cache._pages
    # Attention refuses (here: tensors that are not on a GPU) after pages were taken.
    with pytest.raises(Exception):
        cache.extend(["a", "c"], z(4), z(4), z(4), [3, 1])
    assert cache.seq_len("a") == 6 and cache.seq_len("b") == 6 and "c" not in cache._pages
    assert cache.free_pages == 5  # the copy of the page that a and b shared stays a's
    for s in ("a", "b"):
        for t in range(6):
            assert float(cache.pool[cache._pages[s][t // 4], :, :, t % 4].min()) == 1
    cache.release("a")
    cache.release("b")
    assert cache.free_pages == 8


def _i64(*v):
    return (C.c_int64 * len(v))(*v)


P16 = C.c_void_p(16)


def _chunk(lib, D=128, Hq=8, Hkv=2, page=16, pages=10, scale=0.1, dtype=0, T=4, B=2, q=P16, ss=None,
           ws=P16, ws_n=1 << 40, qst=None):
    qs = _i64(*(qst or (Hq * D, D, 1)))
    ks = _i64(2 * Hkv * page * D, Hkv * page * D, page * D, D if ss is None else ss, 1)
    return lib.akt_chunk_paged_fwd(q, P16, P16, P16, P16, P16, P16, None, B, T, Hq, Hkv, D, page, pages,
                                   pages, qs, ks, scale, 1, dtype, ws, ws_n, None)


@pytest.mark.parametrize("kw,rc,word", [
    (dict(D=96), 2, b"head_dim"), (dict(D=192), 2, b"head_dim"), (dict(Hq=6, Hkv=4), 1, b"multiple"),
    (dict(Hq=129, Hkv=1), 2, b"query heads"), (dict(dtype=1), 1, b"dtype"),
    (dict(scale=float("nan")), 1, b"finite"), (dict(q=C.c_void_p(8)), 1, b"aligned"),
    (dict(qst=(8 * 128, 128, 2)), 1, b"stride"), (dict(qst=(8 * 128 + 4, 128, 1)), 1, b"aligned"),
    (dict(page=0), 1, b"page_size"), (dict(ss=1 << 22), 1, b"slot stride"), (dict(ss=-128), 1, b"slot stride"),
    (dict(pages=1 << 27), 1, b"page table"), (dict(ws=None), 3, b"workspace"), (dict(ws_n=1000), 3, b"workspace"),
    (dict(ws=C.c_void_p(24)), 1, b"workspace"), (dict(q=None), 1, b"pointers"), (dict(T=-1), 1, b"negative"),
    (dict(T=1 << 30), 1, b"large")])
def test_chunk_refusals(kw, rc, word):
    lib = N.load()
    assert _chunk(lib, **kw) == rc
    assert word in lib.akt_last_error()


def test_chunk_workspace_sizes():
    """Small calls ask for little, large ones for two partial slots to each resident workgroup (256
    of eight waves, at D = 256 of four, as assumed without a device), for sequences of many tokens
    and, smaller ones, of few: up to 32 rows to a kv head, whose waves hold a quarter of O each, at
    D = 256 up to 64 and half."""
    ws = N.load().akt_chunk_paged_workspace_size
    zero = -(-N.WORKSPACE_ZERO_BYTES // 256) * 256
    for D, wgs, waves in ((64, 256, 8), (128, 256, 8), (256, 256, 4)):
        o = 32 * D * 4
        many, few = waves * (o + 512), waves * (o // (2 if D == 256 else 4) + 512)
        assert ws(64, 10 ** 4, 32, 8, D, 16, 10 ** 5) == zero + 2 * wgs * (many + few)
        assert ws(1, 10 ** 4, 32, 8, D, 16, 10 ** 5) == zero + 2 * wgs * many
        # 10 tokens of 4 heads: 40 rows, few at D = 256 only.
        assert ws(64, 10, 32, 8, D, 16, 10 ** 5) == zero + 2 * wgs * (few + (0 if D == 256 else many))
        assert ws(64, 8, 32, 8, D, 16, 10 ** 5) == zero + 2 * wgs * few
    slot = lambda D: 8 * (32 * D * 4 + 512)  # noqa: E731
    assert zero < ws(1, 1, 8, 2, 64, 16, 2) < zero + 20 * slot(64)
    assert ws(0, 4, 8, 2, 64, 16, 2) == ws(1, 0, 8, 2, 64, 16, 2) == ws(1, 4, 8, 2, 96, 16, 2) == 0
    lib = N.load()
    assert _chunk(lib, T=0) == 0 and _chunk(lib, B=0) == 0  # nothing to do launches nothing


def _rotary(lib, D=64, rot=64, factor=1.0, dtype=0, q=P16, pos=None, bits=0, S=4, B=1, Hkv=1, inv=P16,
            qst=None):
    qs = _i64(*(qst or (2 * S * D, S * D, D, 1)))
    return lib.akt_rotary_fwd(q, P16, P16, P16, inv, pos, bits, B, 2, Hkv, S, D, rot, qs,
                              _i64(S * D, S * D, D, 1), _i64(0, 1), 0, 0, factor, dtype, None)


@pytest.mark.parametrize("kw,word", [
    (dict(rot=63), b"even"), (dict(rot=66), b"head_dim"), (dict(rot=0), b"even"), (dict(D=60), b"head_dim"),
    (dict(D=1032, rot=8), b"head_dim"), (dict(factor=float("inf")), b"factor"), (dict(dtype=1), b"dtype"),
    (dict(q=C.c_void_p(8)), b"aligned"), (dict(q=None), b"pointers"), (dict(inv=None), b"pointers"),
    (dict(pos=P16, bits=16), b"position_bits"), (dict(S=-1), b"negative"), (dict(qst=(512, 256, 64, 2)), b"stride")])
def test_rotary_refusals(kw, word):
    lib = N.load()
    assert _rotary(lib, **kw) == 1
    assert word in lib.akt_last_error()
    assert _rotary(lib, S=0) == 0 and _rotary(lib, B=0) == 0


def _append(lib, D=64, rot=64, page=16, q=P16, total=4, kst=None, dtype=0):
    s3, s5 = _i64(2 * D, D, 1), _i64(4 * page * D, 2 * page * D, page * D, D, 1)
    return lib.akt_paged_kv_append_rotary(q, P16, P16, P16, P16, P16, P16, P16, P16, P16, 1, total, 2, 2,
                                          D, rot, page, 8, 8, s3, _i64(*kst) if kst else s3, s3, s5, 0, 1.0,
                                          dtype, None)


@pytest.mark.parametrize("kw,word", [
    (dict(rot=3), b"even"), (dict(D=4, rot=4), b"head_dim"), (dict(page=0), b"page_size"),
    (dict(q=None), b"pointers"), (dict(q=C.c_void_p(2)), b"aligned"), (dict(kst=(128, 64, 3)), b"stride"),
    (dict(dtype=7), b"dtype"), (dict(total=-2), b"negative")])
def test_append_rotary_refusals(kw, word):
    lib = N.load()
    assert _append(lib, **kw) == 1
    assert word in lib.akt_last_error()
    assert _append(lib, total=0) == 0


def _copy(lib, pool=P16, n=3, D=64, page=16, Hkv=2, s=None):
    return lib.akt_paged_copy(pool, P16, P16, None, n, Hkv, D, page, 8,
                              _i64(*(s or (2 * Hkv * page * D, Hkv * page * D, page * D, D, 1))), None)


@pytest.mark.parametrize("kw,word", [
    (dict(pool=None), b"pointers"), (dict(pool=C.c_void_p(4)), b"aligned"), (dict(D=12), b"head_dim"),
    (dict(page=0), b"page_size"), (dict(n=-1), b"negative"), (dict(s=(4096, 2048, 1024, 64, 2)), b"stride"),
    (dict(s=(4096, 2048, 1024, -64, 1)), b"strides"), (dict(n=1 << 31), b"too many")])
def test_copy_refusals(kw, word):
    lib = N.load()
    assert _copy(lib, **kw) == 1
    assert word in lib.akt_last_error()
    assert _copy(lib, n=0) == 0


def test_cpu_tensors_and_arguments_are_refused():
    h = torch.float16
    i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    q, pool = torch.zeros(2, 4, 64, dtype=h), torch.zeros(3, 2, 2, 16, 64, dtype=h)
    k = torch.zeros(2, 2, 64, dtype=h)
    inv, factor = rotary_frequencies(64, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        flash_attention_chunk_paged(q, i(0, 2), pool, i(0, 1), i(0), i(2))
    with pytest.raises(ValueError, match="GPU"):
        apply_rotary(torch.zeros(1, 2, 3, 64, dtype=h), None, inv)
    with pytest.raises(ValueError, match="GPU"):
        paged_kv.append_paged_kv_rotary(q, k, k, i(0, 2), pool, i(0, 1), i(0), i(2), inv)
    with pytest.raises(ValueError, match="GPU"):
        paged_kv.copy_pages(pool, i(0), i(1))
    for kw in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=0.0),
               dict(rotary_dim=8, stretch=0.5), dict(rotary_dim=8, scaling="other"),
               dict(rotary_dim=2, scaling="ntk", stretch=2.0), dict(rotary_dim=8, scaling="yarn", stretch=2.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(device="cpu", **kw)


@pytest.mark.gpu
def test_argument_refusals_on_the_device(dev):
    h = torch.float16
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    z = lambda *s, dtype=h: torch.zeros(s, dtype=dtype, device=dev)  # noqa: E731
    pool, q, k = z(3, 2, 2, 16, 64), z(2, 4, 64), z(2, 2, 64)
    inv, _ = rotary_frequencies(64, device=dev)
    chunk = [q, i(0, 2), pool, i(0, 1), i(0), i(2)]
    append = [q, k, k, i(0, 2), pool, i(0, 1), i(0), i(2), inv]
    wrong = [(flash_attention_chunk_paged, chunk, n, bad, err) for n, bad, err in (
        (0, q.float(), TypeError), (0, q.bfloat16(), TypeError), (0, z(2, 4, 128), ValueError),
        (0, z(2, 4, 1, 64), ValueError), (0, z(2, 3, 64), RuntimeError), (1, i(0, 1, 2), ValueError),
        (1, i(0, 2).long(), TypeError), (2, pool[:, :1], ValueError), (2, pool[0], ValueError),
        (3, i(0), ValueError), (4, i(0).cpu(), ValueError), (5, i(2, 2), ValueError))]
    wrong += [(paged_kv.append_paged_kv_rotary, append, n, bad, err) for n, bad, err in (
        (0, q.bfloat16(), TypeError), (0, q[:1], ValueError), (1, z(2, 3, 64), ValueError),
        (2, k[:1], ValueError), (4, pool.float(), TypeError), (4, pool.transpose(3, 4), ValueError),
        (3, i(0, 1, 2), ValueError), (8, inv.float(), TypeError), (8, inv.cpu(), ValueError),
        (8, torch.cat([inv, inv]), RuntimeError), (8, inv[:0], RuntimeError), (8, inv[None], ValueError))]
    wrong += [(paged_kv.copy_pages, [pool, i(0), i(1), i(3)], n, bad, err) for n, bad, err in (
        (0, pool.float(), TypeError), (1, i(0, 1), ValueError), (2, i(1).long(), TypeError), (3, i(1, 2), ValueError))]
    Q, K = z(1, 2, 5, 64), z(1, 1, 5, 64)
    wrong += [(apply_rotary, [Q, K, inv, i(0, 1, 2, 3, 4)], n, bad, err) for n, bad, err in (
        (0, Q.float(), TypeError), (0, Q[0], ValueError), (1, K.bfloat16(), TypeError), (1, z(1, 1, 4, 64), ValueError),
        (3, i(0, 1), ValueError), (3, i(0, 1, 2, 3, 4).float(), TypeError), (3, i(0, 1, 2, 3, 4)[None].expand(2, 5), ValueError))]
    for fn, args, n, bad, err in wrong:
        fn(*args)
        with pytest.raises(err):
            fn(*args[:n], bad, *args[n + 1:])
    torch.cuda.synchronize()


def _state(cache):
    return (list(cache._free), {s: list(p) for s, p in cache._pages.items()}, dict(cache._len),
            list(cache._refs))


def _shared(n=6):
    """Sequences a and b that share n tokens (two pages, the second one partly filled)."""
    cache = PagedKVCache(8, 1, 4, 8, device="cpu")
    cache.append(["a"], torch.ones(n, 1, 8).half(), torch.ones(n, 1, 8).half(), [n])
    cache.fork("a", "b")
    return cache


def _refuse(*args, **kw):
    raise TypeError("refused")


def test_a_refused_append_leaves_the_sequences_as_they_were(host, monkeypatch):
    cache = PagedKVCache(8, 1, 4, 8, device="cpu")
    z = lambda n: torch.zeros(n, 1, 8).half()  # noqa: E731
    cache.append(["a"], z(6), z(6), [6])
    before = _state(cache)
    monkeypatch.setattr(paged_kv, "append_paged_kv", _refuse)  # as for a wrong type or head dim
    with pytest.raises(TypeError):
        cache.append(["a", "c"], z(9), z(9), [4, 5])
    after = _state(cache)
    assert sorted(after[0]) == sorted(before[0]) and after[1:] == before[1:]
    with pytest.raises(TypeError):
        cache.append(["a", "c"], z(0), z(0), [0, 0])
    assert _state(cache)[1:] == before[1:]


def test_an_append_of_too_few_rows_is_refused(host):
    cache = _shared()
    before = _state(cache)
    z = lambda n: torch.zeros(n, 1, 8).half()  # noqa: E731
    for k, v in ((z(3), z(3)), (z(3), z(4)), (z(4), z(3))):
        with pytest.raises(ValueError, match="rows"):
            cache.append(["a", "c"], k, v, [3, 1])
        assert _state(cache) == before
    cache.append(["a", "c"], z(7), z(7), [3, 1])  # rows past the counts belong to no sequence
    assert cache.seq_len("a") == 9 and cache.seq_len("c") == 1


@pytest.mark.parametrize("call", ["append", "extend"])
def test_a_failed_page_copy_changes_nothing(host, monkeypatch, call):
    """The copy of a shared page may be refused (a stream under capture, say): neither sequence then
    holds the page that was meant for it."""
    cache = _shared()
    before, pool = _state(cache), cache.pool.clone()
    x = torch.zeros(3, 1, 8).half()
    monkeypatch.setattr(paged_kv, "copy_pages", _refuse)
    with pytest.raises(TypeError):
        if call == "append":
            cache.append(["a", "c"], x, x, [2, 1])
        else:
            cache.extend(["a", "c"], x, x, x, [2, 1])
    assert _state(cache) == before and torch.equal(cache.pool, pool)


def test_launches_past_the_runtimes_limit_are_refused():
    """Grids of 2^32 work items and more."""
    lib = N.load()
    assert _copy(lib, n=1 << 24) == 1 and b"too many pages" in lib.akt_last_error()
    assert _rotary(lib, S=1 << 30) == 1 and b"too large" in lib.akt_last_error()
    assert _rotary(lib, S=1 << 29, D=72, rot=72) == 1 and b"too large" in lib.akt_last_error()
    assert _append(lib, total=1 << 26) == 1 and b"too many tokens" in lib.akt_last_error()
