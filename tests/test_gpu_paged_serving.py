"""Page copies, and PagedKVCache's steps as a serving loop makes them."""
import math

import pytest
import torch

from attention_kernel_triton_amd import decode_flash_attention_redundant_var_len_paged as pg
from attention_kernel_triton_amd.paged_kv import PagedKVCache, copy_pages
from attention_kernel_triton_amd.rotary import rotary_frequencies
from helpers import assert_close
from oracle import serving

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hkv,page,D", [(8, 16, 128), (1, 1, 64), (3, 7, 72), (2, 64, 256), (5, 100, 1024)])
@pytest.mark.parametrize("partial", [False, True])
def test_copies_are_bit_exact(dev, Hkv, page, D, partial, dtype):
    g = torch.Generator().manual_seed(page + D)
    P, N = 23, 9
    pool = torch.randn(P, 2, Hkv, page, D, generator=g).to(dtype)
    order = torch.randperm(P, generator=g).to(torch.int32)
    src, dst = order[:N].clone(), order[N:2 * N].clone()
    src[2], dst[5], src[6], dst[6] = -1, P, order[20], order[20]  # skipped pairs
    n = torch.randint(-1, page + 2, (N,), generator=g).to(torch.int32) if partial else None
    got = pool.clone().to(dev)
    copy_pages(got, src.to(dev), dst.to(dev), None if n is None else n.to(dev))
    assert torch.equal(got.cpu(), serving.copy_pages(pool, src.tolist(), dst.tolist(), n))


def test_copies_in_a_strided_pool(dev):
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(6, 2, 4, 32, 128, generator=g).half().to(dev)
    before = wide.clone()
    pool = wide[:, :, 1::2, ::2, 64:]
    i32 = dict(dtype=torch.int32, device=dev)
    copy_pages(pool, torch.tensor([0, 4], **i32), torch.tensor([5, 1], **i32),
               torch.tensor([3, 16], **i32))
    want = before.clone()
    want[:, :, 1::2, ::2, 64:] = serving.copy_pages(before[:, :, 1::2, ::2, 64:].cpu(), [0, 4], [5, 1],
                                                    [3, 16]).to(dev)
    assert torch.equal(wide, want)
    copy_pages(pool, torch.zeros(0, **i32), torch.zeros(0, **i32))
    assert torch.equal(wide, want)


def test_copies_past_32_bit_offsets(dev):
    """Pages of a pool of more than 2^32 elements (8.6 GB)."""
    page, Hkv, D = 64, 8, 128
    per = 2 * Hkv * page * D
    P = 2 ** 32 // per + 3
    pool = torch.empty((P, 2, Hkv, page, D), dtype=torch.float16, device=dev)
    pool[0], pool[P - 1], pool[P - 2] = 1.0, 2.0, 3.0
    i32 = dict(dtype=torch.int32, device=dev)
    copy_pages(pool, torch.tensor([P - 1, 0], **i32), torch.tensor([1, P - 2], **i32))
    assert float(pool[1].float().min()) == 2 and float(pool[P - 2].float().max()) == 1
    from attention_kernel_triton_amd.chunk_flash_attention_paged import flash_attention_chunk_paged
    from attention_kernel_triton_amd.paged_kv import append_paged_kv_rotary
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(70, h, D, generator=g).half() for h in (16, 8, 8))
    ap = torch.tensor([0, 70], **i32)
    table = (torch.tensor([0, 2], **i32), torch.tensor([P - 1, P - 2], **i32), torch.tensor([6], **i32))
    inv, _ = rotary_frequencies(D, device=dev)
    qr = append_paged_kv_rotary(q.to(dev), k.to(dev), v.to(dev), ap, pool, *table, inv)
    o = flash_attention_chunk_paged(qr, ap, pool, *table)
    small = pool[P - 2:].clone()
    o2 = flash_attention_chunk_paged(qr, ap, small, table[0], torch.tensor([1, 0], **i32), table[2])
    assert torch.equal(o, o2)
    ref = serving.chunk_attention(qr.cpu(), ap.cpu(), small.cpu(), table[0].cpu(), torch.tensor([1, 0]),
                                  table[2].cpu())
    assert_close(o, ref[0], atol=3 * 2.0 ** -11 * 4.5)
    kr = serving.rotate(k, torch.arange(70)[:, None], inv.cpu())
    assert_close(small[1, 0].transpose(0, 1), kr[:64], atol=2.0 ** -11 * 8 + 3e-5)


class Model:
    """A layer's worth of random projections and the dense history of every sequence."""

    def __init__(self, Hq, Hkv, D, dtype, seed):
        self.g = torch.Generator().manual_seed(seed)
        self.shape, self.dtype, self.hist = (Hq, Hkv, D), dtype, {}

    def tokens(self, n):
        Hq, Hkv, D = self.shape
        mk = lambda h: torch.randn(n, h, D, generator=self.g).to(self.dtype)  # noqa: E731
        return mk(Hq), mk(Hkv), mk(Hkv)

    def add(self, s, k, v):
        old = self.hist.get(s)
        self.hist[s] = (k, v) if old is None else (torch.cat([old[0], k]), torch.cat([old[1], v]))

    def attend(self, s, q, inv, **kw):
        """fp64 attention of the last tokens of s; rotated in fp64 and rounded as the cache is."""
        k, v = self.hist[s]
        n, m = k.shape[0], q.shape[0]
        if inv is not None:
            k = serving.rotate(k, torch.arange(n)[:, None], inv, **kw).to(self.dtype)
            q = serving.rotate(q, torch.arange(n - m, n)[:, None], inv, **kw).to(self.dtype)
        pool = torch.stack([k, v]).permute(0, 2, 1, 3)[None]  # one page
        return serving.chunk_attention(q, [0, m], pool, [0, 1], torch.tensor([0]), [n])


def _tol(dtype):
    """3 u A of the attention (A below 3 here) and, where a rotated element of q or k falls on the
    other side of a rounding than in fp64, a step of it: scores move by up to
    2 u |q||k| scale / sqrt(D) or so, far less than the first."""
    return 4 * torch.finfo(dtype).eps / 2 * 3


@pytest.mark.parametrize("dtype,page,interleaved", [(torch.float16, 16, False), (torch.bfloat16, 7, True)])
def test_a_serving_loop(dev, dtype, page, interleaved):
    """Prompts in chunks, decode steps, a fork that diverges, rejected drafts, a release, a
    compaction: after each step the outputs are those of attention over each history."""
    Hq, Hkv, D = 8, 2, 128
    m = Model(Hq, Hkv, D, dtype, page)
    inv, fac = rotary_frequencies(64, 10000.0, "yarn", 4.0, 64, "cpu")
    kw = dict(interleaved=interleaved, factor=fac)
    cache = PagedKVCache(400 // page + 60, Hkv, page, D, device=dev, dtype=dtype)

    def step(seqs, counts):
        q, k, v = m.tokens(sum(counts))
        o = cache.extend(seqs, q.to(dev), k.to(dev), v.to(dev), counts, inv_freq=inv.to(dev), **kw).cpu()
        t = 0
        for s, n in zip(seqs, counts):
            if n:
                m.add(s, k[t:t + n], v[t:t + n])
                ref = m.attend(s, q[t:t + n], inv, **kw)[0]
                assert_close(o[t:t + n], ref, atol=_tol(dtype), what=f"sequence {s}")
            t += n

    step(["a", "b"], [37, 5])
    step(["a", "b"], [50, 1])
    cache.fork("a", "c")
    m.hist["c"] = m.hist["a"]
    used = cache.free_pages
    step(["a", "c", "b"], [1, 4, 0])   # both write into the shared last page
    assert cache.free_pages == used - 1
    step(["c", "a"], [3, 6])
    cache.truncate("c", 60)             # back into pages that a still holds
    m.hist["c"] = tuple(x[:60] for x in m.hist["c"])
    step(["c", "a", "b"], [2, 1, 1])
    cache.release("a")
    del m.hist["a"]
    cache.fork("c", "d")
    m.hist["d"] = m.hist["c"]
    step(["d"], [9])
    cache.release("b")
    del m.hist["b"]
    moved = cache.compact()
    assert moved > 0 and cache.compact() == 0
    live = {p for s in ("c", "d") for p in cache._pages[s]}
    assert live == set(range(cache.pool.shape[0] - cache.free_pages))
    cache.pool[len(live):] = math.nan   # nothing lives there
    step(["d", "c"], [1, 1])
    cache.release("c")
    cache.release("d")
    assert cache.free_pages == cache.pool.shape[0] and not any(cache._refs)


def test_a_forked_sequence_decodes(dev):
    """fork, append and the single-token decode: the fork's tokens do not show in the original."""
    m = Model(4, 1, 64, torch.float16, 3)
    cache = PagedKVCache(20, 1, 16, 64, device=dev)
    _, k, v = m.tokens(21)
    cache.append([0], k.to(dev), v.to(dev), [21])
    m.add(0, k, v)
    cache.fork(0, 1)
    m.hist[1] = m.hist[0]
    for s in (1, 0):
        q, k, v = m.tokens(1)
        indptr, indices, last = cache.append([s], k.to(dev), v.to(dev), [1])
        m.add(s, k, v)
        o = pg.flash_attention_decode_paged(q[:, :, None].to(dev), cache.pool, indptr, indices, last)
        assert_close(o, m.attend(s, q, None)[0])
    o = cache.extend([0, 1], *(x.to(dev) for x in m.tokens(0)), [0, 0])
    assert o.shape == (0, 4, 64)


def test_extend_without_rotation_and_with_lse(dev):
    m = Model(4, 2, 64, torch.float16, 5)
    cache = PagedKVCache(20, 2, 16, 64, device=dev)
    q, k, v = m.tokens(30)
    o, lse = cache.extend([7], q.to(dev), k.to(dev), v.to(dev), [30], causal=False, softmax_scale=0.2,
                          return_lse=True)
    pool = torch.stack([k, v]).permute(0, 2, 1, 3)[None]
    ref = serving.chunk_attention(q, [0, 30], pool, [0, 1], torch.tensor([0]), [30], False, 0.2)
    assert_close(o, ref[0])
    assert_close(lse, ref[1], atol=1e-4)


def test_refused_growth_changes_nothing(dev):
    cache = PagedKVCache(3, 1, 4, 64, device=dev)
    z = lambda n: torch.zeros(n, 1, 64, dtype=torch.float16, device=dev)  # noqa: E731
    cache.append([0], z(6), z(6), [6])
    cache.fork(0, 1)
    state = (list(cache._free), {s: list(p) for s, p in cache._pages.items()}, dict(cache._len),
             list(cache._refs))
    for seqs, counts in (([0, 1], [1, 9]), ([2, 0], [1, 3]), ([0, 1], [3, 1])):
        with pytest.raises(MemoryError):
            cache.append(seqs, z(sum(counts)), z(sum(counts)), counts)
        assert state == (cache._free, cache._pages, cache._len, cache._refs)
    for seqs, counts in (([0, 0], [1, 1]), ([0], [-1]), ([0, 1], [1])):
        with pytest.raises(ValueError):
            cache.append(seqs, z(2), z(2), counts)
        assert state == (cache._free, cache._pages, cache._len, cache._refs)
    cache.append([0, 1], z(2), z(2), [1, 1])  # one copy, the other keeps the page
    assert cache.free_pages == 0 and cache.seq_len(1) == 7
