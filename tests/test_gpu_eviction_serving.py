"""PagedKVCache's steps with sums of attention weight, evictions and shared prefixes, as a serving
loop makes them, against fp64 attention over the tokens that each head still holds."""
import math

import pytest
import torch

from attention_kernel_triton_amd.kept_index import select_heaviest
from attention_kernel_triton_amd.paged_kv import PagedKVCache, append_paged_kv_rotary
from attention_kernel_triton_amd.rotary import rotary_frequencies
from attention_kernel_triton_amd.sparsetoken_decode_flash_attention_redundant_var_len_paged import (
    sparsetoken_flash_attention_decode_paged)
from helpers import assert_close
from oracle import serving

pytestmark = pytest.mark.gpu


class Model:
    """Each sequence's tokens by kv head: K (not rotated), V, positions, and sums."""

    def __init__(self, Hq, Hkv, D, dtype, inv, seed, **kw):
        self.g = torch.Generator().manual_seed(seed)
        self.Hq, self.Hkv, self.D, self.dtype, self.inv, self.kw = Hq, Hkv, D, dtype, inv, kw
        self.hist, self.next = {}, {}

    def tokens(self, n):
        mk = lambda h: torch.randn(n, h, self.D, generator=self.g).to(self.dtype)  # noqa: E731
        return mk(self.Hq), mk(self.Hkv), mk(self.Hkv)

    def add(self, s, k, v):
        n, at = k.shape[0], self.next.get(s, 0)
        pos = torch.arange(at, at + n).expand(self.Hkv, n)
        new = [k.transpose(0, 1), v.transpose(0, 1), pos, torch.zeros(self.Hkv, n, dtype=torch.float64)]
        old = self.hist.get(s)
        self.hist[s] = new if old is None else [torch.cat((a, b), 1) for a, b in zip(old, new)]
        self.next[s] = at + n

    def fork(self, s, t):
        self.hist[t], self.next[t] = list(self.hist[s]), self.next[s]

    def keep(self, s, ind):
        pick = lambda x: torch.stack([x[h, ind[h].long()] for h in range(self.Hkv)])  # noqa: E731
        self.hist[s] = [pick(x) for x in self.hist[s]]

    def attend(self, s, q, window=None):
        """O [m, Hq, D] of the last tokens of s; adds the weights that they give to the sums."""
        k, v, pos, w = self.hist[s]
        m, n, G = q.shape[0], k.shape[1], self.Hq // self.Hkv
        O = torch.zeros(m, self.Hq, self.D, dtype=torch.float64)
        w = w.clone()
        qr = serving.rotate(q, torch.arange(self.next[s] - m, self.next[s])[:, None], self.inv, **self.kw)
        for h in range(self.Hq):
            kr = serving.rotate(k[h // G], pos[h // G], self.inv, **self.kw).to(self.dtype).double()
            sc = qr[:, h].to(self.dtype).double() @ kr.t() / math.sqrt(self.D)
            sc[torch.arange(n) > torch.arange(n - m, n)[:, None]] = -math.inf
            p = torch.softmax(sc, -1)
            O[:, h] = p @ v[h // G].double()
            w[h // G] += p[m - min(m, window) if window is not None else 0:].sum(0)
        self.hist[s][3] = w
        return O


def _tol(dtype):
    """As in tests/test_gpu_paged_serving.py: 3 u A of the attention, and elements of q and k that
    round otherwise than in fp64."""
    return 4 * torch.finfo(dtype).eps / 2 * 3


@pytest.mark.parametrize("dtype,page,interleaved", [(torch.float16, 16, False), (torch.bfloat16, 7, True)])
@pytest.mark.parametrize("shared", [False, True])
def test_a_serving_loop_with_evictions(dev, dtype, page, interleaved, shared):
    Hq, Hkv, D = 8, 2, 128
    inv, _ = rotary_frequencies(64, 10000.0, device="cpu")
    m = Model(Hq, Hkv, D, dtype, inv, page, interleaved=interleaved)
    cache = PagedKVCache(900 // page + 60, Hkv, page, D, device=dev, dtype=dtype, weight_rows=6,
                         weight_len=256)

    def step(seqs, counts, observe=None):
        q, k, v = m.tokens(sum(counts))
        o = cache.extend(seqs, q.to(dev), k.to(dev), v.to(dev), counts, inv_freq=inv.to(dev),
                         interleaved=interleaved, shared_prefix=shared, observe=observe).cpu()
        t = 0
        for s, n in zip(seqs, counts):
            if n:
                m.add(s, k[t:t + n], v[t:t + n])
                assert_close(o[t:t + n], m.attend(s, q[t:t + n], observe), atol=_tol(dtype), what=f"sequence {s}")
                got = cache.weights[cache._rows[s], :, :cache.seq_len(s)].cpu()
                # An element of q or k that rounds otherwise moves a weight by some 2 u |q||k| scale /
                # sqrt(D), u = eps / 2, of itself: |q||k| scale / sqrt(D) is about 1, up to 4 in the tail.
                want = m.hist[s][3]
                assert float(((got - want).abs() / (want + 1e-3)).max()) <= 8 * torch.finfo(dtype).eps
                assert not cache.weights[cache._rows[s], :, cache.seq_len(s):].any()
            t += n

    def evict(seqs, keep, first, recent):
        long = [s for s in seqs if cache.seq_len(s) > keep]
        old = {s: cache.weights[cache._rows[s]].cpu() for s in long}
        lens = {s: cache.seq_len(s) for s in long}
        assert cache.evict(seqs, keep, first, recent) == sum(lens[s] - keep for s in long)
        for s in long:
            m.keep(s, serving.heaviest(old[s][None], [lens[s]], keep, first, recent)[0][0])
            assert cache.seq_len(s) == keep and cache.next_position(s) == m.next[s]

    step(["a", "b"], [120, 9])
    step(["a", "b"], [1, 1])
    for t in "cd":
        cache.fork("a", t)
        m.fork("a", t)
    step(["a", "c", "d", "b"], [1, 4, 1, 1])
    evict(["c", "b"], 70, 2, 10)               # c's pages are a's too
    step(["a", "c", "d", "b"], [1, 1, 1, 1])
    evict(["a", "c", "d"], 60, 0, 30)
    step(["a", "c", "d"], [2, 1, 1])
    step(["b", "d"], [40, 1], observe=5)
    cache.truncate("d", 61)
    m.hist["d"], m.next["d"] = [x[:, :61] for x in m.hist["d"]], m.next["d"] - (m.hist["d"][0].shape[1] - 61)
    step(["d", "a"], [3, 1])
    cache.fork("d", "e")
    m.fork("d", "e")
    cache.compact()
    step(["d", "e"], [1, 1])
    evict(["a", "b", "c", "d", "e"], 33, 4, 8)
    step(["a", "b", "c", "d", "e"], [1, 1, 1, 1, 2])
    for s in "abcde":
        cache.release(s)
    assert cache.free_pages == cache.pool.shape[0] and not any(cache._refs)
    assert len(cache._free_rows) == 6 and not cache._dropped


def test_a_selection_serves_the_sparse_decode(dev):
    """Without eviction: the heaviest tokens' list, a row for each query head, is a sparse decode's."""
    cache = PagedKVCache(40, 2, 16, 128, device=dev, weight_rows=2, weight_len=400)
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(300, h, 128, generator=g).half() for h in (8, 2, 2))
    cache.extend([0], q.to(dev), k.to(dev), v.to(dev), [300], observe=64)
    n = torch.tensor([300], dtype=torch.int32, device=dev)
    rows = torch.tensor([cache._rows[0]], dtype=torch.int32, device=dev)
    ind, nnz = select_heaviest(cache.weights, n, 50, first=4, recent=16, rows=rows)
    indptr, indices, last = cache.page_table([0])
    o = sparsetoken_flash_attention_decode_paged(
        q[-1:, :, None].to(dev), cache.pool, indptr, indices,
        ind.repeat_interleave(4, 1).contiguous(), nnz.repeat_interleave(4, 1).contiguous())
    for h in range(8):
        at = ind[0, h // 4].cpu().long()
        kk, vv = k[at, h // 4].double(), v[at, h // 4].double()
        p = torch.softmax(kk @ q[-1, h].double() / math.sqrt(128), 0)
        assert_close(o[0, h].reshape(-1), p @ vv)


def test_without_sums_or_shared_pages_extend_is_as_before(dev):
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(40, h, 64, generator=g).half().to(dev) for h in (4, 2, 2))
    outs = []
    for kw, ext in (({}, {}), ({"weight_rows": 2, "weight_len": 64}, {}),
                    ({"weight_rows": 2, "weight_len": 64}, {"observe": 0}), ({}, {"shared_prefix": True})):
        cache = PagedKVCache(10, 2, 16, 64, device=dev, **kw)
        outs.append(cache.extend([3, 4], q, k, v, [30, 10], return_lse=True, **ext))
        only = cache.extend([3], q[:1], k[:1], v[:1], [1], **ext)
        assert only.shape == (1, 4, 64)
        if ext.get("observe") == 0:
            assert not cache.weights.any() and not cache._rows
    for o, lse in outs[1:3]:
        assert torch.equal(o, outs[0][0]) and torch.equal(lse, outs[0][1])
    assert float((outs[3][0] - outs[0][0]).abs().max()) <= 6 * 2.0 ** -11 * 4.5


def test_a_refused_step_leaves_sums_and_rows(dev):
    cache = PagedKVCache(10, 2, 16, 64, device=dev, weight_rows=1, weight_len=64)
    z = lambda n, h: torch.randn(n, h, 64, dtype=torch.float16, device=dev)  # noqa: E731
    cache.extend([0], z(5, 4), z(5, 2), z(5, 2), [5])
    sums = cache.weights.clone()
    with pytest.raises(MemoryError, match="rows"):
        cache.extend([0, 1], z(2, 4), z(2, 2), z(2, 2), [1, 1])
    with pytest.raises(RuntimeError):
        cache.extend([0], z(2, 4), z(2, 2), z(2, 2), [2], softmax_scale=math.inf)
    assert cache.seq_len(0) == 5 and 1 not in cache._pages and torch.equal(cache.weights, sums)
    cache.release(0)
    with pytest.raises(RuntimeError):
        cache.extend([2], z(2, 4), z(2, 2), z(2, 2), [2], softmax_scale=math.inf)
    assert not cache._rows and cache._free_rows == [0] and 2 not in cache._pages
    with pytest.raises(ValueError):
        cache.extend([2], z(2, 4), z(2, 2), z(2, 2), [2], observe=-1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,rot", [(128, 64), (80, 36)])
def test_positions_with_an_offset(dev, D, rot, dtype):
    """append_paged_kv_rotary at offsets equals the oracle's rotation, and plain calls are unchanged."""
    g = torch.Generator().manual_seed(D)
    inv, _ = rotary_frequencies(rot, device="cpu")
    q, k, v = (torch.randn(9, h, D, generator=g).to(dtype) for h in (4, 2, 2))
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    t = (i(0, 4, 9), torch.zeros(6, 2, 2, 8, D, dtype=dtype, device=dev), i(0, 2, 3), i(4, 1, 2), i(6, 5))
    call = lambda pool, **kw: append_paged_kv_rotary(  # noqa: E731
        q.to(dev), k.to(dev), v.to(dev), t[0], pool, *t[2:], inv.to(dev), **kw)
    pool = t[1].clone()
    off = i(1000, 0)
    qr = call(pool, position_offset=off)
    pos = torch.tensor([10, 11, 12, 13, 0, 1, 2, 3, 4]) + torch.tensor([1000] * 4 + [0] * 5)
    u = torch.finfo(dtype).eps / 2
    # One rounding of |x| below 5 and fp32 products of turns of about 2^-24.
    assert_close(qr, serving.rotate(q, pos[:, None], inv), atol=8 * u + 4e-6)
    kr = serving.rotate(k, pos[:, None], inv)
    assert_close(pool[1, 0, :, 2:6].transpose(0, 1), kr[:4], atol=8 * u + 4e-6)
    p0, p1 = t[1].clone(), t[1].clone()
    a, b = call(p0), call(p1, position_offset=i(0, 0))
    assert torch.equal(a, b) and torch.equal(p0, p1) and torch.equal(a[4:], qr[4:])
    for err, bad in ((TypeError, off.long()), (ValueError, off[:1]), (ValueError, off.cpu())):
        with pytest.raises(err):
            call(t[1].clone(), position_offset=bad)
