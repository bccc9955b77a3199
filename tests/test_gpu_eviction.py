"""The attention that cached tokens draw, the choice of the heaviest, and their move, each against
the oracle.

Sums.  A term exp(s - l) with s an fp32 sum of D products: s is off by up to (D + 2) 2^-24 |q| |k|
scale, the scale's and log2(e)'s roundings, l's product and the fma add up to 4 2^-24 each of |s|
and |l|, exp2 a few 2^-24.  Sums of a lane's terms go 16 at a time into a running total of a
sequence's blocks of 32 rows: (rows / 32 + 24) 2^-24 of the sum, then one addition to the old sum.
Selections and moves are exact.
"""
import math

import pytest
import torch

from attention_kernel_triton_amd.attention_weights_paged import accumulate_attention_weights_paged
from attention_kernel_triton_amd.kept_index import select_heaviest
from attention_kernel_triton_amd.paged_kv import keep_tokens
from oracle import serving

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def i32(v, dev=None):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# --------------------------------------------------------------------------- sums
class Step:
    """Sequences of ctx[i] cached and n[i] new tokens, their normalisers, and sums so far."""

    def __init__(self, ctx, n, Hq, Hkv, D, page, dtype=F16, causal=True, seed=0, room=5, more=2):
        g = torch.Generator().manual_seed(1000 * seed + sum(ctx) + 7 * sum(n) + D + page)
        lens = [c + m for c, m in zip(ctx, n)]
        counts = [-(-x // page) for x in lens]
        P = sum(counts) + 3
        self.indices = torch.randperm(P, generator=g)[:sum(counts)].to(torch.int32)
        self.indptr = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
        self.last = i32([(x - 1) % page + 1 if x else 0 for x in lens])
        self.q_indptr = torch.tensor([0] + list(n)).cumsum(0).to(torch.int32)
        self.pool = torch.randn(P, 2, Hkv, page, D, generator=g).to(dtype)
        self.q = torch.randn(sum(n), Hq, D, generator=g).to(dtype)
        self.causal, self.lens = causal, lens
        self.rows = torch.randperm(len(n) + more, generator=g)[:len(n)].to(torch.int32)
        self.weights = torch.rand(len(n) + more, Hkv, max(lens) + room, generator=g)
        self.lse = serving.chunk_attention(self.q, self.q_indptr, self.pool, self.indptr, self.indices,
                                           self.last, causal)[1].float()

    def table(self, dev=None):
        t = (self.pool, self.indptr, self.indices, self.last)
        return t if dev is None else [x.to(dev) for x in t]

    def run(self, dev, **kw):
        w = self.weights.to(dev)
        accumulate_attention_weights_paged(w, self.q.to(dev), self.q_indptr.to(dev), self.lse.to(dev),
                                           *self.table(dev), rows=self.rows.to(dev),
                                           causal=self.causal, **kw)
        return w.cpu()

    def check(self, dev, scale=None, window=None):
        got = self.run(dev, softmax_scale=scale, window=window)
        want, added, far, norm = serving.attention_weights(
            self.weights, self.q, self.q_indptr, self.lse, *self.table(), rows=self.rows,
            causal=self.causal, scale=scale, window=window)
        D, rows = self.q.shape[-1], max(self.q_indptr.diff().tolist()) * self.q.shape[1] // self.pool.shape[2]
        eps = 2.0 ** -24
        tol = eps * ((D + 8) * far + 4 * norm + (rows / 32 + 32) * added + want.abs()) + 1e-30
        fin = torch.isfinite(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.double()[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)])
        over = ((got.double() - want).abs() - tol)[fin]
        assert over.numel() == 0 or float(over.max()) <= 0, float(over.max())
        assert torch.equal(got[added == 0], self.weights[added == 0])  # others stay as they were
        return got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,page,Hq,Hkv", [(64, 16, 8, 2), (128, 16, 8, 2), (256, 16, 4, 2),
                                           (128, 24, 6, 2), (64, 1, 5, 1), (256, 7, 2, 2),
                                           (128, 64, 14, 2), (64, 48, 12, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_sums_of_mixed_batches(dev, D, page, Hq, Hkv, dtype, causal):
    Step([0, 12, 300, 77, 0, 1000], [5, 1, 33, 0, 1, 3], Hq, Hkv, D, page, dtype, causal).check(dev)


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("ctx", [0, 1, 31, 63, 64, 65, 255, 256, 257, 600])
def test_sums_by_chunk_and_context_lengths(dev, n, ctx):
    Step([ctx], [n], 8, 2, 64, 16).check(dev)


@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 16, 33, 128])
def test_sums_by_query_heads_per_kv_head(dev, G):
    Step([200, 40], [1, 9], 2 * G if G <= 32 else G, 2 if G <= 32 else 1, 64, 16).check(dev)


def test_sums_of_a_prompt_in_many_blocks(dev):
    Step([500, 3], [700, 20], 8, 2, 128, 32, BF16).check(dev)
    Step([100], [900], 4, 1, 256, 16).check(dev)


@pytest.mark.parametrize("B", [64, 65, 200, 1030])
def test_sums_of_many_sequences(dev, B):
    g = torch.Generator().manual_seed(B)
    n = torch.randint(0, 4, (B,), generator=g).tolist()
    n[B - 3] = 30
    ctx = torch.randint(0, 90, (B,), generator=g).tolist()
    n[B // 2:B // 2 + 20] = [0] * 20
    Step(ctx, n, 4, 2, 64, 16).check(dev)


@pytest.mark.parametrize("window", [0, 1, 5, 32, 100])
@pytest.mark.parametrize("causal", [True, False])
def test_sums_of_the_last_tokens(dev, window, causal):
    s = Step([100, 0, 40], [40, 77, 3], 8, 2, 64, 16, causal=causal)
    got = s.check(dev, window=window)
    if window == 100:
        assert torch.equal(got, s.run(dev))


@pytest.mark.parametrize("scale", [0.02, 0.3, -0.1, 0.0])
def test_sums_by_scale(dev, scale):
    s = Step([70, 5], [3, 8], 4, 2, 64, 16)
    s.lse = serving.chunk_attention(s.q, s.q_indptr, *s.table(), True, scale)[1].float()
    s.check(dev, scale=scale)


def test_each_row_draws_one_in_all(dev):
    """The weights of a row sum to 1, so those of a (sequence, head) sum to its rows' number."""
    s = Step([300, 40, 0], [1, 7, 50], 8, 2, 128, 16)
    s.weights.zero_()
    total = s.run(dev)[s.rows.long()].double().sum(-1)
    want = torch.tensor([1.0, 7.0, 50.0], dtype=torch.float64)[:, None] * 4
    assert float(((total - want) / want).abs().max()) < 1e-5


def test_sums_of_values_that_are_not_finite(dev):
    """Behind the last token, in keys that some rows do not see, in keys that they see, in a row
    of q, in a normaliser: each reaches the tokens of the rows that see it, and no others."""
    s = Step([30, 100], [5, 1], 4, 2, 64, 16)
    s.pool[s.indices[2].long(), :, :, 3:] = math.nan  # 35 tokens: behind the last
    s.check(dev)
    s.pool[s.indices[2].long(), 0, :, 2] = math.nan  # token 34: one row sees it
    s.check(dev)
    s.pool[s.indices[3].long(), 0, 1, 5, 7] = math.inf
    s.check(dev)
    s.q[1, 2, 3] = math.nan
    s.check(dev)
    s.lse[2, 0], s.lse[3, 1], s.lse[0, 3] = -math.inf, math.inf, math.nan
    s.check(dev)


def test_sums_with_bad_pages_rows_and_tables(dev):
    s = Step([40, 70, 20], [1, 3, 2], 4, 2, 64, 16)
    s.indices[1], s.indices[5] = -1, 10 ** 6
    s.rows[2] = -1
    s.check(dev)
    s.rows[1] = 99
    s.check(dev)
    a = {"w": s.weights.to(dev), "q": s.q.to(dev), "qi": s.q_indptr.to(dev), "lse": s.lse.to(dev)}
    a.update(zip(("pool", "ip", "ind", "last"), s.table(dev)))
    for name, bad in (("ip", [0, 10 ** 6, 3, -5]), ("ip", [9, 3, 9, 0]), ("last", [10 ** 6, -3, 0]),
                      ("qi", [-4, 1, 90, 2])):
        b = dict(a)
        b[name] = i32(bad, dev)
        accumulate_attention_weights_paged(*b.values())
    torch.cuda.synchronize()


def test_sums_in_short_and_strided_rows(dev):
    """A row that ends before its sequence takes the sums of the first tokens only."""
    s = Step([100, 20], [1, 4], 8, 2, 64, 16)
    s.weights = s.weights[:, :, :60].clone()
    got = s.check(dev)
    wide = torch.zeros(2 * s.weights.shape[0], 4, 100)
    view = wide[::2, 1::2, 7:67]
    view.copy_(s.weights)
    d = wide.to(dev)
    wq = torch.zeros(s.q.shape[0], 16, 128, dtype=F16)
    wq[:, 1::2, 64:] = s.q
    accumulate_attention_weights_paged(d[::2, 1::2, 7:67], wq.to(dev)[:, 1::2, 64:],
                                       s.q_indptr.to(dev), s.lse.to(dev), *s.table(dev),
                                       rows=s.rows.to(dev))
    assert torch.equal(d.cpu()[::2, 1::2, 7:67], got)
    d[::2, 1::2, 7:67] = 0
    assert not d.any()


def test_sums_do_not_depend_on_the_run_and_replay(dev):
    s = Step([3000, 40], [33, 200], 8, 2, 128, 16)
    first = s.run(dev)
    assert torch.equal(first, s.run(dev))
    w = s.weights.to(dev)
    a = [s.q.to(dev), s.q_indptr.to(dev), s.lse.to(dev), *s.table(dev)]
    rows = s.rows.to(dev)
    twice = w.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        accumulate_attention_weights_paged(w, *a, rows=rows)
    for i in range(3):  # each replay adds the same again
        g.replay()
        accumulate_attention_weights_paged(twice, *a, rows=rows)
        torch.cuda.synchronize()
        assert torch.equal(w, twice)
        if i == 0:
            assert torch.equal(w.cpu(), first)
    side = torch.cuda.Stream(dev)
    w2 = s.weights.to(dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        accumulate_attention_weights_paged(w2, *a, rows=rows)
    torch.cuda.synchronize()
    assert torch.equal(w2.cpu(), first)


def test_sums_refusals(dev):
    s = Step([10, 4], [1, 2], 4, 2, 64, 16)
    a = {"w": s.weights.to(dev), "q": s.q.to(dev), "qi": s.q_indptr.to(dev), "lse": s.lse.to(dev)}
    a.update(zip(("pool", "ip", "ind", "last"), s.table(dev)))
    kw = {"rows": s.rows.to(dev)}

    def call(**over):
        accumulate_attention_weights_paged(*{**a, **{k: v for k, v in over.items() if k in a}}.values(),
                                           **{**kw, **{k: v for k, v in over.items() if k not in a}})

    call()
    for err, over in ((TypeError, {"w": a["w"].half()}), (ValueError, {"w": a["w"].cpu()}),
                      (ValueError, {"w": a["w"][:, :1]}), (ValueError, {"w": a["w"][..., ::2]}),
                      (ValueError, {"w": a["w"][:1].expand_as(a["w"])}),
                      (ValueError, {"w": a["w"][:, :1].expand_as(a["w"])}),
                      (ValueError, {"w": a["w"][:1], "rows": None}), (TypeError, {"lse": a["lse"].half()}),
                      (ValueError, {"lse": a["lse"][:1]}), (ValueError, {"lse": a["lse"].cpu()}),
                      (TypeError, {"q": a["q"].float()}), (TypeError, {"pool": a["pool"].bfloat16()}),
                      (TypeError, {"rows": kw["rows"].long()}), (ValueError, {"rows": kw["rows"][:1]}),
                      (ValueError, {"window": -1}), (RuntimeError, {"softmax_scale": math.nan}),
                      (ValueError, {"ip": a["ip"][:2]}), (ValueError, {"q": a["q"][:, :, :32]})):
        with pytest.raises(err):
            call(**over)


# --------------------------------------------------------------------------- selection
def check_select(dev, w, lengths, keep, first=0, recent=0, rows=None):
    got = select_heaviest(w.to(dev), i32(lengths, dev), keep, first=first, recent=recent,
                          rows=None if rows is None else i32(rows, dev))
    want = serving.heaviest(w, lengths, keep, first, recent, rows)
    for g, x in zip(got, want):
        assert g.dtype == torch.int32 and torch.equal(g.cpu(), x)


@pytest.mark.parametrize("L", [1, 2, 63, 64, 65, 1000, 1024, 1025, 2049, 4095, 4096, 4097, 9000, 17000, 33000])
@pytest.mark.parametrize("share", [0.0, 0.02, 0.5, 0.97])
def test_selections(dev, L, share):
    g = torch.Generator().manual_seed(L)
    w = torch.exp(2 * torch.randn(3, 2, L, generator=g))
    keep = int(L * share)
    lengths = [L, max(1, L - 3), L // 2]
    check_select(dev, w, lengths, keep)
    if keep >= 6:
        check_select(dev, w, lengths, keep, first=2, recent=4)
        check_select(dev, w, lengths, keep, first=0, recent=keep)
        check_select(dev, w, lengths, keep, first=keep)
        check_select(dev, w, lengths, keep, first=1, recent=keep - 2)


@pytest.mark.parametrize("kind", ["equal", "few", "zeros", "signed", "specials", "tiny"])
def test_selections_among_equal_and_unusual_sums(dev, kind):
    g = torch.Generator().manual_seed(1)
    w = torch.randn(2, 3, 5000, generator=g)
    if kind == "equal":
        w = torch.ones_like(w)
    elif kind == "few":
        w = torch.randint(0, 3, w.shape, generator=g).float()
    elif kind == "zeros":
        w = torch.where(torch.rand(w.shape, generator=g) < 0.5, 0.0, -0.0) + (w > 2).float() * 0
        w = torch.copysign(torch.zeros_like(w), torch.randn(w.shape, generator=g))
        w[0, 0, ::7] = 1e-38
    elif kind == "specials":
        for i, x in enumerate((math.nan, -math.nan, math.inf, -math.inf, 0.0, -0.0)):
            w[:, :, i::11] = x
        w[0, 0] = torch.where(torch.isnan(w[0, 0]), torch.copysign(w[0, 0], torch.tensor(-1.0)), w[0, 0])
    elif kind == "tiny":
        w = w * 2.0 ** -140  # below the normal range
    for keep in (1, 10, 1000, 4321):
        check_select(dev, w, [5000, 4444], keep, first=1 if keep > 1 else 0, recent=min(keep // 2, 50))


def test_selection_rows_and_lengths(dev):
    g = torch.Generator().manual_seed(2)
    w = torch.rand(6, 2, 500, generator=g)
    check_select(dev, w, [500, 3, 0, 499, 200, 900, -5], 100, first=4, recent=16,
                 rows=[5, 0, 1, 1, 3, 2, 4])
    check_select(dev, w, [500, 400], 50, rows=[-1, 6])
    check_select(dev, w, [500, 400], 0)
    check_select(dev, w[:, :, :0], [0, 3], 4)
    wide = torch.rand(12, 4, 1030, generator=g)
    check_select(dev, wide[::2, 1::2, 13:513], [500, 477], 60)
    a = select_heaviest(wide.to(dev)[::2, 1::2, 13:513], i32([500, 477], dev), 60)
    b = select_heaviest(wide[::2, 1::2, 13:513].contiguous().to(dev), i32([500, 477], dev), 60)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for B, H in ((0, 2), (2, 0)):
        ind, nnz = select_heaviest(torch.zeros(3, H, 10, device=dev), torch.zeros(B, dtype=torch.int32, device=dev), 5)
        assert ind.shape == (B, H, 5) and nnz.shape == (B, H, 1)


def test_selection_of_long_rows(dev):
    g = torch.Generator().manual_seed(3)
    w = torch.exp(2 * torch.randn(2, 1, 120001, generator=g))
    w[1] = torch.round(w[1] * 4) / 4
    for L, lengths in ((120001, [120001, 100000]), (65536, [65536, 65535]), (65537, [65537, 40000])):
        for first, recent in ((4, 77), (0, 12345), (12000, 300)):
            check_select(dev, w[:, :, :L].contiguous(), lengths, 12345, first, recent)


def test_selection_replays(dev):
    g = torch.Generator().manual_seed(4)
    w = torch.rand(4, 2, 3000, generator=g).to(dev)
    n = i32([3000, 2000, 50, 2999], dev)
    select_heaviest(w, n, 100, first=1, recent=9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ind, nnz = select_heaviest(w, n, 100, first=1, recent=9)
    for _ in range(3):
        w.copy_(torch.rand(4, 2, 3000, generator=g))
        graph.replay()
        want = select_heaviest(w, n, 100, first=1, recent=9)
        torch.cuda.synchronize()
        assert torch.equal(ind, want[0]) and torch.equal(nnz, want[1])


def test_selection_refusals(dev):
    w, n = torch.rand(2, 2, 50, device=dev), i32([50, 40], dev)
    for err, args, kw in ((ValueError, (w, n, 5), {"first": 3, "recent": 3}), (ValueError, (w, n, -1), {}),
                          (ValueError, (w, n, 5), {"first": -1}), (TypeError, (w.half(), n, 5), {}),
                          (TypeError, (w, n.long(), 5), {}), (ValueError, (w.cpu(), n, 5), {}),
                          (ValueError, (w, n.cpu(), 5), {}), (ValueError, (w[0], n, 5), {}),
                          (ValueError, (w[..., ::2], n, 5), {}), (ValueError, (w[:1], n, 5), {}),
                          (ValueError, (w, n, 5), {"rows": i32([1], dev)})):
        with pytest.raises(err):
            select_heaviest(*args, **kw)


# --------------------------------------------------------------------------- moves
class Kept:
    def __init__(self, lens, keep, Hkv, D, page, dtype=F16, seed=0, extra=3, rows=True):
        g = torch.Generator().manual_seed(1000 * seed + sum(lens) + D + page + keep)
        counts = [-(-x // page) for x in lens]
        P = sum(counts) + extra
        order = torch.randperm(P, generator=g).to(torch.int32)
        self.indices, self.free = order[:sum(counts)].clone(), order[sum(counts):]
        self.indptr = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
        self.last = i32([(x - 1) % page + 1 if x else 0 for x in lens])
        self.pool = torch.randn(P, 2, Hkv, page, D, generator=g).to(dtype)
        B = len(lens)
        self.ind = torch.full((B, Hkv, keep), -1, dtype=torch.int32)
        self.nnz = torch.zeros(B, Hkv, 1, dtype=torch.int32)
        for b, n in enumerate(lens):
            for h in range(Hkv):
                k = min(n, keep - (h % 2) * (keep // 3))  # heads may keep different numbers
                self.ind[b, h, :k] = torch.randperm(n, generator=g)[:k].sort().values.to(torch.int32)
                self.nnz[b, h] = k
        self.weights = torch.rand(B + 2, Hkv, max(lens) + 4, generator=g)
        self.rows = torch.randperm(B + 2, generator=g)[:B].to(torch.int32)

    def check(self, dev, dst=None, weights=True):
        pool, w = self.pool.to(dev), self.weights.to(dev)
        keep_tokens(pool, self.indptr.to(dev), self.indices.to(dev), self.last.to(dev),
                    self.ind.to(dev), self.nnz.to(dev),
                    dst_page_indices=None if dst is None else dst.to(dev),
                    weights=w if weights else None, rows=self.rows.to(dev) if weights else None)
        want, ww = serving.keep_tokens(self.pool, self.indptr, self.indices, self.last, self.ind,
                                       self.nnz, dst, self.weights if weights else None, self.rows)
        bits = lambda x: x.view(torch.int16)  # noqa: E731  (NaNs are moved too)
        assert torch.equal(bits(pool.cpu()), bits(want))
        assert torch.equal(w.cpu(), ww if weights else self.weights)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Hkv,page,D", [(8, 16, 128), (1, 1, 64), (3, 7, 72), (2, 64, 256), (2, 100, 8),
                                        (1, 24, 1024)])
def test_moves_are_bit_exact(dev, Hkv, page, D, dtype):
    Kept([300, 5, 0, 129, 77], 60, Hkv, D, page, dtype).check(dev)
    Kept([300, 5, 0, 129, 77], 60, Hkv, D, page, dtype).check(dev, weights=False)


# Batches of the in-place walk: lists shorter, as long as, and longer than one; one token dropped
# near the front, in the middle, at the end.
@pytest.mark.parametrize("n", [511, 512, 513, 1023, 1024, 1025, 2048, 3000])
@pytest.mark.parametrize("drop", ["first", "middle", "last", "half", "front"])
def test_moves_of_long_lists(dev, n, drop):
    c = Kept([n + 1], n, 2, 64, 16)
    at = {"first": 0, "middle": n // 2, "last": n}.get(drop)
    t = torch.arange(n + 1, dtype=torch.int32)
    kept = t[t != at] if at is not None else t[::2] if drop == "half" else t[n // 2:]
    c.ind[:], c.nnz[:] = -1, len(kept)
    c.ind[..., :len(kept)] = kept
    c.check(dev)


def test_moves_of_sums_longer_than_a_batch(dev):
    c = Kept([20000], 15000, 1, 8, 64)
    c.check(dev)


def test_moves_into_other_pages(dev):
    """A shared page's place is taken by a free one; the pages that were read stay as they are."""
    c = Kept([100, 90], 40, 2, 64, 16, extra=6)
    dst = c.indices.clone()
    dst[0], dst[2], dst[int(c.indptr[1]) + 1] = c.free[0], c.free[1], c.free[2]
    c.check(dev, dst)
    c.ind[0, :, :40], c.nnz[0] = torch.arange(40, dtype=torch.int32), 40  # nothing moves but the page
    c.check(dev, dst)


def test_entries_that_cannot_be_served_are_skipped(dev):
    c = Kept([100, 90, 40], 30, 2, 64, 16)
    c.ind[0, 0, 5], c.ind[0, 0, 7], c.ind[0, 1, 9], c.ind[1, 0, 3] = 4, -1, 100, 10 ** 6
    c.ind[1, 1, 10] = c.ind[1, 1, 11]  # a token twice
    c.nnz[1, 0], c.nnz[2, 0], c.nnz[2, 1] = 99, -4, 0
    c.indices[1], c.indices[int(c.indptr[1])] = -1, 10 ** 6
    c.rows[2] = 55
    c.check(dev)


def test_sums_shorter_than_their_sequences(dev):
    c = Kept([100, 90], 70, 2, 64, 16)
    c.weights = c.weights[:, :, :50].clone()
    c.check(dev)


def test_moves_in_strided_tensors(dev):
    c = Kept([100, 90], 40, 2, 64, 16)
    wide = torch.randn(c.pool.shape[0], 2, 4, 32, 128).half()
    wide[:, :, 1::2, ::2, 64:] = c.pool
    d, w = wide.to(dev), torch.zeros(8, 4, 200)
    w[::2, 1::2, 3:3 + c.weights.shape[2]] = c.weights
    dw = w.to(dev)
    keep_tokens(d[:, :, 1::2, ::2, 64:], c.indptr.to(dev), c.indices.to(dev), c.last.to(dev),
                c.ind.to(dev), c.nnz[..., 0].to(dev), weights=dw[::2, 1::2, 3:3 + c.weights.shape[2]],
                rows=c.rows.to(dev))
    want, ww = serving.keep_tokens(c.pool, c.indptr, c.indices, c.last, c.ind, c.nnz, None, c.weights, c.rows)
    wide[:, :, 1::2, ::2, 64:] = want
    w[::2, 1::2, 3:3 + c.weights.shape[2]] = ww
    assert torch.equal(d.cpu(), wide) and torch.equal(dw.cpu(), w)


def test_moves_replay(dev):
    """Each replay moves the tokens that the list names again, as the eager call does."""
    c = Kept([300, 200], 150, 2, 64, 16)
    a = [x.to(dev) for x in (c.indptr, c.indices, c.last, c.ind, c.nnz)]
    pool, w, rows = c.pool.to(dev), c.weights.to(dev), c.rows.to(dev)
    pool2, w2 = pool.clone(), w.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        keep_tokens(pool, *a, weights=w, rows=rows)
    for _ in range(3):
        g.replay()
        keep_tokens(pool2, *a, weights=w2, rows=rows)
        torch.cuda.synchronize()
        assert torch.equal(pool, pool2) and torch.equal(w, w2)


def test_move_refusals(dev):
    c = Kept([30, 20], 10, 2, 64, 16)
    a = {k: getattr(c, k).to(dev) for k in ("pool", "indptr", "indices", "last", "ind", "nnz")}

    def call(dst=None, weights=None, rows=None, **kw):
        keep_tokens(*{**a, **kw}.values(), dst_page_indices=dst, weights=weights, rows=rows)

    w = c.weights.to(dev)
    for err, kw in ((TypeError, {"pool": a["pool"].float()}), (ValueError, {"pool": a["pool"].cpu()}),
                    (TypeError, {"ind": a["ind"].long()}), (ValueError, {"ind": a["ind"][:, :1]}),
                    (ValueError, {"nnz": a["nnz"][:1]}), (ValueError, {"dst": a["indices"][:-1]}),
                    (ValueError, {"weights": w[:1]}), (TypeError, {"weights": w.double()}),
                    (ValueError, {"weights": w, "rows": i32([1], dev)}),
                    (ValueError, {"weights": w[:, :1].expand_as(w)}),
                    (ValueError, {"indptr": a["indptr"][:2]}), (ValueError, {"pool": a["pool"][..., ::2]})):
        with pytest.raises(err):
            call(**kw)


def test_past_32_bit_offsets(dev):
    """Pages and sums of tensors of more than 2^32 (2^31) elements."""
    page, Hkv, D = 64, 8, 128
    P = 2 ** 32 // (2 * Hkv * page * D) + 3
    pool = torch.empty((P, 2, Hkv, page, D), dtype=F16, device=dev)
    g = torch.Generator().manual_seed(5)
    small = torch.randn(3, 2, Hkv, page, D, generator=g).half()
    pool[P - 3:] = small.to(dev)
    L = 2 ** 20
    N = 2 ** 31 // (Hkv * L) + 2
    sums = torch.zeros((N, Hkv, L), device=dev)
    t = [i32([0, 3]), i32([P - 1, P - 3, P - 2]), i32([60])]
    s = [t[0], i32([2, 0, 1]), t[2]]
    n = 188
    q = torch.randn(5, 16, D, generator=g).half()
    qi, rows = i32([0, 5]), i32([N - 1])
    lse = serving.chunk_attention(q, qi, small, *s)[1].float()
    to = lambda v: [x.to(dev) for x in v]  # noqa: E731
    accumulate_attention_weights_paged(sums, *to([q, qi, lse]), pool, *to(t), rows=rows.to(dev))
    near = torch.zeros(1, Hkv, 200, device=dev)
    accumulate_attention_weights_paged(near, *to([q, qi, lse, small, *s]))
    assert torch.equal(sums[N - 1, :, :200], near[0]) and float(near.sum()) > 79
    ind, nnz = select_heaviest(sums, i32([n], dev), 70, first=1, recent=5, rows=rows.to(dev))
    want = serving.heaviest(near.cpu(), [n], 70, 1, 5)
    assert torch.equal(ind.cpu(), want[0]) and torch.equal(nnz.cpu(), want[1])
    keep_tokens(pool, *to(t), ind, nnz, weights=sums, rows=rows.to(dev))
    moved, w = serving.keep_tokens(small, *s, *want, weights=near.cpu())
    assert torch.equal(pool[P - 3:].cpu(), moved) and torch.equal(sums[N - 1, :, :200].cpu(), w[0])
