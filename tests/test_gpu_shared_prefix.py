"""Attention with shared prefixes against the fp64 oracle.

Tolerances as for chunk attention (tests/test_gpu_chunk.py): the two parts' probabilities are
rounded to the type in numerator and normaliser, their sums are joined in 32 bits (the factors
2^(m - M) of two maxima are as exact as the probabilities' own exponents), and O is rounded once.
"""
import ctypes as C
import math

import pytest
import torch

from attention_kernel_triton_amd import _native as N
from attention_kernel_triton_amd.chunk_flash_attention_paged import flash_attention_chunk_paged
from attention_kernel_triton_amd.shared_prefix_flash_attention_paged import (
    flash_attention_shared_prefix_paged)
from oracle import serving

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


class Case:
    """Groups of sequences over prefixes, own tokens ctx[i] + n[i], all behind a permuted pool.
    groups: (sequences, prefix tokens) of each; `before` sequences have none, nor do those left."""

    def __init__(self, groups, ctx, n, Hq, Hkv, D, page, dtype=F16, before=0, seed=0, slack=0):
        g = torch.Generator().manual_seed(1000 * seed + sum(ctx) + 7 * sum(n) + D + page)
        lens = [c + m for c, m in zip(ctx, n)]
        own = [-(-x // page) for x in lens]
        shared = [-(-x // page) for _, x in groups]
        P = sum(own) + sum(shared) + 3
        order = torch.randperm(P, generator=g).to(torch.int32)
        ints = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
        starts = lambda v: torch.tensor([0] + list(v)).cumsum(0).to(torch.int32)  # noqa: E731
        tail = lambda v: ints([(x - 1) % page + 1 if x else 0 for x in v])  # noqa: E731
        self.indptr, self.indices, self.last = starts(own), order[:sum(own)].clone(), tail(lens)
        self.prefix_indptr = starts(shared)
        self.prefix_indices = order[sum(own):sum(own) + sum(shared)].clone()
        self.prefix_last = tail([x for _, x in groups])
        self.group_indptr = starts([k for k, _ in groups]) + before
        self.q_indptr = starts(n)
        self.pool = torch.randn(P, 2, Hkv, page, D, generator=g).to(dtype)
        self.q = torch.randn(sum(n) + slack, Hq, D, generator=g).to(dtype)
        self.longest = max(lens) + max([x for _, x in groups] + [0])

    names = ("q", "q_indptr", "pool", "indptr", "indices", "last", "group_indptr", "prefix_indptr",
             "prefix_indices", "prefix_last")

    def args(self, dev=None):
        return [getattr(self, k) if dev is None else getattr(self, k).to(dev) for k in self.names]

    def check(self, dev, causal=True, scale=None):
        a = self.args(dev)
        o, lse = flash_attention_shared_prefix_paged(*a, causal=causal, softmax_scale=scale,
                                                     return_lse=True)
        only = flash_attention_shared_prefix_paged(*a, causal=causal, softmax_scale=scale)
        ref = serving.shared_prefix_attention(*self.args(), causal, scale)
        T = int(self.q_indptr[-1])
        compare(self, o.cpu()[:T], lse.cpu()[:T], [x[:T] for x in ref])
        assert torch.equal(only[:T].view(torch.int16), o[:T].view(torch.int16))


def compare(c, o, lse, ref):
    O, L, A, C = ref
    D, N = c.q.shape[-1], c.longest
    u = torch.finfo(c.q.dtype).eps / 2
    ds = (D + 8) * 2.0 ** -24 * C
    vmax = float(c.pool.double().nan_to_num(0, 0, 0).abs().max())
    small = N * 2.0 ** -25 * vmax if c.q.dtype == F16 else 0.0
    tol = (3 * u + 2 * ds[..., None] + 1e-6) * A + small + 1e-7
    fin = torch.isfinite(O)
    assert torch.equal(torch.isnan(o), torch.isnan(O))
    assert torch.equal(o.double()[~fin & ~torch.isnan(O)], O[~fin & ~torch.isnan(O)])
    err = ((o.double() - O).abs() - tol)[fin]
    assert err.numel() == 0 or float(err.max()) <= 0, (float(err.max()), o.shape)
    assert torch.equal(lse == -math.inf, L == -math.inf)
    t = ds + (N + 40) * 2.0 ** -24 + 4 * 2.0 ** -23 * L.abs().nan_to_num(0, 0, 0) + 1e-6
    fin = torch.isfinite(L)
    over = ((lse.double() - L).abs() - t)[fin]
    assert over.numel() == 0 or float(over.max()) <= 0, float(over.max())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,page,Hq,Hkv", [(64, 16, 8, 2), (128, 16, 8, 2), (256, 16, 4, 2),
                                           (128, 24, 6, 2), (64, 1, 5, 1), (256, 7, 2, 2),
                                           (128, 64, 14, 2), (64, 48, 12, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_groups_and_sequences_without_one(dev, D, page, Hq, Hkv, dtype, causal):
    Case([(3, 200), (1, 33), (2, 0)], [0, 12, 300, 77, 5, 0, 100, 31, 2], [5, 1, 33, 0, 1, 3, 1, 2, 1],
         Hq, Hkv, D, page, dtype, before=1).check(dev, causal)


# Rows of a group around a wave's and a unit's, prefixes around a step, a block and a page.
@pytest.mark.parametrize("B", [1, 2, 7, 8, 9, 16, 17, 33, 65, 130])
@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 32, 127, 128, 129, 600])
def test_group_and_prefix_sizes(dev, B, prefix):
    Case([(B, prefix)], [i % 40 for i in range(B)], [1] * B, 8, 2, 64, 16).check(dev)


@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 16, 33, 128])
def test_query_heads_per_kv_head(dev, G):
    Case([(5, 300)], [40, 0, 3, 100, 9], [1, 2, 1, 1, 7], 2 * G if G <= 32 else G,
         2 if G <= 32 else 1, 64, 16).check(dev)


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F16), (256, F16)])
def test_long_prefix_over_many_workgroups(dev, D, dtype):
    Case([(12, 7003)], [10 * i for i in range(12)], [1] * 12, 8, 2, D, 16, dtype).check(dev)
    Case([(2, 3001), (20, 900)], [5] * 22, [40, 3] + [2] * 20, 8, 2, D, 32, dtype).check(dev)


def test_prompts_behind_a_prefix(dev):
    Case([(3, 700)], [0, 0, 0], [150, 300, 77], 8, 2, 128, 16, BF16).check(dev)


def test_more_sequences_and_groups_than_lanes(dev):
    g = torch.Generator().manual_seed(0)
    B = 150
    n = torch.randint(0, 4, (B,), generator=g).tolist()
    ctx = torch.randint(0, 60, (B,), generator=g).tolist()
    Case([(2, i % 50) for i in range(70)], ctx, n, 4, 2, 64, 16, before=3).check(dev)


def test_more_sequences_than_the_kernel_keeps_places_of(dev):
    g = torch.Generator().manual_seed(1)
    B = 1000
    n = torch.randint(0, 3, (B,), generator=g).tolist()
    n[400], n[990] = 40, 70
    ctx = torch.randint(0, 20, (B,), generator=g).tolist()
    Case([(9, i % 40) for i in range(100)], ctx, n, 2, 1, 64, 16, before=5).check(dev)


def test_own_keys_or_prefix_may_be_missing(dev):
    """No own token beyond the contract (a table without pages), empty prefixes, no groups at all."""
    c = Case([(2, 100), (1, 0)], [0, 5, 0], [1, 1, 1], 8, 2, 64, 16)
    c.indptr[1:] -= c.indptr[1].clone()  # sequence 0 loses its page: it sees the prefix only
    c.indices = c.indices[1:].clone()
    c.last[0] = 0
    c.check(dev)
    c = Case([], [3, 40], [1, 2], 8, 2, 64, 16)
    c.check(dev)
    c = Case([(2, 0)], [0, 0], [1, 1], 8, 2, 64, 16)
    c.indptr[:], c.last[:] = 0, 0  # nothing at all to see
    c.check(dev)


def test_equals_chunk_attention_over_whole_tables(dev):
    """A prefix of whole pages in front of each table, read per sequence, gives the same sums."""
    c = Case([(4, 320)], [50, 0, 17, 200], [1, 3, 1, 1], 8, 2, 128, 16)
    o, lse = flash_attention_shared_prefix_paged(*c.args(dev), return_lse=True)
    own = [c.indices[int(a):int(b)] for a, b in zip(c.indptr[:-1], c.indptr[1:])]
    whole = torch.cat([torch.cat((c.prefix_indices, x)) for x in own]).to(dev)
    indptr = torch.tensor([0] + [20 + len(x) for x in own]).cumsum(0).to(torch.int32).to(dev)
    o2, lse2 = flash_attention_chunk_paged(c.q.to(dev), c.q_indptr.to(dev), c.pool.to(dev), indptr,
                                           whole, c.last.to(dev), return_lse=True)
    # Each is within 3 u A of the truth, and A <= |V| here.
    assert float((o - o2).abs().max()) <= 2 * 3 * 2.0 ** -11 * float(c.pool.abs().max())
    assert float((lse - lse2).abs().max()) <= 1e-5


@pytest.mark.parametrize("scale", [0.01, 1.0, -0.2, 0.0])
def test_scales(dev, scale):
    c = Case([(4, 100)], [20, 3, 0, 60], [1, 1, 2, 1], 4, 2, 64, 16)
    c.check(dev, scale=scale)


def test_values_that_are_not_finite(dev):
    """In the pages behind a last token, in keys that rows do not see, and in keys that they see."""
    c = Case([(2, 37)], [10, 50], [3, 1], 4, 2, 64, 16)
    c.pool[c.prefix_indices[-1].long(), :, :, 37 % 16:] = math.nan
    c.pool[c.indices[0].long(), :, :, 13:] = math.inf  # behind the last token
    c.check(dev)
    c.pool[c.indices[0].long(), 1, :, 12] = math.inf  # the last new token's V: one row sees it
    c.check(dev)
    c.pool[c.prefix_indices[1].long(), 1, 0, 3] = math.nan
    c.check(dev)


def test_bad_pages_and_tables(dev):
    c = Case([(2, 100)], [40, 70], [1, 1], 4, 2, 64, 16)
    c.indices[1], c.prefix_indices[2], c.prefix_indices[4] = -1, 10 ** 6, -7
    c.check(dev)
    a = dict(zip(c.names, c.args(dev)))
    for name, bad in (("group_indptr", [5, -3]), ("group_indptr", [2, 0]), ("prefix_indptr", [9, 2]),
                      ("prefix_indptr", [-5, 10 ** 6]), ("prefix_last", [10 ** 6]),
                      ("q_indptr", [-4, 1, 90])):
        b = dict(a)
        b[name] = torch.tensor(bad, dtype=torch.int32, device=dev)
        o = flash_attention_shared_prefix_paged(*b.values())
        assert o.shape == c.q.shape


def test_strided_tensors_and_rows_of_no_sequence(dev):
    c = Case([(3, 90)], [4, 30, 9], [1, 2, 1], 4, 2, 64, 16, slack=3)
    P = c.pool.shape[0]
    wide = torch.zeros(P, 2, 4, 32, 128, dtype=F16)
    wide[:, :, 1::2, ::2, 64:] = c.pool
    wq = torch.zeros(c.q.shape[0], 8, 192, dtype=F16)
    wq[:, ::2, 64:128] = c.q
    a = c.args(dev)
    a[0], a[2] = wq.to(dev)[:, ::2, 64:128], wide.to(dev)[:, :, 1::2, ::2, 64:]
    o, lse = flash_attention_shared_prefix_paged(*a, return_lse=True)
    o2, lse2 = flash_attention_shared_prefix_paged(*c.args(dev), return_lse=True)
    assert torch.equal(o[:4], o2[:4]) and torch.equal(lse[:4], lse2[:4])


@pytest.mark.parametrize("word", [-1, 0x7fffffff, 6, 0])
@pytest.mark.parametrize("D,n", [(64, 1), (128, 9), (256, 2)])
def test_a_workspace_may_hold_anything_behind_its_counters(dev, D, n, word):
    """Rows of no sequence, and rows that no part writes because q_indptr is not in order, name no
    slots: whatever the workspace holds, they lead nowhere, and rows of no sequence stay."""
    c = Case([(3, 700)], [4, 300, 9], [n, 2, n], 4, 2, D, 16, slack=5)
    a = c.args(dev)
    T, Hq = c.q.shape[:2]
    lib = N.load()
    sizes = (3, T, Hq, 2, D, 16, a[4].numel())
    size = lib.akt_shared_prefix_paged_workspace_size(*sizes, 1, a[8].numel())
    i64 = lambda x: (C.c_int64 * len(x))(*x)  # noqa: E731
    ptr = lambda x: C.c_void_p(x.data_ptr())  # noqa: E731

    def call(q_indptr, group_indptr):
        ws = torch.full((-(-size // 4),), word, dtype=torch.int32, device=dev)
        ws[:N.WORKSPACE_ZERO_BYTES // 4] = 0
        o = torch.full((T, Hq, D), 7.0, dtype=F16, device=dev)
        lse = torch.full((T, Hq), 7.0, device=dev)
        t = dict(zip(c.names, a), q_indptr=q_indptr, group_indptr=group_indptr)
        rc = lib.akt_shared_prefix_paged_fwd(
            *(ptr(t[k]) for k in ("q", "q_indptr", "pool", "indptr", "indices", "last", "group_indptr",
                                  "prefix_indptr", "prefix_indices", "prefix_last")), ptr(o), ptr(lse),
            *sizes, 1, a[8].numel(), c.pool.shape[0], i64(a[0].stride()), i64(a[2].stride()), D ** -0.5, 1,
            0, ptr(ws), size, C.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0
        torch.cuda.synchronize()
        return o, lse

    o, lse = call(a[1], a[6])
    o2, lse2 = flash_attention_shared_prefix_paged(*a, return_lse=True)
    end = int(c.q_indptr[-1])
    assert torch.equal(o[:end], o2[:end]) and torch.equal(lse[:end], lse2[:end])
    assert bool((o[end:] == 7).all()) and bool((lse[end:] == 7).all())
    i32 = dict(dtype=torch.int32, device=dev)
    o, lse = call(torch.tensor([0, T - 1, 2, T - 2], **i32), torch.tensor([1, 3], **i32))
    assert bool((o[T - 1:] == 7).all()) and bool((lse[T - 1:] == 7).all())


def test_results_do_not_depend_on_the_run_or_the_stream(dev):
    c = Case([(9, 5000), (20, 300)], [20] * 30, [1] * 9 + [30] + [2] * 20, 8, 2, 128, 16)
    a = c.args(dev)
    first = flash_attention_shared_prefix_paged(*a, return_lse=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(flash_attention_shared_prefix_paged(*a, return_lse=True))
    torch.cuda.synchronize()
    for o, lse in outs:
        assert torch.equal(o, first[0]) and torch.equal(lse, first[1])


def test_captured_calls_replay(dev):
    """Two graphs, each with a call of its own, replayed in turn with eager calls between."""
    cases = [Case([(6, 900)], [30] * 6, [1] * 6, 8, 2, 128, 16),
             Case([(2, 100), (3, 40)], [3] * 5, [4, 1, 1, 60, 1], 8, 2, 64, 16)]
    args = [c.args(dev) for c in cases]
    want = [flash_attention_shared_prefix_paged(*a, return_lse=True) for a in args]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(flash_attention_shared_prefix_paged(*a, return_lse=True))
        graphs.append(g)
    for i in range(4):
        for g, out in zip(graphs, outs):
            out[0].zero_()
            g.replay()
        eager = flash_attention_shared_prefix_paged(*args[i % 2])
        torch.cuda.synchronize()
        assert torch.equal(eager, want[i % 2][0])
        for out, w in zip(outs, want):
            assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])


def test_nothing_to_do(dev):
    c = Case([(1, 20)], [3], [1], 4, 2, 64, 16)
    a = c.args(dev)
    assert flash_attention_shared_prefix_paged(a[0][:0], torch.zeros(2, dtype=torch.int32, device=dev),
                                               *a[2:]).shape == (0, 4, 64)
    z = torch.zeros(1, dtype=torch.int32, device=dev)
    e = torch.zeros(0, dtype=torch.int32, device=dev)
    flash_attention_shared_prefix_paged(a[0], z, a[2], z, e, e, z, z, e, e)  # no sequences
    torch.cuda.synchronize()


def test_refusals(dev):
    a = dict(zip(Case.names, Case([(2, 20)], [3, 4], [1, 1], 4, 2, 64, 16).args(dev)))

    def call(**kw):
        return flash_attention_shared_prefix_paged(*{**a, **kw}.values())

    for err, kw in ((TypeError, {"q": a["q"].float()}), (TypeError, {"pool": a["pool"].bfloat16()}),
                    (ValueError, {"q": a["q"].cpu()}), (ValueError, {"group_indptr": a["group_indptr"].cpu()}),
                    (TypeError, {"prefix_indices": a["prefix_indices"].long()}),
                    (ValueError, {"group_indptr": a["group_indptr"][:1]}),
                    (ValueError, {"prefix_indptr": torch.cat([a["prefix_indptr"]] * 2)}),
                    (ValueError, {"prefix_last": torch.cat([a["prefix_last"]] * 2)}),
                    (ValueError, {"last": a["last"][:1]}), (ValueError, {"q": a["q"][..., :32]}),
                    (RuntimeError, {"q": a["q"][:, :3]})):
        with pytest.raises(err):
            call(**kw)
    with pytest.raises(RuntimeError):
        flash_attention_shared_prefix_paged(*a.values(), softmax_scale=math.inf)
    wide = torch.randn(4, 2, 2, 16, 96, dtype=torch.float16, device=dev)
    with pytest.raises(RuntimeError, match="head_dim"):
        call(q=torch.randn(2, 4, 96, dtype=torch.float16, device=dev), pool=wide)
