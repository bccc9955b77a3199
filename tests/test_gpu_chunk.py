"""Chunk attention over a paged cache against the fp64 oracle.

Tolerances follow from the arithmetic.  With u the half step of the 16-bit type (2^-11 in fp16,
2^-8 in bf16) and A = softmax |V|: P rounded to the type in numerator and normaliser moves O by
at most 2 u A, its own rounding by u |O| <= u A.  The scores are fp32 sums of D products:
ds <= (D + 8) 2^-24 |q| |k| scale, which moves O by at most 2 ds A and the LSE by ds.  An fp16
probability below its normal range is off by up to 2^-25 against a row maximum of at least 1.
The LSE is a sum of N fp32 terms (N 2^-24) and a few roundings of its own.
"""
import math

import pytest
import torch

from attention_kernel_triton_amd import decode_flash_attention_redundant_var_len_paged as pg
from attention_kernel_triton_amd.chunk_flash_attention_paged import flash_attention_chunk_paged
from attention_kernel_triton_amd.merge_states import merge_states
from oracle import serving

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


class Case:
    """Sequences of ctx[i] cached and n[i] new tokens over a permuted page table."""

    def __init__(self, ctx, n, Hq, Hkv, D, page, dtype=F16, seed=0, extra=3, slack=0):
        g = torch.Generator().manual_seed(1000 * seed + sum(ctx) + 7 * sum(n) + D + page)
        lens = [c + m for c, m in zip(ctx, n)]
        counts = [-(-x // page) for x in lens]
        self.lens, self.n = lens, n
        P = sum(counts) + extra
        self.indices = torch.randperm(P, generator=g)[:sum(counts)].to(torch.int32)
        self.indptr = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
        self.last = torch.tensor([(x - 1) % page + 1 if x else 0 for x in lens], dtype=torch.int32)
        self.q_indptr = torch.tensor([0] + list(n)).cumsum(0).to(torch.int32)
        self.pool = torch.randn(P, 2, Hkv, page, D, generator=g).to(dtype)
        self.q = torch.randn(sum(n) + slack, Hq, D, generator=g).to(dtype)
        self.page = page

    def slot(self, b, t):
        """(page, slot) of token t of sequence b."""
        return int(self.indices[int(self.indptr[b]) + t // self.page]), t % self.page

    def args(self, dev):
        return [x.to(dev) for x in (self.q, self.q_indptr, self.pool, self.indptr, self.indices,
                                    self.last)]

    def run(self, dev, **kw):
        o, lse = flash_attention_chunk_paged(*self.args(dev), return_lse=True, **kw)
        only = flash_attention_chunk_paged(*self.args(dev), **kw)
        return o.cpu(), lse.cpu(), only.cpu()

    def oracle(self, causal=True, scale=None):
        return serving.chunk_attention(self.q, self.q_indptr, self.pool, self.indptr, self.indices,
                                       self.last, causal, scale)

    def check(self, dev, causal=True, scale=None):
        o, lse, only = self.run(dev, causal=causal, softmax_scale=scale)
        compare(self, o, lse, self.oracle(causal, scale))
        compare(self, only, None, self.oracle(causal, scale))


def compare(c, o, lse, ref):
    O, L, A, C = ref
    D, N = c.q.shape[-1], max(c.lens)
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
    if lse is not None:
        empty = L == -math.inf
        assert torch.equal(lse == -math.inf, empty)
        t = ds + (N + 40) * 2.0 ** -24 + 4 * 2.0 ** -23 * L.abs().nan_to_num(0, 0, 0) + 1e-6
        fin = torch.isfinite(L)
        over = ((lse.double() - L).abs() - t)[fin]
        assert over.numel() == 0 or float(over.max()) <= 0, float(over.max())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,page,Hq,Hkv", [(64, 16, 8, 2), (128, 16, 8, 2), (256, 16, 4, 2),
                                           (128, 24, 6, 2), (64, 1, 5, 1), (256, 7, 2, 2),
                                           (128, 64, 14, 2), (64, 48, 12, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_mixed_batches(dev, D, page, Hq, Hkv, dtype, causal):
    Case([0, 12, 300, 77, 0, 1000], [5, 1, 33, 0, 1, 3], Hq, Hkv, D, page, dtype).check(dev, causal)


# Rows of a unit around its wave and unit edges, steps and tiles cut at every place, and
# sequences that begin with the chunk.
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 130, 257])
@pytest.mark.parametrize("ctx", [0, 1, 31, 32, 127, 128, 129, 600])
def test_chunk_and_context_lengths(dev, n, ctx):
    Case([ctx], [n], 8, 2, 64, 16).check(dev)


@pytest.mark.parametrize("G", [1, 2, 3, 5, 6, 7, 8, 12, 16, 31, 33, 64, 100, 128])
@pytest.mark.parametrize("n,ctx", [(1, 200), (5, 40), (70, 10)])
def test_query_heads_per_kv_head(dev, G, n, ctx):
    Case([ctx, ctx + 3], [n, 1], 2 * G if G <= 32 else G, 2 if G <= 32 else 1, 64, 16).check(dev)


# Long sequences alone (one unit's keys over many workgroups), with one token and with several
# row blocks.
@pytest.mark.parametrize("n,ctx,Hq,Hkv,D,page,dtype", [
    (1, 9000, 4, 1, 128, 16, F16), (1, 20001, 8, 2, 64, 32, BF16), (40, 7000, 8, 2, 128, 16, F16),
    (130, 5000, 4, 2, 256, 24, F16), (300, 3000, 8, 1, 128, 128, BF16), (3, 6000, 16, 1, 256, 16, BF16)])
@pytest.mark.parametrize("causal", [True, False])
def test_units_cut_over_workgroups(dev, n, ctx, Hq, Hkv, D, page, dtype, causal):
    Case([ctx], [n], Hq, Hkv, D, page, dtype).check(dev, causal)


# More sequences than a wave has lanes, many of them without new tokens or without tokens.
@pytest.mark.parametrize("B", [64, 65, 200])
def test_many_sequences(dev, B):
    g = torch.Generator().manual_seed(B)
    n = torch.randint(0, 4, (B,), generator=g).tolist()
    ctx = torch.randint(0, 90, (B,), generator=g).tolist()
    n[B // 2:B // 2 + 20] = [0] * 20
    Case(ctx, n, 4, 2, 64, 16).check(dev)
    Case(ctx, n, 4, 2, 128, 8, BF16).check(dev, causal=False)


def test_one_long_chunk_beside_single_tokens(dev):
    Case([100] * 5 + [0] + [900] * 6, [1] * 5 + [777] + [1] * 6, 8, 2, 128, 16).check(dev)


def test_results_do_not_depend_on_the_run(dev):
    a = Case([5000, 40, 3000], [33, 200, 1], 8, 2, 128, 16).args(dev)
    first = flash_attention_chunk_paged(*a, return_lse=True)
    for _ in range(5):
        again = flash_attention_chunk_paged(*a, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_single_tokens_agree_with_the_paged_decode(dev):
    c = Case([300, 17, 2000, 0], [1, 1, 1, 1], 8, 2, 128, 16)
    q, _, pool, indptr, indices, last = c.args(dev)
    o, lse = flash_attention_chunk_paged(*c.args(dev), return_lse=True)
    ro, rl = pg.flash_attention_decode_paged(q.unsqueeze(2), pool, indptr, indices, last,
                                             return_lse=True)
    # Both are within 3 u A of the exact result, A below 3 here.
    assert float((o - ro).abs().max()) <= 6 * 2.0 ** -11 * 3
    assert float((lse - rl).abs().max()) <= 1e-4


def test_parts_of_a_context_merge_into_the_whole(dev):
    """Attention over the first 512 tokens (not causal) and, as a cache of their own, over the
    rest (causal) merge into attention over all."""
    c = Case([900], [20], 8, 2, 128, 16)
    whole, wl, _ = c.run(dev)
    q, qp, pool, indptr, indices, last = c.args(dev)
    i32 = dict(dtype=torch.int32, device=dev)
    a = flash_attention_chunk_paged(q, qp, pool, torch.tensor([0, 32], **i32), indices[:32],
                                    torch.tensor([16], **i32), causal=False, return_lse=True)
    b = flash_attention_chunk_paged(q, qp, pool, torch.tensor([0, indices.numel() - 32], **i32),
                                    indices[32:], last, return_lse=True)
    o, lse = merge_states(torch.stack([a[0], b[0]]), torch.stack([a[1], b[1]]))
    assert float((o.cpu() - whole).abs().max()) <= 9 * 2.0 ** -11 * 3
    assert float((lse.cpu() - wl).abs().max()) <= 1e-5


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.0])
def test_scales(dev, scale):
    Case([50, 200], [9, 1], 8, 2, 64, 16).check(dev, scale=scale)


def test_rows_that_see_nothing(dev):
    """Sequences without pages, and (a table that breaks the contract) more new tokens than
    tokens: zeros and -inf, and the rows that see keys keep theirs."""
    c = Case([0, 30, 0], [4, 3, 0], 8, 2, 64, 16)
    c.q_indptr = torch.tensor([0, 3, 43, 44], dtype=torch.int32)
    c.q = torch.randn(44, 8, 64, generator=torch.Generator().manual_seed(4)).half()
    for causal in (True, False):
        o, lse, only = c.run(dev, causal=causal)
        O, L, A, C = c.oracle(causal)
        compare(c, o, lse, (O, L, A, C))
        compare(c, only, None, (O, L, A, C))
        assert float(o[43:].abs().max()) == 0 and bool((lse[43:] == -math.inf).all())


def test_rows_of_no_sequence_are_left_alone(dev):
    c = Case([5, 60], [2, 3], 8, 2, 64, 16, slack=7)
    c.q[5:] = math.nan
    o, lse, _ = c.run(dev)
    ref = c.oracle()
    compare(c, o[:5], lse[:5], tuple(x[:5] for x in ref))


@pytest.mark.parametrize("page", [16, 8])
@pytest.mark.parametrize("n", [1, 6, 70])
def test_pages_outside_the_pool_are_skipped(dev, page, n):
    c = Case([150, 400, 40], [n, n, n], 8, 2, 64, page)
    for i in (0, 3, 5, 20):
        c.indices[i] = [-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1][i % 4]
    c.indices[int(c.indptr[2]):int(c.indptr[3])] = -5  # a sequence of nothing else
    c.check(dev)
    c.check(dev, causal=False)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D,page,dtype,n", [(64, 16, F16, 5), (128, 24, BF16, 40), (256, 16, F16, 9),
                                            (128, 16, BF16, 3)])
def test_masked_values_never_reach_a_row(dev, D, page, dtype, n, bad):
    """K and V of slots past the length, and of the last two new tokens, hold values that are not
    finite: rows that do not see them stay exact."""
    c = Case([70, 200], [n, n], 4, 2, D, page, dtype)
    for b in range(2):
        length = c.lens[b]
        for t in range(length, -(-length // page) * page):
            p, s = c.slot(b, t)
            c.pool[p, :, :, s] = bad
        for t in (length - 2, length - 1):
            p, s = c.slot(b, t)
            c.pool[p, 1, :, s] = bad
            c.pool[p, 0, 1, s] = bad
    o, lse, only = c.run(dev)
    O, L, A, C = c.oracle()
    keep = torch.ones(2 * n, dtype=torch.bool)
    for b in range(2):
        keep[b * n + n - 2:b * n + n] = False
    assert bool(torch.isfinite(O[keep]).all())
    ref = tuple(x[keep] for x in (O, L, A, C))
    compare(c, o[keep], lse[keep], ref)
    compare(c, only[keep], None, ref)
    assert not bool(torch.isfinite(o[~keep]).any())


def test_a_value_that_is_seen_comes_through(dev):
    """An infinity in V at a key that all rows see gives infinities, a NaN gives NaN."""
    c = Case([200], [4], 4, 1, 64, 16)
    p, s = c.slot(0, 3)
    c.pool[p, 0, 0, s] = c.q[0, 0]  # a score that is not small for one head
    c.pool[p, 1, 0, s, 5] = math.inf
    c.pool[p, 1, 0, s, 9] = math.nan
    o, _, _ = c.run(dev)
    assert bool(torch.isnan(o[:, :, 9]).all())
    assert bool((o[0, 0, 5] == math.inf).all())
    rest = [d for d in range(64) if d not in (5, 9)]
    assert bool(torch.isfinite(o[:, :, rest]).all())


def test_large_scores_raise_the_running_max(dev):
    """Scores that grow along the keys by far more than the slack, and fall again."""
    c = Case([700], [40], 8, 2, 128, 16)
    g = torch.Generator().manual_seed(2)
    for t in range(740):
        p, s = c.slot(0, t)
        c.pool[p, 0, :, s] *= 1 + 8 * math.sin(t / 110.0) ** 2
    c.q *= 3
    c.check(dev)


def test_strided_tensors(dev):
    """q as a view of a fused projection, the pool as every other head of a wider one."""
    c = Case([40, 333], [7, 1], 8, 2, 64, 16)
    ref = c.run(dev)[0]
    q, qp, pool, indptr, indices, last = c.args(dev)
    wide = torch.full((pool.shape[0], 2, 4, 16, 64), 9.0, dtype=F16, device=dev)
    wide[:, :, ::2] = pool
    qw = torch.zeros((8, 12, 64), dtype=F16, device=dev)
    qw[:, 2:10] = q
    o = flash_attention_chunk_paged(qw[:, 2:10], qp, wide[:, :, ::2], indptr, indices, last)
    assert torch.equal(o.cpu(), ref)
    slots = torch.zeros((pool.shape[0], 2, 2, 32, 64), dtype=F16, device=dev)
    slots[:, :, :, ::2] = pool
    o = flash_attention_chunk_paged(q, qp, slots[:, :, :, ::2], indptr, indices, last)
    assert torch.equal(o.cpu(), ref)


def test_empty_calls(dev):
    c = Case([0], [0], 4, 2, 64, 16)
    o, lse, _ = c.run(dev)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    i32 = dict(dtype=torch.int32, device=dev)
    q = torch.zeros((3, 4, 64), dtype=F16, device=dev)
    pool = torch.zeros((2, 2, 2, 16, 64), dtype=F16, device=dev)
    none = torch.zeros(0, **i32)
    flash_attention_chunk_paged(q, torch.zeros(1, **i32), pool, torch.zeros(1, **i32), none, none)
    o = flash_attention_chunk_paged(q, torch.tensor([0, 3], **i32), pool, torch.tensor([0, 0], **i32),
                                    none, torch.zeros(1, **i32))
    assert float(o.abs().max()) == 0


def test_another_stream(dev):
    c = Case([400, 3000], [9, 1], 8, 2, 64, 16)
    ref = c.run(dev)[0]
    a = c.args(dev)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        o = flash_attention_chunk_paged(*a)
    st.synchronize()
    assert torch.equal(o.cpu(), ref)


@pytest.mark.parametrize("B,n,D,Hq,Hkv", [(1, 1, 128, 8, 8), (2, 16, 128, 32, 8), (4, 7, 64, 8, 8),
                                          (5, 1, 128, 8, 8), (3, 3, 128, 4, 1)])
def test_few_units_share_the_workgroups(dev, B, n, D, Hq, Hkv):
    """Few units over all workgroups, on both sides of an eighth of them."""
    Case([6000 + 131 * i for i in range(B)], [n] * B, Hq, Hkv, D, 16).check(dev)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_around_the_borders(dev, D, dtype):
    """Sequences of few and of many rows to a kv head beside each other."""
    Case([900, 40, 2000, 0, 500, 1300, 70], [31, 32, 33, 63, 64, 65, 1], 2, 2, D, 16, dtype).check(dev)


def test_two_streams_at_once(dev):
    """Calls that overlap on two streams each have a workspace of their own."""
    cases = [Case([9000, 50, 2000], [1, 300, 5], 16, 4, 128, 16, seed=s) for s in range(2)]
    args = [c.args(dev) for c in cases]
    want = [flash_attention_chunk_paged(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    out = []
    for _ in range(8):
        for st, a in zip(streams, args):
            with torch.cuda.stream(st):
                out.append(flash_attention_chunk_paged(*a))
    torch.cuda.synchronize()
    for i, o in enumerate(out):
        assert torch.equal(o, want[i % 2])


def test_padded_batch(dev):
    """Sequences with neither tokens nor pages between the others, rows of q past the last one."""
    c = Case([300, 0, 0, 2000, 0, 77, 0], [200, 0, 1, 2, 0, 0, 0], 8, 2, 64, 16, slack=5)
    o, lse, _ = c.run(dev)
    O, L, A, C = c.oracle()
    m = sum(c.n)
    c.q = c.q[:m]
    compare(c, o[:m], lse[:m], (O[:m], L[:m], A[:m], C[:m]))


def test_graph_replays_follow_the_tables(dev):
    """A captured call replayed on changed tables and inputs, beside eager calls and a second
    graph captured on the same stream."""
    cases = [Case([3000, 40], [9, 1], 8, 2, 64, 16, seed=s) for s in range(3)]
    short = Case([700, 1500], [4, 6], 8, 2, 64, 16)  # the same shapes, other lengths
    static = [x.clone() for x in cases[0].args(dev)]
    other = [x.clone() for x in cases[1].args(dev)]
    flash_attention_chunk_paged(*static)
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        oa = flash_attention_chunk_paged(*static)
    with torch.cuda.graph(gb):
        ob = flash_attention_chunk_paged(*other)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for c in (cases[0], cases[2], short, cases[0]):
        new = c.args(dev)
        P, T = static[2].shape[0], static[4].numel()
        static[0].copy_(new[0])
        static[1].copy_(new[1])
        static[2][:new[2].shape[0]].copy_(new[2][:P])
        static[3].copy_(new[3])
        static[4][:min(T, new[4].numel())].copy_(new[4][:T])
        static[5].copy_(new[5])
        want = flash_attention_chunk_paged(*[x.clone() for x in static])
        wantb = flash_attention_chunk_paged(*other)
        torch.cuda.synchronize()
        for _ in range(3):
            oa.zero_()
            ob.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(sa):
                ga.replay()
            with torch.cuda.stream(sb):
                gb.replay()
            torch.cuda.synchronize()
            assert torch.equal(oa, want) and torch.equal(ob, wantb)


def plant(c, b, heads, first, bad):
    """Writes `bad` into V of keys first .. first + 43 of sequence b (those that it has) for each kv
    head in `heads`, a dim of its own for every key.  Returns (key, kv head, dim) of each."""
    out = []
    for h in heads:
        for i in range(44):
            t = first + i
            if 0 <= t < c.lens[b]:
                p, s = c.slot(b, t)
                c.pool[p, 1, h, s, i] = bad
                out.append((t, h, i))
    return out


# Keys on both sides of the last one that every row of a unit sees: up to 40 before it, 3 after.
# 300 tokens of 4 heads to a kv head are several units, of which the `unit`-th is looked at.
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 24), (256, 16)])
@pytest.mark.parametrize("n,ctx,unit", [(1, 200, 0), (1, 95, 0), (1, 4100, 0), (3, 45, 0), (3, 128, 0),
                                        (3, 3001, 0), (12, 250, 0), (40, 7, 0), (40, 190, 0),
                                        (300, 101, 0), (300, 101, 2), (300, 3000, 1)])
def test_values_that_rows_see_come_through_at_the_diagonal(dev, n, ctx, unit, D, page, dtype, bad):
    """A value of V that is not finite reaches the rows that see its key, and no others.  A positive
    probability times it is the value itself, so each dim of O is finite or exactly that."""
    c = Case([ctx, 33], [n, 1], 8, 2, D, page, dtype)
    clean = c.pool.clone()
    tokens = 32 * (8 if D <= 128 else 4) // 4
    planted = plant(c, 0, (0, 1), ctx + unit * tokens - 40, bad)
    planted = [(0, n, ctx, *x) for x in planted]
    planted += [(n, 1, 33, *x) for x in plant(c, 1, (1,), 33 - 40, bad)]  # a single token beside it
    o, lse, only = c.run(dev)
    c.pool, clean = clean, c.pool
    O, L, A, C = c.oracle()
    for row, m, pos, t, h, i in planted:
        O[row + max(0, t - pos):row + m, 4 * h:4 * h + 4, i] = bad
    compare(c, o, lse, (O, L, A, C))
    compare(c, only, None, (O, L, A, C))


@pytest.mark.parametrize("n", [1, 5, 40, 300])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_values_come_through_where_every_token_sees_all(dev, n, D):
    c = Case([150], [n], 8, 2, D, 16)
    clean = c.pool.clone()
    planted = plant(c, 0, (0, 1), 150 - 40, math.inf)
    o, lse, only = c.run(dev, causal=False)
    c.pool = clean
    O, L, A, C = c.oracle(False)
    for t, h, i in planted:
        O[:, 4 * h:4 * h + 4, i] = math.inf
    compare(c, o, lse, (O, L, A, C))
    compare(c, only, None, (O, L, A, C))
