"""Rotary positions, dense and appended to a paged cache, against the fp64 oracle.

Tolerances: with u the half step of the 16-bit type, the output is off by its own rounding,
u |y|, and by 32-bit work: products and sums of a cos - b sin (4 x 2^-24 (|a| + |b|)), the
angle's fraction rounded to 32 bits of a turn (2 pi 2^-25), and v_sin_f32 / v_cos_f32, which
are documented to about 2^-20 of absolute error: 1.5e-6 (|a| + |b|) |factor| in all.
"""
import math

import pytest
import torch

from attention_kernel_triton_amd.paged_kv import append_paged_kv, append_paged_kv_rotary
from attention_kernel_triton_amd.rotary import apply_rotary, rotary_frequencies
from oracle import serving

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def check(got, x, ref, rot, factor=1.0):
    got, x = got.cpu(), x.cpu()
    assert got.dtype == x.dtype and got.shape == x.shape
    u = torch.finfo(x.dtype).eps / 2
    pair = 2 * x.double().abs().amax(-1, keepdim=True) * abs(factor)
    tiny = torch.finfo(x.dtype).smallest_normal * u
    tol = u * 1.001 * ref.abs() + 1.5e-6 * pair + tiny
    err = (got.double() - ref).abs() - tol
    assert float(err.max()) <= 0, float(err.max())
    assert torch.equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,Hq,Hkv,S,D,rot", [
    (2, 8, 2, 77, 64, 64), (1, 4, 4, 1, 128, 128), (3, 6, 2, 33, 128, 64), (1, 5, 1, 130, 256, 64),
    (2, 3, 1, 9, 16, 16), (1, 2, 1, 5, 1024, 512), (2, 4, 2, 19, 128, 60), (1, 2, 2, 40, 64, 2),
    (1, 3, 1, 7, 72, 72), (1, 2, 1, 11, 40, 32), (1, 2, 1, 3, 8, 6), (1, 33, 7, 300, 32, 32)])
def test_dense(dev, B, Hq, Hkv, S, D, rot, interleaved, dtype):
    g = torch.Generator().manual_seed(B + Hq + S + D + rot)
    Q = torch.randn(B, Hq, S, D, generator=g).to(dtype)
    K = torch.randn(B, Hkv, S, D, generator=g).to(dtype)
    inv, factor = rotary_frequencies(rot, device="cpu")
    for pos, transpose, fac in ((None, False, 1.0),
                                (torch.randint(0, 10 ** 6, (B, S), generator=g), True, 1.3),
                                (torch.randint(-50, 2 ** 31 - 1, (S,), generator=g).int(), False, -0.5)):
        kw = dict(interleaved=interleaved, factor=fac, transpose=transpose)
        q, k = apply_rotary(Q.to(dev), K.to(dev), inv.to(dev),
                            positions=None if pos is None else pos.to(dev), **kw)
        p = torch.arange(S)[None] if pos is None else (pos if pos.dim() == 2 else pos[None])
        for got, x in ((q, Q), (k, K)):
            assert got.is_contiguous()
            check(got, x, serving.rotate(x, p[:, None], inv, **kw), rot, fac)


def test_k_may_be_left_out(dev):
    Q = torch.randn(1, 3, 20, 64, generator=torch.Generator().manual_seed(1)).half()
    inv, _ = rotary_frequencies(64, device=dev)
    q, k = apply_rotary(Q.to(dev), None, inv)
    assert k is None
    check(q, Q, serving.rotate(Q, torch.arange(20), inv.cpu()), 64)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [64, 20])
def test_transpose_is_the_gradient(dev, rot, interleaved):
    """<y, R x> = <R^T y, x>, against the formula's gradient by autograd in fp64 and against
    differences of the forward."""
    g = torch.Generator().manual_seed(rot)
    X = torch.randn(2, 3, 10, 64, generator=g).half()
    Y = torch.randn(2, 3, 10, 64, generator=g).half()
    inv, _ = rotary_frequencies(rot, device="cpu")
    kw = dict(interleaved=interleaved, factor=1.25)
    grad, _ = apply_rotary(Y.to(dev), None, inv.to(dev), transpose=True, **kw)
    x64 = X.double().requires_grad_()
    y = x64.clone()
    r = rot
    ang = torch.arange(10)[:, None].double() * inv
    first = slice(0, r, 2) if interleaved else slice(0, r // 2)
    second = slice(1, r, 2) if interleaved else slice(r // 2, r)
    a, b = x64[..., first], x64[..., second]
    y[..., first] = 1.25 * (a * ang.cos() - b * ang.sin())
    y[..., second] = 1.25 * (a * ang.sin() + b * ang.cos())
    y.backward(Y.double())
    check(grad, Y, x64.grad, rot, 1.25)
    # Differences along a direction: the map is linear, so a whole step is exact but for
    # roundings of the two outputs (u |.| each, values below 8).
    E = torch.randn(X.shape, generator=g).half()
    f1, _ = apply_rotary((X + E).to(dev), None, inv.to(dev), **kw)
    f0, _ = apply_rotary(X.to(dev), None, inv.to(dev), **kw)
    step = (X + E).double() - X.double()
    lhs = ((f1.cpu().double() - f0.cpu().double()) * Y.double()).sum()
    rhs = (grad.cpu().double() * step).sum()
    n = X.numel()
    bound = 2.0 ** -11 * 8 * 3 * n * 4.5
    assert abs(float(lhs - rhs)) <= bound
    assert abs(float(lhs - rhs)) <= 6 * 2.0 ** -11 * 8 * math.sqrt(n) * 4.5  # roundings are independent


def test_dense_strides_and_streams(dev):
    """Token-major projections seen as [B, H, S, D], and positions with strides."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 30, 10, 64, generator=g).half().to(dev)  # [B, S, heads, D]
    Q, K = x[:, :, :8].transpose(1, 2), x[:, :, 8:].transpose(1, 2)
    inv, _ = rotary_frequencies(64, device=dev)
    pos = torch.randint(0, 999, (30, 2), generator=g).to(dev).t()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        q, k = apply_rotary(Q, K, inv, positions=pos)
    st.synchronize()
    for got, t in ((q, Q), (k, K)):
        check(got, t, serving.rotate(t.cpu(), pos.cpu()[:, None], inv.cpu()), 64)
    odd = torch.randn(1, 2, 5, 65, generator=g).half().to(dev)[..., 1:]  # rows not 16-byte aligned
    q, _ = apply_rotary(odd, None, inv)
    check(q, odd, serving.rotate(odd.cpu(), torch.arange(5), inv.cpu()), 64)


def test_values_that_are_not_finite_stay_in_their_pair(dev):
    for rot in (64, 20):
        Q = torch.ones(1, 1, 2, 64).half()
        Q[0, 0, 1, 3] = math.nan
        Q[0, 0, 1, 63] = math.inf
        inv, _ = rotary_frequencies(rot, device=dev)
        q, _ = apply_rotary(Q.to(dev), None, inv)
        bad = ~torch.isfinite(q.cpu()[0, 0])
        want = {3, 3 + rot // 2, 63} | ({31} if rot == 64 else set())
        assert {int(d) for d in bad[1].nonzero()} == want and not bool(bad[0].any())


def test_empty_dense(dev):
    inv, _ = rotary_frequencies(64, device=dev)
    q, k = apply_rotary(torch.zeros(0, 2, 5, 64).half().to(dev), torch.zeros(0, 1, 5, 64).half().to(dev),
                        inv)
    assert q.shape == (0, 2, 5, 64) and k.shape == (0, 1, 5, 64)
    q, _ = apply_rotary(torch.zeros(2, 2, 0, 64).half().to(dev), None, inv)
    assert q.shape == (2, 2, 0, 64)


@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "yarn"])
def test_frequencies(scaling):
    inv, factor = rotary_frequencies(64, 10000.0, scaling, 1.0 if scaling is None else 4.0, 4096, "cpu")
    plain = torch.tensor([10000.0 ** (-f / 32) for f in range(32)], dtype=torch.float64)
    assert inv.dtype == torch.float64 and inv.shape == (32,)
    if scaling is None:
        want = plain
    elif scaling == "linear":
        want = plain / 4
    elif scaling == "ntk":
        want = plain * torch.tensor([4.0 ** (-f / 31) for f in range(32)], dtype=torch.float64)
    else:
        turns = 4096 * plain / (2 * math.pi)
        mix = torch.tensor([min(1.0, max(0.0, (float(t) - 1) / 31)) for t in turns], dtype=torch.float64)
        want = plain * (mix + (1 - mix) / 4)
        assert float(inv[0]) == 1.0 and abs(float(inv[-1] / plain[-1]) - 0.25) < 1e-12
    assert torch.allclose(inv, want, rtol=1e-13)
    assert factor == (0.1 * math.log(4.0) + 1 if scaling == "yarn" else 1.0)


def _table(g, lens, page, extra=2):
    counts = [-(-n // page) for n in lens]
    indices = torch.randperm(sum(counts) + extra, generator=g)[:sum(counts)].to(torch.int32)
    indptr = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    last = torch.tensor([(n - 1) % page + 1 if n else 0 for n in lens], dtype=torch.int32)
    return indptr, indices, last, sum(counts) + extra


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,rot,page", [(8, 2, 128, 128, 16), (3, 1, 64, 32, 1), (4, 4, 256, 64, 24),
                                               (6, 2, 64, 20, 16), (5, 5, 80, 80, 7), (2, 1, 1024, 1024, 4),
                                               (1, 1, 768, 768, 4), (70, 10, 128, 112, 16)])
def test_append(dev, Hq, Hkv, D, rot, page, interleaved, dtype):
    g = torch.Generator().manual_seed(Hq + D + rot + page)
    n = [3, 0, 1, 40, 0, 17] + [1] * 70
    ctx = [0, 5, 200, 9, 0, 33] + torch.randint(0, 60, (70,), generator=g).tolist()
    indptr, indices, last, P = _table(g, [a + b for a, b in zip(ctx, n)], page)
    T, slack = sum(n), 5
    ap = torch.tensor([0] + n).cumsum(0).to(torch.int32)
    q = torch.randn(T + slack, Hq, D, generator=g).to(dtype)
    kv = torch.randn(T + slack, 2, Hkv, D, generator=g).to(dtype)
    pool = torch.randn(P, 2, Hkv, page, D, generator=g).to(dtype)
    inv, _ = rotary_frequencies(rot, 500000.0, device="cpu")
    bad = int(indices[int(indptr[3])])  # the first page of a sequence whose rows begin after it
    if ctx[3] + n[3] > page:
        indices[int(indptr[4]) - 1] = P + 3
    gp = pool.clone().to(dev)
    kvd = kv.to(dev)
    got = append_paged_kv_rotary(q.to(dev), kvd[:, 0], kvd[:, 1], ap.to(dev), gp, indptr.to(dev),
                                 indices.to(dev), last.to(dev), inv.to(dev),
                                 interleaved=interleaved, factor=1.1)
    pos = torch.cat([torch.arange(c, c + m) for c, m in zip(ctx, n)])
    kw = dict(interleaved=interleaved, factor=1.1)
    check(got[:T], q[:T], serving.rotate(q[:T], pos[:, None], inv, **kw), rot, 1.1)
    kr = serving.rotate(kv[:T, 0], pos[:, None], inv, **kw)
    out, touched = gp.cpu(), torch.zeros(P, page, dtype=torch.bool)
    t = 0
    for b, (c, m) in enumerate(zip(ctx, n)):
        for i in range(m):
            pg = int(indices[int(indptr[b]) + (c + i) // page])
            if 0 <= pg < P:
                s = (c + i) % page
                touched[pg, s] = True
                check(out[pg, 0, :, s], kv[t, 0], kr[t], rot, 1.1)
                assert torch.equal(out[pg, 1, :, s], kv[t, 1])
            t += 1
    keep = ~touched[:, None, None, :, None].expand_as(out)
    assert torch.equal(out[keep], pool[keep])
    assert bad >= 0


def test_append_at_far_positions(dev):
    """A page table whose pages repeat: positions past 10^6 without a pool of that size."""
    g = torch.Generator().manual_seed(8)
    page, length = 1 << 12, (1 << 20) + 77
    np_ = -(-length // page)
    indices = torch.zeros(np_, dtype=torch.int32)
    indices[-1] = 1
    ap = torch.tensor([0, 5], dtype=torch.int32)
    q, k, v = (torch.randn(5, 2, 64, generator=g).half() for _ in range(3))
    pool = torch.zeros(2, 2, 2, page, 64).half().to(dev)
    inv, _ = rotary_frequencies(64, device="cpu")
    out = append_paged_kv_rotary(q.to(dev), k.to(dev), v.to(dev), ap.to(dev), pool,
                                 torch.tensor([0, np_], dtype=torch.int32, device=dev), indices.to(dev),
                                 torch.tensor([77], dtype=torch.int32, device=dev), inv.to(dev))
    pos = torch.arange(length - 5, length)
    check(out, q, serving.rotate(q, pos[:, None], inv), 64)
    check(pool[1, 0, :, 72:77].transpose(0, 1), k, serving.rotate(k, pos[:, None], inv), 64)
    assert torch.equal(pool[1, 1, :, 72:77].transpose(0, 1).cpu(), v)


def test_tables_outside_the_contract_write_nothing_else(dev):
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(6, 2, 64, generator=g).half().to(dev) for _ in range(3))
    inv, _ = rotary_frequencies(64, device=dev)
    i32 = dict(dtype=torch.int32, device=dev)
    for indptr, last, ap in (([0, 0], [4], [0, 6]),        # no pages
                             ([0, 1], [3], [0, 6]),        # more new tokens than tokens
                             ([-7, 90], [3], [0, 6]),      # outside the table
                             ([0, 2], [2 ** 31 - 1], [5, 2]),
                             ([0, 2], [-4], [-3, 99])):
        pool = torch.zeros((4, 2, 2, 8, 64), dtype=F16, device=dev)
        append_paged_kv_rotary(q, k, v, torch.tensor(ap, **i32), pool, torch.tensor(indptr, **i32),
                               torch.tensor([2, 0], **i32), torch.tensor(last, **i32), inv)
        assert float(pool[[1, 3]].abs().max()) == 0


def test_plain_append_takes_bf16(dev):
    g = torch.Generator().manual_seed(6)
    k, v = (torch.randn(3, 2, 64, generator=g).bfloat16().to(dev) for _ in range(2))
    pool = torch.zeros((2, 2, 2, 4, 64), dtype=BF16, device=dev)
    i32 = dict(dtype=torch.int32, device=dev)
    append_paged_kv(k, v, torch.tensor([0, 3], **i32), pool, torch.tensor([0, 1], **i32),
                    torch.tensor([1], **i32), torch.tensor([3], **i32))
    assert torch.equal(pool[1, 0, :, :3].transpose(0, 1), k)
    assert torch.equal(pool[1, 1, :, :3].transpose(0, 1), v)
    assert float(pool[0].abs().max()) == 0
