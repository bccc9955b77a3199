"""Groups of shared prefixes in numbers around a wave's lanes, and groups whose prefix has no keys, against
the fp64 oracle (tolerances: tests/test_gpu_shared_prefix.py)."""
import ctypes as C

import pytest
import torch

from attention_kernel_triton_amd import _native as N
from attention_kernel_triton_amd.paged_kv import PagedKVCache
from attention_kernel_triton_amd.shared_prefix_flash_attention_paged import (
    flash_attention_shared_prefix_paged)
from test_gpu_shared_prefix import Case

pytestmark = pytest.mark.gpu


# A lane looks at the places of groups that other lanes stored, unless the sequences are a multiple of 64.
@pytest.mark.parametrize("groups,before", [(63, 1), (64, 0), (65, 2), (130, 7), (200, 64)])
def test_groups_around_a_wave(dev, groups, before):
    g = torch.Generator().manual_seed(groups)
    size = torch.randint(1, 4, (groups,), generator=g).tolist()
    B = before + sum(size) + 1
    n = torch.randint(0, 3, (B,), generator=g).tolist()
    n[B // 2] = 21  # a sequence (and so a group) of many rows
    ctx = torch.randint(0, 30, (B,), generator=g).tolist()
    prefix = torch.randint(1, 70, (groups,), generator=g).tolist()
    Case(list(zip(size, prefix)), ctx, n, 4, 2, 64, 16, before=before).check(dev)


def test_a_step_without_a_shared_page_equals_one_without_shared_prefixes(dev):
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(461, h, 128, generator=g).half().to(dev) for h in (8, 2, 2))
    outs = []
    for shared in (False, True):
        cache = PagedKVCache(60, 2, 16, 128, device=dev)
        cache.append([2], k[:50], v[:50], [50])
        outs.append(cache.extend([0, 1, 2], q, k, v, [300, 160, 1], shared_prefix=shared, return_lse=True))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def poisoned(c, dev, word=0x7fffffff):
    """(o, lse) of the case over a workspace that holds `word` behind its counters."""
    a = c.args(dev)
    (T, Hq, D), (P, _, Hkv, page, _) = c.q.shape, c.pool.shape
    sizes = (c.last.numel(), T, Hq, Hkv, D, page, c.indices.numel(), c.prefix_last.numel(),
             c.prefix_indices.numel())
    lib = N.load()
    size = lib.akt_shared_prefix_paged_workspace_size(*sizes)
    ws = torch.full((-(-size // 4),), word, dtype=torch.int32, device=dev)
    ws[:N.WORKSPACE_ZERO_BYTES // 4] = 0
    o, lse = torch.empty_like(a[0]), torch.empty(T, Hq, device=dev)
    i64 = lambda x: (C.c_int64 * len(x))(*x)  # noqa: E731
    ptr = lambda x: C.c_void_p(x.data_ptr())  # noqa: E731
    N.check(lib.akt_shared_prefix_paged_fwd(
        *map(ptr, a), ptr(o), ptr(lse), *sizes, P, i64(a[0].stride()), i64(a[2].stride()), D ** -0.5,
        1, 0, ptr(ws), size,
        C.c_void_p(torch.cuda.current_stream().cuda_stream)), "akt_shared_prefix_paged_fwd")
    torch.cuda.synchronize()
    assert not ws[:N.WORKSPACE_ZERO_BYTES // 4].any()
    return o, lse


# Sequences alone behind a prefix without keys, of few rows and of many (own keys or none), beside
# groups that have keys and one of several sequences that has none.
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G", [1, 4, 33])
def test_prefixes_without_keys(dev, D, G):
    groups = [(1, 0), (1, 0), (2, 90), (1, 0), (3, 0), (1, 17), (1, 0), (0, 0), (1, 0)]
    n = [40, 1, 50, 2, 130, 37, 1, 0, 60, 9, 3, 33]
    c = Case(groups, [0, 60, 100, 5, 7, 0, 33, 20, 12, 0, 80, 4], n, 2 * G if G < 33 else G, 2 if G < 33 else 1,
             D, 16, before=1)
    c.check(dev)
    o, lse = flash_attention_shared_prefix_paged(*c.args(dev), return_lse=True)
    for word in (0x7fffffff, -1, 6):
        o2, lse2 = poisoned(c, dev, word)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_prompts_alone_behind_no_keys_are_divided_as_without_groups(dev):
    B = 16
    c = Case([(1, 0)] * B, [7 * i for i in range(B)], [300] * B, 8, 4, 128, 16)
    plain = Case([], [7 * i for i in range(B)], [300] * B, 8, 4, 128, 16)
    want = flash_attention_shared_prefix_paged(*plain.args(dev), return_lse=True)
    assert torch.equal(c.q, plain.q) and torch.equal(c.pool, plain.pool)
    for o, lse in (flash_attention_shared_prefix_paged(*c.args(dev), return_lse=True), poisoned(c, dev)):
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


def test_prompts_alone_among_more_sequences_than_the_kernel_keeps_places_of(dev):
    n = [1] * 700
    n[5], n[333], n[699] = 50, 70, 33
    Case([(1, 0)] * 600, [i % 9 for i in range(700)], n, 2, 1, 64, 16, before=2).check(dev)


@pytest.mark.parametrize("rows", [1, 700])
def test_the_kernel_timer_counts_both_launches(dev, rows):
    """One thread to a row's dims in the join, or two where rows are few: either is timed."""
    c = Case([(2, 100)], [5, 9], [rows, 1], 32, 8, 64, 16)
    a = c.args(dev)
    flash_attention_shared_prefix_paged(*a)
    torch.cuda.synchronize()
    with N.kernel_timer() as t:
        flash_attention_shared_prefix_paged(*a)
    assert t.launches == 2 and t.total_ms > 0
