"""Groups of shared prefixes in numbers around a wave's lanes, and groups whose prefix has no keys, against
the fp64 oracle (tolerances: tests/test_gpu_shared_prefix.py)."""
import pytest
import torch

from attention_kernel_triton_amd.paged_kv import PagedKVCache
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
