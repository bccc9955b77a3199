"""Which layouts of sums of attention weight are taken where they are written."""
import pytest
import torch

from attention_kernel_triton_amd.attention_weights_paged import accumulate_attention_weights_paged
from attention_kernel_triton_amd.paged_kv import keep_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("strides,apart", [
    ((80, 40, 1), True), ((40, 120, 1), True),  # rows one behind another, by sequence or by head
    ((100, 50, 1), True), ((50, 100, 1), False), ((120, 240, 1), False), ((120, 200, 1), True), ((100, 150, 1), True),
    ((90, 140, 1), True), ((39, 200, 1), False), ((200, 39, 1), False), ((80, 0, 1), False),
    ((80, 1, 1), False), ((60, 100, 1), False), ((60, 80, 1), False)])
def test_rows_that_overlap_are_refused(dev, strides, apart):
    """Three sequences' rows of 40 sums for two heads; two workgroups would write what rows share."""
    buf = torch.zeros(1000, device=dev)
    w = buf.as_strided((3, 2, 40), strides)
    places = {n * strides[0] + h * strides[1] + j for n in range(3) for h in range(2) for j in range(40)}
    assert (len(places) == 240) == apart
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    g = torch.Generator().manual_seed(1)
    pool = torch.randn(6, 2, 2, 16, 64, generator=g).half().to(dev)
    q = torch.randn(3, 4, 64, generator=g).half().to(dev)
    table = (i(0, 1, 3, 5), i(0, 1, 2, 3, 4), i(9, 12, 16))
    ind = i(*range(8)).expand(3, 2, 8).contiguous()
    if not apart:
        with pytest.raises(ValueError, match="same memory"):
            accumulate_attention_weights_paged(w, q, i(0, 1, 2, 3), torch.zeros(3, 4, device=dev), pool, *table)
        with pytest.raises(ValueError, match="same memory"):
            keep_tokens(pool, *table, ind, i(8, 8, 8, 8, 8, 8).view(3, 2), weights=w)
        assert not buf.any()
        return
    plain = torch.zeros(3, 2, 40, device=dev)
    for x in (w, plain):
        accumulate_attention_weights_paged(x, q, i(0, 1, 2, 3), torch.zeros(3, 4, device=dev), pool, *table)
        keep_tokens(pool, *table, ind, i(8, 8, 8, 8, 8, 8).view(3, 2), weights=x)
    assert plain.any() and torch.equal(w, plain)
    outside = torch.ones(1000, dtype=torch.bool)
    outside[list(places)] = False
    assert not buf.cpu()[outside].any()
