"""PagedKVCache's steps on the host: which attention call a step makes, with the kernels' work left out
or done on the CPU."""
import pytest
import torch

from attention_kernel_triton_amd import _ops, paged_kv
from attention_kernel_triton_amd.paged_kv import PagedKVCache


@pytest.fixture
def calls(monkeypatch):
    """The attention calls of the steps, as (name, number of prefixes)."""
    made = []

    def attend(name):
        def call(q, q_indptr, pool, *table, return_lse=False, **kw):
            made.append((name, len(table) - 3 and len(table[-1])))
            return (q, q[..., 0].float()) if return_lse else q
        return call

    monkeypatch.setattr(paged_kv, "append_paged_kv", lambda *a: None)
    monkeypatch.setattr(paged_kv, "copy_pages", lambda *a, **kw: None)
    monkeypatch.setattr(_ops, "chunk_paged", attend("chunk"))
    monkeypatch.setattr(_ops, "shared_prefix_paged", attend("shared"))
    return made


def _z(n):
    return torch.zeros(n, 1, 8).half()


def test_a_step_without_a_shared_page_attends_as_without_shared_prefixes(calls):
    cache = PagedKVCache(40, 1, 4, 8, device="cpu")
    cache.extend(["a", "b"], _z(30), _z(30), _z(30), [21, 9], shared_prefix=True)
    cache.extend(["a"], _z(1), _z(1), _z(1), [1], shared_prefix=True)
    cache.extend([], _z(0), _z(0), _z(0), [], shared_prefix=True)
    assert calls == [("chunk", 0)] * 3
    cache.fork("a", "c")
    step = lambda seqs, n=1, **kw: cache.extend(  # noqa: E731
        seqs, _z(n * len(seqs)), _z(n * len(seqs)), _z(n * len(seqs)), [n] * len(seqs), **kw)
    step(["a", "c", "b"], shared_prefix=True)
    assert calls[-1] == ("shared", 2)
    step(["a", "b", "c"], shared_prefix=True)  # a sequence between: no neighbours share
    assert calls[-1] == ("chunk", 0)
    step(["a", "c"])
    assert calls[-1] == ("chunk", 0)
    out, lse = step(["a", "c"], return_lse=True, shared_prefix=True)
    assert calls[-1] == ("shared", 1) and out.shape == (2, 1, 8) and lse.shape == (2, 1)
