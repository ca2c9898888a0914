"""Workspaces of attention_paged that a batch has outgrown are refused before
anything reaches a GPU, empty ones too; so are streams of another device."""

from types import SimpleNamespace

import pytest
import torch

from kernrelay_amd import ops
from tests.test_paged_refusals import cache, seqs


def handles(table_pages, n):
    c = cache()
    s = seqs(seqs=n, max_new=1, table_pages=table_pages, ld_table=table_pages)
    c.torch_dtype, c.device, s.device, s.rows = torch.bfloat16, 0, 0, None
    return c, s


def space(nbytes, ncnt):
    return dict(ws=torch.empty(nbytes, dtype=torch.uint8), counters=torch.zeros(ncnt, dtype=torch.int32))


@pytest.mark.parametrize("first,then,n", [(2, 4000, 1), (2, 4000, 64), (30, 4000, 64), (4000, 4000, 64)])
def test_a_sequence_that_grows_on_its_first_workspace(monkeypatch, first, then, n):
    monkeypatch.setattr(ops, "_launch_stream", lambda *a: None)
    q = torch.zeros(n, 8, 128, dtype=torch.bfloat16)
    one = handles(first, 1)
    need = ops.attention_paged_workspace(*one, 8)
    c, s = handles(then, n)
    assert (need == (0, 0)) == (first == 2)
    more = ops.attention_paged_workspace(c, s, 8)
    assert more[0] > need[0] or more[1] > need[1]
    with pytest.raises(RuntimeError, match="workspace is too small"):
        ops.attention_paged(c, 0, s, q, torch.empty_like(q), **space(*need))
    if more[1]:  # enough memory, no counters
        with pytest.raises(RuntimeError, match="workspace is too small"):
            ops.attention_paged(c, 0, s, q, torch.empty_like(q), **space(more[0], 0))


def test_workspaces_grow_with_the_batch():
    """What a larger batch of the same rows needs is enough for a smaller one."""
    for n in (1, 3, 40, 200):
        last = 0
        for pages in (1, 5, 40, 1000, 8000):
            nbytes, _ = ops.attention_paged_workspace(*handles(pages, n), 8)
            assert nbytes >= last
            last = nbytes


def test_no_sequences():
    """Arrays of no sequence have no address in torch."""
    c, none = cache(), seqs(seqs=0, table=None, lens=None, starts=None)
    assert ops.attention_paged_workspace(c, none, 8) == (0, 0)
    L, A = ops._lib(), 1 << 20
    assert L.kr_op_attention_paged(c, 0, none, A, 0, A, 0, 4, 8, 0.1, None, 0, None, 0, None) == 0
    assert L.kr_op_attention_paged(c, 0, none, None, 0, None, 0, 0, 8, 0.1, None, 0, None, 0, None) == 0
    assert L.kr_op_cache_compact(c, none, None, 1, 1, None, None) == 0


def test_streams_of_another_device(monkeypatch):
    """A launch there would reach for memory that its device may not have."""
    monkeypatch.setattr(ops, "_RAW", (lambda: 0, lambda dev: 77))
    on = lambda **kw: SimpleNamespace(cuda_stream=5, **kw)  # noqa: E731
    with pytest.raises(ValueError, match="stream is on device 1"):
        ops._launch_stream(on(device_index=1), "cache_copy_pages", 0, 0)
    with pytest.raises(ValueError, match="current device is 0"):
        ops._launch_stream(on(device_index=1), "cache_copy_pages", 1, 1)
    assert ops._launch_stream(on(device_index=0), "cache_copy_pages", 0, 0) == 5
    assert ops._launch_stream(on(), "cache_copy_pages", 0, 0) == 5  # a QueueStream
    assert ops._launch_stream(None, "cache_copy_pages", 0, 0) == 77
