"""Batches of PagedCache at their edges."""

import pytest
import torch

from kernrelay_amd import kvcache, ops
from tests.conftest import announce

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def test_empty_batches(gpu):
    """A step in which no sequence has work: nothing is launched, nothing changes."""
    announce("paged cache, empty batch")
    c = kvcache.PagedCache(2, 8, 16, 2, 64)
    none = torch.empty(0, 4, 64, dtype=BF, device="cuda")
    kv = torch.empty(0, 2, 64, dtype=BF, device="cuda")
    t = torch.ones(8, 64, device="cuda")
    for news in ({}, {c.tables.add(): 0}):
        seqs, positions, slots = c.batch(news)
        assert ops.attention_paged_workspace(c.handle, seqs, 4) == (0, 0)
        ops.qk_norm_rope_cache(ops.make_rope(t, t), c.handle, 1, none, kv, kv, none.clone(), positions, slots)
        ops.attention_paged(c.handle, 1, seqs, none, none.clone())
        ops.attention_paged(c.handle, 1, seqs, none, none.clone(), ws=torch.empty(0, dtype=torch.uint8, device="cuda"),
                            counters=torch.zeros(0, dtype=torch.int32, device="cuda"))
        c.accept(seqs, {s: [] for s in news})
        c.commit(news)
    c.defragment()
    assert c.tables.free_pages() == 8
