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


@pytest.mark.parametrize("rows", [1, 6])
def test_outputs_between_the_inputs(gpu, rows):
    """One buffer for all: the outputs' rows in the columns beside q's, or
    between its rows, as in buffers of their own."""
    announce("paged cache, outputs between the inputs, %d rows" % rows)
    HQ, HKV, D = 8, 2, 64
    W, g = HQ * D, torch.Generator(device="cuda").manual_seed(rows)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)  # noqa: E731
    k_cache, v_cache = normal(1, 4, 16, HKV, D), normal(1, 4, 16, HKV, D)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    seqs = ops.make_seqs(ints([2, 0]), ints(20), ints(0, rows), rows)
    cache, q0, kv0 = ops.make_cache(k_cache, v_cache), normal(rows, HQ, D), normal(rows, HKV, D)
    t = torch.randn(16, D, device="cuda", generator=g)
    rope = ops.make_rope(t, t)
    want = torch.empty_like(q0)
    ops.attention_paged(cache, 0, seqs, q0, want)
    turned = torch.empty_like(q0), torch.empty_like(kv0)
    ops.qk_norm_rope(rope, q0, kv0, *turned)
    row = W + HKV * D
    wide = torch.zeros(rows, 2 * row, dtype=BF, device="cuda")
    q, k = wide[:, :W].view(rows, HQ, D), wide[:, W:row].view(rows, HKV, D)
    for qo, ko in ((wide[:, row:row + W], wide[:, row + W:]), (wide[:, :W], wide[:, W:row])):  # beside, in place
        q.copy_(q0)
        k.copy_(kv0)
        ops.qk_norm_rope(rope, q, k, qo.view(rows, HQ, D), ko.view(rows, HKV, D))
        assert torch.equal(qo.view(rows, HQ, D), turned[0]) and torch.equal(ko.view(rows, HKV, D), turned[1])
    q.copy_(q0)
    out = wide[:, row:row + W].view(rows, HQ, D)
    ops.attention_paged(cache, 0, seqs, q, out)
    assert torch.equal(out, want)
    # other strides: out's rows are the even ones of a twice as dense buffer, q's every fourth odd one
    dense = torch.zeros(8 * rows, W, dtype=BF, device="cuda")
    q, out = dense[1::4][:rows].view(rows, HQ, D), dense[::2][:rows].view(rows, HQ, D)
    q.copy_(q0)
    ops.attention_paged(cache, 0, seqs, q, out)
    assert torch.equal(out, want)
    if rows > 1:
        with pytest.raises(RuntimeError, match="out overlaps q"):
            ops.attention_paged(cache, 0, seqs, q, dense[1::2][:rows].view(rows, HQ, D))
