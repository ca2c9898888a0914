"""Batches of PagedCache at their edges."""

import pytest
import torch

from kernrelay_amd import kvcache, ops
from tests.conftest import announce
from tests.test_gpu_paged import Batch

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


@pytest.mark.parametrize("form", ["step", "tree", "many"])
def test_two_graphs_on_one_workspace(gpu, form):
    """Captured calls that share a workspace, replayed one after the other in
    changing order with eager calls between them: the bits of each alone."""
    announce("attention_paged two graphs, one workspace, " + form)
    if form == "many":  # hundreds of units, one long among them: tickets
        lens = [20] * 100
        lens[40] = 9000
        a, b = (Batch(41 + i, 28, 4, 128, BF, 16, lens, [1] * 100) for i in range(2))
    elif form == "step":
        a, b = Batch(41, 28, 4, 128, BF, 16, [3000, 40], [1, 1]), Batch(42, 8, 2, 128, BF, 16, [900, 2500, 7], [1, 1, 1])
    else:
        a, b = Batch(41, 8, 2, 128, BF, 16, [3000, 40], [30, 9], "tree"), Batch(42, 8, 2, 128, BF, 16, [2000], [70], "tree")
    want = [x.run() for x in (a, b)]
    need = [ops.attention_paged_workspace(x.cache, x.seqs, x.HQ) for x in (a, b)]
    ws = torch.full((max(n for n, _ in need),), 255, dtype=torch.uint8, device="cuda")
    counters = torch.zeros(max(n for _, n in need), dtype=torch.int32, device="cuda")
    assert ws.numel() > 0 and (counters.numel() > 0) == (form == "many")
    outs, graphs = [torch.empty_like(x.q) for x in (a, b)], []
    call = lambda x, o: ops.attention_paged(x.cache, 1, x.seqs, x.q, o, ws=ws, counters=counters)  # noqa: E731
    for x, o in zip((a, b), outs):
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(x, o)
    for order in ((0, 1), (1, 0), (0, 0, 1, 1), (1, 0, 1)):
        for o in outs:
            o.fill_(9.0)
        for i in order:
            graphs[i].replay()
            eager = torch.empty_like(outs[1 - i])
            call((a, b)[1 - i], eager)
            assert torch.equal(eager, want[1 - i])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert int(counters.abs().sum()) == 0


def test_compact_one_row_to_many(gpu):
    """A path that names a draft more than once: each place gets its row."""
    announce("cache_compact, a draft named twice")
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(2, 4, 8, 2, 64, device="cuda", generator=g).to(BF) for _ in range(2))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    was = [c.clone() for c in (k, v)]
    seqs = ops.make_seqs(ints([[2, 0]]), ints([5]), ints([0, 6]), 6)
    ops.cache_compact(ops.make_cache(k, v), seqs, ints([[4, 0, 4, 1]]), ints([4]))
    for now, old in zip((k, v), was):
        rows, old_rows = (torch.cat((c[:, 2], c[:, 0]), 1) for c in (now, old))
        for i, j in enumerate((4, 0, 4, 1)):
            old_rows[:, 5 + i] = torch.cat((old[:, 2], old[:, 0]), 1)[:, 5 + j]
        assert torch.equal(rows, old_rows) and torch.equal(now[:, [1, 3]], old[:, [1, 3]])
