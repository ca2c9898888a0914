"""Eviction by weight against a plain restatement, bit for bit."""

import math
import random

import pytest
import torch

from kernrelay_amd import ops
from tests.conftest import announce

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def ints(v, dt=torch.int32):
    return torch.tensor(v, dtype=dt, device="cuda")


def kept(w, n, budget, sinks, recent):
    """Which token stands at each place afterwards; w: the weights as floats."""
    if n <= budget:
        return list(range(n)) + [-1] * (budget - n)
    end, low = budget - recent, n - recent
    order = sorted(range(sinks, low), key=lambda j: (-w[j] if w[j] == w[j] else math.inf, w[j] != w[j], j))
    best = set(order[:end - sinks])
    movers = sorted(j for j in best if j >= end)
    out = [j for j in range(end)]
    for j in range(sinks, end):
        if j not in best:
            out[j] = movers.pop(0)
    assert not movers
    return out + list(range(low, n))


class Case:
    def __init__(self, seed, lens, heads=2, D=64, layers=2, page=8, dt=BF, width=None, heads_first=False, entries=None):
        rng = random.Random(seed)
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.page = lens, page
        need = [(n + page - 1) // page for n in lens]
        total = sum(need) + 3
        order = rng.sample(range(total), total)
        self.table, at = [], 0
        for n in need:
            self.table.append(order[at:at + n] + [-1] * (max(need + [1]) - n))
            at += n
        shape = (layers, total, heads, page, D) if heads_first else (layers, total, page, heads, D)
        self.k, self.v = (torch.randn(shape, device="cuda", generator=self.g).to(dt) for _ in range(2))
        if heads_first:
            self.k, self.v = self.k.transpose(2, 3), self.v.transpose(2, 3)
        width = max(lens) + 2 if width is None else width
        self.w = torch.rand(layers, heads, len(lens) + 2, width + 1, device="cuda", generator=self.g)[..., :width]
        self.w = self.w.transpose(1, 2)
        self.entry = rng.sample(range(len(lens) + 2), len(lens)) if entries is None else entries
        self.cache = ops.make_cache(self.k, self.v)
        self.seqs = ops.make_seqs(ints(self.table).view(len(lens), -1), ints(lens), ints([0] * (len(lens) + 1)), 0)

    def run(self, budget, sinks=0, recent=0):
        keep = torch.full((self.k.shape[0], len(self.lens), self.k.shape[3], budget), 77, dtype=torch.int32, device="cuda")
        ops.cache_evict(self.cache, self.seqs, ops.make_weights(self.w, entry=ints(self.entry)), keep, sinks=sinks,
                        recent=recent)
        return keep

    def check(self, budget, sinks=0, recent=0):
        was = [t.clone() for t in (self.k, self.v, self.w)]
        keep = self.run(budget, sinks, recent)
        want = [t.clone() for t in was]
        for layer in range(self.k.shape[0]):
            for b, n in enumerate(self.lens):
                there = 0 <= self.entry[b] < self.w.shape[1] and n <= self.w.shape[3]
                for h in range(self.k.shape[3]):
                    if there:
                        of = kept(was[2][layer, self.entry[b], h].tolist(), n, budget, sinks, recent)
                    else:
                        of = list(range(min(n, budget))) + [-1] * (budget - n)
                    assert keep[layer, b, h].tolist() == of, (layer, b, h)
                    if n <= budget or not there:
                        continue
                    place = lambda i: (ints(self.table[b], torch.int64)[i // self.page], i % self.page)  # noqa: E731
                    to, of = torch.arange(budget, device="cuda"), ints(of, torch.int64)
                    (a, c), (e, f) = place(to), place(of)
                    ok = ((a >= 0) & (a < self.k.shape[1]) & (e >= 0) & (e < self.k.shape[1])) & (to != of)
                    for new, old in zip(want[:2], was[:2]):
                        new[layer, a[ok], c[ok], h] = old[layer, e[ok], f[ok], h]
                    want[2][layer, self.entry[b], h, :budget] = was[2][layer, self.entry[b], h][of]
        bits = {BF: torch.int16, HF: torch.int16, torch.float32: torch.int32}
        for a, b in zip((self.k, self.v, self.w), want):
            assert torch.equal(a.contiguous().view(bits[a.dtype]), b.contiguous().view(bits[b.dtype]))
        return keep


@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (7, 0, 0), (20, 3, 5), (20, 20, 0),
                                                 (20, 0, 20), (20, 7, 13), (39, 2, 30), (64, 4, 8)])
@pytest.mark.parametrize("kw", [dict(D=64, page=8), dict(D=128, page=7, dt=HF, heads_first=True), dict(D=128, page=1, heads=1)])
def test_small(gpu, budget, sinks, recent, kw):
    announce("evict %s %s" % ((budget, sinks, recent), kw))
    Case(budget + sinks, [0, 1, 2, 8, 19, 20, 21, 22, 40, 65, 100], **kw).check(budget, sinks, recent)


@pytest.mark.parametrize("kind", ["equal", "few", "zeros", "odd", "spread", "sorted", "reverse"])
def test_orders_of_weights(gpu, kind):
    """Ties go to the first; 0 and -0 are equal; a NaN is below -infinity."""
    announce("evict weights %s" % kind)
    x = Case(17, [150, 97, 300], layers=1)
    if kind == "equal":
        x.w.fill_(0.5)
    elif kind == "few":
        x.w.copy_((x.w * 4).floor())
    elif kind == "zeros":
        x.w.copy_(torch.where(x.w < 0.5, 0.0, -0.0))
    elif kind == "odd":
        bad = torch.tensor([math.nan, math.inf, -math.inf, 0.0, 1e-42, -1.0], device="cuda")
        x.w.copy_(bad[(x.w * 6).long()])
    elif kind == "spread":
        x.w.copy_((x.w * 200 - 100).exp2())
    else:
        x.w.copy_(x.w.sort(dim=3, descending=kind == "reverse").values)
    x.check(60, 2, 10)


@pytest.mark.parametrize("lens,budget,sinks,recent,kw", [
    ([5000, 1024, 1025, 3100], 1024, 0, 0, dict()),
    ([4097, 2500], 2100, 16, 900, dict(D=128, page=64)),
    ([70000], 5000, 4, 1000, dict(page=128, layers=1, heads=1)),
    ([70000, 66000], 65000, 0, 64, dict(page=128, layers=1, heads=1)),
    ([1300] * 5, 1290, 4, 700, dict(heads=8, layers=3, dt=HF)),   # the recent ones' new places are their old ones
])
def test_long(gpu, lens, budget, sinks, recent, kw):
    announce("evict long %s" % ((lens, budget, sinks, recent),))
    x = Case(3, lens, **kw)
    x.w.copy_(torch.where(x.w < 0.3, 0.25, x.w))  # many equal ones, too
    x.check(budget, sinks, recent)


def test_again_and_again(gpu):
    """Each time over the budget by a few tokens; nothing is moved that may stay."""
    announce("evict again")
    x = Case(5, [90, 90], page=16)
    for more in (20, 3, 1, 10):
        x.lens = [64 + more, 64 + more // 2]
        x.seqs = ops.make_seqs(ints(x.table), ints(x.lens), ints([0, 0, 0]), 0)
        keep = x.check(64, 2, 8)
        at = torch.arange(64, device="cuda")
        moved = (keep != at).sum(dim=3)
        assert int(moved.max()) <= 8 + more


def test_left_alone(gpu):
    """Entries outside the weights, more tokens than columns, pages that are none."""
    announce("evict alone")
    x = Case(8, [50, 60, 70, 40], width=60, entries=[2, -1, 4, 0], page=4)
    x.table[0][5], x.table[0][9] = -1, 10 ** 6
    x.seqs = ops.make_seqs(ints(x.table), ints(x.lens), ints([0] * 5), 0)
    x.check(30, 1, 6)


def test_lengths_that_are_none(gpu):
    announce("evict lengths")
    x = Case(9, [50, 60, 70], width=60)
    x.lens = [50, 0, 50]
    table = x.table
    x.seqs = ops.make_seqs(ints(table), ints([50, -5, 2 ** 31 - 1]), ints([0] * 4), 0)
    was = [t.clone() for t in (x.k, x.v, x.w)]
    keep = x.run(30, 1, 6)
    assert keep[:, 1].eq(-1).all() and bool((keep[:, 2] == torch.arange(30, device="cuda")).all())
    for layer in range(2):
        for h in range(2):
            assert keep[layer, 0, h].tolist() == kept(was[2][layer, x.entry[0], h].tolist(), 50, 30, 1, 6)
    others = [e for e in range(x.w.shape[1]) if e != x.entry[0]]
    assert torch.equal(x.w[:, others], was[2][:, others])
    mine = set(table[0])
    pages = [p for p in range(x.k.shape[1]) if p not in mine]
    assert torch.equal(x.k[:, pages], was[0][:, pages]) and torch.equal(x.v[:, pages], was[1][:, pages])


@pytest.mark.parametrize("n,budget", [(700, 300), (30000, 9000)])
def test_one_entry_twice(gpu, n, budget):
    """Against the contract: which tokens stay is open, but lists name tokens of
    their sequence, and what is around them stays."""
    announce("evict twice %d" % n)
    x = Case(5, [n] * 4, layers=2, entries=[1, 1, 1, 1], page=16)
    x.w.copy_((x.w * 9).floor())
    others, was = [0, 2, 3, 4, 5], x.w.clone()
    room = torch.full((2 * 4 * 2 * budget + 4096,), 77, dtype=torch.int32, device="cuda")
    keep = room[2048:-2048].view(2, 4, 2, budget)
    ops.cache_evict(x.cache, x.seqs, ops.make_weights(x.w, entry=ints(x.entry)), keep, sinks=3, recent=50)
    assert bool(room[:2048].eq(77).all()) and bool(room[-2048:].eq(77).all())
    assert int(keep.min()) >= 0 and int(keep.max()) < n
    assert bool((keep[..., :3] == ints([0, 1, 2])).all()) and bool((keep[..., -50:] == torch.arange(n - 50, n, device="cuda")).all())
    assert torch.equal(x.w[:, others], was[:, others])


def test_no_sequences(gpu):
    x = Case(8, [5])
    seqs = ops.make_seqs(torch.empty(0, 3, dtype=torch.int32, device="cuda"), ints([]), ints([0]), 0)
    ops.cache_evict(x.cache, seqs, ops.make_weights(x.w), torch.empty(2, 0, 2, 4, dtype=torch.int32, device="cuda"))


def test_captured(gpu):
    announce("evict captured")
    x = Case(6, [80, 50], page=16)
    lens = ints(x.lens)
    x.seqs = ops.make_seqs(ints(x.table), lens, ints([0, 0, 0]), 0)
    h = ops.make_weights(x.w, entry=ints(x.entry))
    keep = torch.zeros(2, 2, 2, 40, dtype=torch.int32, device="cuda")
    first = [t.clone() for t in (x.k, x.v, x.w)]

    def back():
        for t, f in zip((x.k, x.v, x.w), first):
            t.copy_(f)

    ops.cache_evict(x.cache, x.seqs, h, keep, sinks=1, recent=5)
    back()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_evict(x.cache, x.seqs, h, keep, sinks=1, recent=5)
    for ls in ([80, 50], [41, 40], [60, 77], [3, 80]):
        lens.copy_(ints(ls))
        x.lens = ls
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (keep, x.k, x.v, x.w)]
        back()
        assert torch.equal(x.check(40, 1, 5), got[0])
        for a, b in zip((x.k, x.v, x.w), got[1:]):
            assert torch.equal(a, b)
        back()
