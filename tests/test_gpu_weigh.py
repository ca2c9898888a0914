"""Attention weight per cached token against float64.

Tolerances. A score is an fp32 sum of D products, scaled: off by at most
dS = (D + 8) 2^-24 scale max sum |q k|. The exponent's argument is
s log2(e) - lse log2(e) in fp32, off by less than 2^-22 (|s| + |lse|) for the
products' and the constants' roundings, and the hardware's 2^x by 2^-21: a
weight is off by their sum, relatively. A key's sum adds a row at a time in
each of 32 lanes and pieces of it after that: below (rows / 32 + 64) 2^-24 of
the sum. The old weight's product and sum round once each.
The logarithm of a row's sum: its relative error dS + 2^-18 (as the
attention's tests have it), and 2^-22 (1 + |lse|) for the logarithm, the sum
with the maximum and the change of base.
"""

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


def normal(g, *shape, dt=BF):
    return torch.randn(*shape, device="cuda", generator=g).to(dt)


class Batch:
    """A launch over a cache: random pages, ragged sequences."""

    def __init__(self, seed, lens, news, HQ, HKV, D, dt=BF, page=16, tree=False, layers=2, heads_first=False,
                 spare_rows=0, pad_table=0):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        rng = random.Random(seed)
        self.lens, self.news, self.HQ, self.HKV, self.D, self.page = lens, news, HQ, HKV, D, page
        need = [(a + b + page - 1) // page for a, b in zip(lens, news)]
        total = sum(need) + 3
        order = rng.sample(range(total), total)
        width = max(need + [1])
        self.table, at = [], 0
        for n in need:
            self.table.append(order[at:at + n] + [-1] * (width - n + pad_table))
            at += n
        if heads_first:
            self.k, self.v = (normal(self.g, layers, total, HKV, page, D, dt=dt).transpose(2, 3) for _ in range(2))
        else:
            self.k, self.v = (normal(self.g, layers, total, page, HKV, D, dt=dt) for _ in range(2))
        self.starts = [sum(news[:i]) for i in range(len(news) + 1)]
        rows = self.starts[-1] + spare_rows
        self.q = normal(self.g, max(rows, 1), HQ * D + 16, dt=dt)[:rows, :HQ * D].view(rows, HQ, D)
        self.tree, self.seen = None, None
        if tree:
            words = (max(news) + 63) // 64
            self.seen, bits = [], []
            for n in news:
                see = []
                for i in range(n):
                    p = rng.randint(max(0, i - 4), i - 1) if i else -1
                    see.append((see[p] if p >= 0 else 0) | (1 << i))
                self.seen += see
            for s in self.seen + [0] * spare_rows:
                bits.append([((s >> (64 * w)) & (2 ** 64 - 1)) - ((s >> (64 * w + 63) & 1) << 64) for w in range(words)])
            self.tree = ints(bits, torch.int64).view(rows, words)
        self.cache = ops.make_cache(self.k, self.v)
        self.seqs = ops.make_seqs(ints(self.table).view(len(lens), -1), ints(lens), ints(self.starts), max(news + [0]),
                                  tree=self.tree)

    def keys(self, layer, b, n, src=None):
        """[n, HKV, D] in float64, and which of them are there."""
        src = self.k if src is None else src
        at = torch.arange(n, device="cuda")
        ids = ints(self.table[b], torch.int64)[at // self.page] if n else at
        ok = (ids >= 0) & (ids < src.shape[1])
        return src[layer][ids.clamp(0, src.shape[1] - 1), at % self.page].double(), ok

    def hidden(self, b, n, total):
        """[n, total]: which keys the new tokens do not see."""
        at, i = torch.arange(total, device="cuda"), torch.arange(n, device="cuda")
        j = at - self.lens[b]
        if self.seen is None:
            return j[None] > i[:, None]
        rows = [[k < self.lens[b] or (self.seen[self.starts[b] + r] >> (k - self.lens[b])) & 1 for k in range(total)]
                for r in range(n)]
        return ~torch.tensor(rows, dtype=torch.bool, device="cuda").view(n, total)

    def lse(self, layer, scale):
        """Exact, in float64; -inf for rows that see nothing."""
        out = torch.zeros(self.q.shape[0], self.HQ, dtype=torch.float64, device="cuda")
        big = 0.0
        for b, n in enumerate(self.news):
            total = self.lens[b] + n
            k, ok = self.keys(layer, b, total)
            hide = self.hidden(b, n, total) | ~ok
            for h in range(self.HQ):
                kh = k[:, h // (self.HQ // self.HKV)]
                qh = self.q[self.starts[b]:self.starts[b + 1], h].double()
                s = (qh @ kh.t()) * scale
                out[self.starts[b]:self.starts[b + 1], h] = torch.logsumexp(s.masked_fill(hide, -math.inf), -1)
                if total and n:
                    big = max(big, float(((qh.abs() @ kh.nan_to_num(0, 0, 0).abs().t()) * scale).max()))
        return out, big


def check_weigh(x, layer, w, old, entry, lse, scale=None, last=0, decay=1.0, paths=None, lim=None):
    """w [entries, HKV, width] after the call, old before it."""
    scale = x.D ** -0.5 if scale is None else scale
    want, tol = old.double().clone(), torch.zeros_like(old, dtype=torch.float64)
    for b, ctx in enumerate(x.lens):
        rows = list(range(x.news[b])) if paths is None else paths[b]
        n = len(rows)
        if n == 0 or entry[b] is None:
            continue
        total = ctx + n
        k, ok = x.keys(layer, b, total)
        hide = x.hidden(b, n, total) if paths is None else torch.arange(total, device="cuda")[None] - ctx > torch.arange(
            n, device="cuda")[:, None]
        hide = hide | ~ok
        skip = max(n - last, 0) if last else 0
        cols = min(total, w.shape[2])
        for g in range(x.HKV):
            got = torch.zeros(total, dtype=torch.float64, device="cuda")
            err = torch.zeros_like(got)
            for h in range(g * (x.HQ // x.HKV), (g + 1) * (x.HQ // x.HKV)):
                for i in range(skip, n):
                    row = x.starts[b] + rows[i]
                    if rows[i] < 0 or rows[i] >= x.news[b] or lse[row, h] == -math.inf:
                        continue
                    s = (k[:, g] @ x.q[row, h].double()) * scale
                    mag = (k[:, g].abs() @ x.q[row, h].double().abs()) * scale
                    e = torch.exp(s - lse[row, h].double())
                    rel = (x.D + 8) * 2.0 ** -24 * mag + 2.0 ** -22 * (s.abs() + lse[row, h].abs()) + 2.0 ** -21
                    got += torch.where(hide[i], 0.0, e)
                    err += torch.where(hide[i], 0.0, e * rel)
            err += got * ((n * x.HQ // x.HKV) / 32 + 64) * 2.0 ** -24
            was = old[entry[b], g, :cols].double()
            cached = torch.arange(cols, device="cuda") < ctx
            keep = torch.where(cached & (decay != 0.0), decay * was, 0.0)
            want[entry[b], g, :cols] = keep + got[:cols]
            tol[entry[b], g, :cols] = err[:cols] * 1.01 + 2.0 ** -23 * (keep.abs() + got[:cols]) + 1e-38
    same = torch.isnan(want) & torch.isnan(w)
    bad = ~(((w.double() - want).abs() <= tol) | same | (w.double() == want))
    assert not bool(bad.any()), (bad.nonzero()[:5], w[bad][:5], want[bad][:5], tol[bad][:5])


def weigh(x, layer, w, lse, entry=None, **kw):
    h = ops.make_weights(w, entry=entry)
    ws = torch.full((ops.attention_paged_weigh_workspace(x.cache, x.seqs, x.HQ),), 255, dtype=torch.uint8, device="cuda")
    ops.attention_paged_weigh(x.cache, layer, x.seqs, x.q, lse, h, ws, **kw)


@pytest.mark.parametrize("kw", [
    dict(lens=[1], news=[1], HQ=4, HKV=4, D=64),
    dict(lens=[0], news=[1], HQ=2, HKV=1, D=128, dt=HF),
    dict(lens=[0, 31, 32, 33, 127, 128, 129], news=[1] * 7, HQ=7, HKV=1, D=64, page=7),
    dict(lens=[300, 5, 0, 64], news=[1, 0, 3, 1], HQ=8, HKV=2, D=128, page=1, spare_rows=2),
    dict(lens=[700, 200], news=[40, 33], HQ=14, HKV=2, D=64, page=24, dt=HF, heads_first=True),
    dict(lens=[0], news=[300], HQ=4, HKV=2, D=128, page=16),
    dict(lens=[90, 500], news=[65, 70], HQ=4, HKV=1, D=128, page=32, tree=True),
    dict(lens=[3, 0, 40], news=[5, 17, 1], HQ=28, HKV=4, D=128, page=16, tree=True, dt=HF),
    dict(lens=[20] * 70, news=[1] * 70, HQ=4, HKV=2, D=64, page=8, pad_table=40),
])
def test_weights_of_new_tokens(gpu, kw):
    announce("weigh %s" % kw)
    x = Batch(11, **kw)
    n = len(x.lens)
    width = max(a + b for a, b in zip(x.lens, x.news)) + 3
    entry = list(range(n + 1))[::-1][:n]
    # rows of the weights inside a wider tensor, heads outside entries
    w = torch.rand(x.k.shape[0], x.HKV, n + 1, width + 5, device="cuda", generator=x.g)[..., :width].transpose(1, 2)
    for layer in range(x.k.shape[0]):
        old = w.clone()
        lse, _ = x.lse(layer, x.D ** -0.5)
        weigh(x, layer, w, lse.float(), ints(entry))
        check_weigh(x, layer, w[layer], old[layer], entry, lse.float())
        assert torch.equal(w[1 - layer], old[1 - layer])
        again = old.clone()
        weigh(x, layer, again, lse.float(), ints(entry))
        assert torch.equal(again, w)  # the same bits at every call


@pytest.mark.parametrize("last", [1, 3, 64, 10 ** 6])
@pytest.mark.parametrize("decay", [0.0, 0.5])
def test_last_and_decay(gpu, last, decay):
    announce("weigh last %d decay %g" % (last, decay))
    x = Batch(3, [400, 0, 77], [100, 70, 2], 8, 2, 64)
    w = torch.rand(1 + 1, 3, 2, 505, device="cuda", generator=x.g)
    if decay == 0.0:
        w[0, 0, 0, 5] = math.nan  # the old value is not read
    old = w.clone()
    lse, _ = x.lse(0, 0.3)
    weigh(x, 0, w, lse.float(), last=last, decay=decay, scale=0.3)
    check_weigh(x, 0, w[0], old[0], [0, 1, 2], lse.float(), scale=0.3, last=last, decay=decay)


@pytest.mark.parametrize("last", [0, 2])
@pytest.mark.parametrize("tree", [False, True])
def test_accepted_paths(gpu, tree, last):
    announce("weigh paths %s %d" % (tree, last))
    x = Batch(5, [130, 0, 61, 9], [24, 9, 70, 4], 14, 2, 64, page=8, tree=tree)
    paths = [[0, 2, 5, 23], [0], [0, 1, 64, 69, 70, -3], []]  # (two that name no row count nothing)
    width = 8
    lse, _ = x.lse(1, x.D ** -0.5)
    w = torch.rand(2, 4, 2, 150, device="cuda", generator=x.g)
    old = w.clone()
    path = ints([p + [-1] * (width - len(p)) for p in paths])
    weigh(x, 1, w, lse.float(), path=path, path_lens=ints([len(p) for p in paths]), last=last)
    check_weigh(x, 1, w[1], old[1], [0, 1, 2, 3], lse.float(), paths=paths, last=last)


@pytest.mark.parametrize("form", ["causal", "tree", "path"])
@pytest.mark.parametrize("HQ,HKV", [(8, 1), (2, 1)])
def test_more_sequences_than_a_wave_has_lanes(gpu, form, HQ, HKV):
    """130 of them, in the form for many rows and the one for few."""
    announce("weigh 130 %s %d" % (form, HQ))
    rng = random.Random(130)
    lens, news = [rng.randint(0, 90) for _ in range(130)], [rng.choice((0, 1, 5, 13)) for _ in range(130)]
    x = Batch(130, lens, news, HQ, HKV, 64, page=8, layers=1, tree=form != "causal")
    lse, _ = x.lse(0, x.D ** -0.5)
    entry = list(range(130))[::-1]
    w = torch.rand(130, HKV, 105, device="cuda", generator=x.g)
    old, kw, paths = w.clone(), {}, None
    if form == "path":
        paths = [sorted(rng.sample(range(n), rng.randint(0, n))) for n in news]
        kw = dict(path=ints([p + [-1] * (13 - len(p)) for p in paths]), path_lens=ints([len(p) for p in paths]))
    weigh(x, 0, w, lse.float(), ints(entry), **kw)
    check_weigh(x, 0, w, old, entry, lse.float(), paths=paths)


@pytest.mark.parametrize("rows", ["few", "many"])
def test_narrow_weights_and_odd_batches(gpu, rows):
    """Columns for some of the tokens only; starts that do not ascend and lengths that are
    none leave everything inside."""
    announce("weigh narrow %s" % rows)
    x = Batch(8, [300, 40, 90], [3, 2, 1] if rows == "few" else [60, 2, 41], 8, 2, 64, page=8)
    lse, _ = x.lse(0, x.D ** -0.5)
    pad = torch.full((2, 5, 2, 140), 3.5, device="cuda")
    w = pad[:, 1:4, :, :129]
    weigh(x, 0, w, lse.float())
    check_weigh(x, 0, w[0], torch.full_like(w[0], 3.5), [0, 1, 2], lse.float())
    pad[:, 1:4, :, :129] = 3.5
    assert bool((pad == 3.5).all())
    n = x.q.shape[0]
    for lens, starts in (([2 ** 31 - 1, -7, 90], [0, 1, 2, n]), ([300, 40, 90], [n, 0, -9, 2 ** 31 - 1]),
                         ([300, 40, 90], [5, 2, n + 100, 1])):
        x.seqs = ops.make_seqs(ints(x.table), ints(lens), ints(starts), max(x.news))
        weigh(x, 0, w, lse.float(), ints([0, 2, 1]))
        pad[:, 1:4, :, :129] = 3.5
        assert bool((pad == 3.5).all())


def test_what_nobody_sees(gpu):
    """Pages that are none, keys that are no numbers behind the sequences and in masked
    places, rows that see nothing, entries outside, columns past the width."""
    announce("weigh hidden")
    x = Batch(7, [200, 45, 30, 50], [1, 6, 4, 2], 4, 2, 128, page=16, tree=True)
    x.table[0][3] = -1
    x.table[0][7] = x.k.shape[1] + 9
    x.table[2] = [-1] * len(x.table[2])  # nothing is there
    x.seqs = ops.make_seqs(ints(x.table), ints(x.lens), ints(x.starts), 6, tree=x.tree)
    bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda").to(BF)
    used = {p for t in x.table for p in t}
    for p in set(range(x.k.shape[1])) - used:
        x.k[:, p] = bad[p % 3]
    last = x.table[3][(50 + 2) // 16]
    x.k[:, last, (50 + 2) % 16:] = math.nan     # behind the last token
    x.seen[x.starts[1] + 3] &= ~(1 << 1)         # the draft that the others do not see holds NaN
    for r in range(6):
        x.seen[x.starts[1] + r] &= ~(1 << 1)
    x.k[:, x.table[1][(45 + 1) // 16], (45 + 1) % 16] = math.nan
    x.tree.copy_(ints([[s] for s in x.seen], torch.int64))
    lse, _ = x.lse(0, x.D ** -0.5)
    assert bool((lse[x.starts[2]:x.starts[3]] == -math.inf).all())
    w = torch.rand(2, 3, 2, 190, device="cuda", generator=x.g)
    old = w.clone()
    weigh(x, 0, w, lse.float(), ints([1, 2, 0, 3]))  # the last one's entry is outside
    check_weigh(x, 0, w[0], old[0], [1, 2, 0, None], lse.float())
    assert bool(torch.isfinite(w).all())


def test_nothing_to_do(gpu):
    announce("weigh nothing")
    x = Batch(1, [4, 9], [0, 0], 4, 2, 64)
    w = torch.rand(2, 2, 2, 20, device="cuda")
    old = w.clone()
    weigh(x, 0, w, torch.zeros(0, 4, device="cuda"))
    x = Batch(1, [4, 9], [0, 0], 4, 2, 64, spare_rows=3)
    weigh(x, 0, w, torch.zeros(3, 4, device="cuda"))
    assert torch.equal(w, old)


def test_starts_that_go_back_and_forth(gpu):
    """Half of 1024 sequences claim all 2048 rows, a million tokens each: more row
    tiles of key tiles than a launch counts. Nothing is worked on."""
    announce("weigh starts")
    n, page, rows, HQ = 1024, 1024, 2048, 32
    k = torch.zeros(1, 2, page, 1, 64, device="cuda", dtype=BF)
    cache = ops.make_cache(k, k.clone())
    table = torch.full((n, 1024), -1, dtype=torch.int32, device="cuda")
    seqs = ops.make_seqs(table, ints([page * 1024 - rows] * n), ints([0, rows] * (n // 2) + [0]), rows)
    w = torch.rand(1, 1, page * 1024, device="cuda")
    old = w.clone()
    h = ops.make_weights(w, entry=ints([0] * n))
    ws = torch.empty(ops.attention_paged_weigh_workspace(cache, seqs, HQ), dtype=torch.uint8, device="cuda")
    q = torch.zeros(rows, HQ, 64, device="cuda", dtype=BF)
    ops.attention_paged_weigh(cache, 0, seqs, q, torch.zeros(rows, HQ, device="cuda"), h, ws)
    torch.cuda.synchronize()
    assert torch.equal(w, old)


@pytest.mark.parametrize("D,HQ,HKV,lens,news", [(128, 28, 4, [5000, 3100], [300, 1]), (64, 14, 2, [20000], [1]),
                                                (128, 32, 8, [2500], [64]), (64, 4, 4, [0], [1100])])
def test_long_ones_add_up(gpu, D, HQ, HKV, lens, news):
    """Every row's weights sum to 1, so a head's columns sum to its rows; and against
    float64 products."""
    announce("weigh long %s" % ((D, HQ, HKV, lens, news),))
    x = Batch(9, lens, news, HQ, HKV, D, page=64, layers=1)
    lse, big = x.lse(0, D ** -0.5)
    w = torch.full((1, len(lens), HKV, max(a + b for a, b in zip(lens, news)) + 1), -7.0, device="cuda")
    weigh(x, 0, w, lse.float(), decay=0.0)
    rel = (D + 8) * 2.0 ** -24 * big + 2.0 ** -22 * 2 * (big + float(lse.abs().max())) + 2.0 ** -21
    G = HQ // HKV
    for b, n in enumerate(news):
        total = lens[b] + n
        k, _ = x.keys(0, b, total)
        hide = x.hidden(b, n, total)
        assert bool((w[0, b, :, total:] == -7.0).all())
        for g in range(HKV):
            want = torch.zeros(total, dtype=torch.float64, device="cuda")
            for h in range(g * G, (g + 1) * G):
                rows = slice(x.starts[b], x.starts[b + 1])
                s = (x.q[rows, h].double() @ k[:, g].t()) * D ** -0.5
                want += (s - lse[rows, h].float().double()[:, None]).masked_fill(hide, -math.inf).exp().sum(0)
            tol = want * (rel + (n * G / 32 + 64) * 2.0 ** -24) * 1.01
            got = w[0, b, g, :total].double()
            assert bool(((got - want).abs() <= tol).all())
            assert abs(float(want.sum()) - n * G) < 1e-4 * n * G


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("kw", [
    dict(lens=[0, 1, 40], news=[1, 1, 1], HQ=4, HKV=2, D=64),
    dict(lens=[900], news=[1], HQ=28, HKV=4, D=128),                       # cut into pieces, by a second launch
    dict(lens=[3000] + [40] * 99, news=[1] * 100, HQ=8, HKV=2, D=64, layers=1),  # by tickets
    dict(lens=[300] * 60, news=[1] * 60, HQ=8, HKV=4, D=128, layers=1),    # four key streams
    dict(lens=[500, 3], news=[9, 11], HQ=14, HKV=2, D=64, tree=True),
    dict(lens=[700, 0], news=[200, 31], HQ=8, HKV=2, D=128),
])
def test_attention_gives_its_rows_sums(gpu, kw, dt):
    """lse beside the same results; and what the weights are made of."""
    announce("attention lse %s %s" % (kw, dt))
    x = Batch(21, dt=dt, spare_rows=1, **kw)
    nbytes, ncnt = ops.attention_paged_workspace(x.cache, x.seqs, x.HQ)
    want, big = x.lse(0, x.D ** -0.5)
    for cut in (False, True):
        ws = torch.full((nbytes,), 170, dtype=torch.uint8, device="cuda") if cut else None
        cnt = torch.zeros(ncnt, dtype=torch.int32, device="cuda") if cut else None
        out, plain = (torch.full(x.q.shape, 3.0, dtype=dt, device="cuda") for _ in range(2))
        pad = torch.full((x.q.shape[0], x.HQ + 3), 5.0, device="cuda")
        lse = pad[:, :x.HQ]
        ops.attention_paged(x.cache, 0, x.seqs, x.q, out, ws=ws, counters=cnt, lse=lse)
        ops.attention_paged(x.cache, 0, x.seqs, x.q, plain, ws=ws, counters=cnt)
        assert torch.equal(out, plain)
        n = x.starts[-1]
        assert bool((pad[:, x.HQ:] == 5.0).all()) and bool((lse[n:] == 5.0).all())
        tol = (x.D + 8) * 2.0 ** -24 * big + 2.0 ** -18 + 2.0 ** -22 * (1 + want[:n].abs())
        assert bool(((lse[:n].double() - want[:n]).abs() <= tol).all())


def test_lse_of_a_row_that_sees_nothing(gpu):
    announce("attention lse empty")
    x = Batch(2, [0, 20], [2, 1], 4, 2, 64, tree=True)
    x.tree[1] = 0
    lse, out = torch.zeros(3, 4, device="cuda"), torch.ones_like(x.q)
    ops.attention_paged(x.cache, 0, x.seqs, x.q, out, lse=lse)
    assert bool((lse[1] == -math.inf).all()) and bool((out[1] == 0).all())
    assert bool(torch.isfinite(lse[[0, 2]]).all())


def test_captured(gpu):
    """A captured attention and its weights, replayed over other lengths and pages."""
    announce("weigh captured")
    x = Batch(4, [90, 30], [1, 2], 8, 2, 64, page=8, pad_table=9)
    lens = ints(x.lens)
    x.seqs = ops.make_seqs(ints(x.table), lens, ints(x.starts), 2)
    nbytes, ncnt = ops.attention_paged_workspace(x.cache, x.seqs, 8)
    ws, cnt = torch.empty(nbytes, dtype=torch.uint8, device="cuda"), torch.zeros(ncnt, dtype=torch.int32, device="cuda")
    wws = torch.empty(ops.attention_paged_weigh_workspace(x.cache, x.seqs, 8), dtype=torch.uint8, device="cuda")
    out, lse = torch.empty_like(x.q), torch.empty(3, 8, device="cuda")
    w = torch.zeros(2, 2, 2, 120, device="cuda")
    h = ops.make_weights(w)

    def step():
        ops.attention_paged(x.cache, 1, x.seqs, x.q, out, ws=ws, counters=cnt, lse=lse)
        ops.attention_paged_weigh(x.cache, 1, x.seqs, x.q, lse, h, wws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for ls in ([90, 30], [17, 0], [3, 29], [90, 30]):
        lens.copy_(ints(ls))
        w.fill_(0.25)
        graph.replay()
        torch.cuda.synchronize()
        got = w.clone()
        w.fill_(0.25)
        step()
        assert torch.equal(got, w)
        x.lens = ls
        check_weigh(x, 1, got[1], torch.full_like(got[1], 0.25), [0, 1], lse)
