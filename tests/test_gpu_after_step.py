"""The calls of a program that drafts and evicts, together: prompt, attention with
its rows' sums, weights, drafts verified, accepted and weighed, eviction, over
several steps, against a plain simulation in float64 that keeps each head's
tokens in lists.

Attention's bound is that of its own tests in a coarse form: outputs are rounded
once to bf16 and the scores' error is far below that, so 2^-8 |o| + 2^-8 sum p |v|
covers it. Weights: (D + 8) 2^-24 of the score's terms and a few 2^-20 more,
below 2^-12 relatively; each step adds its own.
"""

import random

import pytest
import torch

from kernrelay_amd import kvcache, ops
from tests.conftest import announce
from tests.test_gpu_evict import kept

pytestmark = pytest.mark.gpu

LAYERS, HQ, HKV, D, V = 2, 8, 2, 64, 600
G = HQ // HKV


def test_drafts_and_evictions_step_by_step(gpu):
    announce("after a step")
    gen = torch.Generator(device="cuda").manual_seed(0)
    rng = random.Random(0)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen).bfloat16()  # noqa: E731
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device="cuda")  # noqa: E731
    cache = kvcache.PagedCache(LAYERS, 40, 8, HKV, D)
    D2 = torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D
    ang = torch.arange(400, dtype=torch.float64, device="cuda")[:, None] * 1e4 ** -D2
    ang = torch.cat((ang, ang), 1)
    rope = ops.make_rope(ang.cos().float(), ang.sin().float())
    ids = [cache.tables.add() for _ in range(3)]
    w = torch.zeros(LAYERS, 5, HKV, 120, device="cuda")
    entry = ints([4, 0, 2])
    weights = ops.make_weights(w, entry=entry)
    # the simulation: [layer][sequence][head] -> keys, values, weights
    sim = {s: [[dict(k=torch.zeros(0, D, dtype=torch.float64, device="cuda"),
                     v=torch.zeros(0, D, dtype=torch.float64, device="cuda"),
                     w=torch.zeros(0, dtype=torch.float64, device="cuda")) for _ in range(HKV)] for _ in range(LAYERS)]
           for s in ids}
    place = {s: 0 for s in ids}
    evictions = 0

    def rotate(x, pos):
        h = x.shape[-1] // 2
        turned = torch.cat((-x[..., h:], x[..., :h]), -1)
        return x * ang.cos()[pos][:, None] + turned * ang.sin()[pos][:, None]

    def attend(news, tree=None, depths=None, seen=None):
        """One launch over all layers: handle, and for each layer what the rows were."""
        seqs, positions, slots = cache.batch(news, tree=tree, depths=depths)
        rows = sum(news.values())
        nbytes, ncnt = ops.attention_paged_workspace(cache.handle, seqs, HQ)
        ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        cnt = torch.zeros(ncnt, dtype=torch.int32, device="cuda")
        want = [place[s] + (i if depths is None else depths[s][i]) for s, n in news.items() for i in range(n)]
        assert positions.tolist() == want
        kept_rows = []
        for layer in range(LAYERS):
            q, k, v = randn(rows, HQ, D), randn(rows, HKV, D), randn(rows, HKV, D)
            qo, out, lse = torch.empty_like(q), torch.empty_like(q), torch.empty(rows, HQ, device="cuda")
            ops.qk_norm_rope_cache(rope, cache.handle, layer, q, k, v, qo, positions, slots)
            ops.attention_paged(cache.handle, layer, seqs, qo, out, ws=ws, counters=cnt, lse=lse)
            pos = ints(want, torch.int64)
            kr = rotate(k.double(), pos).bfloat16().double()
            assert bool(((qo.double() - rotate(q.double(), pos)).abs() <= 2.0 ** -7 * q.double().abs().amax()).all())
            at = 0
            for s, n in news.items():
                for h in range(HQ):
                    c = sim[s][layer][h // G]
                    for i in range(n):
                        sees = list(range(i + 1)) if seen is None else [j for j in range(n) if (seen[s][i] >> j) & 1]
                        r = [at + j for j in sees]
                        kk, vv = torch.cat((c["k"], kr[r, h // G])), torch.cat((c["v"], v.double()[r, h // G]))
                        a = (kk @ qo[at + i, h].double()) * D ** -0.5
                        p = torch.softmax(a, 0)
                        o, mag = p @ vv, p @ vv.abs()
                        assert bool(((out[at + i, h].double() - o).abs() <= 2.0 ** -8 * 1.1 * (mag + o.abs()) + 2.0 ** -7 * mag).all())
                        assert abs(float(lse[at + i, h]) - float(torch.logsumexp(a, 0))) < 2.0 ** -6
                at += n
            kept_rows.append((qo, lse, kr, v.double()))
        return seqs, kept_rows

    def weigh(seqs, news, kept_rows, paths=None, last=0):
        """Weighs on the GPU and in the simulation, whose lists get the tokens."""
        wws = torch.empty(ops.attention_paged_weigh_workspace(cache.handle, seqs, HQ), dtype=torch.uint8, device="cuda")
        kw = {}
        if paths is not None:
            width = max(len(p) for p in paths.values())
            kw = dict(path=ints([p + [-1] * (width - len(p)) for p in paths.values()]),
                      path_lens=ints([len(p) for p in paths.values()]))
        for layer, (qo, lse, kr, v) in enumerate(kept_rows):
            ops.attention_paged_weigh(cache.handle, layer, seqs, qo, lse, weights, wws, last=last, **kw)
            at = 0
            for b, (s, n) in enumerate(news.items()):
                rows = [at + i for i in (range(n) if paths is None else paths[s])]
                for g in range(HKV):
                    c = sim[s][layer][g]
                    n0 = c["k"].shape[0]
                    c["k"], c["v"] = torch.cat((c["k"], kr[rows, g])), torch.cat((c["v"], v[rows, g]))
                    c["w"] = torch.cat((c["w"], torch.zeros(len(rows), dtype=torch.float64, device="cuda")))
                    for i, r in enumerate(rows):
                        if last and i < len(rows) - last:
                            continue
                        for h in range(g * G, (g + 1) * G):
                            a = (c["k"][:n0 + i + 1] @ qo[r, h].double()) * D ** -0.5
                            c["w"][:n0 + i + 1] += torch.exp(a - lse[r, h].double())
                at += n

    def compare():
        for b, s in enumerate(ids):
            n = cache.tables.tokens(s)
            pages = ints(cache.tables.pages_of(s), torch.int64)
            at = torch.arange(n, device="cuda")
            for layer in range(LAYERS):
                for g in range(HKV):
                    c = sim[s][layer][g]
                    assert c["k"].shape[0] == n
                    for src, name in ((cache.k, "k"), (cache.v, "v")):
                        got = src[layer, pages[at // 8], at % 8, g].double()
                        assert bool(((got - c[name]).abs() <= 2.0 ** -7 * c[name].abs() + 1e-30).all())
                    got = w[layer, entry[b], g, :n].double()
                    assert bool(((got - c["w"]).abs() <= 2.0 ** -11 * c["w"] + 1e-6).all())

    # the prompts: only their last tokens' looks count
    news = dict(zip(ids, (50, 7, 33)))
    seqs, rows = attend(news)
    cache.commit(news)
    weigh(seqs, news, rows, last=5)
    for s, n in news.items():
        place[s] += n
    compare()
    for step in range(7):
        news = {s: rng.randint(1, 9) for s in ids}
        par = {s: [-1] + [rng.randint(max(0, i - 3), i - 1) for i in range(1, n)] for s, n in news.items()}
        depths = {s: [0] * n for s, n in news.items()}
        seen = {s: [0] * n for s, n in news.items()}
        for s, n in news.items():
            for i, p in enumerate(par[s]):
                depths[s][i] = depths[s][p] + 1 if p >= 0 else 0
                seen[s][i] = (seen[s][p] if p >= 0 else 0) | (1 << i)
        tree = ints([[x] for s in ids for x in seen[s]], torch.int64)
        seqs, rows = attend(news, tree=tree, depths=depths, seen=seen)
        R = sum(news.values())
        logits = torch.randn(R, V, device="cuda", generator=gen) * 4
        starts = [0]
        for n in news.values():
            starts.append(starts[-1] + n)
        above = ints([starts[b] + max(p, 0) for b, s in enumerate(ids) for p in par[s]], torch.int64)
        tokens = logits[above].topk(2, 1).indices.gather(1, torch.randint(0, 2, (R, 1), device="cuda", generator=gen))[:, 0]
        path, lens, nxt = torch.empty(3, 9, dtype=torch.int32, device="cuda"), ints([0] * 3), ints([0] * 3, torch.int64)
        nbytes, ncnt = ops.verify_drafts_workspace(seqs, logits)
        ops.verify_drafts(seqs, logits, tokens, torch.rand(R, device="cuda", generator=gen),
                          torch.rand(3, device="cuda", generator=gen), path, lens, nxt,
                          torch.empty(nbytes, dtype=torch.uint8, device="cuda"),
                          torch.zeros(ncnt, dtype=torch.int32, device="cuda"),
                          parents=ints([p for s in ids for p in par[s]]))
        paths = {s: p[:n] for s, p, n in zip(ids, path.tolist(), lens.tolist())}
        assert all(p[0] == 0 and par[s][b] == a for s, p in paths.items() for a, b in zip(p, p[1:]))
        assert bool((nxt >= 0).all())
        cache.accept(seqs, paths)
        weigh(seqs, news, rows, paths=paths)
        for s in ids:
            place[s] += len(paths[s])
        compare()
        if step % 2 == 1:
            old = w.clone()
            tok = [cache.tables.tokens(s) for s in ids]
            keep = cache.evict(ids, weights, 40, sinks=2, recent=9)
            for b, s in enumerate(ids):
                if tok[b] <= 40:
                    continue
                evictions += 1
                for layer in range(LAYERS):
                    for g in range(HKV):
                        of = kept(old[layer, entry[b], g].tolist(), tok[b], 40, 2, 9)
                        assert keep[layer, b, g].tolist() == of
                        c = sim[s][layer][g]
                        for name in ("k", "v", "w"):
                            c[name] = c[name][ints(of, torch.int64)]
            compare()
    assert evictions >= 4


def test_forks_keep_their_tokens(gpu):
    """One of two forks is trimmed: the other's pages are as they were."""
    announce("evict a fork")
    gen = torch.Generator(device="cuda").manual_seed(1)
    cache = kvcache.PagedCache(1, 30, 8, 2, 64)
    a = cache.tables.add()
    cache.batch({a: 50})
    cache.commit({a: 50})
    cache.k.copy_(torch.randn(cache.k.shape, device="cuda", generator=gen))
    cache.v.copy_(torch.randn(cache.v.shape, device="cuda", generator=gen))
    b = cache.fork(a)

    def rows(s, n):
        at = torch.arange(n, device="cuda")
        pages = torch.tensor(cache.tables.pages_of(s), device="cuda")
        return torch.stack((cache.k[0, pages[at // 8], at % 8], cache.v[0, pages[at // 8], at % 8])).clone()

    was = rows(a, 50)
    w = torch.rand(1, 2, 2, 60, device="cuda", generator=gen)
    keep = cache.evict([b], ops.make_weights(w, entry=torch.tensor([1], dtype=torch.int32, device="cuda")), 20, recent=4)
    assert torch.equal(rows(a, 50), was)
    now = rows(b, 20)
    for h in range(2):
        assert torch.equal(now[:, :, h], was[:, keep[0, 0, h].long(), h])
    assert not set(cache.tables.pages_of(a)) & set(cache.tables.pages_of(b))


def test_entries_are_read_before_tokens_go(gpu):
    """A sequence that would lose tokens without weights of its own is refused, and all
    stays; with them it is trimmed."""
    announce("evict entries")
    gen = torch.Generator(device="cuda").manual_seed(2)
    cache = kvcache.PagedCache(1, 30, 8, 2, 64)
    ids = [cache.tables.add() for _ in range(2)]
    news = dict(zip(ids, (50, 30)))
    cache.batch(news)
    cache.commit(news)
    cache.k.copy_(torch.randn(cache.k.shape, device="cuda", generator=gen))
    w = torch.rand(1, 3, 2, 60, device="cuda", generator=gen)
    was, old = cache.k.clone(), w.clone()
    entry = torch.zeros(2, dtype=torch.int32, device="cuda")
    weights = ops.make_weights(w, entry=entry)
    for bad in ([0, 3], [-1, 0], [1, 1]):
        entry.copy_(torch.tensor(bad, dtype=torch.int32))
        with pytest.raises(ValueError, match="entry of its own"):
            cache.evict(ids, weights, 20, recent=4)
    assert torch.equal(cache.k, was) and torch.equal(w, old) and [cache.tables.tokens(s) for s in ids] == [50, 30]
    entry.copy_(torch.tensor([2, -1], dtype=torch.int32))
    keep = cache.evict(ids, weights, 40, recent=4)  # (the second has too few tokens to lose any)
    assert [cache.tables.tokens(s) for s in ids] == [40, 30]
    for h in range(2):
        assert keep[0, 0, h].tolist() == kept(old[0, 2, h].tolist(), 50, 40, 0, 4)
        assert keep[0, 1, h].tolist() == list(range(30)) + [-1] * 10
