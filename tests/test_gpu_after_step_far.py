"""The calls after a step at addresses past 32 bits, on other streams, and from
graphs that share a workspace: each against the same call in the ordinary place."""

import random

import pytest
import torch

from kernrelay_amd import ops
from tests.conftest import announce
from tests.test_gpu_evict import kept

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def ints(v, dt=torch.int32):
    return torch.tensor(v, dtype=dt, device="cuda")


def randn(g, *shape, dt=BF):
    return torch.randn(*shape, device="cuda", generator=g).to(dt)


def pages_of(cache, ids):
    return cache[:, ids].clone()


@pytest.mark.parametrize("new", [1, 40])
def test_pages_and_weights_past_32_bits(gpu, new):
    """Pages from 2^31 elements on of a cache, weights of an entry there, beside a small
    cache and weights with the same tokens."""
    announce("far pages %d" % new)
    g = torch.Generator(device="cuda").manual_seed(new)
    H, G, D, page, pages, layers = 2, 4, 128, 16, 550000, 1
    far = [torch.empty(layers, pages, page, H, D, dtype=BF, device="cuda") for _ in range(2)]
    assert far[0].numel() > 2 ** 31
    lens, used = [70, 33], [9, 8]
    ids = [pages - 1 - 7 * i for i in range(sum(used))]
    for t in far:
        t[:, ids] = randn(g, layers, len(ids), page, H, D)
    near = [pages_of(t, ids) for t in far]
    width = 200
    room = torch.empty(2 ** 31 + 2 ** 20, device="cuda")
    wide = room.as_strided((layers, 3, H, width), (0, 2 ** 30, 256, 1))  # (entry 2 begins at 2^31)
    wide.copy_(torch.rand(layers, 3, H, width, device="cuda", generator=g))
    small = wide.clone()
    rows = 2 * new
    q, lse = randn(g, rows, H * G, D), torch.randn(rows, H * G, device="cuda", generator=g) + 9
    tables = {"far": [ids[:9], ids[9:] + [-1]], "near": [list(range(9)), list(range(9, 17)) + [-1]]}
    out = []
    for kv, w, where in ((far, wide, "far"), (near, small, "near")):
        cache = ops.make_cache(*kv)
        seqs = ops.make_seqs(ints(tables[where]), ints(lens), ints([0, new, rows]), new)
        h = ops.make_weights(w, entry=ints([2, 0]))
        ws = torch.empty(ops.attention_paged_weigh_workspace(cache, seqs, H * G), dtype=torch.uint8, device="cuda")
        ops.attention_paged_weigh(cache, 0, seqs, q, lse, h, ws)
        weighed = w.clone()
        done = ops.make_seqs(ints(tables[where]), ints([n + new for n in lens]), ints([0, 0, 0]), 0)
        keep = torch.empty(layers, 2, H, 24, dtype=torch.int32, device="cuda")
        ops.cache_evict(cache, done, h, keep, sinks=2, recent=5)
        out.append((weighed, w.clone(), keep, *(pages_of(t, ids if where == "far" else list(range(17))) for t in kv)))
    for a, b in zip(*out):
        assert torch.equal(a, b)
    for b, e in enumerate((2, 0)):
        for head in range(H):
            assert out[0][2][0, b, head].tolist() == kept(out[0][0][0, e, head].tolist(), lens[b] + new, 24, 2, 5)


@pytest.mark.parametrize("draft", [False, True])
def test_logits_past_32_bits(gpu, draft):
    announce("far logits %s" % draft)
    g = torch.Generator(device="cuda").manual_seed(3)
    V, rows, ld = 9001, 4, 750000011
    x = randn(g, rows, V, dt=HF) * 3
    p = torch.softmax(x.float(), 1).to(HF) if draft else None
    tokens, u, u_next = x.float().argmax(1).roll(1, 0), torch.full((rows,), 0.01, device="cuda"), ints([0], torch.float32)
    u_next.fill_(0.7)
    got = []
    room = [torch.empty(3 * ld + V, dtype=HF, device="cuda") for _ in range(2 if draft else 1)]
    for far in (False, True):
        ts = [x, p]
        if far:
            for i, r in enumerate(room):
                wide = r.as_strided((rows, V), (ld, 1))
                wide.copy_(ts[i])
                ts[i] = wide
        seqs = ops.make_seqs(ints([[0]]), ints([0]), ints([0, rows]), rows)
        nbytes, ncnt = ops.verify_drafts_workspace(seqs, ts[0], draft=ts[1])
        path, n, nxt = torch.empty(1, rows, dtype=torch.int32, device="cuda"), ints([0]), ints([0], torch.int64)
        ops.verify_drafts(seqs, ts[0], tokens, u, u_next, path, n, nxt, torch.empty(nbytes, dtype=torch.uint8, device="cuda"),
                          torch.zeros(ncnt, dtype=torch.int32, device="cuda"), draft=ts[1])
        got.append((path.tolist(), n.tolist(), nxt.tolist()))
    assert got[0] == got[1] and got[0][1] == [rows]  # (each draft is its row's largest: accepted)


def test_graphs_that_share_a_workspace(gpu):
    """Two captured steps over many rows, each with its own handles, and eager calls in
    between: one workspace for all, one after the other."""
    announce("shared workspace")
    g = torch.Generator(device="cuda").manual_seed(8)
    rng = random.Random(8)
    H, G, D, page = 2, 4, 64, 16
    k, v = randn(g, 1, 200, page, H, D), randn(g, 1, 200, page, H, D)
    cache = ops.make_cache(k, v)
    steps = []
    for new, n in ((50, 3), (17, 5)):
        ids = rng.sample(range(200), n * 20)
        lens = ints([rng.randint(1, 250) for _ in range(n)])
        seqs = ops.make_seqs(ints(ids).view(n, 20), lens, ints([new * i for i in range(n + 1)]), new)
        q = randn(g, new * n, H * G, D)
        steps.append(dict(seqs=seqs, q=q, out=torch.empty_like(q), lse=torch.empty(new * n, H * G, device="cuda"),
                          w=torch.zeros(1, n, H, 320, device="cuda"), lens=lens, n=n))
    need = [ops.attention_paged_workspace(cache, s["seqs"], H * G) for s in steps]
    ws = torch.empty(max(b for b, _ in need), dtype=torch.uint8, device="cuda")
    cnt = torch.zeros(max(c for _, c in need) + 1, dtype=torch.int32, device="cuda")
    wws = torch.empty(max(ops.attention_paged_weigh_workspace(cache, s["seqs"], H * G) for s in steps), dtype=torch.uint8,
                      device="cuda")
    assert wws.numel() > 0

    def run(s):
        ops.attention_paged(cache, 0, s["seqs"], s["q"], s["out"], ws=ws, counters=cnt, lse=s["lse"])
        ops.attention_paged_weigh(cache, 0, s["seqs"], s["q"], s["lse"], ops.make_weights(s["w"]), wws)

    graphs = []
    for s in steps:
        run(s)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run(s)
    for i in range(6):
        s, other = steps[i % 2], steps[1 - i % 2]
        s["lens"].copy_(ints([rng.randint(1, 250) for _ in range(s["n"])]))
        s["w"].fill_(0.5)
        graphs[i % 2].replay()
        run(other)
        torch.cuda.synchronize()
        got = s["w"].clone()
        s["w"].fill_(0.5)
        wws.fill_(255)
        run(s)
        torch.cuda.synchronize()
        assert torch.equal(got, s["w"])


def test_evictions_on_two_streams(gpu):
    """Of different sequences of one cache, at the same time, each on a stream of its own."""
    announce("evict streams")
    g = torch.Generator(device="cuda").manual_seed(2)
    rng = random.Random(2)
    layers, H, D, page = 3, 2, 64, 8
    k, v = randn(g, layers, 700, page, H, D), randn(g, layers, 700, page, H, D)
    cache = ops.make_cache(k, v)
    ids = rng.sample(range(700), 600)
    w = torch.rand(layers, 2, H, 2400, device="cuda", generator=g)
    first = w.clone()
    lens = [2400, 1999]
    tables = [ids[:300], ids[300:]]
    streams, keeps = [torch.cuda.Stream() for _ in range(2)], []
    for b, s in enumerate(streams):
        seqs = ops.make_seqs(ints([tables[b]]), ints([lens[b]]), ints([0, 0]), 0)
        keeps.append((seqs, ops.make_weights(w, entry=ints([b])),
                      torch.empty(layers, 1, H, 900, dtype=torch.int32, device="cuda")))
    was = k.clone()
    torch.cuda.synchronize()
    for (seqs, h, keep), s in zip(keeps, streams):
        ops.cache_evict(cache, seqs, h, keep, sinks=4, recent=300, stream=s)
    torch.cuda.synchronize()
    for b, (_, _, keep) in enumerate(keeps):
        t = ints(tables[b], torch.int64)
        to = torch.arange(900, device="cuda")
        for layer in range(layers):
            for head in range(H):
                of = kept(first[layer, b, head].tolist(), lens[b], 900, 4, 300)
                assert keep[layer, 0, head].tolist() == of
                of = ints(of, torch.int64)
                assert torch.equal(k[layer, t[to // page], to % page, head], was[layer, t[of // page], of % page, head])
                assert torch.equal(w[layer, b, head, :900], first[layer, b, head][of])
