"""Page tables when tokens go: positions, pages given back and shared ones, and
what PagedCache.evict refuses (no GPU)."""

from types import SimpleNamespace

import pytest
import torch

from kernrelay_amd import kvcache
from kernrelay_amd.kvcache import PageTables


def grown(t, n):
    s = t.add()
    t.reserve({s: n})
    t.commit(s, n)
    return s


def test_positions_go_on_and_pages_come_back():
    t = PageTables(10, 4)
    a = grown(t, 30)
    assert (t.position(a), t.free_pages()) == (30, 2)
    t.evict(a, 30)
    assert (t.tokens(a), t.position(a), t.free_pages()) == (30, 30, 2)  # nothing to do
    t.evict(a, 9)
    assert (t.tokens(a), t.position(a), t.free_pages()) == (9, 30, 7)
    t.reserve({a: 4})
    t.commit(a, 4)
    t.evict(a, 9)
    assert (t.tokens(a), t.position(a)) == (9, 34)
    b = t.fork(a)
    assert (t.tokens(b), t.position(b)) == (9, 34)
    t.free(a)
    t.free(b)
    assert t.free_pages() == 10 and t.position(t.add()) == 0


def test_shared_pages_are_copied():
    t = PageTables(12, 4)
    a = grown(t, 18)
    b, c = t.fork(a), t.fork(a)
    before = t.pages_of(a)
    src, dst = t.own({a: 10, b: 6})
    # a takes copies of its first three, b of its first two; c keeps the old ones
    assert src == before[:3] + before[:2] and len(set(dst)) == 5 and not set(dst) & set(before)
    assert t.pages_of(a) == dst[:3] + before[3:] and t.pages_of(b) == dst[3:] + before[2:]
    assert t.pages_of(c) == before
    src, dst = t.own({c: 8})
    assert (src, dst) == ([], [])  # nobody else holds them now
    for s in (a, b, c):
        t.free(s)
    assert t.free_pages() == 12


def test_the_last_holder_keeps_its_page():
    t = PageTables(6, 4)
    a = grown(t, 8)
    b = t.fork(a)
    before = t.pages_of(a)
    src, dst = t.own({a: 8, b: 8})
    assert src == before and t.pages_of(b) == before and t.pages_of(a) == dst


def test_too_few_pages_change_nothing():
    t = PageTables(3, 4)
    a = grown(t, 8)
    b = t.fork(a)
    with pytest.raises(MemoryError, match="needs 2 pages, 1 of 3"):
        t.own({a: 8})
    assert t.pages_of(a) == t.pages_of(b)
    with pytest.raises(ValueError, match="budget"):
        t.evict(a, 0)


class Calls:
    def __init__(self, monkeypatch):
        self.made = []
        note = lambda name: lambda *a, **kw: self.made.append((name, a))  # noqa: E731
        monkeypatch.setattr(kvcache.ops, "make_cache", lambda k, v: SimpleNamespace(device=0))
        monkeypatch.setattr(kvcache.ops, "make_seqs", lambda *a, **kw: SimpleNamespace(args=a))
        for name in ("cache_copy_pages", "cache_compact", "cache_evict"):
            monkeypatch.setattr(kvcache.ops, name, note(name))
        monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def weights(**kw):
    f = dict(layers=2, heads=3, width=64, entries=4, seqs=None, device=0)
    f.update(kw)
    return SimpleNamespace(**f)


def make(monkeypatch, sizes):
    calls = Calls(monkeypatch)
    cache = kvcache.PagedCache(2, 32, 4, 3, 64, device="cpu")
    seqs = []
    for n in sizes:
        s = cache.tables.add()
        cache.batch({s: n})
        cache.commit({s: n})
        seqs.append(s)
    calls.made.clear()
    return calls, cache, seqs


def test_evict(monkeypatch):
    calls, cache, (a, b) = make(monkeypatch, [30, 7])
    c = cache.fork(a)
    keep = cache.evict([b, a], weights(), 10, sinks=1, recent=2)
    assert keep.shape == (2, 2, 3, 10)
    assert [m[0] for m in calls.made] == ["cache_copy_pages", "cache_evict"]
    table, lens = calls.made[1][1][1].args[:2]
    assert lens.tolist() == [7, 30] and table.shape == (2, 8)
    assert len(calls.made[0][1][1]) == 3  # the pages of a's ten tokens are c's too
    assert [cache.tables.tokens(s) for s in (a, b, c)] == [10, 7, 30]
    _, positions, slots = cache.batch({a: 2, b: 1})
    assert positions.tolist() == [30, 31, 7] and len(set(slots.tolist())) == 3
    cache.commit({a: 2, b: 1})


@pytest.mark.parametrize("kw,args,text", [
    (dict(layers=1), {}, "layers"), (dict(heads=2), {}, "heads"), (dict(device=1), {}, "device"),
    (dict(entries=1), {}, "entry"), (dict(seqs=3), {}, "entry"), (dict(width=29), {}, "columns"),
    ({}, dict(budget=0), "budget"), ({}, dict(sinks=6, recent=5), "budget"), ({}, dict(sinks=-1), "budget"),
    ({}, dict(recent=-1), "budget"), ({}, dict(twice=True), "twice"),
])
def test_evict_refuses_and_changes_nothing(monkeypatch, kw, args, text):
    calls, cache, (a, b) = make(monkeypatch, [30, 7])
    cache.fork(a)
    args = dict(args)
    ids = [a, a] if args.pop("twice", False) else [a, b]
    pages = cache.tables.pages_of(a)
    with pytest.raises(ValueError, match=text):
        cache.evict(ids, weights(**kw), args.pop("budget", 10), **args)
    assert calls.made == [] and cache.tables.pages_of(a) == pages and cache.tables.tokens(a) == 30
    with pytest.raises(KeyError):
        cache.evict([99], weights(), 10)


def test_batches_from_before_are_out_of_date(monkeypatch):
    _, cache, (a, b) = make(monkeypatch, [30, 7])
    seqs, _, _ = cache.batch({a: 3, b: 3})
    cache.evict([a, b], weights(), 10)
    with pytest.raises(ValueError, match="out of date"):
        cache.accept(seqs, {a: [0], b: [0]})
    with pytest.raises(ValueError, match="out of date"):
        cache.commit({b: 3, a: 1})
    assert cache.tables.tokens(b) == 7
    cache.commit({b: 3, a: 0})
    cache.batch({a: 1})
    cache.commit({a: 1})
    assert (cache.tables.tokens(a), cache.tables.position(a)) == (11, 31)


def test_not_while_a_graph_is_captured(monkeypatch):
    _, cache, (a, _) = make(monkeypatch, [30, 7])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(ValueError, match="captured"):
        cache.evict([a], weights(), 10)


@pytest.mark.parametrize("entry,ok", [
    ([2, 0, 1], True), ([2, 0, -1], True), ([2, 0, 2], True),  # (the last has too few tokens to lose any)
    ([4, 0, 1], False), ([0, -1, 1], False), ([3, 3, 1], False),
])
def test_sequences_that_lose_tokens_have_weights_of_their_own(monkeypatch, entry, ok):
    """The device leaves a sequence without weights alone, and two of one entry move
    its weights twice: the tables would say otherwise."""
    calls, cache, ids = make(monkeypatch, [30, 20, 7])
    w = weights(seqs=3, keep=(None, torch.tensor(entry, dtype=torch.int32)))
    pages = [cache.tables.pages_of(s) for s in ids]
    if ok:
        cache.evict(ids, w, 10)
        assert [cache.tables.tokens(s) for s in ids] == [10, 10, 7]
        return
    with pytest.raises(ValueError, match="entry of its own"):
        cache.evict(ids, w, 10)
    assert calls.made == [] and [cache.tables.tokens(s) for s in ids] == [30, 20, 7]
    assert [cache.tables.pages_of(s) for s in ids] == pages


def test_a_batch_that_was_kept_before_an_eviction_is_out_of_date_too(monkeypatch):
    """As many tokens on the same pages as when it was made: accept refuses it all the
    same, before any row moves."""
    calls, cache, (a, b) = make(monkeypatch, [9, 7])
    seqs, _, _ = cache.batch({a: 2, b: 3})
    cache.commit({a: 2})
    cache.evict([a], weights(), 9)
    assert cache.tables.tokens(a) == 9
    calls.made.clear()
    for path in ([], [0], [1]):
        with pytest.raises(ValueError, match="out of date"):
            cache.accept(seqs, {a: path, b: [0, 1]})
    assert calls.made == [] and (cache.tables.tokens(a), cache.tables.tokens(b)) == (9, 7)
