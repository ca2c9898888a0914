"""Page bookkeeping of the paged cache (no GPU): pages are never shared by
accident, never lost, and copies are asked for exactly where a shared page
would be written."""

import random
from types import SimpleNamespace

import pytest
import torch

from kernrelay_amd import kvcache
from kernrelay_amd.kvcache import PageTables


class Mirror:
    """What each sequence's tokens are, kept beside the tables: page contents
    as plain lists that only the tables' own answers touch."""

    def __init__(self, pages, page_size):
        self.t = PageTables(pages, page_size)
        self.mem = [None] * (pages * page_size)
        self.want = {}
        self.stamp = 0

    def copy(self, src, dst):
        n = self.t.page_size
        assert len(set(dst)) == len(dst) and not set(dst) & set(src)
        for a, b in zip(src, dst):
            self.mem[b * n:(b + 1) * n] = self.mem[a * n:(a + 1) * n]

    def append(self, wants, keep=None):
        self.copy(*self.t.reserve(wants))
        for s, n in wants.items():
            new = []
            for slot in self.t.slots(s, n):
                self.stamp += 1
                self.mem[slot] = self.stamp
                new.append(self.stamp)
            k = n if keep is None else keep
            self.want[s] = self.want[s] + new[:k]
            self.t.commit(s, k)

    def check(self):
        n = self.t.page_size
        for s, want in self.want.items():
            ids = self.t.pages_of(s)
            assert self.t.tokens(s) == len(want) and len(ids) == -(-len(want) // n)
            assert [self.mem[ids[i // n] * n + i % n] for i in range(len(want))] == want
        used = {p for s in self.want for p in self.t.pages_of(s)}
        assert self.t.free_pages() == self.t.pages - len(used)


@pytest.mark.parametrize("page_size", [1, 3, 16])
@pytest.mark.parametrize("seed", range(4))
def test_random_histories(page_size, seed):
    rng = random.Random(seed)
    m = Mirror(40, page_size)
    for _ in range(300):
        act = rng.choice(("add", "append", "append", "drafts", "fork", "free", "defragment"))
        live = list(m.want)
        try:
            if act == "add" or not live:
                m.want[m.t.add()] = []
            elif act == "append":
                m.append({s: rng.randint(0, 2 * page_size) for s in rng.sample(live, rng.randint(1, len(live)))})
            elif act == "drafts":
                s = rng.choice(live)
                n = rng.randint(1, 3 * page_size)
                m.append({s: n}, keep=rng.randint(0, n))
            elif act == "fork":
                s = rng.choice(live)
                m.want[m.t.fork(s)] = list(m.want[s])
            elif act == "free":
                s = rng.choice(live)
                m.t.free(s)
                del m.want[s]
            else:
                m.copy(*m.t.defragment())
                used = {p for s in m.want for p in m.t.pages_of(s)}
                assert used == set(range(len(used)))
        except MemoryError:
            pass
        m.check()


def test_both_forks_write_at_once():
    """Two holders of one page that write in one batch: one copies, one keeps."""
    m = Mirror(8, 4)
    a = m.t.add()
    m.want[a] = []
    m.append({a: 6})
    b = m.t.fork(a)
    m.want[b] = list(m.want[a])
    m.append({a: 1, b: 1})
    m.check()
    assert m.t.pages_of(a)[0] == m.t.pages_of(b)[0] and m.t.pages_of(a)[1] != m.t.pages_of(b)[1]
    assert m.t.free_pages() == 5


def test_full_pool_changes_nothing():
    t = PageTables(3, 2)
    a, b = t.add(), t.add()
    t.reserve({a: 4})
    t.commit(a, 4)
    with pytest.raises(MemoryError, match="needs 3 pages, 1 of 3"):
        t.reserve({b: 5, a: 0})
    assert t.free_pages() == 1 and t.pages_of(b) == []


def test_refusals():
    with pytest.raises(ValueError):
        PageTables(0, 4)
    t = PageTables(2, 2)
    a = t.add()
    with pytest.raises(KeyError):
        t.free(7)
    with pytest.raises(ValueError, match="no room"):
        t.slots(a, 1)
    with pytest.raises(ValueError, match="no room"):
        t.commit(a, 1)
    with pytest.raises(ValueError, match="negative"):
        t.reserve({a: -1})
    t.free(a)
    with pytest.raises(KeyError):
        t.tokens(a)


class Calls:
    """Stands for the GPU calls: what would have been launched."""

    def __init__(self, monkeypatch):
        self.made = []
        note = lambda name: lambda *a, **kw: self.made.append(name)  # noqa: E731
        monkeypatch.setattr(kvcache.ops, "make_cache", lambda k, v: SimpleNamespace(device=0))
        monkeypatch.setattr(kvcache.ops, "make_seqs", lambda *a, **kw: SimpleNamespace())
        for name in ("cache_copy_pages", "cache_compact"):
            monkeypatch.setattr(kvcache.ops, name, note(name))
        monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


@pytest.mark.parametrize("between", ["defragment", "free", "accept", "batch", "commit"])
def test_accept_refuses_a_batch_whose_pages_moved(monkeypatch, between):
    """Its page table is the batch's: rows would move on pages that are not the
    sequences' any more."""
    calls = Calls(monkeypatch)
    cache = kvcache.PagedCache(1, 16, 4, 1, 64, device="cpu")
    hole, a, b = (cache.tables.add() for _ in range(3))
    for s in (hole, a, b):
        cache.batch({s: 5})
        cache.commit({s: 5})
    seqs, _, _ = cache.batch({a: 6, b: 2})
    if between == "defragment":
        cache.free(hole)
        cache.defragment()
    elif between == "free":
        cache.free(b)
    elif between == "accept":
        cache.accept(seqs, {a: [1, 3], b: [0]})
    elif between == "batch":
        cache.batch({a: 9})
    else:
        cache.commit({a: 1, b: 2})
    made, held = list(calls.made), {s: cache.tables.tokens(s) for s in (a,)}
    with pytest.raises((ValueError, KeyError)):
        cache.accept(seqs, {a: [1, 3], b: [0]})
    assert calls.made == made and cache.tables.tokens(a) == held[a]


def test_accept_after_a_fork(monkeypatch):
    """A fork in between shares the tokens that were; the drafts stay their own."""
    Calls(monkeypatch)
    cache = kvcache.PagedCache(1, 16, 4, 1, 64, device="cpu")
    a = cache.tables.add()
    cache.batch({a: 5})
    cache.commit({a: 5})
    seqs, _, _ = cache.batch({a: 3})
    b = cache.fork(a)
    cache.accept(seqs, {a: [0, 2]})
    assert (cache.tables.tokens(a), cache.tables.tokens(b)) == (7, 5)


def test_commit_is_all_or_nothing(monkeypatch):
    Calls(monkeypatch)
    cache = kvcache.PagedCache(1, 16, 4, 1, 64, device="cpu")
    a, b = cache.tables.add(), cache.tables.add()
    cache.batch({a: 3, b: 3})
    with pytest.raises(ValueError, match="no room"):
        cache.commit({a: 3, b: 30})
    assert cache.tables.tokens(a) == 0


def test_tables_stay_as_they_are_while_a_graph_is_captured(monkeypatch):
    """The copies that a reservation needs would only run with the graph."""
    Calls(monkeypatch)
    cache = kvcache.PagedCache(1, 16, 4, 1, 64, device="cpu")
    a = cache.tables.add()
    seqs, _, _ = cache.batch({a: 3})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    free = cache.tables.free_pages()
    for call in (lambda: cache.batch({a: 9}), lambda: cache.accept(seqs, {a: [1]}), cache.defragment):
        with pytest.raises(ValueError, match="captured"):
            call()
    assert cache.tables.free_pages() == free and cache.tables.tokens(a) == 0
