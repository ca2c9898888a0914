"""Accepted paths of PagedCache against the positions that their drafts' keys
were rotated for, and batches that are refused (no GPU: the launches are stood
in for)."""

import warnings

import pytest
import torch

from kernrelay_amd import kvcache
from tests.test_kvcache import Calls


@pytest.fixture
def cache(monkeypatch):
    """A cache with one sequence of 5 tokens, and the launches it would make."""
    calls = Calls(monkeypatch)
    c = kvcache.PagedCache(1, 16, 4, 1, 64, device="cpu")
    c.calls, c.seq = calls, c.tables.add()
    c.batch({c.seq: 5})
    c.commit({c.seq: 5})
    return c


TREE = torch.zeros(5, 1, dtype=torch.int64)
DEPTHS = [0, 1, 1, 2, 2]


@pytest.mark.parametrize("path", [[], [0], [0, 1], [0, 2, 4]])
def test_paths_that_go_down(cache, path):
    seqs, positions, _ = cache.batch({cache.seq: 5}, tree=TREE, depths={cache.seq: DEPTHS})
    assert positions.tolist() == [5 + d for d in DEPTHS]
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        cache.accept(seqs, {cache.seq: path})
    # the i-th kept draft's key was rotated for the place it has now
    assert [positions[d] for d in path] == list(range(5, cache.tables.tokens(cache.seq)))


@pytest.mark.parametrize("path", [[1], [0, 3], [1, 0], [0, 1, 2], [3, 4]])
def test_paths_that_skip_or_turn_back(cache, path):
    seqs, _, _ = cache.batch({cache.seq: 5}, tree=TREE, depths={cache.seq: DEPTHS})
    made = list(cache.calls.made)
    with pytest.raises(ValueError, match="draft by draft"):
        cache.accept(seqs, {cache.seq: path})
    assert cache.calls.made == made and cache.tables.tokens(cache.seq) == 5
    cache.accept(seqs, {cache.seq: [0, 2]})


def test_a_tree_needs_depths(cache):
    """Siblings would stand at one position after the other."""
    free = cache.tables.free_pages()
    with pytest.raises(ValueError, match="depths"):
        cache.batch({cache.seq: 5}, tree=TREE)
    assert cache.tables.free_pages() == free


def test_a_chain_that_is_not_kept_from_its_start_warns(cache):
    seqs, _, _ = cache.batch({cache.seq: 4})
    with pytest.warns(RuntimeWarning, match="chain"):
        cache.accept(seqs, {cache.seq: [0, 2]})
    seqs, _, _ = cache.batch({cache.seq: 4})
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        cache.accept(seqs, {cache.seq: [0, 1, 2]})


@pytest.mark.parametrize("tree,depths,error", [
    (TREE.int(), DEPTHS, ValueError), (TREE[:, 0], DEPTHS, ValueError), (TREE[:4], DEPTHS, ValueError),
    (torch.zeros(9, 0, dtype=torch.int64), DEPTHS, ValueError),
    (torch.zeros(1, 1, dtype=torch.int64).expand(5, 1), DEPTHS, ValueError),
    (torch.zeros(5, 1, dtype=torch.int64, device="meta"), DEPTHS, ValueError),
    (TREE, DEPTHS[:4], ValueError), (TREE, ["a"] * 5, TypeError), (TREE, [None] * 5, TypeError)])
def test_a_refused_batch_changes_nothing(cache, tree, depths, error):
    """Not the tables, nor the pages that a fork shares."""
    twin = cache.fork(cache.seq)
    held = cache.tables.free_pages(), cache.tables.pages_of(cache.seq), list(cache.calls.made)
    with pytest.raises(error):
        cache.batch({cache.seq: 5}, tree=tree, depths={cache.seq: depths})
    with pytest.raises(KeyError):
        cache.batch({cache.seq: 5, twin + 9: 1})
    with pytest.raises(ValueError):
        cache.batch({cache.seq: 5, twin: -1})
    assert (cache.tables.free_pages(), cache.tables.pages_of(cache.seq), cache.calls.made) == held
    cache.batch({cache.seq: 5}, tree=TREE, depths={cache.seq: DEPTHS})
    assert len(cache.calls.made) == len(held[2]) + 1 and cache.tables.pages_of(cache.seq) != held[1]


def test_drafts_that_a_later_batch_wrote_over(cache):
    """Two batches on the same page: the rows are the second's."""
    first, _, _ = cache.batch({cache.seq: 2}, tree=TREE, depths={cache.seq: [0, 1]})
    second, _, slots = cache.batch({cache.seq: 2}, tree=TREE, depths={cache.seq: [0, 0]})
    made = list(cache.calls.made)
    with pytest.raises(ValueError, match="out of date"):
        cache.accept(first, {cache.seq: [0, 1]})
    assert cache.calls.made == made and cache.tables.tokens(cache.seq) == 5
    other = cache.tables.add()
    cache.batch({other: 3, cache.seq: 0})  # no new tokens of the sequence
    cache.accept(second, {cache.seq: [1]})
    assert cache.tables.tokens(cache.seq) == 6
    cache.free(cache.seq)
    with pytest.raises(KeyError):
        cache.accept(second, {cache.seq: []})
