"""A paged key/value cache: whose page is whose (PageTables, plain host
bookkeeping) and the pages themselves on the GPU (PagedCache), with the calls
that write, read and move them (ops.qk_norm_rope_cache, ops.attention_paged,
ops.cache_copy_pages, ops.cache_compact, ops.cache_evict).

No counterpart in the reference, which stops at the prompt's last row. Pages
are shared by forked sequences and copied when one of them writes; a sequence
takes pages as its tokens come and gives them back when it ends.
"""

import heapq
import warnings

from . import ops


class PageTables:
    """Which pages hold which sequence's tokens. Page ids are handed out lowest
    first. Every method either does all it says or raises and changes nothing."""

    def __init__(self, pages, page_size):
        if pages < 1 or page_size < 1:
            raise ValueError("needs at least one page of one token")
        self.pages, self.page_size = pages, page_size
        self._free = list(range(pages))  # a heap
        self._refs = [0] * pages
        self._seqs = {}                  # id -> [tokens, page ids]
        self._gone = {}                  # id -> tokens evicted so far, where there are any
        self._next = 0

    def _seq(self, seq):
        try:
            return self._seqs[seq]
        except KeyError:
            raise KeyError("no sequence %r" % (seq,)) from None

    def free_pages(self):
        return len(self._free)

    def tokens(self, seq):
        return self._seq(seq)[0]

    def position(self, seq):
        """Of the sequence's next token: its tokens and those evicted."""
        return self._seq(seq)[0] + self._gone.get(seq, 0)

    def pages_of(self, seq):
        return list(self._seq(seq)[1])

    def add(self):
        """A new, empty sequence's id."""
        seq, self._next = self._next, self._next + 1
        self._seqs[seq] = [0, []]
        return seq

    def fork(self, seq):
        """A new sequence with the same tokens, on the same pages."""
        tokens, ids = self._seq(seq)
        keep = ids[:-(-tokens // self.page_size)]
        new = self.add()
        self._seqs[new] = [tokens, keep]
        if seq in self._gone:
            self._gone[new] = self._gone[seq]
        for p in keep:
            self._refs[p] += 1
        return new

    def _drop(self, ids):
        for p in ids:
            self._refs[p] -= 1
            if self._refs[p] == 0:
                heapq.heappush(self._free, p)

    def free(self, seq):
        """Ends a sequence; pages that no other one shares are free again."""
        self._drop(self._seq(seq)[1])
        del self._seqs[seq]
        self._gone.pop(seq, None)

    def reserve(self, wants):
        """Room for wants[seq] more tokens of each sequence: new pages, and own
        copies of shared pages that the tokens would write to. Returns the pages
        to copy as (sources, copies). MemoryError if the pages do not suffice."""
        need = 0
        plan = []
        left = {}  # shared page -> holders that keep it
        for seq, n in wants.items():
            if n < 0:
                raise ValueError("a negative number of tokens")
            tokens, ids = self._seq(seq)
            own = []
            if n > 0:
                for at in range(tokens // self.page_size, len(ids)):
                    holders = left.setdefault(ids[at], self._refs[ids[at]])
                    if holders > 1:
                        own.append(at)
                        left[ids[at]] = holders - 1
            more = max(0, -(-(tokens + n) // self.page_size) - len(ids))
            plan.append((seq, own, more))
            need += len(own) + more
        if need > len(self._free):
            raise MemoryError("needs %d pages, %d of %d are free" % (need, len(self._free), self.pages))
        src, dst = [], []
        for seq, own, more in plan:
            tokens, ids = self._seqs[seq]
            for at in own:
                new = self._take()
                if at * self.page_size < tokens:  # (behind the last token there is nothing to copy)
                    src.append(ids[at])
                    dst.append(new)
                self._refs[ids[at]] -= 1
                ids[at] = new
            ids.extend(self._take() for _ in range(more))
        return src, dst

    def _take(self):
        p = heapq.heappop(self._free)
        self._refs[p] = 1
        return p

    def slots(self, seq, n):
        """Cache slots of the sequence's next n tokens (reserved before)."""
        tokens, ids = self._seq(seq)
        if n < 0 or tokens + n > len(ids) * self.page_size:
            raise ValueError("sequence %r has no room for %d more tokens" % (seq, n))
        return [ids[t // self.page_size] * self.page_size + t % self.page_size for t in range(tokens, tokens + n)]

    def commit(self, seq, n):
        """The next n tokens are the sequence's; pages behind them are given back."""
        s = self._seq(seq)
        if n < 0 or s[0] + n > len(s[1]) * self.page_size:
            raise ValueError("sequence %r has no room for %d more tokens" % (seq, n))
        s[0] += n
        keep = -(-s[0] // self.page_size)
        self._drop(s[1][keep:])
        del s[1][keep:]

    def own(self, counts):
        """Own copies of the shared pages that hold the first counts[seq] tokens of
        each sequence. Returns the pages to copy as (sources, copies).
        MemoryError if the pages do not suffice."""
        plan = []
        left = {}  # shared page -> holders that keep it
        for seq, n in counts.items():
            ids = self._seq(seq)[1]
            for at in range(min(-(-n // self.page_size), len(ids))):
                holders = left.setdefault(ids[at], self._refs[ids[at]])
                if holders > 1:
                    plan.append((ids, at))
                    left[ids[at]] = holders - 1
        if len(plan) > len(self._free):
            raise MemoryError("needs %d pages, %d of %d are free" % (len(plan), len(self._free), self.pages))
        src, dst = [], []
        for ids, at in plan:
            new = self._take()
            src.append(ids[at])
            dst.append(new)
            self._refs[ids[at]] -= 1
            ids[at] = new
        return src, dst

    def evict(self, seq, budget):
        """The sequence has `budget` tokens if it had more; pages behind them are given back."""
        s = self._seq(seq)
        if budget < 1:
            raise ValueError("a budget holds at least one token")
        if s[0] > budget:
            self._gone[seq] = self._gone.get(seq, 0) + s[0] - budget
            s[0] = budget
            keep = -(-budget // self.page_size)
            self._drop(s[1][keep:])
            del s[1][keep:]

    def defragment(self):
        """Moves the pages in use to the lowest ids; returns (sources, copies)."""
        used = self.pages - len(self._free)
        to = sorted(p for p in self._free if p < used)
        of = [p for p in range(used, self.pages) if self._refs[p]]
        moved = dict(zip(of, to))
        for a, b in moved.items():
            self._refs[b], self._refs[a] = self._refs[a], 0
        for s in self._seqs.values():
            s[1][:] = [moved.get(p, p) for p in s[1]]
        self._free = list(range(used, self.pages))
        return of, to


class PagedCache:
    """The pages on the current GPU, [layers, pages, page_size, heads, head_dim]
    for keys and values, and their tables. Calls go to the current stream."""

    def __init__(self, layers, pages, page_size, heads, head_dim, dtype=None, device="cuda"):
        import torch
        dtype = torch.bfloat16 if dtype is None else dtype
        self.tables = PageTables(pages, page_size)
        shape = (layers, pages, page_size, heads, head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        self.handle = ops.make_cache(self.k, self.v)
        self._batches, self._last = 0, {}  # how many there were; the last one with new tokens of a sequence
        self._evicted = set()              # sequences that lost tokens after their last batch

    def _state(self, seq):
        """What a batch's rows of a sequence depend on."""
        # (the position too: an eviction can bring back the tokens and pages of before)
        return self._last.get(seq), self.tables.tokens(seq), self.tables.position(seq), self.tables.pages_of(seq)

    def _current(self):
        """Before the tables change: the calls that follow must reach the pages,
        and now (a captured copy would only run with its graph)."""
        import torch
        if torch.cuda.is_current_stream_capturing():
            raise ValueError("the tables cannot change while a graph is captured")
        if torch.cuda.current_device() != self.handle.device:
            raise ValueError("the cache is on device %d, the current device is %d" % (
                self.handle.device, torch.cuda.current_device()))

    def _ints(self, values, dtype):
        import torch
        return torch.tensor(values, dtype=dtype).to(self.k.device)

    def batch(self, news, tree=None, depths=None):
        """The next launch's sequences: news[seq] new tokens of each, in order.
        Reserves their pages (copying shared ones). tree [rows, words] int64:
        ops.make_seqs; depths[seq]: each draft's depth below the sequence's last
        token (needed with a tree; None: 0, 1, 2, ..). Returns (handle,
        positions, slots), good until one of the sequences ends, gets tokens or
        is in another batch with new tokens, or the pages are defragmented."""
        import torch
        self._current()
        if tree is not None:
            if depths is None:
                raise ValueError("a tree needs the depths of its drafts")
            ops.check_tree(tree, max(news.values(), default=0), "batch")
            if tree.shape[0] < sum(news.values()) or tree.device != self.k.device:
                raise ValueError("the tree must have a row for each new token, on the cache's device")
        if depths is not None and any(len(depths[s]) != n for s, n in news.items()):
            raise ValueError("depths must give one depth for each new token")
        # (all that can be refused is, before the tables change)
        positions = self._ints([self.tables.position(s) + (i if depths is None else depths[s][i])
                                for s, n in news.items() for i in range(n)], torch.int64)
        src, dst = self.tables.reserve(news)
        ops.cache_copy_pages(self.handle, src, dst)
        ids = [self.tables.pages_of(s) for s in news]
        width = max([1] + [len(i) for i in ids])
        starts, slots = [0], []
        for s, n in news.items():
            starts.append(starts[-1] + n)
            slots += self.tables.slots(s, n)
        seqs = ops.make_seqs(self._ints([i + [-1] * (width - len(i)) for i in ids], torch.int32).view(-1, width),
                             self._ints([self.tables.tokens(s) for s in news], torch.int32),
                             self._ints(starts, torch.int32), max(news.values(), default=0), tree=tree)
        seqs.news = dict(news)
        seqs.depths = None if depths is None else {s: tuple(depths[s]) for s in news}
        self._batches += 1
        self._last.update((s, self._batches) for s, n in news.items() if n > 0)
        self._evicted.difference_update(s for s, n in news.items() if n > 0)
        seqs.held = {s: self._state(s) for s in news}
        return seqs, positions, self._ints(slots, torch.int64)

    def commit(self, news):
        """All new tokens of the last batch are kept."""
        for s, n in news.items():
            if n > 0 and s in self._evicted:
                raise ValueError("the batch is out of date: sequence %r lost tokens since" % (s,))
            self.tables.slots(s, n)  # all have room, or none is kept
        for s, n in news.items():
            self.tables.commit(s, n)

    def accept(self, seqs, paths):
        """Of the drafts of a batch (its handle), paths[seq] are kept, in this
        order: their rows move up behind the sequence's tokens. Every sequence
        of the batch has a path, an empty one where none is kept. Keys stay
        rotated for the positions that batch returned, so the draft kept i-th
        must be one of depth i; a batch without depths cannot tell whether
        others' positions were used, and warns where its own would be wrong."""
        import torch
        self._current()
        if list(paths) != list(seqs.news):
            raise ValueError("paths must be of the batch's sequences, in its order")
        for s, held in seqs.held.items():
            if held != self._state(s):
                raise ValueError("the batch is out of date: sequence %r has other tokens, drafts or pages now" % (s,))
        for s, p in paths.items():
            if len(set(p)) != len(p) or any(not 0 <= i < seqs.news[s] for i in p):
                raise ValueError("the path of sequence %r must name its drafts, each once" % (s,))
            if seqs.depths is not None and any(seqs.depths[s][d] != i for i, d in enumerate(p)):
                raise ValueError("the path of sequence %r must go down draft by draft, from depth 0" % (s,))
        for s, p in paths.items():
            if seqs.depths is None and list(p) != list(range(len(p))):
                warnings.warn("the path of sequence %r skips drafts of a chain: keys written at the batch's positions "
                              "keep those of their old places" % (s,), RuntimeWarning, stacklevel=2)
        width = max([1] + [len(p) for p in paths.values()])
        path = self._ints([list(p) + [-1] * (width - len(p)) for p in paths.values()], torch.int32).view(-1, width)
        ops.cache_compact(self.handle, seqs, path, self._ints([len(p) for p in paths.values()], torch.int32))
        self.commit({s: len(p) for s, p in paths.items()})

    def fork(self, seq):
        return self.tables.fork(seq)

    def free(self, seq):
        self.tables.free(seq)
        self._last.pop(seq, None)
        self._evicted.discard(seq)

    def evict(self, seqs, weights, budget, sinks=0, recent=0):
        """Of each of the sequences (ids, each once) that has more than `budget`
        tokens the first `sinks`, the last `recent` and those with the largest
        weights stay (ops.cache_evict, of every layer and head by itself); the
        pages behind them are free again. weights: a handle (ops.make_weights)
        whose entries are these sequences', in this order: every one that loses
        tokens must have one of its own (the entry vector is read back for that, so
        the call waits for the stream). Positions of later tokens go on as if
        nothing had gone. Batches of the sequences are out of date afterwards.
        Returns keep [layers, seqs, heads, budget]."""
        import torch
        self._current()
        seqs = list(seqs)
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is named twice")
        if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
            raise ValueError("sinks and recent must fit a budget of at least one token")
        tokens = [self.tables.tokens(s) for s in seqs]
        layers, heads = self.k.shape[0], self.k.shape[3]
        if (weights.layers, weights.heads, weights.device) != (layers, heads, self.handle.device):
            raise ValueError("the weights must be of the cache's layers and heads, on its device")
        if weights.entries < len(seqs) if weights.seqs is None else weights.seqs != len(seqs):
            raise ValueError("the weights must have an entry for each sequence")
        if any(n > budget and n > weights.width for n in tokens):
            raise ValueError("a sequence has more tokens than the weights have columns")
        if weights.seqs is not None and any(n > budget for n in tokens):
            # (the vector is on the device, where a sequence without weights is left alone)
            entry = [e for e, n in zip(weights.keep[1].tolist(), tokens) if n > budget]
            if len(set(entry)) != len(entry) or any(not 0 <= e < weights.entries for e in entry):
                raise ValueError("each sequence that loses tokens must have an entry of its own in the weights")
        # (all that can be refused is, before the tables change)
        src, dst = self.tables.own({s: budget for s, n in zip(seqs, tokens) if n > budget})
        ops.cache_copy_pages(self.handle, src, dst)
        ids = [self.tables.pages_of(s) for s in seqs]
        width = max([1] + [len(i) for i in ids])
        handle = ops.make_seqs(self._ints([i + [-1] * (width - len(i)) for i in ids], torch.int32).view(-1, width),
                               self._ints(tokens, torch.int32), self._ints([0] * (len(seqs) + 1), torch.int32), 0)
        keep = torch.empty(layers, len(seqs), heads, budget, dtype=torch.int32, device=self.k.device)
        ops.cache_evict(self.handle, handle, weights, keep, sinks=sinks, recent=recent)
        for s, n in zip(seqs, tokens):
            if n > budget:
                self.tables.evict(s, budget)
                self._evicted.add(s)
        return keep

    def defragment(self):
        self._current()
        src, dst = self.tables.defragment()
        ops.cache_copy_pages(self.handle, src, dst)
