"""Drafts against the target's logits, against a plain restatement in 64 bits.

Outputs are whole numbers and equal: the kernels compute in 64 bits too, so the
two differ only where a random number comes within about 1e-13 of a border.
"""

import math

import numpy as np
import pytest
import torch

from kernrelay_amd import ops
from tests.conftest import announce

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def ints(v, dt=torch.int32):
    return torch.tensor(v, dtype=dt, device="cuda")


def softmax(x, t):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return np.zeros_like(x)
    if not t > 0:
        p = np.zeros_like(x)
        p[int(np.argmax(x))] = 1.0
        return p
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, 0.0 if top == np.inf else np.where(x == -np.inf, 0.0, np.exp((x - top) / t)))
    return w / w.sum()


def walk(x, q, tokens, par, u, u_next, t, width):
    """One sequence: path and next token."""
    n = len(tokens)
    if n == 0:
        return [], -1
    path, p = [0], softmax(x[0], t)
    going = True
    while going and len(path) < width:
        going = False
        for c in range(path[-1] + 1, n):
            if par[c] != path[-1]:
                continue
            y = tokens[c]
            ok = 0 <= y < x.shape[1]
            ask = 1.0 if q is None or not ok else max(float(np.nan_to_num(q[path[-1], y])), 0.0)
            if ok and float(u[c]) * ask < p[y]:
                path.append(c)
                p = softmax(x[c], t)
                going = True
                break
            if q is None:
                left = p.copy()
                if ok:
                    left[y] = 0.0
            else:
                left = np.maximum(p - np.maximum(np.nan_to_num(q[path[-1]].astype(np.float64)), 0.0), 0.0)
            if left.sum() > 0:
                p = left / left.sum()
    if p.sum() == 0:
        return path, -1
    sums = np.cumsum(p)
    over = np.nonzero((sums > float(u_next) * sums[-1]) & (p > 0))[0]
    return path, int(over[0]) if len(over) else int(np.nonzero(p)[0][-1])


class Case:
    def __init__(self, seed, news, V, dt=F32, tree=False, draft=None, temps=(1.0,), pad=0, off=0, spare_rows=0,
                 width=None, peak=3.0, max_new=None):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        rng = np.random.RandomState(seed)
        self.news, self.V = news, V
        self.starts = [sum(news[:i]) for i in range(len(news) + 1)]
        R = self.starts[-1] + spare_rows
        self.x = self._rows(R, V, dt, pad, off)
        self.x.copy_(torch.randn(R, V, device="cuda", generator=self.g) * peak)
        self.par = [[(rng.randint(max(0, i - 3), i) if tree else i - 1) if i else -1 for i in range(n)] for n in news]
        self.parents = ints([p for s in self.par for p in s] + [0] * spare_rows) if tree else None
        above = [self.starts[b] + max(p, 0) for b, s in enumerate(self.par) for p in s] + [0] * spare_rows
        self.draft = None
        if draft is not None:
            self.draft = self._rows(R, V, draft, pad, off)
            self.draft.copy_(torch.softmax(self.x.float() + torch.randn(R, V, device="cuda", generator=self.g) * 0.5, 1))
            q = self.draft.float()[ints(above, torch.int64)] if R else self.draft.float()
            e = -torch.rand(R, V, device="cuda", generator=self.g).clamp(min=1e-30).log()
            self.tokens = (q / e).argmax(1)
        else:
            self.tokens = self.x.float()[ints(above, torch.int64)].topk(min(3, V), 1).indices[:, 0].contiguous() if R else ints([], torch.int64)
            if tree and R:
                pick = torch.randint(0, min(3, V), (R, 1), device="cuda", generator=self.g)
                self.tokens = self.x.float()[ints(above, torch.int64)].topk(min(3, V), 1).indices.gather(1, pick)[:, 0]
        self.u = torch.rand(R, device="cuda", generator=self.g)
        self.u_next = torch.rand(len(news), device="cuda", generator=self.g)
        self.temps = [temps[i % len(temps)] for i in range(len(news))]
        self.width = max(news + [1]) if width is None else width
        self.max_new = max(news + [0]) if max_new is None else max_new

    def _rows(self, R, V, dt, pad, off):
        """[R, V] with `pad` values between rows, `off` values into an allocation."""
        flat = torch.zeros(off + R * (V + pad) + 1, dtype=dt, device="cuda")
        return flat[off:off + R * (V + pad)].view(R, V + pad)[:, :V]

    def handle(self):
        n = len(self.news)
        return ops.make_seqs(torch.zeros(n, 1, dtype=torch.int32, device="cuda"), ints([3] * n), ints(self.starts),
                             self.max_new)

    def run(self):
        n = len(self.news)
        pad = torch.full((n, self.width + 2), 55, dtype=torch.int32, device="cuda")
        path, lens, nxt = pad[:, :self.width], ints([9] * n), ints([9] * n, torch.int64)
        seqs = self.handle()
        nbytes, ncnt = ops.verify_drafts_workspace(seqs, self.x, draft=self.draft)
        ws = torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda")
        cnt = torch.zeros(ncnt, dtype=torch.int32, device="cuda")
        for _ in range(2):  # the workspace may hold anything, the counters are left zero
            ops.verify_drafts(seqs, self.x, self.tokens, self.u, self.u_next, path, lens, nxt, ws, cnt,
                              parents=self.parents, draft=self.draft,
                              temperature=torch.tensor(self.temps, device="cuda") if n else None)
        assert bool((pad[:, self.width:] == 55).all()) and not bool(cnt.any())
        return path.tolist(), lens.tolist(), nxt.tolist()

    def check(self):
        paths, lens, nxt = self.run()
        x = self.x.float().cpu().numpy()
        q = None if self.draft is None else self.draft.float().cpu().numpy()
        tokens, u = self.tokens.tolist(), self.u.tolist()
        seen = 0
        for b, (lo, hi) in enumerate(zip(self.starts, self.starts[1:])):
            hi = min(hi, lo + self.max_new)
            want, token = walk(x[lo:hi], None if q is None else q[lo:hi], tokens[lo:hi], self.par[b][:hi - lo], u[lo:hi],
                               self.u_next[b].item(), self.temps[b], self.width)
            assert paths[b] == want + [-1] * (self.width - len(want)), b
            assert lens[b] == len(want) and nxt[b] == token, (b, nxt[b], token)
            seen += len(want)
        return seen


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("draft", [None, F32, BF])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("V,pad,off", [(5, 0, 0), (1000, 8, 8), (8192, 0, 0), (8193, 0, 1), (30011, 5, 3)])
def test_against_64_bits(gpu, dt, draft, tree, V, pad, off):
    announce("verify %s" % ((dt, draft, tree, V, pad, off),))
    x = Case(V + pad, [1, 5, 0, 9, 2, 13], V, dt, tree, draft, temps=(1.0, 0.7, 0.0, 1.5), pad=pad, off=off, spare_rows=1)
    assert x.check() >= 5


@pytest.mark.parametrize("V", [1, 2, 3, 31])
@pytest.mark.parametrize("draft", [None, F32])
def test_small_vocabularies(gpu, V, draft):
    """Few tokens: siblings are the same ones, refusals leave nothing."""
    announce("verify small %d %s" % (V, draft))
    Case(V, [7, 30, 1, 12] * 5, V, F32, True, draft, temps=(1.0, 0.0, 3.0), peak=1.0).check()


def test_the_path_is_the_targets_own(gpu):
    """Rejection sampling's point: the first token after the root has the target's
    distribution, whether it is a draft or not. 40000 sequences; each token's count
    is within 5 standard deviations."""
    announce("verify distribution")
    N, V = 40000, 6
    for draft in (True, False):
        x = Case(1, [3] * N, V, F32, False, F32 if draft else None)
        x.x.copy_(torch.tensor([0.0, 1.0, 2.0, 0.5, -1.0, -math.inf], device="cuda"))
        q = torch.tensor([0.3, 0.1, 0.2, 0.1, 0.2, 0.1], device="cuda")
        siblings = [-1, 0, 0]
        x.par, x.parents = [siblings] * N, ints(siblings * N)
        if draft:
            x.draft.copy_(q.expand_as(x.draft))
            x.tokens = torch.multinomial(q, 3 * N, replacement=True, generator=x.g)
        else:
            x.tokens = ints([0, 2, 1] * N, torch.int64)
        paths, _, nxt = x.run()
        first = ints([n if p[1] < 0 else -1 for p, n in zip(paths, nxt)], torch.int64)
        took = ints([3 * b + max(p[1], 0) for b, p in enumerate(paths)], torch.int64)
        first = torch.where(first < 0, x.tokens[took], first)
        p = torch.softmax(x.x[0].double(), 0)
        count = torch.bincount(first, minlength=V).double()
        assert bool(((count - N * p).abs() <= 5 * (N * p * (1 - p)).sqrt()).all()), (count / N, p)


def test_odd_logits_and_tokens(gpu):
    """NaN, infinities, rows without any logit, tokens and parents that are none,
    probabilities below zero, random numbers at their ends."""
    announce("verify odd")
    for draft in (None, F32):
        x = Case(9, [6, 6, 6, 6, 6, 6, 3, 3], 700, F32, True, draft, temps=(1.0, 1.0, 0.0, 1.0, math.nan, 1e-30, math.inf, -1.0))
        x.x[0, 3] = math.nan
        x.x[0, 5:300] = -math.inf
        x.x[1] = -math.inf
        x.x[6:12, 40] = math.inf
        x.x[6:12, 699] = math.inf
        x.x[12:18, 7] = math.inf
        x.x[18] = math.nan          # no logit at all
        x.x[24, 100:] = math.nan
        x.x[36:39] = -math.inf
        x.x[36:39, 650] = -3.0
        x.tokens[[2, 8, 20, 31]] = ints([-1, 700, 2 ** 40, -2 ** 62], torch.int64)
        x.par[0][2], x.par[3][4], x.par[4][1] = 2, -7, 9
        x.parents = ints([p for s in x.par for p in s])
        for b, p in ((0, 2), (3, 4), (4, 1)):
            x.par[b][p] = -1        # follows nothing
        if draft:
            x.draft[0, :20] = -0.5
            x.draft[7, 3] = math.nan
            x.draft[13] = 0.0
        x.u[:6] = 0.0
        x.u_next.copy_(torch.tensor([0.0, 1 - 2 ** -24, 0.0, 0.5, 0.0, 0.3, 0.0, 0.9], device="cuda"))
        x.check()


@pytest.mark.parametrize("width", [1, 2, 4])
def test_paths_end_at_the_width(gpu, width):
    announce("verify width %d" % width)
    for draft in (None, F32):
        Case(5, [9, 1, 12, 20], 333, BF, True, draft, width=width, peak=6.0).check()


def test_more_new_tokens_than_said(gpu):
    announce("verify max_new")
    Case(5, [9, 3, 12], 333, BF, True, None, max_new=4, width=12).check()


def test_long_chain(gpu):
    """1024 rows, all accepted; and one of 1000 that is refused at the end."""
    announce("verify long")
    x = Case(2, [1024, 1000], 50, F32, peak=30.0)
    x.u.fill_(0.0)
    x.u[1024 + 999] = 1 - 2 ** -24
    x.tokens[1024 + 999] = int(x.x[1024 + 998].argmin())
    assert x.check() == 1024 + 999


def test_nothing_to_verify(gpu):
    announce("verify nothing")
    x = Case(1, [0, 0], 40)
    assert x.run() == ([[-1], [-1]], [0, 0], [-1, -1])
    x = Case(1, [], 40, spare_rows=2)
    assert x.run() == ([], [], [])


@pytest.mark.parametrize("draft", [None, F32])
@pytest.mark.parametrize("tree", [False, True])
def test_starts_that_do_not_ascend(gpu, draft, tree):
    """Sequences that claim each other's rows: nothing is read or written outside, what
    is no walk is none, and the counters serve the next call."""
    announce("verify starts %s %s" % (draft, tree))
    x = Case(6, [5, 7, 4, 6], 5000, F32, tree, draft)
    good = x.run()
    x.check()
    n = len(x.news)
    seqs = ops.make_seqs(torch.zeros(n, 1, dtype=torch.int32, device="cuda"), ints([3] * n), ints([0, 9, 3, 40, -5]), 8)
    path, lens, nxt = torch.empty(n, 7, dtype=torch.int32, device="cuda"), ints([9] * n), ints([9] * n, torch.int64)
    nbytes, ncnt = ops.verify_drafts_workspace(seqs, x.x, draft=x.draft)
    ws, cnt = torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda"), torch.zeros(ncnt, dtype=torch.int32, device="cuda")

    def call(s, p):
        ops.verify_drafts(s, x.x, x.tokens, x.u, x.u_next, p, lens, nxt, ws, cnt, parents=x.parents, draft=x.draft,
                          temperature=torch.tensor(x.temps, device="cuda"))

    for _ in range(2):
        call(seqs, path)
        assert not bool(cnt.any())
        # (rows 0 to 7 are the first's; the second has none, the third's are the first's in part)
        assert lens[0] >= 1 and lens[1].item() == 0 and lens[3].item() == 0
        assert path[1].tolist() == [-1] * 7 and nxt[1].item() == -1 and nxt[3].item() == -1
        wide = torch.empty(n, x.width, dtype=torch.int32, device="cuda")
        call(x.handle(), wide)
        assert (wide.tolist(), lens.tolist(), nxt.tolist()) == good


@pytest.mark.parametrize("draft", [None, BF])
def test_many_sequences(gpu, draft):
    announce("verify many")
    news = [(i * 7) % 6 for i in range(150)]
    x = Case(3, news, 4099, HF, True, draft, temps=(1.0, 0.0, 0.5))
    x.check()


def test_captured_and_two_at_once(gpu):
    """A captured call replayed over other drafts, and calls on two streams with a
    workspace each."""
    announce("verify captured")
    x = Case(4, [5, 9, 1], 9000, BF, True, F32)
    seqs = x.handle()
    nbytes, ncnt = ops.verify_drafts_workspace(seqs, x.x, draft=x.draft)
    outs = [(torch.empty(3, 9, dtype=torch.int32, device="cuda"), ints([0] * 3), ints([0] * 3, torch.int64),
             torch.empty(nbytes, dtype=torch.uint8, device="cuda"), torch.zeros(ncnt, dtype=torch.int32, device="cuda"))
            for _ in range(2)]

    def call(o, stream=None):
        ops.verify_drafts(seqs, x.x, x.tokens, x.u, x.u_next, *o, parents=x.parents, draft=x.draft, stream=stream)

    call(outs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(outs[0])
    for seed in range(4):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x.x.copy_(torch.randn(x.x.shape, device="cuda", generator=g) * 3)
        x.u.copy_(torch.rand(x.u.shape, device="cuda", generator=g))
        x.u_next.copy_(torch.rand(3, device="cuda", generator=g))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for o, s in zip(outs, streams):
            call(o, s)
        torch.cuda.synchronize()
        want = x.run()
        for o in outs:
            assert tuple(t.tolist() for t in o[:3]) == want
        for t in outs[0][:3]:
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert tuple(t.tolist() for t in outs[0][:3]) == want
        x.temps = [1.0] * 3
        x.check()


def test_sums_at_several_rows(gpu):
    """Sampled trees whose walks refuse drafts at one row, accept a later one there and
    refuse again further down: the sums of both rows, made and known ones."""
    announce("verify sums at several rows")
    n, V = 85, 9001
    x = Case(11, [n] * 24, V, F32, True, F32, temps=(1.0, 0.8), peak=1.5)
    x.par = [[(i - 1) // 4 if i else -1 for i in range(n)] for _ in x.news]
    x.parents = ints([p for s in x.par for p in s])
    above = ints([b * n + max(p, 0) for b, s in enumerate(x.par) for p in s], torch.int64)
    # half of it the target's own opinion, half another's
    t = torch.tensor(x.temps, device="cuda").repeat_interleave(n)[:, None]
    other = torch.randn(x.x.shape, device="cuda", generator=x.g) * 1.5
    x.draft.copy_((torch.softmax(x.x / t, 1) + torch.softmax(other, 1)) / 2)
    x.tokens = (x.draft[above] / -torch.rand(x.x.shape, device="cuda", generator=x.g).clamp(min=1e-30).log()).argmax(1)
    x.check()
    paths, _, _ = x.run()
    later = [sum((c - 1) % 4 > 0 for c in p if c > 0) for p in paths]  # rows where another child than the first was accepted
    assert max(later) >= 2 and sum(k >= 2 for k in later) >= 3, later
