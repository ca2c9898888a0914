"""The paged cache's kernels against float64.

Tolerances. u is half a step of the type (2^-8 bf16, 2^-11 fp16).
* q/k norm + rotation: one rounding, u |y|, plus fp32 arithmetic: the norm's
  sum, root and division and two products are below 2^-20 of each of the two
  terms n1 c, n2 s; fp16 results below its normal range step by 2^-24.
* attention: the weights are rounded to the type before they meet v and the
  result once: u (A + |o|), A = sum p |v| / sum p. A score is an fp32 sum of D
  products, scaled: off by at most dS = (D + 8) 2^-24 scale max_j sum |q k|,
  and so is its weight, relatively (twice: above and below the bar); the
  exponent's argument and the hardware's 2^x add less than 2^-18.
* copies: bit for bit.
"""

import random

import pytest
import torch

from kernrelay_amd import kvcache, ops
from tests.conftest import announce

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
HALF = {BF: 2.0 ** -8, HF: 2.0 ** -11}


def ints(v, dt=torch.int32):
    return torch.tensor(v, dtype=dt, device="cuda")


def normal(gen, *shape, dt=BF, std=1.0, mean=0.0):
    return (torch.randn(*shape, device="cuda", generator=gen) * std + mean).to(dt)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------- q/k norm + rotation
def tables(n, D, dt, g):
    a = torch.rand(n, D, device="cuda", generator=g, dtype=torch.float64) * 6.28
    return a.cos().to(dt), a.sin().to(dt)


def rope_terms(x, gamma, c, s, eps):
    x = x.double()
    if gamma is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * gamma.double()
    h = x.shape[-1] // 2
    turned = torch.cat((-x[..., h:], x[..., :h]), -1)
    a, b = x * c.double()[:, None], turned * s.double()[:, None]
    return a + b, a.abs() + b.abs()


def check_rope(y, x, gamma, c, s, eps=1e-6):
    ref, mag = rope_terms(x, gamma, c, s, eps)
    bound = HALF[y.dtype] * ref.abs() * 1.01 + 2.0 ** -20 * mag + (2.0 ** -25 if y.dtype == HF else 0.0)
    assert bool(((y.double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("D,dt,tdt,norm", [(64, BF, BF, True), (128, HF, torch.float32, True), (128, BF, BF, False),
                                           (256, HF, HF, True), (256, BF, torch.float32, False)])
@pytest.mark.parametrize("rows,HQ,HKV", [(1, 4, 4), (37, 14, 2), (130, 7, 1)])
def test_qk_norm_rope(gpu, rows, HQ, HKV, D, dt, tdt, norm):
    announce("qk_norm_rope %s" % ((rows, HQ, HKV, D, dt, tdt, norm),))
    g = gen(rows + D)
    qkv = normal(g, rows, (HQ + 2 * HKV) * D + 8, dt=dt)  # q and k as views of a wider row
    q, k = qkv[:, :HQ * D].view(rows, HQ, D), qkv[:, HQ * D:(HQ + HKV) * D].view(rows, HKV, D)
    c, s = tables(200, D, tdt, g)
    gains = [normal(g, D, dt=dt, std=0.3, mean=1.0) for _ in range(2)] if norm else [None, None]
    pos = torch.randint(0, 200, (rows,), device="cuda", generator=g)
    pad = torch.full((rows + 2, HQ * D + 16), 7.0, dtype=dt, device="cuda")
    qo, ko = pad[:rows, :HQ * D].view(rows, HQ, D), torch.empty(rows, HKV, D, dtype=dt, device="cuda")
    rope = ops.make_rope(c, s, *gains, eps=1e-5)
    ops.qk_norm_rope(rope, q, k, qo, ko, positions=pos)
    check_rope(qo, q, gains[0], c[pos], s[pos], 1e-5)
    check_rope(ko, k, gains[1], c[pos], s[pos], 1e-5)
    assert torch.all(pad[rows:] == 7.0) and torch.all(pad[:, HQ * D:] == 7.0)
    # in place, and rows at their own index
    q2, k2 = q.clone(), k.clone()
    ops.qk_norm_rope(rope, q2, k2, q2, k2)
    check_rope(q2, q, gains[0], c[:rows], s[:rows], 1e-5)
    check_rope(k2, k, gains[1], c[:rows], s[:rows], 1e-5)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dt", [BF, HF])
def test_chain_has_the_separate_calls_bits(gpu, D, dt):
    announce("qk_norm_rope chain %d %s" % (D, dt))
    g, rows, HQ, HKV = gen(D), 211, 6, 2
    q, k = normal(g, rows, HQ, D, dt=dt), normal(g, rows, HKV, D, dt=dt)
    c, s = tables(rows, D, dt, g)
    gq, gk = (normal(g, D, dt=dt, std=0.1, mean=1.0) for _ in range(2))
    want = []
    for x, w in ((q, gq), (k, gk)):
        y = torch.empty_like(x)
        ops.rowop("rmsnorm", x.view(-1, D), y.view(-1, D), gamma=w)
        ops.rope(y, rows, x.shape[1], D, c, s)
        want.append(y)
    got = torch.empty_like(q), torch.empty_like(k)
    ops.qk_norm_rope(ops.make_rope(c, s, gq, gk, chain=True), q, k, *got)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for x, y in ((q, torch.empty_like(q)), (k, torch.empty_like(k))):  # no norm: the rotation alone
        want = x.clone()
        ops.rope(want, rows, x.shape[1], D, c, s)
        ops.qk_norm_rope(ops.make_rope(c, s, chain=True), x, k, y, torch.empty_like(k))
        assert torch.equal(y, want)


def test_rope_strange_rows(gpu):
    """Zero rows, huge rows, and positions outside the tables."""
    announce("qk_norm_rope strange rows")
    g, D = gen(5), 128
    q, k = normal(g, 5, 2, D), normal(g, 5, 1, D)
    q[0] = 0.0
    q[1] *= 2.0 ** 40
    k[2] *= 2.0 ** -60
    c, s = tables(9, D, torch.float32, g)
    gq, gk = normal(g, D, std=0.1, mean=1.0), normal(g, D, std=0.1, mean=1.0)
    pos = ints([0, 8, 3, 9, -1], torch.int64)
    qo, ko = torch.full_like(q, 3.0), torch.full_like(k, 3.0)
    ops.qk_norm_rope(ops.make_rope(c, s, gq, gk), q, k, qo, ko, positions=pos)
    check_rope(qo[:3], q[:3], gq, c[pos[:3]], s[pos[:3]])
    check_rope(ko[:3], k[:3], gk, c[pos[:3]], s[pos[:3]])
    assert torch.all(qo[3:] == 0.0) and torch.all(ko[3:] == 0.0) and torch.all(qo[0] == 0.0)


@pytest.mark.parametrize("layout", ["tokens", "heads", "inside"])
@pytest.mark.parametrize("page,D,dt,rows", [(1, 64, BF, 5), (24, 128, HF, 61), (16, 128, BF, 300)])
def test_rope_cache(gpu, page, D, dt, rows, layout):
    announce("qk_norm_rope_cache %s" % ((page, D, dt, rows, layout),))
    g, HQ, HKV, layers = gen(page), 6, 3, 2
    pages = rows // page + 3
    k_cache, v_cache = (paged_tensor(layers, pages, page, HKV, D, dt, layout) for _ in range(2))
    before = k_cache.clone(), v_cache.clone()
    qkv = normal(g, rows, HQ + 2 * HKV, D, dt=dt)
    q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:]
    c, s = tables(400, D, dt, g)
    gq, gk = (normal(g, D, dt=dt, std=0.1, mean=1.0) for _ in range(2))
    pos = torch.randint(0, 400, (rows,), device="cuda", generator=g)
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:rows]
    slots[rows // 2] = -1
    slots[rows // 3] = pages * page
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    ops.qk_norm_rope_cache(ops.make_rope(c, s, gq, gk), ops.make_cache(k_cache, v_cache), 1, q, k, v, qo, pos, slots)
    check_rope(qo, q, gq, c[pos], s[pos])
    there = (slots >= 0) & (slots < pages * page)
    at = slots[there] // page, slots[there] % page
    check_rope(k_cache[1][at], k[there], gk, c[pos[there]], s[pos[there]])
    assert torch.equal(v_cache[1][at], v[there])
    k_cache[1][at] = before[0][1][at]  # all else is as it was
    v_cache[1][at] = before[1][1][at]
    for now, was in zip((k_cache, v_cache), before):
        assert torch.equal(now.contiguous().view(torch.int16), was.contiguous().view(torch.int16))


# ------------------------------------------------------------------ attention
def paged_tensor(layers, pages, page, HKV, D, dt, layout):
    """A cache full of NaN: what nobody wrote must reach nobody."""
    full = lambda *s: torch.full(s, float("nan"), dtype=dt, device="cuda")  # noqa: E731
    if layout == "heads":
        return full(layers, pages, HKV, page, D).transpose(2, 3)
    if layout == "inside":  # k and v rows side by side, pages of a larger pool
        return full(layers, pages + 1, page + 2, HKV + 1, D + 8)[:, 1:, 1:-1, :HKV, :D]
    return full(layers, pages, page, HKV, D)


class Batch:
    """Sequences of `lens` cached and `news` new tokens on pages in random
    order, the rest of the cache NaN."""

    def __init__(self, seed, HQ, HKV, D, dt, page, lens, news, form="causal", layout="tokens", gap=0, words=None,
                 spare=0):
        self.g, self.rng = gen(seed), random.Random(seed)
        self.HQ, self.HKV, self.D, self.dt, self.page, self.lens, self.news = HQ, HKV, D, dt, page, lens, news
        need = [-(-(a + b) // page) for a, b in zip(lens, news)]
        self.pages = sum(need) + 2
        order = list(range(self.pages))
        self.rng.shuffle(order)
        width = max(need + [1]) + spare
        self.table, at = [], 0
        for n in need:
            self.table.append(order[at:at + n] + [-1] * (width - n))
            at += n
        self.k, self.v = (paged_tensor(2, self.pages, page, HKV, D, dt, layout) for _ in range(2))
        self.starts = [gap]
        for n in news:
            self.starts.append(self.starts[-1] + n)
        self.rows = self.starts[-1] + gap
        self.seen = []  # per row of the launch: which new tokens it sees
        for n in news:
            for i in range(n):
                if form == "causal":
                    self.seen.append([j <= i for j in range(n)])
                elif form == "none":
                    self.seen.append([False] * n)
                else:
                    self.seen.append([j == i or self.rng.random() < 0.4 for j in range(n)])
        for b, (a, n) in enumerate(zip(lens, news)):
            ids = ints(self.table[b][:need[b]], torch.int64)
            for cache in (self.k, self.v):
                rows = torch.full((need[b] * page, HKV, D), float("nan"), dtype=dt, device="cuda")
                rows[:a + n] = normal(self.g, a + n, HKV, D, dt=dt)
                cache[1][ids] = rows.view(need[b], page, HKV, D)
        tree = None
        if form != "causal":
            words = words or max(1, -(-max(news) // 64))
            tree = torch.zeros(self.rows, words, dtype=torch.int64)
            for r, see in enumerate(self.seen):
                for j, x in enumerate(see):
                    if x:
                        tree[gap + r, j // 64] |= (1 << (j % 64)) - ((1 << 64) if j % 64 == 63 else 0)
            tree = tree.cuda()
        self.tree = tree
        self.q = normal(self.g, self.rows, HQ, D, dt=dt)
        self.cache = ops.make_cache(self.k, self.v)
        self.dev = [ints(self.table).view(len(lens), width), ints(self.lens), ints(self.starts)]
        self.seqs = ops.make_seqs(*self.dev, max(news, default=0), tree=tree)

    def space(self):
        nbytes, ncnt = ops.attention_paged_workspace(self.cache, self.seqs, self.HQ)
        return dict(ws=torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda"),
                    counters=torch.zeros(ncnt, dtype=torch.int32, device="cuda"))

    def run(self, scale=None, cut=True, **kw):
        out = torch.full_like(self.q, 9.0)
        ops.attention_paged(self.cache, 1, self.seqs, self.q, out, scale=scale, **(self.space() if cut else {}), **kw)
        return out

    def check(self, out, scale=None, usable=None):
        scale = self.D ** -0.5 if scale is None else scale
        G, u, r = self.HQ // self.HKV, HALF[self.dt], 0
        for b, (a, n) in enumerate(zip(self.lens, self.news)):
            if n == 0:
                continue
            lo = self.starts[b]
            ids = ints([p if 0 <= p < self.pages else 0 for p in self.table[b][:-(-(a + n) // self.page)]], torch.int64)
            k, v = (c[1][ids].reshape(-1, self.HKV, self.D)[:a + n].double().permute(1, 0, 2) for c in (self.k, self.v))
            sees = torch.ones(n, a + n, dtype=torch.bool)
            sees[:, a:] = torch.tensor(self.seen[r:r + n])
            r += n
            for j in range(a + n):
                if not 0 <= self.table[b][j // self.page] < self.pages:
                    sees[:, j] = False
            sees = sees.cuda()
            k, v = k.nan_to_num(0.0, 0.0, 0.0), v
            q = self.q[lo:lo + n].double().view(n, self.HKV, G, self.D).permute(1, 2, 0, 3)  # [HKV, G, n, D]
            s = torch.matmul(q, k[:, None].transpose(2, 3)) * scale
            dS = (self.D + 8) * 2.0 ** -24 * scale * torch.matmul(q.abs(), k[:, None].abs().transpose(2, 3)).amax(-1)
            s = s.masked_fill(~sees, float("-inf"))
            top = s.amax(-1, keepdim=True)
            p = (s - top.masked_fill(top == float("-inf"), 0.0)).exp()
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            clean = v[:, None].nan_to_num(0.0, 0.0, 0.0)
            ref, A = torch.matmul(p, clean), torch.matmul(p, clean.abs())
            # a row that sees a value that is no number has it; the others do not
            special = (~v.isfinite()).any(-1)
            for h in range(self.HKV):
                for j in special[h].nonzero().flatten().tolist():
                    extra = sees[:, j].double()[None, :, None] * torch.where(v[h, j].isfinite(), 0.0, v[h, j])
                    ref[h] = torch.where(sees[:, j][None, :, None], ref[h] + extra, ref[h])
            bound = u * (A + ref.abs()) * 1.01 + A * (2 * dS[..., None] + 2.0 ** -18)
            bound = bound + (2.0 ** -24 if self.dt == HF else 0.0)
            got = out[lo:lo + n].double().view(n, self.HKV, G, self.D).permute(1, 2, 0, 3)
            fine = ref.isfinite()
            assert bool(((got - ref).abs() <= bound)[fine].all()), "sequence %d off by %g of the bound" % (
                b, float(((got - ref).abs() / bound)[fine].max()))
            assert torch.equal(got[~fine].isnan(), ref[~fine].isnan())
            assert torch.equal(got[~fine].nan_to_num(0.0), ref[~fine].nan_to_num(0.0))
        assert torch.all(out[:self.starts[0]] == 9.0) and torch.all(out[self.starts[-1]:] == 9.0)


STEPS = [(14, 2, 64, BF, 16, [37], [1]), (28, 4, 128, BF, 16, [0, 1, 63, 64, 65, 700], [1] * 6),
         (32, 8, 128, HF, 24, [5000, 31], [1, 1]), (8, 8, 64, HF, 7, [100, 257], [1, 1]),
         (40, 1, 128, BF, 64, [333, 20], [1, 1]), (28, 4, 128, BF, 1, [150], [1]),
         (12, 4, 64, BF, 128, [20000, 0, 3, 9000], [1, 1, 1, 1])]


@pytest.mark.parametrize("HQ,HKV,D,dt,page,lens,news", STEPS)
@pytest.mark.parametrize("cut", [True, False])
def test_attention_step(gpu, HQ, HKV, D, dt, page, lens, news, cut):
    announce("attention_paged step %s" % ((HQ, HKV, D, dt, page, lens, cut),))
    b = Batch(1, HQ, HKV, D, dt, page, lens, news)
    b.check(b.run(cut=cut))


MANY = [(28, 4, 128, BF, 16, [40, 1000, 0], [16, 5, 9]), (32, 8, 128, HF, 24, [2900, 77, 64], [61, 64, 1]),
        (14, 2, 64, BF, 8, [130, 0], [100, 130]), (4, 4, 128, BF, 32, [33, 95, 0, 200], [32, 0, 33, 2]),
        (16, 2, 64, HF, 5, [3000], [8]), (20, 4, 128, HF, 48, [1, 127, 128, 129], [12, 13, 6, 7])]


@pytest.mark.parametrize("form", ["causal", "tree"])
@pytest.mark.parametrize("HQ,HKV,D,dt,page,lens,news", MANY)
def test_attention_trees_and_chunks(gpu, HQ, HKV, D, dt, page, lens, news, form):
    announce("attention_paged %s %s" % (form, (HQ, HKV, D, dt, page, lens, news)))
    b = Batch(2, HQ, HKV, D, dt, page, lens, news, form=form, gap=3)
    b.check(b.run())
    b.check(b.run(cut=False))


@pytest.mark.parametrize("lens,news", [([600], [700]), ([0, 300], [513, 90])])
def test_attention_long_chunks(gpu, lens, news):
    announce("attention_paged chunk %s %s" % (lens, news))
    b = Batch(3, 14, 2, 64, BF, 16, lens, news)
    b.check(b.run())
    b = Batch(3, 7, 1, 128, HF, 40, lens, news)
    b.check(b.run())


@pytest.mark.parametrize("D,HQ,HKV,dt", [(128, 28, 4, BF), (64, 14, 2, HF)])
@pytest.mark.parametrize("most", [1, 9, 17])
def test_attention_uneven_batches(gpu, most, D, HQ, HKV, dt):
    """One long sequence among many short ones, some without new tokens, in 32,
    64 and 128 packed rows: its units are cut though there are hundreds; every
    call leaves the counters zero and gives the same bits."""
    announce("attention_paged uneven %s" % ((most, D, HQ, HKV, dt),))
    rng = random.Random(most)
    n = 400 // HKV
    lens = [rng.randint(0, 40) for _ in range(n)]
    lens[n // 3] = 9000
    news = [rng.choice((0, 1, most, most)) for _ in range(n)]
    news[n // 3] = most
    b = Batch(15, HQ, HKV, D, dt, 16, lens, news, form="causal" if most == 1 else "tree")
    sp = b.space()
    assert sp["counters"].numel() > 0
    outs = []
    for _ in range(3):
        out = torch.full_like(b.q, 9.0)
        ops.attention_paged(b.cache, 1, b.seqs, b.q, out, **sp)
        outs.append(out)
    b.check(outs[0])
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    assert int(sp["counters"].abs().sum()) == 0
    b.check(b.run(cut=False))


@pytest.mark.parametrize("D,HQ,HKV,dt", [(128, 28, 4, HF), (64, 14, 2, BF)])
@pytest.mark.parametrize("longest", [30000, 300])
def test_attention_one_unit_per_cu(gpu, longest, D, HQ, HKV, dt):
    """As many units of few rows as the device has CUs, one long sequence among
    them (cut) or none (whole)."""
    announce("attention_paged one unit per cu %s" % ((longest, D, HQ, HKV, dt),))
    rng = random.Random(longest)
    n = 240 // HKV
    lens = [rng.randint(0, 300) for _ in range(n)]
    lens[7] = longest
    b = Batch(16, HQ, HKV, D, dt, 24, lens, [1] * n)
    b.check(b.run())
    assert torch.equal(b.run(), b.run())
    b.check(b.run(cut=False))


@pytest.mark.parametrize("lens,news", [([3000, 10, 5, 0], [40, 20, 0, 7]), ([2000, 0, 30], [1, 0, 1]),
                                       ([0, 1800, 64, 9], [9, 15, 0, 2])])
def test_attention_workspace_may_hold_anything(gpu, lens, news):
    """Fewer units than the handles allow for, on a workspace that reads as notes
    of cut units (each number 2: all inside the tensors, of a row that belongs
    to no sequence): they have no part, and that row stays as it was."""
    announce("attention_paged old workspace %s" % ((lens, news),))
    b = Batch(17, 8, 2, 128, BF, 16, lens, news, gap=3)
    sp = b.space()
    assert sp["ws"].numel() > 0
    for _ in range(2):
        sp["ws"].view(torch.int32).fill_(2)
        out = torch.full_like(b.q, 9.0)
        ops.attention_paged(b.cache, 1, b.seqs, b.q, out, **sp)
        b.check(out)


@pytest.mark.parametrize("layout", ["heads", "inside"])
def test_attention_layouts(gpu, layout):
    announce("attention_paged layout " + layout)
    for D, HQ, HKV, news in ((128, 8, 2, [1, 1]), (64, 12, 3, [30, 9])):
        b = Batch(4, HQ, HKV, D, BF, 24, [300, 71], news, form="tree", layout=layout, words=3, spare=2)
        b.check(b.run())


def test_attention_strided_rows(gpu):
    announce("attention_paged strided rows")
    b = Batch(5, 8, 2, 128, BF, 16, [90, 40], [7, 3])
    wide = torch.zeros(b.rows, 8 * 128 + 64, dtype=BF, device="cuda")
    q = wide[:, 64:].view(b.rows, 8, 128)
    q.copy_(b.q)
    pad = torch.full((b.rows, 8 * 128 + 8), 9.0, dtype=BF, device="cuda")
    out = pad[:, :1024].view(b.rows, 8, 128)
    ops.attention_paged(b.cache, 1, b.seqs, q, out, **b.space())
    b.check(out)
    assert torch.all(pad[:, 1024:] == 9.0)
    assert torch.equal(out, b.run())


def test_rows_that_see_nothing(gpu):
    """No cached token and an empty mask: zeros, whatever the cache holds."""
    announce("attention_paged empty rows")
    for news in ([1, 1], [40, 3]):
        b = Batch(6, 8, 2, 128, BF, 16, [0, 20], news, form="none")
        out = b.run()
        assert torch.all(out[:news[0]] == 0.0)
        b.check(out)
    b = Batch(6, 8, 2, 128, BF, 16, [70, 20], [1, 1])
    b.table[0] = [-1, b.pages, -7, 1 << 30, -1]  # no page at all
    b.dev[0].copy_(ints([r + [-1] * (b.dev[0].shape[1] - len(r)) for r in b.table]))
    out = b.run()
    assert torch.all(out[0] == 0.0)
    b.check(out)


@pytest.mark.parametrize("bad", [-1, 1 << 20])
def test_keys_of_bad_pages_are_seen_by_nobody(gpu, bad):
    announce("attention_paged bad pages %d" % bad)
    for news in ([1, 1], [21, 8]):
        b = Batch(7, 8, 2, 128, BF, 24, [500, 200], news)
        b.table[0][3] = bad
        b.table[1][0] = bad
        b.dev[0].copy_(ints(b.table))
        b.check(b.run())


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("D", [64, 128])
def test_hidden_values_have_no_part(gpu, value, D):
    """Drafts whose keys or values are no numbers: the rows that do not see them
    are as they would be without, and those that do have them."""
    announce("attention_paged hidden %s D=%d" % (value, D))
    for HQ, HKV, news in ((4, 2, [9, 5]), (8, 2, [40, 12])):
        b = Batch(8, HQ, HKV, D, BF, 16, [50, 0], news, form="tree")
        for s, j, cols in ((0, 4, slice(0, 3)), (0, 7, slice(D - 1, D)), (1, 3, slice(0, D))):
            pos = b.lens[s] + j
            b.v[1, b.table[s][pos // 16], pos % 16, 1, cols] = value
        b.check(b.run())
        # a key that nobody but its own row sees
        row = sum(b.news[:1]) + 1
        for r in range(b.starts[1], b.starts[2]):
            b.seen[r][1] = r == row
        b2 = b
        t = b2.tree.cpu()
        for r in range(b.starts[1], b.starts[2]):
            t[r, 0] = (int(t[r, 0]) & ~2) | (2 if r == row else 0)
        b2.tree.copy_(t)
        pos = b.lens[1] + 1
        b2.k[1, b.table[1][pos // 16], pos % 16, :] = value
        out, ref = b2.run(), b2
        keep = [r for r in range(b.rows) if r != row]
        b2.k[1, b.table[1][pos // 16], pos % 16, :] = 0.0
        clean = ref.run()
        assert torch.equal(out[keep].view(torch.int16), clean[keep].view(torch.int16))


def test_scores_far_apart(gpu):
    """Large scores: the running maximum moves, small weights vanish, none overflow."""
    announce("attention_paged large scores")
    for news in ([1], [33]):
        b = Batch(9, 8, 2, 128, BF, 16, [900], news)
        b.k[1].mul_(torch.linspace(0.1, 12.0, b.pages, device="cuda", dtype=BF)[:, None, None, None])
        b.check(b.run(scale=0.5), scale=0.5)
        b.check(b.run(scale=2.0 ** -30), scale=2.0 ** -30)


def test_device_arrays_that_lead_outside(gpu):
    """Lengths, starts and tokens past the handle's bounds end at the bounds."""
    announce("attention_paged clamps")
    b = Batch(10, 8, 2, 128, BF, 16, [40, 40], [4, 4])
    want = b.run()
    b.dev[2].copy_(ints([0, 4, 1000]))  # rows that the launch does not have
    assert torch.equal(b.run(), want)
    b.dev[2].copy_(ints([-5, -2, 3]))   # negative starts
    out = b.run()
    assert torch.all(out[3:] == 9.0)
    b.dev[2].copy_(ints([0, 4, 8]))
    b.dev[1].copy_(ints([-3, 1 << 30]))  # a negative length counts as none; one past the table ends with it
    out = b.run()
    b.dev[1].copy_(ints([0, 40]))
    assert torch.equal(out[:4], b.run()[:4]) and bool(out[:4].isfinite().all())


@pytest.mark.parametrize("news,most", [([3, 2], 1), ([40, 20], 17)])
def test_new_tokens_past_max_new_are_not_worked(gpu, news, most):
    """The first max_new tokens of a sequence are as in a launch of theirs, and
    the rows behind them as they were."""
    announce("attention_paged past max_new %s %d" % (news, most))
    b = Batch(18, 8, 2, 128, HF, 16, [100, 30], news)
    seqs, out = ops.make_seqs(*b.dev, most), torch.full_like(b.q, 9.0)
    ops.attention_paged(b.cache, 1, seqs, b.q, out)
    for s, n in enumerate(news):
        lo, n = b.starts[s], min(n, most)
        assert torch.all(out[lo + n:b.starts[s + 1]] == 9.0)
        alone = torch.full_like(b.q, 9.0)
        starts = ints([lo if i <= s else lo + n for i in range(3)])
        ops.attention_paged(b.cache, 1, ops.make_seqs(b.dev[0], b.dev[1], starts, most), b.q, alone)
        assert torch.equal(out[lo:lo + n], alone[lo:lo + n])
        assert torch.all(alone[:lo] == 9.0) and torch.all(alone[lo + n:] == 9.0)


def test_far_pages(gpu):
    """Offsets past 2^31 elements within a layer, and past 2^32 over the layers."""
    announce("attention_paged far pages")
    g, HKV, D, page = gen(11), 8, 128, 64
    pages = (1 << 31) // (page * HKV * D) + 40
    k, v = (torch.empty(2, pages, page, HKV, D, dtype=BF, device="cuda") for _ in range(2))
    ids = [pages - 1, 3, pages - 20, pages - 2]
    for c in (k, v):
        c[1, ints(ids, torch.int64)] = normal(g, 4, page, HKV, D)
    L = 200
    cache = ops.make_cache(k, v)
    seqs = ops.make_seqs(ints([ids]), ints([L]), ints([0, 2]), 2)
    q, out = normal(g, 2, 8, D), torch.empty(2, 8, D, dtype=BF, device="cuda")
    ops.attention_paged(cache, 1, seqs, q, out)
    small_k, small_v = (c[1:, ints(ids, torch.int64)].contiguous() for c in (k, v))
    near, want = ops.make_cache(small_k, small_v), torch.empty_like(out)
    ops.attention_paged(near, 0, ops.make_seqs(ints([[0, 1, 2, 3]]), ints([L]), ints([0, 2]), 2), q, want)
    assert torch.equal(out, want)
    # writes and copies there too
    slots = ints([(pages - 1) * page + 5, (pages - 20) * page + 63], torch.int64)
    kk, vv = normal(g, 2, HKV, D), normal(g, 2, HKV, D)
    c, s = tables(4, D, BF, g)
    ops.qk_norm_rope_cache(ops.make_rope(c, s), cache, 1, q, kk, vv, out, None, slots)
    assert torch.equal(v[1, pages - 1, 5], vv[0]) and torch.equal(v[1, pages - 20, 63], vv[1])
    ops.cache_copy_pages(cache, [pages - 1], [pages - 30])
    assert torch.equal(k[1, pages - 30], k[1, pages - 1]) and torch.equal(v[1, pages - 30], v[1, pages - 1])


def test_replayed_graph_follows_its_arrays(gpu):
    """Captured once, replayed with other lengths, pages and starts between
    eager calls; each replay has the eager call's bits."""
    announce("attention_paged graph")
    for news in ([1, 1, 1], [20, 3, 11]):
        b = Batch(12, 28, 4, 128, BF, 16, [700, 90, 2000], news, spare=3)
        sp, out = b.space(), torch.full_like(b.q, 9.0)
        call = lambda: ops.attention_paged(b.cache, 1, b.seqs, b.q, out, **sp)  # noqa: E731
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        for lens in ([700, 90, 2000], [3, 80, 1500], [650, 0, 2], [700, 90, 2000]):
            b.lens = lens
            b.dev[1].copy_(ints(lens))
            out.fill_(9.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, b.run())
            assert int(sp["counters"].abs().sum()) == 0


def test_two_calls_side_by_side(gpu):
    """Two streams, a workspace each, many times over: the bits of one alone."""
    announce("attention_paged two streams")
    a = Batch(13, 28, 4, 128, BF, 16, [3000, 500], [1, 1])
    b = Batch(14, 32, 8, 128, HF, 24, [1500, 2500], [17, 40], form="tree")
    want = a.run(), b.run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(x.q) for x in (a, b)]
    spaces = [x.space() for x in (a, b)]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, st, o, sp in zip((a, b), streams, outs, spaces):
            ops.attention_paged(x.cache, 1, x.seqs, x.q, o, stream=st, **sp)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


# ---------------------------------------------------------- copies, compaction
@pytest.mark.parametrize("layout", ["tokens", "heads", "inside"])
@pytest.mark.parametrize("page,HKV,D,n", [(16, 4, 128, 3), (1, 1, 64, 9), (24, 2, 64, 500), (7, 3, 128, 40)])
def test_copy_pages(gpu, page, HKV, D, n, layout):
    announce("cache_copy_pages %s" % ((page, HKV, D, n, layout),))
    rng, pages, layers = random.Random(n), 2 * n + 3, 3
    k, v = (paged_tensor(layers, pages, page, HKV, D, BF, layout) for _ in range(2))
    k.copy_(normal(gen(1), *k.shape))
    v.copy_(normal(gen(2), *v.shape))
    ids = rng.sample(range(pages), 2 * n)
    src, dst = ids[:n], ids[n:]
    src[-1] = src[0]  # one page may be copied more than once
    want = [c.clone() for c in (k, v)]
    for w in want:
        w[:, ints(dst, torch.int64)] = w[:, ints(src, torch.int64)]
    ops.cache_copy_pages(ops.make_cache(k, v), src, dst)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    if layout == "inside":  # nothing beside the pages
        assert torch.all(torch.isnan(k._base[:, 0])) and torch.all(torch.isnan(k._base[..., D:]))


@pytest.mark.parametrize("width", [1, 8, 13, 40, 200])
@pytest.mark.parametrize("page,HKV,D,layout", [(16, 4, 128, "tokens"), (5, 3, 64, "heads"), (24, 1, 128, "inside")])
def test_compact(gpu, page, HKV, D, layout, width):
    announce("cache_compact %s" % ((page, HKV, D, layout, width),))
    rng, layers = random.Random(width), 2
    lens, drafts = [0, 37, 100], max(width, 3) + 20
    need = [-(-(a + drafts) // page) for a in lens]
    pages = sum(need) + 1
    order = rng.sample(range(pages), pages)
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (max(need) - n))
        at += n
    k, v = (paged_tensor(layers, pages, page, HKV, D, BF, layout) for _ in range(2))
    k.copy_(normal(gen(1), *k.shape))
    v.copy_(normal(gen(2), *v.shape))
    # ascending, shuffled (all are read before any is written), with a hole
    paths = [sorted(rng.sample(range(drafts), width)), rng.sample(range(drafts), width),
             [-1 if i == width // 2 else x for i, x in enumerate(sorted(rng.sample(range(drafts), width)))]]
    counts = [width, width + 5, max(0, width - 2)]
    want = [c.clone() for c in (k, v)]
    for b, a in enumerate(lens):
        for i in range(min(counts[b], width)):
            j = paths[b][i]
            if j >= 0:
                for w, c in zip(want, (k, v)):
                    w[:, table[b][(a + i) // page], (a + i) % page] = c[:, table[b][(a + j) // page], (a + j) % page]
    seqs = ops.make_seqs(ints(table), ints(lens), ints([0, 1, 2, 3]), drafts)
    ops.cache_compact(ops.make_cache(k, v), seqs, ints(paths), ints(counts))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_compact_leads_nowhere(gpu):
    """Paths off the table, pages that are none, negative counts: nothing moves."""
    announce("cache_compact bad paths")
    k, v = (normal(gen(3), 1, 6, 8, 2, 64) for _ in range(2))
    was = k.clone(), v.clone()
    seqs = ops.make_seqs(ints([[0, 1], [2, -1], [3, 99], [4, 5]]), ints([4, 4, 4, 1 << 30]), ints([0] * 5), 1)
    path = ints([[1 << 30, 12, 2147483647], [4, 5, 6], [4, 5, 9], [0, 1, 2]])
    ops.cache_compact(ops.make_cache(k, v), seqs, path, ints([3, 3, 3, 3]))
    ops.cache_compact(ops.make_cache(k, v), seqs, path.clamp(max=3), ints([-1, 0, -2147483648, 3]))
    assert torch.equal(k, was[0]) and torch.equal(v, was[1])


# ------------------------------------------------------------- all of it together
def test_drafts_forks_and_steps(gpu):
    """A small decoder's cache as a server uses it: a prompt in two chunks, a
    fork, drafted trees with some accepted, single tokens, a sequence that
    ends, a defragmented pool. Every attention is checked against the tokens
    that the sequence is known to hold, with keys and values kept beside."""
    announce("paged cache, all together")
    HQ, HKV, D, page, layers = 8, 2, 64, 8, 2
    g, rng = gen(21), random.Random(21)
    cache = kvcache.PagedCache(layers, 64, page, HKV, D, dtype=HF)
    cos, sin = tables(512, D, torch.float32, g)
    gq, gk = (normal(g, D, dt=HF, std=0.1, mean=1.0) for _ in range(2))
    rope = ops.make_rope(cos, sin, gq, gk)
    held = {}  # sequence -> per layer (k, v) rows in 64 bits

    def launch(news, seen=None, depths=None):
        """All new tokens through both layers; seen[s][i]: drafts that i sees."""
        tree = None
        if seen is not None:
            tree = ints([[sum(1 << j for j in see)] for s in news for see in seen[s]], torch.int64)
        seqs, positions, slots = cache.batch(news, tree=tree, depths=depths)
        T = sum(news.values())
        rows = {}
        for layer in range(layers):
            qkv = normal(g, T, HQ + 2 * HKV, D, dt=HF)
            q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:]
            qo, out = (torch.empty(T, HQ, D, dtype=HF, device="cuda") for _ in range(2))
            ops.qk_norm_rope_cache(rope, cache.handle, layer, q, k, v, qo, positions, slots)
            nbytes, ncnt = ops.attention_paged_workspace(cache.handle, seqs, HQ)
            ops.attention_paged(cache.handle, layer, seqs, qo, out,
                                ws=torch.empty(nbytes, dtype=torch.uint8, device="cuda"),
                                counters=torch.zeros(ncnt, dtype=torch.int32, device="cuda"))
            kr = rope_terms(k, gk, cos[positions], sin[positions], 1e-6)[0].to(HF).double()
            at = 0
            for s, n in news.items():
                old = held[s][layer]
                ks, vs = torch.cat((old[0], kr[at:at + n])), torch.cat((old[1], v[at:at + n].double()))
                L = old[0].shape[0]
                hidden = torch.ones(n, L + n, dtype=torch.bool)
                hidden[:, :L] = False
                for i in range(n):
                    hidden[i, [L + j for j in (range(i + 1) if seen is None else seen[s][i])]] = False
                for h in range(HQ):
                    a = qo[at:at + n, h].double() @ ks[:, h // 4].t() / 8.0
                    p = a.masked_fill(hidden.cuda(), float("-inf")).softmax(-1)
                    want, A = p @ vs[:, h // 4], p @ vs[:, h // 4].abs()
                    # k itself was rounded either way at a step's edge: its products move by
                    # at most 2u sum |q k| / 8 (< 2u 64 * 16 / 8: here |q k| sums stay below 60)
                    bound = HALF[HF] * (A + want.abs()) * 1.01 + A * (2 * HALF[HF] * 60 / 8 + 2.0 ** -10)
                    assert bool(((out[at:at + n, h].double() - want).abs() <= bound).all())
                rows.setdefault(s, []).append((ks[L:], vs[L:]))
                at += n
        return seqs, rows

    def keep(rows, paths):
        for s, path in paths.items():
            for layer in range(layers):
                held[s][layer] = tuple(torch.cat((o, r[list(path)])) for o, r in zip(held[s][layer], rows[s][layer]))

    def tokens(news):
        seqs, rows = launch(news)
        cache.commit(news)
        keep(rows, {s: range(n) for s, n in news.items()})

    def drafts(sizes):
        seen, depths, paths = {}, {}, {}
        for s, n in sizes.items():
            par = [-1] + [rng.randint(-1, i - 1) for i in range(1, n)]
            up = []
            for i, p in enumerate(par):
                up.append((up[p] if p >= 0 else []) + [i])
            seen[s], depths[s] = up, [len(u) - 1 for u in up]
            paths[s] = rng.choice(up)
        seqs, rows = launch(sizes, seen, depths)
        cache.accept(seqs, paths)
        keep(rows, paths)

    def add():
        s = cache.tables.add()
        held[s] = [(torch.empty(0, HKV, D, dtype=torch.float64, device="cuda"),) * 2 for _ in range(layers)]
        return s

    a, b = add(), add()
    tokens({a: 29, b: 11})
    tokens({a: 14, b: 1})
    c = cache.fork(a)
    held[c] = list(held[a])
    drafts({a: 9, b: 6, c: 12})
    tokens({a: 1, b: 1, c: 1})
    drafts({c: 30, b: 2})
    cache.free(a)
    cache.defragment()
    tokens({b: 1, c: 20})
    drafts({b: 17, c: 1})
    tokens({c: 1, b: 1})
    seqs, _, _ = cache.batch({b: 3, c: 2})
    for bad in ({c: [0], b: [1]}, {b: [1]}, {b: [3], c: []}, {b: [1, 1], c: []}, {b: [-1], c: []}):
        with pytest.raises(ValueError):
            cache.accept(seqs, bad)
    cache.accept(seqs, {b: [], c: []})
    used = sum(-(-cache.tables.tokens(s) // page) for s in (b, c))
    assert cache.tables.free_pages() == 64 - used
