"""What a program does with the paged cache after the attention of a step, as
measurable cases.

* verify: drafted tokens, a chain or a tree for each sequence, are held against
  the target's logits with given random numbers (rejection sampling): the path
  that is accepted and the token that follows it. Drafts come as they are or
  with the probabilities that they were drawn from;
* weigh: the attention weight that each cached token gets from a launch's new
  tokens, added to what it got before, key head by key head;
* evict: the tokens of a sequence that got least go, layer by layer and head by
  head, and what is left moves together, with its weights.

Head counts and vocabularies are those of the three model shapes the framework
prefills. Inputs: keys and queries N(0, 1), pages handed out in random order;
logits N(0, 1.5) under a dozen tokens that stand out, so that the first has
about half of the probability.
"""

import math
import random

import torch

own = False

# query heads, kv heads, head size, layers, vocabulary
SHAPES = {"0.5b": (14, 2, 64, 24, 151936), "7b": (28, 4, 128, 28, 152064), "8b": (32, 8, 128, 36, 151936)}
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
PEAKS = 12  # tokens that stand out in a row of logits


def listed():
    return [
        # one conversation's four drafts, taken as they are: latency
        dict(name="verify_one_0.5b_5", op="verify", vocab=151936, seqs=1, new=5, tree=False, draft="", dtype="bf16"),
        # a batch of chains that a small model drew
        dict(name="verify_sampled_7b_32x7", op="verify", vocab=152064, seqs=32, new=7, tree=False, draft="fp32",
             dtype="bf16"),
        # a batch of trees, wide logits
        dict(name="verify_tree_8b_16x24", op="verify", vocab=151936, seqs=16, new=24, tree=True, draft="",
             dtype="fp32"),
        # trees whose branches were drawn, a small odd vocabulary
        dict(name="verify_sampled_tree_6x13", op="verify", vocab=32003, seqs=6, new=13, tree=True, draft="fp32",
             dtype="fp16"),
        # the first tokens of one short conversation: latency
        dict(name="weigh_one_0.5b_37", op="weigh", model="0.5b", seqs=1, ctx=37, new=1, last=0, form="causal", page=16,
             dtype="bf16"),
        # a busy server's decoding step, lengths ragged
        dict(name="weigh_step_7b_64x4000", op="weigh", model="7b", seqs=64, ctx=4000, new=1, last=0, form="causal",
             page=16, dtype="bf16"),
        # what the last tokens of a long document look at, before most of it goes
        dict(name="weigh_window_8b_64x32000", op="weigh", model="8b", seqs=1, ctx=31500, new=500, last=64,
             form="causal", page=24, dtype="fp16"),
        # every token of a prompt's next chunk
        dict(name="weigh_chunk_7b_2048", op="weigh", model="7b", seqs=1, ctx=8000, new=2048, last=0, form="causal",
             page=32, dtype="bf16"),
        # one short conversation that just went over its budget
        dict(name="evict_one_0.5b_700", op="evict", model="0.5b", seqs=1, ctx=700, budget=512, sinks=4, recent=64,
             page=24, dtype="fp16"),
        # a batch that is trimmed every few tokens
        dict(name="evict_trim_8b_16x530", op="evict", model="8b", seqs=16, ctx=530, budget=512, sinks=4, recent=128,
             page=16, dtype="bf16"),
        # a batch of prompts cut to a third
        dict(name="evict_7b_8x3000", op="evict", model="7b", seqs=8, ctx=3000, budget=1000, sinks=4, recent=100,
             page=16, dtype="bf16"),
        # one long document cut to an eighth
        dict(name="evict_8b_1x32000", op="evict", model="8b", seqs=1, ctx=32000, budget=4000, sinks=16, recent=501,
             page=64, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("verify", "weigh", "evict"))
    model = rng.choice(tuple(SHAPES))
    page = rng.choice((8, 16, 24, 32, 64, 128))
    dtype = rng.choice(("bf16", "fp16"))
    if op == "verify":
        vocab = rng.choice((SHAPES[model][4], _log_int(rng, 1000, 152064)))
        new = _log_int(rng, 1, 40)
        draft = rng.choice(("", "", "fp32", dtype))
        rows = 384 if not draft else 200
        return dict(op=op, vocab=vocab, seqs=_log_int(rng, 1, max(1, min(64, rows // new))), new=new,
                    tree=rng.random() < 0.5, draft=draft, dtype=rng.choice((dtype, "fp32")))
    if op == "weigh":
        form = rng.choice(("causal", "causal", "tree", "path"))
        if form == "causal" and rng.random() < 0.5:
            new, seqs = _log_int(rng, 2, 1500), rng.randint(1, 2)
            ctx = _log_int(rng, 1, 8000 // seqs)
            last = rng.choice((0, _log_int(rng, 1, new)))
        else:
            new = 1 if form == "causal" else _log_int(rng, 2, 100)
            seqs = _log_int(rng, 1, 64)
            ctx = _log_int(rng, 8, (120000 if form == "causal" else 60000) // seqs)
            last = 0
        return dict(op=op, model=model, seqs=seqs, ctx=ctx, new=new, last=last, form=form, page=page, dtype=dtype)
    seqs = _log_int(rng, 1, 16)
    ctx = _log_int(rng, 64, 24000 // seqs)
    budget = _log_int(rng, 32, ctx)
    sinks = rng.randint(0, budget // 8)
    return dict(op=op, model=model, seqs=seqs, ctx=ctx, budget=budget, sinks=sinks,
                recent=rng.randint(0, budget // 2 - sinks), page=page, dtype=dtype)


# -------------------------------------------------------------------- inputs
def _normal(gen, *shape, dtype, std=1.0):
    """Large ones too: drawn in the type itself."""
    return torch.empty(*shape, device=gen.device, dtype=dtype).normal_(0.0, std, generator=gen)


def _uniform(gen, *shape):
    return torch.rand(*shape, device=gen.device, generator=gen)


def _dealt(most, n, tag):
    """n ragged sizes that the case fixes: one is `most`, the others from half of it up."""
    deal = random.Random(tag)
    return [most] + [deal.randint((most + 1) // 2, most) for _ in range(n - 1)]


def _pages(counts, page, rng, device):
    """A page table over a pool in random order; -1 behind a sequence's last page."""
    need = [(n + page - 1) // page for n in counts]
    total = sum(need) + 2
    order = list(range(total))
    rng.shuffle(order)
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (max(need) - n))
        at += n
    return torch.tensor(table, dtype=torch.int32, device=device), total


def _parents(n, rng):
    """Each draft hangs on a random earlier one; the first is the sequence's last token."""
    return [-1] + [rng.randint(max(0, i - 6), i - 1) for i in range(1, n)]


def _sizes(case, rng):
    """Cached and new tokens of each sequence, dealt out by the seed."""
    order = rng.sample(range(case["seqs"]), case["seqs"])
    lens = _dealt(case["ctx"], case["seqs"], "%(seqs)d %(ctx)d" % case)
    new = _dealt(case["new"], case["seqs"], "%(seqs)d %(ctx)d %(new)d" % case)
    return [lens[i] for i in order], [new[i] for i in order]


def prepare(case, seed):
    device = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=device).manual_seed(seed)
    rng = random.Random(seed)
    s = dict(case=case)
    {"verify": _prepare_verify, "weigh": _prepare_weigh, "evict": _prepare_evict}[case["op"]](s, gen, rng)
    if own:  # the handles that a program keeps
        from kernrelay_amd import ops
        s["seqs"] = ops.make_seqs(s["table"], s["lens"], s["starts"], s["max_new"], tree=s.get("tree"))
        if case["op"] == "verify":
            nbytes, ncnt = ops.verify_drafts_workspace(s["seqs"], s["logits"], draft=s["draft"])
            s["ws"] = torch.empty(nbytes, dtype=torch.uint8, device=device)
            s["counters"] = torch.zeros(ncnt, dtype=torch.int32, device=device)
        else:
            s["cache"] = ops.make_cache(s["k_cache"], s["v_cache"])
            s["weights"] = ops.make_weights(s["mass"], entry=s["entry"])
        if case["op"] == "weigh":
            nbytes = ops.attention_paged_weigh_workspace(s["cache"], s["seqs"], s["q"].shape[1])
            s["ws"] = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return s


def _prepare_verify(s, gen, rng):
    case, dev = s["case"], gen.device
    B, V = case["seqs"], case["vocab"]
    new = _dealt(case["new"], B, "%(seqs)d %(new)d" % case)
    rng.shuffle(new)
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device=dev)  # noqa: E731
    starts = [sum(new[:i]) for i in range(B + 1)]
    R = starts[-1]
    s["starts"], s["lens"], s["table"] = ints(starts), ints([100] * B), ints([[0]] * B)
    s["max_new"] = max(new)
    logits = _normal(gen, R, V, dtype=torch.float32, std=1.5)
    peaks = torch.randint(0, V, (R, PEAKS), device=dev, generator=gen)
    height = 14.0 - math.log(152064 / V) - 1.2 * torch.arange(PEAKS, device=dev)
    logits.scatter_(1, peaks, (height + _normal(gen, R, PEAKS, dtype=torch.float32)))
    s["logits"] = logits.to(DT[case["dtype"]])
    parents = [_parents(n, rng) if case["tree"] else [-1] + list(range(n - 1)) for n in new]
    above = ints([starts[b] + max(p, 0) for b in range(B) for p in parents[b]], torch.int64)  # the parent's row
    s["parents"] = ints([p for par in parents for p in par]) if case["tree"] else None
    s["draft"] = None
    if case["draft"]:  # a smaller model's opinion, and tokens drawn from it
        q = torch.softmax(logits + _normal(gen, R, V, dtype=torch.float32, std=0.5), dim=1)
        s["draft"] = q.to(DT[case["draft"]])
        q = s["draft"].float()[above]
        s["tokens"] = (q.log() - (-_uniform(gen, R, V).clamp(min=1e-30).log()).log()).argmax(dim=1)
    else:  # a drafter's best guesses, now and then a wrong one
        nth = ints([sum(1 for p in par[:i] if p == par[i]) % PEAKS for par in parents for i in range(len(par))],
                   torch.int64)
        best = logits.topk(PEAKS, dim=1).indices[above].gather(1, nth[:, None])[:, 0]
        wrong = torch.randint(0, V, (R,), device=dev, generator=gen)
        s["tokens"] = torch.where(_uniform(gen, R) < 0.85, best, wrong)
    s["u"], s["u_next"] = _uniform(gen, R), _uniform(gen, B)
    s["temperature"] = torch.tensor([rng.choice((0.0, 0.7, 1.0, 1.0)) for _ in range(B)], device=dev)
    s["path"] = torch.empty(B, case["new"], dtype=torch.int32, device=dev)
    s["path_lens"] = torch.empty(B, dtype=torch.int32, device=dev)
    s["next"] = torch.empty(B, dtype=torch.int64, device=dev)


def _prepare_weigh(s, gen, rng):
    case, dev = s["case"], gen.device
    HQ, HKV, D = SHAPES[case["model"]][:3]
    B, dt, page = case["seqs"], DT[case["dtype"]], case["page"]
    lens, new = _sizes(case, rng)
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device=dev)  # noqa: E731
    s["table"], total = _pages([a + b for a, b in zip(lens, new)], page, rng, dev)
    starts = [sum(new[:i]) for i in range(B + 1)]
    s["lens"], s["starts"], s["max_new"] = ints(lens), ints(starts), max(new)
    s["k_cache"] = _normal(gen, 1, total, page, HKV, D, dtype=dt)
    s["v_cache"] = torch.zeros_like(s["k_cache"])
    s["q"] = _normal(gen, starts[-1], HQ, D, dtype=dt)
    s["path"] = s["path_lens"] = s["tree"] = None
    if case["form"] == "tree":
        words = (max(new) + 63) // 64
        rows = []
        for n in new:
            seen = []
            for i, p in enumerate(_parents(n, rng)):
                seen.append((seen[p] if p >= 0 else 0) | (1 << i))
            rows += [[((b >> (64 * w)) & (2 ** 64 - 1)) - ((b >> (64 * w + 63) & 1) << 64) for w in range(words)]
                     for b in seen]
        s["tree"] = ints(rows, torch.int64)
    if case["form"] == "path":  # accepted drafts, moved together already: new token i came as row path[i]
        paths = []
        for n in new:
            at, path = 0, []
            while at < n:
                path.append(at)
                at += rng.randint(1, 7)
            paths.append(path)
        width = max(len(p) for p in paths)
        s["path"] = ints([p + [-1] * (width - len(p)) for p in paths])
        s["path_lens"] = ints([len(p) for p in paths])
    entries = B + 2
    s["entry"] = ints(rng.sample(range(entries), B))  # which of the program's slots the sequences have
    s["mass"] = torch.exp(_normal(gen, 1, entries, HKV, max(a + b for a, b in zip(lens, new)) + 5, dtype=torch.float32,
                                  std=1.5)) * 0.05
    # what the attention of these tokens left: the logarithm of each row's sum
    score, row, there = _scores(s)
    s["lse"] = torch.zeros(starts[-1], HQ, device=dev)
    lse = torch.logsumexp(score, dim=-1).permute(0, 3, 1, 2).flatten(2)  # [B, N, HQ]
    s["lse"][row[there]] = lse[there]


def _prepare_evict(s, gen, rng):
    case, dev = s["case"], gen.device
    _, HKV, D, layers, _ = SHAPES[case["model"]]
    B, page = case["seqs"], case["page"]
    lens = _dealt(case["ctx"], B, "%(seqs)d %(ctx)d" % case)
    rng.shuffle(lens)
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device=dev)  # noqa: E731
    s["table"], total = _pages(lens, page, rng, dev)
    s["lens"], s["starts"], s["max_new"] = ints(lens), ints([0] * (B + 1)), 0
    s["k_cache"], s["v_cache"] = (_normal(gen, layers, total, page, HKV, D, dtype=DT[case["dtype"]]) for _ in range(2))
    s["entry"] = ints(rng.sample(range(B + 2), B))
    s["mass"] = torch.exp(_normal(gen, layers, B + 2, HKV, max(lens) + 5, dtype=torch.float32, std=1.5)) * 0.05
    s["keep"] = torch.empty(layers, B, HKV, case["budget"], dtype=torch.int32, device=dev)


# --------------------------------------------------------------- plain forms
def _probabilities(logits, temperature):
    """Softmax over the row's temperature; 0: the first of the largest has it all."""
    x, t = logits.double(), temperature.double()[:, None]
    top = x.amax(dim=1, keepdim=True)
    w = torch.exp((x - top) / t.masked_fill(t == 0.0, 1.0))
    at = torch.arange(x.shape[1], device=x.device)
    first = torch.where(x == top, at, x.shape[1]).amin(dim=1, keepdim=True)
    return torch.where(t == 0.0, (at == first).double(), w / w.sum(dim=1, keepdim=True))


def _plain_verify(s):
    starts, tokens, u = s["starts"].long(), s["tokens"], s["u"].double()
    dev, R, B = tokens.device, s["tokens"].shape[0], s["starts"].shape[0] - 1
    row = torch.arange(R, device=dev)
    seq = torch.searchsorted(starts, row, right=True) - 1
    i = row - starts[seq]
    above = row - 1 if s["parents"] is None else starts[seq] + s["parents"].long()
    above = torch.where(i == 0, -1, above)                     # [R]: row of the parent, none for the first
    at = above.clamp(min=0)
    p = _probabilities(s["logits"], s["temperature"][seq])
    before = (above[:, None] == above) & (above[:, None] >= 0) & (row[:, None] > row)  # earlier drafts of that parent
    if s["draft"] is None:
        px = p[at, tokens].masked_fill((before & (tokens[:, None] == tokens)).any(dim=1), 0.0)
        passes = u * (1.0 - (before.double() * px).sum(dim=1)).clamp(min=0.0) < px
        left = p.index_put((at[above >= 0], tokens[above >= 0]), p.new_zeros(()))
        gone = left.sum(dim=1, keepdim=True) == 0.0
        left = torch.where(gone, p, left)
    else:
        q, nth = s["draft"].double(), before.sum(dim=1)
        passes, left = torch.zeros(R, dtype=torch.bool, device=dev), p
        for k in range(int(nth.max()) + 1):                    # each parent's k-th draft
            here = row[(above >= 0) & (nth == k)]
            par, x = above[here], tokens[here]
            passes[here] = u[here] * q[par, x] < left[par, x]
            rest = (left[par] - q[par]).clamp_(min=0.0)
            total = rest.sum(dim=1, keepdim=True)
            left = left.index_put((par,), torch.where(total > 0.0, rest / total.masked_fill(total == 0.0, 1.0), left[par]))
    taken = (passes & ~(before & passes).any(dim=1)) | (above < 0)
    reach = torch.eye(R, device=dev)                           # [R, R]: the column is the row itself or above it
    reach[row[above >= 0], above[above >= 0]] = 1.0
    for _ in range(max(1, s["max_new"] - 1).bit_length()):
        reach = (reach @ reach).clamp_(max=1.0)
    kept = (reach * (~taken).float()).sum(dim=1) == 0.0
    count = torch.zeros(B, dtype=torch.long, device=dev).index_add(0, seq, kept.long())
    nth = kept.long().cumsum(0) - (count.cumsum(0) - count)[seq] - 1
    s["path"].fill_(-1)
    s["path"][seq[kept], nth[kept]] = i[kept].int()
    s["path_lens"].copy_(count)
    stop = torch.zeros(B, dtype=torch.long, device=dev).scatter_reduce(0, seq[kept], row[kept], "amax")
    sums = left[stop].cumsum(dim=1)
    past = (sums <= s["u_next"].double()[:, None] * sums[:, -1:]).sum(dim=1)
    last = torch.where(left[stop] > 0.0, torch.arange(left.shape[1], device=dev), -1).amax(dim=1)
    s["next"].copy_(torch.minimum(past, last))
    return s["path"], s["path_lens"], s["next"]


def _scores(s):
    """Scaled scores [B, HKV, G, N, L] of each sequence's new tokens, -inf where a token does not see a key or does not
    count; the tokens' rows [B, N] and which there are."""
    q, table, tree, path = s["q"], s["table"].long().clamp(min=0), s["tree"], s["path"]
    dev, B = q.device, s["table"].shape[0]
    HQ, D = q.shape[1:]
    HKV = s["k_cache"].shape[3]
    starts, lens = s["starts"].long(), s["lens"].long()
    new = starts[1:] - starts[:-1] if path is None else s["path_lens"].long()
    last = s["case"]["last"] or s["max_new"]
    first = (new - last).clamp(min=0)                               # the first that counts
    N = min(last, s["max_new"] if path is None else path.shape[1])
    i = first[:, None] + torch.arange(N, device=dev)                # [B, N]
    there = i < new[:, None]
    row = starts[:-1, None] + (i if path is None else path.long()[:, :N])
    row = row.clamp(0, q.shape[0] - 1)
    k = s["k_cache"][0][table].flatten(1, 2).float().transpose(1, 2)  # [B, HKV, L, D]
    L = k.shape[2]
    at = torch.arange(L, device=dev) - lens[:, None]                # [B, L]: which new token, cached below 0
    if tree is None:
        sees = at[:, None, :] <= i[:, :, None]
    else:
        j = at.clamp(0, 64 * tree.shape[1] - 1)
        word = tree[row].gather(2, (j // 64)[:, None, :].expand(B, N, L))
        sees = (at < 0)[:, None, :] | ((word >> (j % 64)[:, None, :]) & 1).bool()
    sees = sees & (at < new[:, None])[:, None, :] & there[:, :, None]  # [B, N, L]
    qh = q[row].float().view(B, N, HKV, HQ // HKV, D).permute(0, 2, 3, 1, 4).reshape(B, HKV, -1, D)
    score = (qh @ k.transpose(2, 3).contiguous() * D ** -0.5).view(B, HKV, HQ // HKV, N, L)
    return score.masked_fill_(~sees[:, None, None], -math.inf), row, there


def _plain_weigh(s):
    score, row, there = _scores(s)
    B, HKV, G, N, L = score.shape
    lse = s["lse"][row].view(B, N, HKV, G).permute(0, 2, 3, 1)[..., None]
    got = score.sub_(lse).exp_().sum(dim=(2, 3))                    # [B, HKV, L]
    mass = s["mass"][0]
    width = min(L, mass.shape[2])
    lens = s["lens"].long()
    new = (s["starts"][1:] - s["starts"][:-1]).long() if s["path"] is None else s["path_lens"].long()
    at = torch.arange(width, device=lens.device)
    old = mass[s["entry"].long(), :, :width]
    now = torch.where((at < lens[:, None])[:, None], old + got[..., :width], got[..., :width])
    mass[s["entry"].long(), :, :width] = torch.where((at < (lens + new)[:, None])[:, None], now, old)
    return s["mass"]


def _plain_evict(s):
    case, table, lens = s["case"], s["table"].long(), s["lens"].long()
    k_cache, v_cache, mass = s["k_cache"], s["v_cache"], s["mass"]
    layers, _, page, HKV, _ = k_cache.shape
    budget, sinks, recent = case["budget"], case["sinks"], case["recent"]
    dev, end = lens.device, case["budget"] - case["recent"]
    entry = s["entry"].long()
    m = mass[:, entry]                                              # [layers, B, HKV, width]
    at = torch.arange(m.shape[3], device=dev)
    low = (lens - recent)[:, None, None]                            # [B, 1, 1]: the recent tokens begin
    middle = (at >= sinks) & (at < low)
    order = m.masked_fill(~middle, -math.inf).sort(dim=3, descending=True, stable=True).indices
    most = torch.zeros_like(m, dtype=torch.bool).scatter_(3, order[..., :end - sinks], True) & middle
    hole, mover = ~most & (at >= sinks) & (at < end), most & (at >= end)
    # the n-th hole gets the n-th mover
    n = mover.cumsum(dim=3) - 1
    movers = torch.zeros_like(order).scatter_(3, torch.where(mover, n, m.shape[3] - 1), at.expand_as(order) * mover)
    of = torch.where(hole, movers.gather(3, (hole.cumsum(dim=3) - 1).clamp(min=0)), at)
    of = torch.where((at >= end) & (at < budget), at - budget + lens[:, None, None], of)[..., :budget]
    to = at[:budget].expand_as(of)
    over = (lens > budget)[:, None, None]
    of = torch.where(over, of, to)
    s["keep"].copy_(torch.where(of < lens[:, None, None], of, -1))
    layer, seq, head = (torch.arange(n, device=dev).view(v) for n, v in
                        ((layers, (-1, 1, 1, 1)), (len(lens), (-1, 1, 1)), (HKV, (-1, 1))))
    there = (of != to) & over
    layer, seq, head = (t.expand_as(of)[there] for t in (layer, seq, head))
    of, to = of[there], to[there]
    here, away = (layer, table[seq, to // page], to % page, head), (layer, table[seq, of // page], of % page, head)
    k_cache[here] = k_cache[away]
    v_cache[here] = v_cache[away]
    mass[layer, entry[seq], head, to] = mass[layer, entry[seq], head, of]
    return s["keep"], k_cache, v_cache, mass


_PLAIN = {"verify": _plain_verify, "weigh": _plain_weigh, "evict": _plain_evict}


# ----------------------------------------------------------------------- run
def _own(s):
    from kernrelay_amd import ops
    case = s["case"]
    if case["op"] == "verify":
        ops.verify_drafts(s["seqs"], s["logits"], s["tokens"], s["u"], s["u_next"], s["path"], s["path_lens"],
                          s["next"], s["ws"], s["counters"], parents=s["parents"], draft=s["draft"],
                          temperature=s["temperature"])
        return s["path"], s["path_lens"], s["next"]
    if case["op"] == "weigh":
        ops.attention_paged_weigh(s["cache"], 0, s["seqs"], s["q"], s["lse"], s["weights"], s["ws"], last=case["last"],
                                  path=s["path"], path_lens=s["path_lens"])
        return s["mass"]
    ops.cache_evict(s["cache"], s["seqs"], s["weights"], s["keep"], sinks=case["sinks"], recent=case["recent"])
    return s["keep"], s["k_cache"], s["v_cache"], s["mass"]


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------- work
def work(case):
    # ragged batches: sizes run from half to the whole, three quarters in the mean
    part = 1.0 if case["seqs"] == 1 else 0.75
    B = case["seqs"]
    if case["op"] == "verify":
        # the rows down to the first draft that is not accepted, about three below the first; the draft's row there
        V, size = case["vocab"], 4 if case["dtype"] == "fp32" else 2
        rows = B * min(1 if case["new"] == 1 else part * case["new"], 4.0)
        dsize = {"": 0, "fp32": 4}.get(case["draft"], 2)
        return {"bytes": V * (rows * size + B * dsize), "flops": 4 * rows * V}
    HQ, HKV, D, layers, _ = SHAPES[case["model"]]
    if case["op"] == "weigh":
        ctx, new = part * case["ctx"], 1 if case["new"] == 1 else part * case["new"]
        rows = new / 4 if case["form"] == "path" else new
        rows = max(1.0, min(rows, case["last"] or rows))
        keys = ctx + (1 if case["form"] == "path" else new)
        seen = rows * (keys - rows / 2 if case["form"] == "causal" else ctx + 1 + math.log2(new) / 2)
        return {"bytes": B * (keys * HKV * (2 * D + 8) + rows * HQ * (2 * D + 4)), "flops": B * 2 * seen * HQ * D}
    lens = [n for n in _dealt(case["ctx"], B, "%(seqs)d %(ctx)d" % case)]
    over = [n for n in lens if n > case["budget"]]
    middle = case["budget"] - case["sinks"] - case["recent"]
    # of the tokens that stay, those that stand where they may stay need not move
    moved = sum(middle * (1 - middle / max(1, n - case["sinks"] - case["recent"])) + case["recent"] for n in over)
    return {"bytes": layers * HKV * (4 * sum(over) + 4 * B * case["budget"] + moved * (2 * 2 * 2 * D + 4)) + 4,
            "flops": 0}


# --------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    return {"verify": _exact_verify, "weigh": _exact_weigh, "evict": _exact_evict}[case["op"]](s)


def _exact_verify(s):
    starts, tokens, u = s["starts"].tolist(), s["tokens"].tolist(), s["u"].tolist()
    paths, nexts = [], []
    for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
        n, t = hi - lo, s["temperature"][b].item()
        par = [i - 1 for i in range(n)] if s["parents"] is None else s["parents"][lo:hi].tolist()
        path, more = [0], True
        while more:
            x = s["logits"][lo + path[-1]].double()
            if t > 0:
                p = torch.softmax(x / t, dim=0)
            else:
                p = torch.zeros_like(x)
                p[int((x == x.max()).nonzero()[0])] = 1.0
            more = False
            for c in (c for c in range(1, n) if par[c] == path[-1]):
                tok = tokens[lo + c]
                q = s["draft"][lo + path[-1]].double() if s["draft"] is not None else None
                ask = 1.0 if q is None else q[tok].item()
                if u[lo + c] * ask < p[tok].item():
                    path.append(c)
                    more = True
                    break
                rest = p.clone()
                if q is None:
                    rest[tok] = 0.0
                else:
                    rest = torch.relu(rest - q)
                if rest.sum() > 0:
                    p = rest / rest.sum()
        sums = torch.cumsum(p, 0)
        over = (sums > s["u_next"][b].double() * sums[-1]).nonzero()
        nexts.append(int(over[0]) if len(over) else int(p.nonzero()[-1]))
        paths.append(path)
    dev, width = s["tokens"].device, s["path"].shape[1]
    return (torch.tensor([p + [-1] * (width - len(p)) for p in paths], dtype=torch.int32, device=dev),
            torch.tensor([len(p) for p in paths], dtype=torch.int32, device=dev), torch.tensor(nexts, device=dev))


def _exact_weigh(s):
    HQ, D = s["q"].shape[1:]
    page, HKV = s["k_cache"].shape[2:4]
    dev, last = s["q"].device, s["case"]["last"]
    lens, starts, table, entry = (s[n].tolist() for n in ("lens", "starts", "table", "entry"))
    mass = s["mass"].double()
    for b, ctx in enumerate(lens):
        rows = list(range(starts[b], starts[b + 1]))
        if s["path"] is not None:
            rows = [starts[b] + p for p in s["path"][b].tolist()[:s["path_lens"][b].item()]]
        n = len(rows)
        ids = torch.tensor(table[b][:(ctx + n + page - 1) // page], device=dev)
        k = s["k_cache"][0].index_select(0, ids).reshape(-1, HKV, D)[:ctx + n].double()
        hidden = torch.zeros(n, ctx + n, dtype=torch.bool, device=dev)
        if s["tree"] is None:
            hidden[:, ctx:] = torch.ones(n, n, dtype=torch.bool, device=dev).triu(1)
        else:
            bits = [[(int(w[j // 64]) >> (j % 64)) & 1 == 0 for j in range(n)] for w in s["tree"][rows].tolist()]
            hidden[:, ctx:] = torch.tensor(bits, device=dev)
        if last and last < n:
            rows, hidden = rows[-last:], hidden[-last:]
        mass[0, entry[b], :, ctx:ctx + n] = 0.0
        at = torch.tensor(rows, device=dev)
        for h in range(HQ):
            g = h // (HQ // HKV)
            a = s["q"][at, h].double() @ k[:, g].t() / math.sqrt(D)
            a[hidden] = -math.inf
            mass[0, entry[b], g, :ctx + n] += (a - s["lse"][at, h].double()[:, None]).exp().sum(dim=0)
    return mass


def _exact_evict(s):
    case = s["case"]
    page = s["k_cache"].shape[2]
    budget, sinks, recent = case["budget"], case["sinks"], case["recent"]
    lens, entry = s["lens"].tolist(), s["entry"].tolist()
    layers, B, HKV, _ = s["keep"].shape
    dev, end = s["keep"].device, budget - recent
    keep = torch.full((layers, B, HKV, budget), -1, dtype=torch.int64, device=dev)
    k, v, mass = s["k_cache"].clone(), s["v_cache"].clone(), s["mass"].double()
    for b, n in enumerate(lens):
        place = lambda i: (s["table"][b].long()[i // page], i % page)  # noqa: E731
        if n <= budget:
            keep[:, b, :, :n] = torch.arange(n, device=dev)
            continue
        for ly in range(layers):
            for h in range(HKV):
                old = s["mass"][ly, entry[b], h]
                rank = torch.argsort(-old[sinks:n - recent].double(), stable=True)[:end - sinks] + sinks
                of = torch.arange(budget, device=dev)
                stays = torch.zeros(budget, dtype=torch.bool, device=dev)
                stays[rank[rank < end]] = True
                stays[:sinks] = True
                of[:end][~stays[:end]] = rank[rank >= end].sort().values
                of[end:] = torch.arange(n - recent, n, device=dev)
                keep[ly, b, h] = of
                to = torch.arange(budget, device=dev)
                for new, was in ((k, s["k_cache"]), (v, s["v_cache"])):
                    a, c = place(to)
                    e, f = place(of)
                    new[ly, a, c, h] = was[ly, e, f, h]
                mass[ly, entry[b], h, :budget] = old[of].double()
    return keep.int(), k.double(), v.double(), mass
