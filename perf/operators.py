"""The paged cache's operators as measurable cases: what writes a key/value
cache, what reads it and what moves its pages.

* rope: per-head RMSNorm of q and k with the position rotation in one pass,
  to plain tensors (a prompt's prefill) or, k and v, to their cache slots;
* attend: attention of each sequence's new tokens over its pages: one token,
  a tree of drafted tokens under a bit mask, or a causal chunk of a prompt;
* copy: whole pages copied to others, every layer's (forked sequences);
* compact: the rows of accepted drafts moved to the front of the drafted ones.

Head counts are those of the three model shapes the framework prefills.
Inputs: activations, keys and values N(0, 1), norm gains 1 + N(0, 0.02), pages
handed out in random order.
"""

import math
import random

import torch

own = False

# query heads, kv heads, head size, layers
HEADS = {"0.5b": (14, 2, 64, 24), "7b": (28, 4, 128, 28), "8b": (32, 8, 128, 36)}
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # a prompt of the longest configured length, q/k norms, no cache
        dict(name="rope_prompt_8b_s4096", op="rope", model="8b", rows=4096, norm=True, cache=False, dtype="bf16",
             table="bf16", pos=4096, page=0),
        # one decoding step of 48 sequences, no norms: latency
        dict(name="rope_step_7b_48", op="rope", model="7b", rows=48, norm=False, cache=True, dtype="bf16",
             table="bf16", pos=8192, page=16),
        # a mixed batch of prompts' chunks and steps, fp16, odd sizes, wide tables
        dict(name="rope_mixed_0.5b_1501", op="rope", model="0.5b", rows=1501, norm=True, cache=True, dtype="fp16",
             table="fp32", pos=32768, page=24),
        # the first tokens of one short conversation: latency
        dict(name="attend_one_0.5b_37", op="attend", model="0.5b", seqs=1, ctx=37, new=1, form="step", page=16,
             dtype="bf16"),
        # a busy server's decoding step, lengths ragged
        dict(name="attend_step_7b_64x4000", op="attend", model="7b", seqs=64, ctx=4000, new=1, form="step", page=16,
             dtype="bf16"),
        # one long document's next token
        dict(name="attend_long_8b_120001", op="attend", model="8b", seqs=1, ctx=120001, new=1, form="step", page=64,
             dtype="bf16"),
        # drafted trees of a small batch, fp16, odd pages
        dict(name="attend_tree_8b_8x61", op="attend", model="8b", seqs=8, ctx=2900, new=61, form="tree", page=24,
             dtype="fp16"),
        # the next chunk of a long prompt
        dict(name="attend_chunk_7b_2048", op="attend", model="7b", seqs=1, ctx=8000, new=2048, form="causal", page=32,
             dtype="bf16"),
        # a fork's last page
        dict(name="copy_fork_8b_3", op="copy", model="8b", pages=40, pairs=3, page=16, dtype="bf16"),
        # many forks, or a pool that is defragmented
        dict(name="copy_many_7b_130", op="copy", model="7b", pages=300, pairs=130, page=16, dtype="bf16"),
        # accepted drafts of one short conversation: latency
        dict(name="compact_0.5b_1x4", op="compact", model="0.5b", seqs=1, ctx=21, new=13, accept=4, page=24,
             dtype="fp16"),
        # accepted drafts of a batch
        dict(name="compact_7b_32x9", op="compact", model="7b", seqs=32, ctx=40, new=24, accept=9, page=16,
             dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("rope", "attend", "attend", "attend", "copy", "compact"))
    model = rng.choice(tuple(HEADS))
    page = rng.choice((8, 16, 24, 32, 64, 128))
    dtype = rng.choice(("bf16", "fp16"))
    if op == "rope":
        cache = rng.random() < 0.6
        return dict(op=op, model=model, rows=_log_int(rng, 1, 4096), norm=rng.random() < 0.6, cache=cache,
                    dtype=dtype, table=rng.choice((dtype, "fp32")), pos=_log_int(rng, 4096, 65536),
                    page=page if cache else 0)
    if op == "attend":
        form = rng.choice(("step", "tree", "causal"))
        if form == "causal":
            new, seqs = _log_int(rng, 2, 1500), rng.randint(1, 2)
            ctx = _log_int(rng, 1, 8000 // seqs)
        else:
            new = 1 if form == "step" else _log_int(rng, 2, 100)
            seqs = _log_int(rng, 1, 64)
            ctx = _log_int(rng, 8, (120000 if form == "step" else 60000) // seqs)
        return dict(op=op, model=model, seqs=seqs, ctx=ctx, new=new, form=form, page=page, dtype=dtype)
    if op == "copy":
        pairs = _log_int(rng, 1, 100)
        return dict(op=op, model=model, pages=2 * pairs + rng.randint(1, 20), pairs=pairs, page=rng.choice((8, 16, 24)),
                    dtype=dtype)
    new = _log_int(rng, 2, 60)
    return dict(op=op, model=model, seqs=_log_int(rng, 1, 32), ctx=_log_int(rng, 4, 100), new=new,
                accept=rng.randint(1, min(new, 12)), page=rng.choice((8, 16, 24)), dtype=dtype)


# -------------------------------------------------------------------- inputs
def _normal(gen, *shape, dtype, std=1.0, mean=0.0):
    return torch.empty(*shape, device=gen.device, dtype=torch.float32).normal_(mean, std, generator=gen).to(dtype)


def _many(gen, *shape, dtype):
    """Large caches: drawn in the type itself."""
    return torch.empty(*shape, device=gen.device, dtype=dtype).normal_(0.0, 1.0, generator=gen)


def _tables(rows, D, dtype, device):
    inv = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=device) / D)
    a = torch.arange(rows, dtype=torch.float64, device=device)[:, None] * inv
    a = torch.cat((a, a), dim=1)
    return a.cos().to(dtype), a.sin().to(dtype)


def _batch(case, rng):
    """Cached and new tokens of each sequence: ragged lengths that the case fixes, dealt out by the seed."""
    n, deal = case["seqs"], random.Random("%(seqs)d %(ctx)d %(new)d" % case)
    lens = [case["ctx"]] + [deal.randint((case["ctx"] + 1) // 2, case["ctx"]) for _ in range(n - 1)]
    new = [case["new"]] + [deal.randint((case["new"] + 1) // 2, case["new"]) for _ in range(n - 1)]
    order = rng.sample(range(n), n)
    return [lens[i] for i in order], [new[i] for i in order]


def _pages(lens, new, page, rng, device):
    """A page table over a pool in random order; -1 behind a sequence's last page."""
    need = [(a + b + page - 1) // page for a, b in zip(lens, new)]
    total = sum(need) + 2
    order = list(range(total))
    rng.shuffle(order)
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (max(need) - n))
        at += n
    return torch.tensor(table, dtype=torch.int32, device=device), total


def _trees(new, rng, device):
    """Each draft hangs on a random earlier one; bit j of row i: j is i or above it. Also the drafts' parents."""
    words = (max(new) + 63) // 64
    rows, parents = [], []
    for n in new:
        seen, par = [], []
        for i in range(n):
            p = -1 if i == 0 else rng.randint(max(0, i - 6), i - 1)
            par.append(p)
            seen.append((seen[p] if p >= 0 else 0) | (1 << i))
        parents.append(par)
        rows += [[((s >> (64 * w)) & (2 ** 64 - 1)) - ((s >> (64 * w + 63) & 1) << 64) for w in range(words)]
                 for s in seen]
    return torch.tensor(rows, dtype=torch.int64, device=device), parents


def prepare(case, seed):
    device = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=device).manual_seed(seed)
    rng = random.Random(seed)
    HQ, HKV, D, layers = HEADS[case["model"]]
    dt = DT[case["dtype"]]
    s = dict(case=case)
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device=device)  # noqa: E731
    if case["op"] == "rope":
        T = case["rows"]
        qkv = _normal(gen, T, HQ + 2 * HKV, D, dtype=dt)  # the fused projection's rows
        s["q"], s["k"], s["v"] = qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:]
        s["cos"], s["sin"] = _tables(case["pos"], D, DT[case["table"]], device)
        s["gq"], s["gk"] = ((_normal(gen, D, dtype=dt, std=0.02, mean=1.0) for _ in range(2)) if case["norm"]
                            else (None, None))
        s["q_out"] = torch.empty(T, HQ, D, dtype=dt, device=device)
        if case["cache"]:
            ps = case["page"]
            pages = (T + ps - 1) // ps + 2
            s["positions"] = ints([rng.randrange(case["pos"]) for _ in range(T)], torch.int64)
            s["slots"] = ints(rng.sample(range(pages * ps), T), torch.int64)
            s["k_cache"], s["v_cache"] = (_many(gen, 1, pages, ps, HKV, D, dtype=dt) for _ in range(2))
        else:
            s["k_out"] = torch.empty(T, HKV, D, dtype=dt, device=device)
    elif case["op"] == "copy":
        s["k_cache"], s["v_cache"] = (_many(gen, layers, case["pages"], case["page"], HKV, D, dtype=dt)
                                      for _ in range(2))
        ids = rng.sample(range(case["pages"]), 2 * case["pairs"])
        s["src"], s["dst"] = ids[:case["pairs"]], ids[case["pairs"]:]  # a scheduler's lists
    else:
        lens, new = _batch(case, rng)
        table, total = _pages(lens, new, case["page"], rng, device)
        n = 1 if case["op"] == "attend" else layers
        s["k_cache"], s["v_cache"] = (_many(gen, n, total, case["page"], HKV, D, dtype=dt) for _ in range(2))
        starts = [sum(new[:i]) for i in range(len(new) + 1)]
        s["table"], s["lens"], s["starts"] = table, ints(lens), ints(starts)
        s["max_new"] = max(new)
        s["tree"] = None
        if case["op"] == "attend":
            if case["form"] == "tree":
                s["tree"], _ = _trees(new, rng, device)
            s["q"] = _normal(gen, sum(new), HQ, D, dtype=dt)
            s["out"] = torch.empty(sum(new), HQ, D, dtype=dt, device=device)
        else:
            _, parents = _trees(new, rng, device)
            paths = []
            for par in parents:  # the longest accepted: the path up from a late draft, at most `accept` long
                path, i = [], len(par) - 1
                while i >= 0:
                    path.append(i)
                    i = par[i]
                paths.append(path[::-1][:case["accept"]])
            s["path"] = ints([p + [-1] * (case["accept"] - len(p)) for p in paths])
            s["path_lens"] = ints([len(p) for p in paths])
    if own:  # the handles that a program keeps
        from kernrelay_amd import ops
        if "k_cache" in s:
            s["cache"] = ops.make_cache(s["k_cache"], s["v_cache"])
        if "cos" in s:
            s["rope"] = ops.make_rope(s["cos"], s["sin"], q_gamma=s["gq"], k_gamma=s["gk"], eps=EPS)
        if "table" in s:
            s["seqs"] = ops.make_seqs(s["table"], s["lens"], s["starts"], s["max_new"], tree=s["tree"])
        if case["op"] == "attend":
            nbytes, ncnt = ops.attention_paged_workspace(s["cache"], s["seqs"], HQ)
            s["ws"] = torch.empty(nbytes, dtype=torch.uint8, device=device)
            s["counters"] = torch.zeros(ncnt, dtype=torch.int32, device=device)
    return s


# --------------------------------------------------------------- plain forms
def _rotated(x, gamma, cos, sin):
    y = x.float()
    if gamma is not None:
        y = y * torch.rsqrt((y * y).mean(dim=-1, keepdim=True) + EPS) * gamma.float()
    h = y.shape[-1] // 2
    turned = torch.cat((-y[..., h:], y[..., :h]), dim=-1)
    return (y * cos.float()[:, None] + turned * sin.float()[:, None]).to(x.dtype)


def _plain_rope(s):
    at = s["positions"] if "positions" in s else slice(0, s["q"].shape[0])
    cos, sin = s["cos"][at], s["sin"][at]
    s["q_out"].copy_(_rotated(s["q"], s["gq"], cos, sin))
    k = _rotated(s["k"], s["gk"], cos, sin)
    if "slots" not in s:
        s["k_out"].copy_(k)
        return s["q_out"], s["k_out"]
    page = s["k_cache"].shape[2]
    where = (0, s["slots"] // page, s["slots"] % page)
    s["k_cache"][where] = k
    s["v_cache"][where] = s["v"]
    return s["q_out"], s["k_cache"], s["v_cache"]


def _plain_attend(s):
    q, table, tree = s["q"], s["table"].long().clamp(min=0), s["tree"]
    dev, N = q.device, s["max_new"]
    HQ, D = q.shape[1:]
    HKV = s["k_cache"].shape[3]
    B = table.shape[0]
    starts, lens = s["starts"].long(), s["lens"].long()
    new = starts[1:] - starts[:-1]
    i = torch.arange(N, device=dev)
    row = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)         # [B, N]
    k = s["k_cache"][0][table].flatten(1, 2).float().transpose(1, 2)  # [B, HKV, L, D]
    v = s["v_cache"][0][table].flatten(1, 2).float().transpose(1, 2)
    L = k.shape[2]
    at = torch.arange(L, device=dev) - lens[:, None]                # [B, L]: which draft, cached below 0
    if tree is None:
        sees = at[:, None, :] <= i[None, :, None]
    else:
        j = at.clamp(0, 64 * tree.shape[1] - 1)
        word = tree[row].gather(2, (j // 64)[:, None, :].expand(B, N, L))
        sees = (at < 0)[:, None, :] | ((word >> (j % 64)[:, None, :]) & 1).bool()
    sees = sees & (at < new[:, None])[:, None, :]                   # [B, N, L]
    qh = q[row].float().view(B, N, HKV, HQ // HKV, D).permute(0, 2, 3, 1, 4).reshape(B, HKV, -1, D)
    score = qh @ k.transpose(2, 3).contiguous() * D ** -0.5          # [B, HKV, G*N, L]
    score = score.view(B, HKV, HQ // HKV, N, L).masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    score = score.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = score.sum(dim=-1, keepdim=True)
    o = (score.view(B, HKV, -1, L) @ v.contiguous()).view(B, HKV, HQ // HKV, N, D)
    o = o / total.masked_fill(total == 0.0, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, N, HQ, D)[i[None, :] < new[:, None]]
    s["out"].copy_(o)
    return s["out"]


def _plain_copy(s):
    src, dst = (torch.tensor(s[n], device=s["k_cache"].device) for n in ("src", "dst"))
    s["k_cache"][:, dst] = s["k_cache"][:, src]
    s["v_cache"][:, dst] = s["v_cache"][:, src]
    return s["k_cache"], s["v_cache"]


def _plain_compact(s):
    page = s["k_cache"].shape[2]
    path, lens = s["path"].long(), s["lens"].long()
    i = torch.arange(path.shape[1], device=path.device)
    there = i < s["path_lens"].long()[:, None]
    to, of = lens[:, None] + i, lens[:, None] + path
    seq = torch.arange(path.shape[0], device=path.device)[:, None].expand_as(path)[there]
    to, of = to[there], of[there]
    table = s["table"].long()
    to, of = (table[seq, to // page], to % page), (table[seq, of // page], of % page)
    s["k_cache"][:, to[0], to[1]] = s["k_cache"][:, of[0], of[1]]
    s["v_cache"][:, to[0], to[1]] = s["v_cache"][:, of[0], of[1]]
    return s["k_cache"], s["v_cache"]


_PLAIN = {"rope": _plain_rope, "attend": _plain_attend, "copy": _plain_copy, "compact": _plain_compact}


# ----------------------------------------------------------------------- run
def _own(s):
    from kernrelay_amd import ops
    op = s["case"]["op"]
    if op == "rope":
        if "slots" in s:
            ops.qk_norm_rope_cache(s["rope"], s["cache"], 0, s["q"], s["k"], s["v"], s["q_out"], s["positions"],
                                   s["slots"])
            return s["q_out"], s["k_cache"], s["v_cache"]
        ops.qk_norm_rope(s["rope"], s["q"], s["k"], s["q_out"], s["k_out"])
        return s["q_out"], s["k_out"]
    if op == "attend":
        ops.attention_paged(s["cache"], 0, s["seqs"], s["q"], s["out"], ws=s["ws"], counters=s["counters"])
        return s["out"]
    if op == "copy":
        ops.cache_copy_pages(s["cache"], s["src"], s["dst"])
    else:
        ops.cache_compact(s["cache"], s["seqs"], s["path"], s["path_lens"])
    return s["k_cache"], s["v_cache"]


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------- work
def work(case):
    HQ, HKV, D, layers = HEADS[case["model"]]
    if case["op"] == "rope":
        T = case["rows"]
        tables = 2 * min(T, case["pos"]) * D * (4 if case["table"] == "fp32" else 2)
        values = T * D * (HQ + HKV + (HKV if case["cache"] else 0))
        return {"bytes": 4 * values + tables + (16 * T if case["cache"] else 0), "flops": 7 * T * D * (HQ + HKV)}
    if case["op"] == "copy":
        return {"bytes": 2 * case["pairs"] * 2 * layers * case["page"] * HKV * D * 2, "flops": 0}
    # ragged batches: lengths run from half to the whole, three quarters in the mean
    part = 1.0 if case["seqs"] == 1 else 0.75
    if case["op"] == "compact":
        rows = case["seqs"] * max(1.0, min(case["accept"], part * case["new"] / 3.5))
        return {"bytes": 2 * rows * 2 * layers * HKV * D * 2, "flops": 0}
    ctx = part * case["ctx"]
    new = 1 if case["new"] == 1 else part * case["new"]
    seen = new * (ctx + (new + 1) / 2 if case["form"] == "causal" else ctx + 1 + math.log2(new) / 2)
    return {"bytes": case["seqs"] * (2 * (ctx + new) * HKV * D * 2 + 2 * new * HQ * D * 2),
            "flops": case["seqs"] * 4 * seen * HQ * D}


# --------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "attend": _exact_attend, "copy": _exact_copy, "compact": _exact_compact}[case["op"]](s)


def _exact_rope(s):
    T, HQ, D = s["q"].shape
    at = s["positions"] if "positions" in s else torch.arange(T, device=s["q"].device)
    c, n = s["cos"].double().index_select(0, at), s["sin"].double().index_select(0, at)
    outs = []
    for x, g in ((s["q"], s["gq"]), (s["k"], s["gk"])):
        x = x.double()
        if g is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * g.double()
        lo, hi = x[..., :D // 2], x[..., D // 2:]
        c1, c2, n1, n2 = (t[:, None, w] for t in (c, n) for w in (slice(0, D // 2), slice(D // 2, D)))
        outs.append(torch.cat((lo * c1 - hi * n1, hi * c2 + lo * n2), -1))
    if "slots" not in s:
        return tuple(outs)
    caches = []
    for cache, rows in ((s["k_cache"], outs[1]), (s["v_cache"], s["v"].double())):
        flat = cache.double().view(-1, *cache.shape[3:])
        flat.index_copy_(0, s["slots"], rows)
        caches.append(flat.view(cache.shape))
    return outs[0], caches[0], caches[1]


def _exact_attend(s):
    HQ, D = s["q"].shape[1:]
    page, HKV = s["k_cache"].shape[2:4]
    lens, starts, table = s["lens"].tolist(), s["starts"].tolist(), s["table"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b, ctx in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        n = hi - lo
        ids = torch.tensor(table[b][:(ctx + n + page - 1) // page], device=out.device)
        k, v = (c[0].index_select(0, ids).reshape(-1, HKV, D)[:ctx + n].double() for c in
                (s["k_cache"], s["v_cache"]))
        hidden = torch.zeros(n, ctx + n, dtype=torch.bool, device=out.device)
        if s["tree"] is None:
            hidden[:, ctx:] = torch.ones(n, n, dtype=torch.bool, device=out.device).triu(1)
        else:
            bits = [[(int(w[j // 64]) >> (j % 64)) & 1 == 0 for j in range(n)] for w in s["tree"][lo:hi].tolist()]
            hidden[:, ctx:] = torch.tensor(bits, device=out.device)
        for h in range(HQ):
            g = h // (HQ // HKV)
            a = s["q"][lo:hi, h].double() @ k[:, g].t() / math.sqrt(D)
            a[hidden] = -math.inf
            out[lo:hi, h] = torch.softmax(a, dim=-1) @ v[:, g]
    return out


def _exact_copy(s):
    outs = []
    for cache in (s["k_cache"], s["v_cache"]):
        new = cache.clone()
        for a, b in zip(s["src"], s["dst"]):
            new[:, b] = cache[:, a]
        outs.append(new)
    return tuple(outs)


def _exact_compact(s):
    page = s["k_cache"].shape[2]
    lens, paths, counts, table = (s[n].tolist() for n in ("lens", "path", "path_lens", "table"))
    outs = []
    for cache in (s["k_cache"], s["v_cache"]):
        new = cache.clone()
        for b, ctx in enumerate(lens):
            for i in range(counts[b]):
                to, of = ctx + i, ctx + paths[b][i]
                new[:, table[b][to // page], to % page] = cache[:, table[b][of // page], of % page]
        outs.append(new)
    return tuple(outs)
