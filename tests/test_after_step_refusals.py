"""What the calls after a step over the paged cache refuse, before anything
reaches a GPU: the C entries get addresses that nothing reads, the wrappers CPU
tensors."""

import ctypes

import pytest
import torch

from kernrelay_amd import ops
from tests.test_paged_refusals import BAD_CACHES, BAD_SEQS, cache, refused, seqs

A = 1 << 20
W = 1 << 30    # away from the cache at A
FAR = 1 << 40


def weights(**kw):
    f = dict(w=W, layer_stride=3 * 4 * 70, entry_stride=4 * 70, head_stride=70, layers=2, entries=3, heads=4, width=64,
             entry=None)
    f.update(kw)
    return ops.KrWeights(**f)


def drafts(**kw):
    f = dict(logits=A, ld_logits=100, draft=None, ld_draft=0, tokens=W, parents=None, u=W + 4096, u_next=W + 8192,
             temperature=None, dtype=ops.KR_BF16, draft_dtype=0, vocab=100, rows=7)
    f.update(kw)
    return ops.KrDrafts(**f)


def far_seqs(**kw):
    """Arrays away from the cache's and the weights'."""
    f = dict(table=FAR + (8 << 20), lens=FAR + (9 << 20), starts=FAR + (10 << 20))
    f.update(kw)
    return seqs(**f)


def weigh(c=None, s=None, w=None, layer=0, q=FAR, ldq=0, lse=FAR + (1 << 20), ld_lse=0, rows=5, HQ=8, scale=0.1, last=0,
          decay=1.0, path=None, ld_path=0, width=0, lens=None):
    return ops._lib().kr_op_attention_paged_weigh(c or cache(), layer, s or far_seqs(), q, ldq, lse, ld_lse, rows, HQ, scale,
                                                  w or weights(), last, decay, path, ld_path, width, lens, None, 0, None)


def evict(c=None, s=None, w=None, budget=10, sinks=0, recent=0, keep=FAR):
    return ops._lib().kr_op_cache_evict(c or cache(), s or far_seqs(), w or weights(), budget, sinks, recent, keep, None)


def verify(d=None, s=None, path=FAR, ld_path=5, width=5, lens=FAR + (1 << 20), nxt=FAR + (2 << 20), ws=FAR + (3 << 20),
           nbytes=1 << 20, cnt=FAR + (5 << 20), ncnt=96):
    return ops._lib().kr_op_verify_drafts(d or drafts(), s or seqs(), path, ld_path, width, lens, nxt, ws, nbytes, cnt,
                                          ncnt, None)


@pytest.mark.parametrize("field,text", BAD_CACHES)
def test_bad_caches(field, text):
    c = cache(**field)
    refused(weigh(c), text)
    refused(evict(c), text)
    refused(ops._lib().kr_op_attention_paged_weigh_workspace(c, seqs(), 8, ctypes.c_size_t(0)), text)
    refused(ops._lib().kr_op_attention_paged_lse(c, 0, seqs(), A, 0, A, 0, A, 0, 5, 8, 0.1, None, 0, None, 0, None), text)


@pytest.mark.parametrize("field,text", BAD_SEQS)
def test_bad_sequences(field, text):
    s = seqs(**field)
    refused(weigh(s=s), text)
    refused(evict(s=s), text)
    refused(verify(s=s), text)


@pytest.mark.parametrize("field,text", [
    (dict(w=None), "needs weights"), (dict(layers=1), "layers or heads"), (dict(heads=3), "layers or heads"),
    (dict(entries=0), "empty"), (dict(width=0), "empty"), (dict(w=W + 2), "misaligned"), (dict(entry=A + 1), "misaligned"),
    (dict(head_stride=63), "overlap"), (dict(entry_stride=4 * 70 - 7), "overlap"), (dict(layer_stride=70), "overlap"),
    (dict(head_stride=-70), "overlap"), (dict(layer_stride=1 << 41), "overlap"),
])
def test_bad_weights(field, text):
    refused(weigh(w=weights(**field)), text)
    refused(evict(w=weights(**field)), text)


@pytest.mark.parametrize("kw,text", [
    (dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(q=None), "missing"), (dict(lse=None), "missing"),
    (dict(q=FAR + 8), "aligned"), (dict(lse=FAR + 2), "aligned"), (dict(ldq=1028), "multiples of 8"),
    (dict(ldq=8), "rows overlap"), (dict(ld_lse=7), "rows overlap"), (dict(rows=-1), "negative"), (dict(last=-1), "negative"),
    (dict(HQ=6), "multiple"), (dict(HQ=0), "multiple"), (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(decay=-0.5), "decay"), (dict(decay=float("nan")), "decay"), (dict(path=A), "lengths"), (dict(lens=A), "lengths"),
    (dict(path=A, lens=A, width=0), "path rows"), (dict(path=A, lens=A, width=4, ld_path=3), "path rows"),
    (dict(q=W), "overlap"), (dict(lse=W + 4), "overlap"), (dict(w=weights(w=A)), "overlap"),
    (dict(s=far_seqs(lens=W + 64)), "overlap"), (dict(s=far_seqs(table=W)), "overlap"),
    (dict(s=far_seqs(starts=W + 4)), "overlap"), (dict(s=far_seqs(tree=W, tree_words=1, ld_tree=1)), "overlap"),
    (dict(w=weights(entry=W)), "overlap"), (dict(path=W, lens=FAR + (4 << 20), width=4, ld_path=4), "overlap"),
    (dict(path=FAR + (4 << 20), lens=W, width=4, ld_path=4), "overlap"),
    (dict(s=seqs(table_pages=1 << 27, ld_table=1 << 27)), "too many tokens"),
])
def test_bad_weigh_calls(kw, text):
    refused(weigh(**kw), text)


# weights that hold as many tokens as the page table; their rows times the key tiles, and the blocks alone
WIDE = dict(w=FAR << 4, layer_stride=1 << 38, entry_stride=1 << 34, head_stride=1 << 30, width=1 << 30)


@pytest.mark.parametrize("kw,s", [(dict(rows=5000), dict(max_new=5000)), (dict(rows=1), dict(seqs=20, max_new=1))])
def test_more_rows_and_keys_than_a_launch_can_count(kw, s):
    s = far_seqs(table_pages=1 << 26, ld_table=1 << 26, **s)
    ws = ctypes.c_size_t(0)
    assert ops._lib().kr_op_attention_paged_weigh_workspace(cache(), s, 8, ctypes.byref(ws)) == 0
    f = dict(q=FAR, lse=FAR + (1 << 30), HQ=8)
    f.update(kw)
    refused(ops._lib().kr_op_attention_paged_weigh(cache(), 0, s, f["q"], 0, f["lse"], 0, f["rows"], 8, 0.1, weights(**WIDE),
                                                   0, 1.0, None, 0, 0, None, FAR + (2 << 30), ws.value, None),
            "too many rows and keys")


@pytest.mark.parametrize("kw,text", [
    (dict(budget=0), "budget"), (dict(sinks=-1), "fit the budget"), (dict(recent=-1), "fit the budget"),
    (dict(sinks=6, recent=5), "fit the budget"), (dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), "fit the budget"),
    (dict(keep=None), "keep"), (dict(keep=FAR + 2), "keep"), (dict(budget=1 << 30), "too large"),
    (dict(keep=W + 64), "overlap"), (dict(keep=A), "overlap"), (dict(w=weights(w=A + 4)), "overlap"),
    (dict(s=far_seqs(lens=FAR + 8)), "overlap"), (dict(s=far_seqs(table=W)), "overlap"), (dict(s=seqs()), "overlap"),
    (dict(w=weights(entry=FAR + 4)), "overlap"),
    (dict(s=seqs(table_pages=1 << 27, ld_table=1 << 27)), "too many tokens"),
])
def test_bad_evictions(kw, text):
    refused(evict(**kw), text)


@pytest.mark.parametrize("field,text", [
    (dict(logits=None), "missing"), (dict(tokens=None), "missing"), (dict(u=None), "missing"), (dict(u_next=None), "missing"),
    (dict(dtype=3), "bf16"), (dict(draft=A, ld_draft=100, draft_dtype=-1), "bf16"), (dict(vocab=0), "size"),
    (dict(rows=-1), "size"), (dict(ld_logits=99), "overlap"), (dict(draft=A, ld_draft=99), "overlap"),
    (dict(ld_logits=1 << 41), "too large"), (dict(vocab=(1 << 30) + 1, ld_logits=1 << 31), "too large"),
    (dict(rows=1 << 30), "too many rows"), (dict(logits=A + 1), "misaligned"), (dict(tokens=W + 4), "misaligned"),
    (dict(u=W + 2), "misaligned"), (dict(parents=W + 1), "misaligned"), (dict(temperature=W + 3), "misaligned"),
])
def test_bad_drafts(field, text):
    refused(verify(drafts(**field)), text)


@pytest.mark.parametrize("kw,text", [
    (dict(width=0), "path rows"), (dict(ld_path=4), "path rows"), (dict(path=None), "output"), (dict(lens=None), "output"),
    (dict(nxt=None), "output"), (dict(nxt=FAR + 4), "misaligned"), (dict(path=FAR + 1), "misaligned"),
    (dict(ws=None), "workspace"), (dict(nbytes=10), "workspace"), (dict(ws=FAR + 8), "workspace"),
    (dict(cnt=None), "workspace"), (dict(ncnt=95), "workspace"), (dict(cnt=FAR + (5 << 20) + 2), "workspace"),
    (dict(cnt=A), "overlap"), (dict(cnt=FAR + (2 << 20)), "overlap"),
    (dict(cnt=None), "workspace"), (dict(ncnt=95), "workspace"), (dict(cnt=FAR + 2), "workspace"), (dict(cnt=A), "overlap"),
    (dict(path=A), "overlap"), (dict(lens=FAR + 4), "overlap"), (dict(nxt=W), "overlap"), (dict(ws=A), "overlap"),
    (dict(s=seqs(max_new=1025)), "1024"),
])
def test_bad_verify_calls(kw, text):
    refused(verify(**kw), text)
    if "s" in kw:
        b, c = ctypes.c_size_t(0), ctypes.c_int(0)
        refused(ops._lib().kr_op_verify_drafts_workspace(drafts(), kw["s"], b, c), text)


def test_lse_is_checked():
    def call(lse=FAR + (1 << 30), ld=0, q=FAR, out=FAR + (1 << 20)):
        return ops._lib().kr_op_attention_paged_lse(cache(), 0, seqs(), q, 0, out, 0, lse, ld, 5, 8, 0.1, None, 0, None, 0, None)
    refused(call(lse=None), "lse is missing")
    refused(call(lse=FAR + (1 << 30) + 2), "misaligned")
    refused(call(ld=7), "lse rows overlap")
    refused(call(lse=FAR + 64), "lse overlaps")
    refused(call(lse=FAR + (1 << 20)), "lse overlaps")
    refused(call(lse=A + 4096), "lse overlaps")
    s = far_seqs()
    refused(ops._lib().kr_op_attention_paged_lse(cache(), 0, s, FAR, 0, FAR + (1 << 20), 0, s.lens, 0, 5, 8, 0.1, None, 0,
                                                 None, 0, None), "lse overlaps")


def test_wrappers_refuse_what_the_entries_cannot_see():
    with pytest.raises(ValueError, match="float32"):
        ops.make_weights(torch.zeros(2, 3, 4, 8, dtype=torch.float64))
    with pytest.raises(ValueError, match="float32"):
        ops.make_weights(torch.zeros(4, 8))
    with pytest.raises(ValueError, match="rows must be contiguous"):
        ops.make_weights(torch.zeros(2, 3, 8, 4).transpose(2, 3))
    with pytest.raises(ValueError, match="empty"):
        ops.make_weights(torch.zeros(2, 0, 4, 8))
    with pytest.raises(ValueError, match="entry"):
        ops.make_weights(torch.zeros(2, 3, 4, 8), entry=torch.zeros(3))
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.make_weights(torch.zeros(2, 3, 4, 8))
    c, s = cache(), seqs()
    c.device = s.device = 0
    c.torch_dtype, s.rows = torch.bfloat16, None
    w = weights()
    w.device, w.seqs = 0, None
    q, lse, ws = torch.zeros(5, 8, 128, dtype=torch.bfloat16), torch.zeros(5, 8), torch.zeros(0, dtype=torch.uint8)
    ints = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    for kw, text in [(dict(q=q[:, :, :64]), "head_dim"), (dict(q=q.half()), "q must be"), (dict(lse=lse.double()), "lse"),
                     (dict(lse=lse[:4]), "lse"), (dict(lse=lse.t().contiguous().t()), "lse"),
                     (dict(path=ints(3, 4)), "lengths"), (dict(path=ints(2, 4), path_lens=ints(3)), "path must"),
                     (dict(path=ints(3, 0), path_lens=ints(3)), "empty"), (dict(path=ints(3, 4), path_lens=ints(2)), "path_lens")]:
        with pytest.raises(ValueError, match=text):
            ops.attention_paged_weigh(c, 0, s, kw.pop("q", q), kw.pop("lse", lse), w, ws, **kw)
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.attention_paged_weigh(c, 0, s, q, lse, w, ws)
    w.seqs = 2
    with pytest.raises(ValueError, match="one entry for each"):
        ops.attention_paged_weigh(c, 0, s, q, lse, w, ws)
    with pytest.raises(ValueError, match="one entry for each"):
        ops.cache_evict(c, s, w, ints(2, 3, 4, 10))
    w.seqs, w.entries = None, 2
    with pytest.raises(ValueError, match="fewer entries"):
        ops.cache_evict(c, s, w, ints(2, 3, 4, 10))
    w.entries = 3
    for keep in (ints(2, 3, 10), ints(2, 2, 4, 10), ints(2, 3, 4, 10).long(), ints(2, 3, 4, 20)[..., ::2]):
        with pytest.raises(ValueError, match="keep"):
            ops.cache_evict(c, s, w, keep)
    w.device = 1
    with pytest.raises(ValueError, match="another device"):
        ops.cache_evict(c, s, w, ints(2, 3, 4, 10))
    with pytest.raises(ValueError, match="lse must be"):
        ops.attention_paged(c, 0, s, q, torch.zeros_like(q), lse=torch.zeros(5, 7))


def test_verify_wrapper():
    s = seqs()
    s.device = 0
    f, i = torch.float32, torch.int32
    good = dict(logits=torch.zeros(7, 50), tokens=torch.zeros(7, dtype=torch.int64), u=torch.zeros(7), u_next=torch.zeros(3),
                path=torch.zeros(3, 5, dtype=i), path_lens=torch.zeros(3, dtype=i),
                next_tokens=torch.zeros(3, dtype=torch.int64), ws=torch.zeros(9, dtype=torch.uint8),
                counters=torch.zeros(0, dtype=i))
    for kw, text in [(dict(logits=torch.zeros(7, 50, 1)), "logits"), (dict(logits=torch.zeros(50, 7).t()), "logits"),
                     (dict(logits=torch.zeros(7, 50)[:, :0]), "logits"), (dict(tokens=torch.zeros(7, dtype=i)), "tokens"),
                     (dict(tokens=torch.zeros(6, dtype=torch.int64)), "tokens"), (dict(u=torch.zeros(7).double()), "u must"),
                     (dict(u_next=torch.zeros(2)), "u_next"), (dict(path=torch.zeros(3, 5)), "path"),
                     (dict(path=torch.zeros(2, 5, dtype=i)), "path"), (dict(path=torch.zeros(3, 0, dtype=i)), "path"),
                     (dict(path_lens=torch.zeros(2, dtype=i)), "path_lens"), (dict(next_tokens=torch.zeros(3, dtype=i)), "next"),
                     (dict(counters=torch.zeros(0)), "counters"), (dict(draft=torch.zeros(7, 49)), "draft"),
                     (dict(draft=torch.zeros(50, 7).t()), "draft"), (dict(parents=torch.zeros(7)), "parents"),
                     (dict(temperature=torch.zeros(3, dtype=f)[:2]), "temperature")]:
        with pytest.raises(ValueError, match=text):
            ops.verify_drafts(s, **{**good, **kw})
    with pytest.raises(TypeError, match="dtype"):
        ops.verify_drafts(s, **{**good, "logits": torch.zeros(7, 50).double()})
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.verify_drafts(s, **good)


@pytest.mark.parametrize("n,tree,ok", [(1 << 21, True, False), (1 << 22, True, False), ((1 << 21) - 1, True, True),
                                       (1 << 22, False, True)])
def test_sampled_trees_of_more_sequences_than_a_launch_can_count(n, tree, ok):
    """The walk of sampled trees takes 1024 threads a sequence, of which the runtime
    counts 2^32 and the launches here 2^31."""
    d = drafts(draft=A + 4096, ld_draft=100, draft_dtype=ops.KR_BF16, parents=W + 16384 if tree else None)
    s = far_seqs(seqs=n, ld_table=4)
    # (what may be launched ends at the workspace)
    refused(verify(d, s, nbytes=0, ncnt=0), "workspace is too small" if ok else "too many sequences")
    b, c = ctypes.c_size_t(0), ctypes.c_int(0)
    rc = ops._lib().kr_op_verify_drafts_workspace(d, s, b, c)
    assert rc == 0 if ok else rc != 0


WS = FAR + (64 << 20)  # more than 32 packed rows: the workspace is written


@pytest.mark.parametrize("kw", [
    dict(q=WS), dict(lse=WS + (1 << 20)), dict(c=cache(k=WS, v=A)), dict(s=dict(table=WS + 64)), dict(s=dict(lens=WS + 64)),
    dict(s=dict(starts=WS + 64)), dict(s=dict(tree=WS, tree_words=1, ld_tree=1)), dict(w=weights(entry=WS + 64)),
    dict(w=weights(w=WS + 64)), dict(path=WS + 64, lens=FAR, width=40, ld_path=40),
    dict(path=FAR, lens=WS + 64, width=40, ld_path=40),
])
def test_weigh_workspaces_on_what_the_call_reads(kw):
    kw = dict(kw)
    s = far_seqs(max_new=40, **kw.pop("s", {}))
    b = ctypes.c_size_t(0)
    c = kw.pop("c", cache())
    assert ops._lib().kr_op_attention_paged_weigh_workspace(c, s, 8, b) == 0 and (1 << 20) < b.value < (4 << 20)
    f = dict(q=FAR + (16 << 20), lse=FAR + (32 << 20), w=weights(), path=None, lens=None, width=0, ld_path=0)
    f.update(kw)
    refused(ops._lib().kr_op_attention_paged_weigh(c, 0, s, f["q"], 0, f["lse"], 0, 120, 8, 0.1, f["w"], 0, 1.0, f["path"],
                                                   f["ld_path"], f["width"], f["lens"], WS, b.value, None), "overlap")


def test_lse_on_the_counters():
    """(which the last piece of a row leaves zero)"""
    s = far_seqs(seqs=256, max_new=1, ld_table=64, table_pages=64)  # (units enough for tickets)
    b, n = ctypes.c_size_t(0), ctypes.c_int(0)
    assert ops._lib().kr_op_attention_paged_workspace(cache(), s, 8, b, n) == 0 and n.value > 0 and b.value > 0
    cnt = FAR + (64 << 20)
    for lse in (cnt - 4, cnt + 4 * n.value - 4):
        refused(ops._lib().kr_op_attention_paged_lse(cache(), 0, s, FAR, 0, FAR + (16 << 20), 0, lse, 0, 256, 8, 0.1,
                                                     FAR + (1 << 30), b.value, cnt, n.value, None), "lse overlaps")
