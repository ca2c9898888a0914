"""What the paged cache's entry points refuse, before anything reaches a GPU:
the C entries get addresses that nothing reads, the wrappers CPU tensors."""

import ctypes

import pytest
import torch

from kernrelay_amd import ops

A = 1 << 20  # a 16-byte aligned address; every call below ends before it is used


def cache(**kw):
    f = dict(k=A, v=A, layer_stride=1 << 20, page_stride=16 * 4 * 128, token_stride=4 * 128, head_stride=128, layers=2,
             pages=8, page_size=16, heads=4, head_dim=128, dtype=ops.KR_BF16)
    f.update(kw)
    return ops.KrCache(**f)


def seqs(**kw):
    f = dict(table=A, ld_table=4, lens=A, starts=A, tree=None, ld_tree=0, table_pages=4, seqs=3, max_new=5,
             tree_words=0)
    f.update(kw)
    return ops.KrSeqs(**f)


def rope(**kw):
    f = dict(cos_t=A, sin_t=A, q_gamma=A, k_gamma=A, positions=64, head_dim=128, table_dtype=ops.KR_BF16, chain=0,
             eps=1e-6)
    f.update(kw)
    return ops.KrRope(**f)


def refused(rc, text):
    assert rc != 0 and text in ops._lib().kr_ops_last_error().decode(), ops._lib().kr_ops_last_error()


BAD_CACHES = [
    (dict(k=None), "needs a cache"), (dict(v=None), "needs a cache"), (dict(dtype=ops.KR_F32), "bf16 or f16"),
    (dict(head_dim=96), "head_dim"), (dict(pages=0), "empty"), (dict(page_size=-1), "empty"),
    (dict(k=A + 8), "aligned"),
    (dict(token_stride=516), "strides"), (dict(head_stride=64), "strides"), (dict(page_stride=0), "strides"),
    (dict(page_stride=1 << 31), "too large"),
]
BAD_SEQS = [
    (dict(table=None), "page table"), (dict(lens=None), "lengths"), (dict(starts=None), "starts"),
    (dict(seqs=-1), "size"),
    (dict(max_new=-2), "size"), (dict(table_pages=0), "size"), (dict(ld_table=3), "overlap"),
    (dict(tree=A, tree_words=0), "tree"), (dict(tree=A, tree_words=2, ld_tree=1), "tree"),
    (dict(tree=A, tree_words=1, ld_tree=1, max_new=65), "too few words"),
]


def attention(c, s, layer=0, q=A, ldq=0, out=A, ldo=0, rows=5, HQ=8, scale=0.1):
    return ops._lib().kr_op_attention_paged(c, layer, s, q, ldq, out, ldo, rows, HQ, scale, None, 0, None, 0, None)


@pytest.mark.parametrize("field,text", BAD_CACHES)
def test_bad_caches(field, text):
    c, L = cache(**field), ops._lib()
    ids = (ctypes.c_int32 * 1)(0)
    refused(attention(c, seqs()), text)
    b, n = ctypes.c_size_t(0), ctypes.c_int(0)
    refused(L.kr_op_attention_paged_workspace(c, seqs(), 8, b, n), text)
    refused(L.kr_op_cache_copy_pages(c, ids, (ctypes.c_int32 * 1)(1), 1, None), text)
    refused(L.kr_op_cache_compact(c, seqs(), A, 4, 4, A, None), text)
    if "head_dim" not in field:
        refused(L.kr_op_qk_norm_rope_cache(rope(), c, 0, A, 0, A, 0, A, 0, A, 0, A, A, 4, 8, None),
                "dtype" if "dtype" in field else text)


@pytest.mark.parametrize("field,text", BAD_SEQS)
def test_bad_sequences(field, text):
    s = seqs(**field)
    refused(attention(cache(), s), text)
    refused(ops._lib().kr_op_cache_compact(cache(), s, A, 4, 4, A, None), text)


@pytest.mark.parametrize("kw,text", [
    (dict(layer=2), "no such layer"), (dict(layer=-1), "no such layer"), (dict(HQ=6), "multiple"),
    (dict(HQ=0), "multiple"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(q=None), "missing"), (dict(out=A + 2), "aligned"), (dict(ldq=1028), "multiples of 8"),
    (dict(rows=-1), "rows")])
def test_attention_arguments(kw, text):
    refused(attention(cache(), seqs(), **kw), text)


def test_attention_long_tables():
    refused(attention(cache(), seqs(table_pages=1 << 27, ld_table=1 << 27)), "too many tokens")


def test_null_handles_and_empty_launches():
    L = ops._lib()
    refused(L.kr_op_attention_paged(None, 0, seqs(), A, 0, A, 0, 1, 8, 0.1, None, 0, None, 0, None), "needs a cache")
    refused(L.kr_op_attention_paged(cache(), 0, None, A, 0, A, 0, 1, 8, 0.1, None, 0, None, 0, None), "page table")
    refused(L.kr_op_qk_norm_rope(0, None, A, 0, A, 0, A, 0, A, 0, None, 4, 8, 2, None), "tables")
    refused(L.kr_op_qk_norm_rope_cache(rope(), None, 0, A, 0, A, 0, A, 0, A, 0, A, A, 4, 8, None), "cache")
    # nothing to do: no launch, no error
    assert attention(cache(), seqs(), rows=0) == 0 and attention(cache(), seqs(seqs=0)) == 0
    assert attention(cache(), seqs(max_new=0)) == 0
    assert L.kr_op_cache_copy_pages(cache(), None, None, 0, None) == 0
    assert L.kr_op_cache_compact(cache(), seqs(), None, 0, 0, None, None) == 0
    assert L.kr_op_qk_norm_rope(0, rope(), A, 0, A, 0, A, 0, A, 0, None, 0, 8, 2, None) == 0


@pytest.mark.parametrize("r,kw,text", [
    (dict(cos_t=None), {}, "tables"), (dict(positions=0), {}, "tables"), (dict(k_gamma=None), {}, "gains"),
    (dict(table_dtype=ops.KR_F16), {}, "tables"), (dict(head_dim=80), {}, "head_dim"), (dict(eps=-1.0), {}, "eps"),
    (dict(sin_t=A + 4), {}, "aligned"), ({}, dict(dtype=ops.KR_F32), "dtype"), ({}, dict(rows=-1), "rows"),
    ({}, dict(HQ=0), "head"), ({}, dict(HKV=0), "head"), ({}, dict(ldq=1028), "multiples of 8"),
    ({}, dict(q=None), "missing"),
    ({}, dict(rows=1 << 30), "too many rows")])
def test_rope_arguments(r, kw, text):
    a = dict(dtype=ops.KR_BF16, q=A, ldq=0, rows=4, HQ=8, HKV=2)
    a.update(kw)
    refused(ops._lib().kr_op_qk_norm_rope(a["dtype"], rope(**r), a["q"], a["ldq"], A, 0, A, 0, A, 0, None, a["rows"],
                                          a["HQ"], a["HKV"], None), text)


def test_rope_cache_arguments():
    L = ops._lib()
    call = lambda r=rope(), c=cache(), layer=0, v=A, slots=A: L.kr_op_qk_norm_rope_cache(  # noqa: E731
        r, c, layer, A, 0, A, 0, v, 0, A, 0, A, slots, 4, 8, None)
    refused(call(r=rope(head_dim=64)), "differ in head_dim")
    refused(call(layer=2), "no such layer")
    refused(call(v=None), "slots and v")
    refused(call(slots=None), "slots and v")


@pytest.mark.parametrize("src,dst,text", [
    ([0], [8], "no such page"), ([-1], [1], "no such page"), ([0, 1], [2, 2], "written twice"),
    ([0, 1], [2, 1], "both read and written"), ([0, 3], [3, 4], "both read and written")])
def test_copy_arguments(src, dst, text):
    ids = ctypes.c_int32 * len(src)
    refused(ops._lib().kr_op_cache_copy_pages(cache(), ids(*src), ids(*dst), len(src), None), text)


def test_copy_and_compact_sizes():
    L = ops._lib()
    refused(L.kr_op_cache_copy_pages(cache(), None, None, 1, None), "ids")
    refused(L.kr_op_cache_copy_pages(cache(), None, None, -1, None), "negative")
    refused(L.kr_op_cache_compact(cache(), seqs(), A, 257, 257, A, None), "at most 256")
    refused(L.kr_op_cache_compact(cache(), seqs(), A, 3, 4, A, None), "overlap")
    refused(L.kr_op_cache_compact(cache(), seqs(), None, 4, 4, A, None), "paths")


def tensors(dt=torch.bfloat16):
    k = torch.zeros(2, 8, 16, 4, 128, dtype=dt)
    return k, torch.zeros_like(k)


def test_wrappers_refuse_shapes_and_types():
    k, v = tensors()
    with pytest.raises(ValueError, match="agree"):
        ops.make_cache(k, v[:, :4])
    with pytest.raises(ValueError, match="agree"):
        ops.make_cache(k, v.half())
    with pytest.raises(ValueError, match="agree"):  # equal shapes, other strides
        ops.make_cache(k, v.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(ValueError, match="contiguous"):
        ops.make_cache(k.transpose(3, 4), v.transpose(3, 4))
    with pytest.raises(ValueError, match="layers"):
        ops.make_cache(k[0, 0], v[0, 0])
    with pytest.raises(RuntimeError, match="device tensors"):  # no CPU fallback
        ops.make_cache(k, v)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="table"):
        ops.make_seqs(i32(3, 4).long(), i32(3), i32(4), 1)
    with pytest.raises(ValueError, match="table"):
        ops.make_seqs(i32(4, 3).t(), i32(3), i32(4), 1)
    with pytest.raises(ValueError, match="lens"):
        ops.make_seqs(i32(3, 4), i32(2), i32(4), 1)
    with pytest.raises(ValueError, match="starts"):
        ops.make_seqs(i32(3, 4), i32(3), i32(3), 1)
    with pytest.raises(ValueError, match="max_new"):
        ops.make_seqs(i32(3, 4), i32(3), i32(4), -1)
    with pytest.raises(ValueError, match="too few words"):
        ops.make_seqs(i32(3, 4), i32(3), i32(4), 65, tree=i32(9, 1).long())
    with pytest.raises(ValueError, match="tree"):
        ops.make_seqs(i32(3, 4), i32(3), i32(4), 5, tree=i32(9, 1))
    t = torch.zeros(64, 128)
    with pytest.raises(ValueError, match="cos and sin"):
        ops.make_rope(t, t[:32])
    with pytest.raises(ValueError, match="gains"):
        ops.make_rope(t, t, q_gamma=torch.ones(128))
    with pytest.raises(ValueError, match="gains"):
        ops.make_rope(t, t, q_gamma=torch.ones(128), k_gamma=torch.ones(64))


def test_wrappers_check_their_tensors():
    """On handles that no call reaches the GPU with."""
    c, s, r = cache(), seqs(), rope()
    c.torch_dtype, c.device, s.device, s.rows, r.device, r.torch_dtype = torch.bfloat16, 0, 0, 4, 0, torch.bfloat16
    c.keep, s.keep = tensors(), [torch.zeros(3, 4, dtype=torch.int32)]
    q = torch.zeros(4, 8, 128, dtype=torch.bfloat16)
    k = torch.zeros(4, 4, 128, dtype=torch.bfloat16)
    n = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="head_dim"):
        ops.qk_norm_rope(r, q[..., :64], k, q, k)
    with pytest.raises(ValueError, match="q_out must be"):
        ops.qk_norm_rope(r, q, k, q[:3], k)
    with pytest.raises(ValueError, match="k must be"):
        ops.qk_norm_rope(r, q, k.half(), q, k)
    with pytest.raises(ValueError, match="gains"):
        ops.qk_norm_rope(r, q.half(), k.half(), q.half(), k.half())
    with pytest.raises(ValueError, match="packed"):
        ops.qk_norm_rope(r, q.transpose(0, 1).contiguous().transpose(0, 1), k, q, k)
    with pytest.raises(ValueError, match="overlap"):
        ops.qk_norm_rope(r, q, k, q[:1].expand(4, 8, 128), k)
    with pytest.raises(ValueError, match="positions"):
        ops.qk_norm_rope(r, q, k, q, k, positions=n.int())
    with pytest.raises(ValueError, match="slots"):
        ops.qk_norm_rope_cache(r, c, 0, q, k, k, q, n, n[:3])
    with pytest.raises(ValueError, match="v must be"):
        ops.qk_norm_rope_cache(r, c, 0, q, k, k[:, :2], q, n, n)
    with pytest.raises(ValueError, match="out must be"):
        ops.attention_paged(c, 0, s, q, q.float())
    with pytest.raises(ValueError, match="too few rows"):
        ops.attention_paged(c, 0, s, torch.zeros(5, 8, 128, dtype=torch.bfloat16), q)
    with pytest.raises(ValueError, match="differ in length"):
        ops.cache_copy_pages(c, [1], [2, 3])
    with pytest.raises(ValueError, match="path must be"):
        ops.cache_compact(c, s, n.view(1, 4), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="path_lens"):
        ops.cache_compact(c, s, torch.zeros(3, 4, dtype=torch.int32), n)


def test_wrappers_refuse_rows_that_overlap():
    """A broadcast row has stride 0: read at its width it would lead past the
    tensor's memory."""
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="overlap"):
        ops.make_seqs(i32(1, 4).expand(3, 4), i32(3), i32(4), 1)
    with pytest.raises(ValueError, match="overlap"):
        ops.make_seqs(i32(3, 4), i32(3), i32(4), 5, tree=i32(1, 2).long().expand(9, 2))
    with pytest.raises(ValueError, match="overlap"):
        ops.make_seqs(i32(9).as_strided((3, 4), (2, 1)), i32(3), i32(4), 1)
    with pytest.raises(ValueError, match="max_new"):  # does not fit the handle
        ops.make_seqs(i32(3, 4), i32(3), i32(4), (1 << 32) + 1)
    c, s = cache(), seqs()
    c.device = s.device = 0
    with pytest.raises(ValueError, match="overlap"):
        ops.cache_compact(c, s, i32(1, 4).expand(3, 4), i32(3))
