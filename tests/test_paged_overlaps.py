"""Outputs that share memory with what a launch reads are refused, before
anything reaches a GPU. (Placements that share none run in
tests/test_gpu_paged_batches.py: here every call must end at its check.)"""

import random

import pytest

from kernrelay_amd import ops
from tests.test_paged_refusals import cache, refused, rope, seqs

Q = 1 << 24       # addresses that nothing reads: far from the cache's
FAR = 1 << 40
D = 128


def attention(q, ldq, out, ldo, rows, HQ, c=None, layer=0):
    return ops._lib().kr_op_attention_paged(c or cache(k=FAR, v=2 * FAR), layer, seqs(), q, ldq, out, ldo, rows, HQ,
                                            0.1, None, 0, None, 0, None)


@pytest.mark.parametrize("seed", range(40))
def test_rows_that_meet(seed):
    """Placements drawn until some element is in both, counted one by one."""
    rng = random.Random(seed)
    while True:
        rows, HQ = rng.choice((1, 2, 3, 7, 20)), rng.choice((4, 8))
        width = HQ * D
        ldq = width + 8 * rng.choice((0, 1, rng.randint(0, 400)))
        ldo = ldq if rng.random() < 0.5 else width + 8 * rng.randint(0, 400)
        shift = 8 * rng.randint(-(rows + 1) * ldo // 8, (rows + 1) * ldq // 8)
        a = {i * ldq + x for i in range(rows) for x in range(0, width, 8)}
        b = {shift + i * ldo + x for i in range(rows) for x in range(0, width, 8)}
        if a & b:
            break
    refused(attention(Q, ldq, Q + 2 * shift, ldo, rows, HQ), "out overlaps q")


def test_out_in_the_cache():
    c = cache(k=FAR, v=FAR + (1 << 20))  # 2 layers of 2 MB each, k and v side by side in them
    layer, size = 2 << 20, 2 * 8 * 16 * 4 * 128
    for l in (0, 1):
        for base in (FAR, FAR + (1 << 20)):
            first, last = base + l * layer, base + l * layer + size - 16
            refused(attention(Q, 0, first, 0, 2, 8, c, l), "out overlaps the cache")
            refused(attention(Q, 0, last, 0, 2, 8, c, l), "out overlaps the cache")
            refused(attention(Q, 0, first - 2 * 2 * 8 * 128 + 16, 0, 2, 8, c, l), "out overlaps the cache")


def plain(q=Q, ldq=0, k=2 * Q, ldk=0, q_out=3 * Q, ldqo=0, k_out=4 * Q, ldko=0, rows=5):
    return ops._lib().kr_op_qk_norm_rope(0, rope(cos_t=FAR, sin_t=FAR), q, ldq, k, ldk, q_out, ldqo, k_out, ldko, None,
                                         rows, 8, 2, None)


def test_rotation_outputs():
    row = 2 * 8 * D
    for kw in (dict(q_out=Q + 16), dict(q_out=Q + row), dict(q_out=Q, ldqo=8 * D + 8), dict(q_out=2 * Q),
               dict(q_out=2 * Q + 512), dict(q_out=2 * Q - row)):
        refused(plain(**kw), "q_out overlaps an input")
    for kw in (dict(k_out=2 * Q + 16), dict(k_out=2 * Q, ldko=3 * D), dict(k_out=Q + row), dict(k_out=3 * Q),
               dict(k_out=3 * Q - 16)):
        refused(plain(**kw), "k_out overlaps")


def test_rotation_into_the_cache():
    def call(q_out, v=3 * Q, c=cache(k=FAR, v=2 * FAR)):
        return ops._lib().kr_op_qk_norm_rope_cache(rope(cos_t=4 * FAR, sin_t=4 * FAR), c, 1, Q, 0, 2 * Q, 0, v, 0, q_out,
                                                   0, 4 * FAR, 4 * FAR, 5, 8, None)
    refused(call(Q + 16), "q_out overlaps an input")
    refused(call(2 * Q), "q_out overlaps an input")
    refused(call(3 * Q + 16), "q_out overlaps an input")
    refused(call(FAR + (2 << 20)), "q_out overlaps the cache")
    refused(call(2 * FAR + (2 << 20) + 64), "q_out overlaps the cache")
