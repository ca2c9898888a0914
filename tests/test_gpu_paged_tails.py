"""attention_paged in fp16 where one key stands far above thousands of others
(an attention sink): what the many small weights add up to must be there.

Bound. Those of tests/test_gpu_paged.py, whose relative half step u of a weight
holds for normal fp16 numbers, and fp16's half step below them: the weights are
kept as 2^7 2^(s - m), so a small one is off by at most 2^-25 / 2^7 = 2^-32 of
the weight of the key that set m, whose own weight is 1 of the sum: 2^-32 sum
|v| of the result.
"""

import pytest
import torch

from kernrelay_amd import ops
from tests.conftest import announce

pytestmark = pytest.mark.gpu

HF, U = torch.float16, 2.0 ** -11


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def run_one(D, L, n, sink, gap, cut, G=4, HKV=2, page=16):
    """One sequence of L cached and n new tokens (causal); key `sink` scores
    about `gap` above the others for every query head. (out, reference, bound)."""
    g = torch.Generator(device="cuda").manual_seed(L + n + D)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    total = L + n
    pages = -(-total // page)
    q = rnd(n, HKV * G, D)
    q[..., 0] = 8.0
    k = 0.1 * rnd(pages * page, HKV, D)
    k[..., 0] = 0.0
    k[sink, :, 0] = gap * D ** 0.5 / 8.0
    v = 1.0 + 0.25 * rnd(pages * page, HKV, D)
    v[sink] = 0.0
    q, k, v = q.to(HF), k.to(HF), v.to(HF)
    table = torch.randperm(pages, device="cuda", generator=g)
    kc, vc = (torch.empty(1, pages, page, HKV, D, dtype=HF, device="cuda") for _ in range(2))
    kc[0, table], vc[0, table] = k.view(pages, page, HKV, D), v.view(pages, page, HKV, D)
    cache = ops.make_cache(kc, vc)
    seqs = ops.make_seqs(table.int()[None], ints([L]), ints([0, n]), n)
    space = {}
    if cut:
        nbytes, ncnt = ops.attention_paged_workspace(cache, seqs, HKV * G)
        assert nbytes > 0
        space = dict(ws=torch.empty(nbytes, dtype=torch.uint8, device="cuda"),
                     counters=torch.zeros(ncnt, dtype=torch.int32, device="cuda"))
    out = torch.full_like(q, 9.0)
    ops.attention_paged(cache, 0, seqs, q, out, **space)

    scale = D ** -0.5
    qd = q.double().view(n, HKV, G, D).permute(1, 2, 0, 3)                      # [HKV, G, n, D]
    kd, vd = (x[:total].double().permute(1, 0, 2)[:, None] for x in (k, v))    # [HKV, 1, total, D]
    s = torch.matmul(qd, kd.transpose(2, 3).contiguous()) * scale
    dS = (D + 8) * 2.0 ** -24 * scale * torch.matmul(qd.abs(), kd.abs().transpose(2, 3).contiguous()).amax(-1)
    sees = torch.arange(total, device="cuda") <= L + torch.arange(n, device="cuda")[:, None]
    p = s.masked_fill(~sees, float("-inf")).softmax(-1)
    ref, A = torch.matmul(p, vd), torch.matmul(p, vd.abs())
    small = 2.0 ** -32 * torch.matmul(sees.double(), vd.abs())
    bound = U * (A + ref.abs()) * 1.01 + A * (2 * dS[..., None] + 2.0 ** -18) + 2.0 ** -24 + small
    return out.double().view(n, HKV, G, D).permute(1, 2, 0, 3), ref, bound


@pytest.mark.parametrize("gap", [10.0, 14.0, 16.0, 17.0, 18.0])
@pytest.mark.parametrize("n", [1, 9, 40])
@pytest.mark.parametrize("D", [64, 128])
def test_sink_above_many(gpu, D, n, gap):
    announce("attention_paged fp16 sink D=%d n=%d gap=%g" % (D, n, gap))
    for sink in (0, 7001):
        for cut in (True, False):
            out, ref, bound = run_one(D, 20000, n, sink, gap, cut)
            over = float(((out - ref).abs() / bound).max())
            assert over <= 1.0, "sink %d, cut %s: %g of the bound" % (sink, cut, over)


@pytest.mark.parametrize("n", [1, 40])
def test_largest_weights_of_a_late_maximum(gpu, n):
    """A key so little above the running maximum that it does not move it: the
    largest weights there are, 2^8 times those of the maximum's key."""
    announce("attention_paged fp16 late maximum n=%d" % n)
    for gap in (4.5, 5.2, 5.6):
        for cut in (True, False):
            out, ref, bound = run_one(128, 3001, n, 2990, gap, cut)
            assert bool(((out - ref).abs() <= bound).all())
