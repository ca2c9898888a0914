"""attention_paged of few rows a key head (single tokens, small trees): the
weights lose nothing on their way to the matrix cores, so that a result is
rounded once.

Bound, with u half a step of the type (2^-8 bf16, 2^-11 fp16): u |o| for the
store; 2 u^2 A, A = sum p |v| / sum p, for what two 16-bit parts leave of a weight
(the first is cut off: the second is below 2u of it, and rounded); a score is an fp32 sum of D products, scaled: off by at most dS = (D + 8) 2^-24
scale max_j sum |q k|, and so is its weight, relatively (twice: above and below
the bar); the exponent's argument, the hardware's 2^x and the 2^-23 that the
second part has over add less than 2^-18. fp16: 2^-24 for results below its
normal range; its second part is off by half a step and the step that it has
over, 1.5 2^-24, where weights are 2^7 2^(s - m), the largest s - m 0 at least:
1.5 2^-31 sum |v|.
"""

import pytest
import torch

from tests.conftest import announce
from tests.test_gpu_paged import BF, HALF, HF, Batch, ints

pytestmark = pytest.mark.gpu

CASES = [(14, 2, 64, BF, 16, [37], [1], "causal"), (28, 4, 128, BF, 16, [0, 1, 63, 64, 65, 700], [1] * 6, "causal"),
         (32, 8, 128, HF, 24, [5000, 31], [1, 1], "causal"), (8, 8, 64, HF, 7, [100, 257], [1, 1], "causal"),
         (16, 2, 64, HF, 5, [3000], [4], "tree"), (28, 4, 128, BF, 32, [900, 20, 0], [4, 3, 2], "tree"),
         (4, 4, 128, BF, 48, [1200, 5], [32, 30], "causal"), (12, 4, 64, BF, 128, [20000, 0, 9000], [1, 1, 1], "causal")]


@pytest.mark.parametrize("HQ,HKV,D,dt,page,lens,news,form", CASES)
@pytest.mark.parametrize("cut", [True, False])
def test_one_rounding(gpu, HQ, HKV, D, dt, page, lens, news, form, cut):
    announce("attention_paged one rounding %s" % ((HQ, HKV, D, dt, page, lens, news, form, cut),))
    b = Batch(31, HQ, HKV, D, dt, page, lens, news, form=form)
    out, scale, u, G, r = b.run(cut=cut), D ** -0.5, HALF[dt], HQ // HKV, 0
    for s, (a, n) in enumerate(zip(lens, news)):
        lo = b.starts[s]
        ids = ints(b.table[s][:-(-(a + n) // page)]).long()
        k, v = (c[1][ids].reshape(-1, HKV, D)[:a + n].double().permute(1, 0, 2)[:, None] for c in (b.k, b.v))
        sees = torch.ones(n, a + n, dtype=torch.bool)
        sees[:, a:] = torch.tensor(b.seen[r:r + n])
        sees, r = sees.cuda(), r + n
        q = b.q[lo:lo + n].double().view(n, HKV, G, D).permute(1, 2, 0, 3)
        kt = k.transpose(2, 3).contiguous()
        p = (torch.matmul(q, kt) * scale).masked_fill(~sees, float("-inf")).softmax(-1)
        dS = (D + 8) * 2.0 ** -24 * scale * torch.matmul(q.abs(), kt.abs()).amax(-1)[..., None]
        ref, A = torch.matmul(p, v), torch.matmul(p, v.abs())
        bound = 1.01 * u * ref.abs() + A * (2 * u * u + 2 * dS + 2.0 ** -18)
        if dt == HF:
            bound = bound + 2.0 ** -24 + 1.5 * 2.0 ** -31 * torch.matmul(sees.double(), v.abs())
        got = out[lo:lo + n].double().view(n, HKV, G, D).permute(1, 2, 0, 3)
        over = float(((got - ref).abs() / bound).max())
        assert over <= 1.0, "sequence %d: %g of the bound" % (s, over)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("D,dt", [(64, HF), (128, BF), (64, BF), (128, HF)])
def test_seen_values_that_are_no_numbers(gpu, D, dt, value):
    """A cached value that every row sees is in every result as it is: an
    infinite one, with the weight 1 or any other, is no NaN."""
    announce("attention_paged seen %s D=%d %s" % (value, D, dt))
    b = Batch(32, 8, 2, D, dt, 16, [900, 40], [2, 3])
    for s, pos, head, cols in ((0, 0, 0, slice(0, 2)), (0, 500, 1, slice(3, 4)), (0, 899, 0, slice(D - 1, D)),
                               (1, 7, 1, slice(0, D))):
        b.v[1, b.table[s][pos // 16], pos % 16, head, cols] = value
    b.check(b.run())
    b.check(b.run(cut=False))
    # all keys alike: every weight is 1 (times the factor of its type)
    b.k[1].nan_to_num_(0.0).zero_()
    b.check(b.run())
    b.check(b.run(cut=False))
