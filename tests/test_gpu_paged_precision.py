"""How exact the paged attention is where its weights range far: a dominant first token (what an attention sink is), and
the errors that remain beside the rounding of the output."""
import pytest
import torch

import paged_ref as R
from smlm_b200 import paged
from test_gpu_paged import BF16, F16, F32, make, roomy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hq,hkv,d,page", [(1, 1, 64, 16), (12, 1, 64, 16), (2, 2, 256, 16), (4, 2, 32, 4),
                                           (9, 1, 128, 32)])
@pytest.mark.parametrize("gap", [15.0, 17.5, 20.0])
@pytest.mark.parametrize("room", [False, True])
def test_weights_far_below_the_largest(dtype, hq, hkv, d, page, gap, room):
    """The first token's score is `gap` above all others and its value is 0, so the output is what the small weights
    carry. Each weight is held to 16 bits or more (2^-16 of it; fp16: or to 2^-40 of the largest weight), exponents of
    up to 30 in fp32 add less than 2^-17, the fp32 sums n 2^-24, and the output is rounded once."""
    lens = [32, 600, 7]
    q, k, v, table, lengths = make(lens, hq, hkv, d, page, dtype, seed=d + hq, stale=0.0)
    q.zero_()
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    v.copy_((v.float() * 100 + 700).to(dtype))
    first = table[:, 0].long()
    k[first, :, 0, 0] = gap
    v[first, :, 0] = 0.0
    out, lse = paged.paged_attention(q, k, v, roomy(table, page) if room else table, lengths, scale=1.0, return_lse=True)
    ref, rlse, mag, _ = R.attention(q, k, v, table, lengths, 1.0)
    n = torch.tensor(lens, dtype=torch.float64).view(-1, 1, 1)
    bound = R.UNIT[dtype] * ref.abs() + mag * (2.0 ** -15 + n * 2.0 ** -24) + 2.0 ** -25
    if dtype == F16:
        bound = bound + n * 2.0 ** -40 * float(v.abs().max())
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    # the logarithm of a sum of 1 and small weights around the exponent `gap`: both rounded to fp32
    assert bool(((lse.double().cpu() - rlse).abs() <= 2.0 ** -21 * rlse.abs() + 2.0 ** -20).all())
