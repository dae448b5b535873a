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


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq,hkv,d,n", [(6, 6, 64, 24), (12, 1, 64, 24), (2, 2, 256, 24), (6, 6, 64, 500)])
def test_rounding_the_output_is_the_only_error_that_shows(dtype, hq, hkv, d, n):
    """The squared error is that of the float64 result rounded to the type: weights rounded once to the type would add
    half as much again at 24 tokens."""
    q, k, v, table, lengths = make([n] * 32, hq, hkv, d, 16, dtype, seed=n + d)
    out = paged.paged_attention(q, k, v, table, lengths).double().cpu()
    ref = R.attention(q, k, v, table, lengths, d ** -0.5)[0]
    rounded = ref.to(dtype).double()
    assert float((out - ref).square().mean()) <= 1.1 * float((rounded - ref).square().mean())


@pytest.mark.parametrize("n", [900, 20000])
def test_fp32_error_of_long_sums(n):
    """The root mean square error of fp32 caches is below 2^-20 of the outputs'."""
    q, k, v, table, lengths = make([n], 6, 2, 64, 16, F32, seed=n)
    out = paged.paged_attention(q, k, v, table, lengths).double().cpu()
    ref = R.attention(q, k, v, table, lengths, 0.125)[0]
    assert float((out - ref).square().mean().sqrt()) <= 2.0 ** -20 * float(ref.square().mean().sqrt())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("room", [False, True])
def test_peaked_scores_over_values_with_a_common_part(dtype, room):
    """Scores of tens and values around 4: the weights have to add up to the sum they are divided by. The products are
    exact in fp32, their sum of 64 terms is off by at most 64 2^-24 of its terms' sizes (fp32 caches: 2^-19)."""
    q, k, v, table, lengths = make([40, 333, 1500], 8, 2, 64, 16, dtype, seed=11, stale=0.0)
    q, v = (q.float() * 6).to(dtype), (v.float() * 0.25 + 4).to(dtype)
    out = paged.paged_attention(q, k, v, roomy(table, 16) if room else table, lengths)
    ref, _, mag, reach = R.attention(q, k, v, table, lengths, 0.125)
    score = 2.0 ** -19 if dtype == F32 else 64 * 2.0 ** -24
    n = lengths.double().cpu().view(-1, 1, 1)
    bound = R.UNIT[dtype] * ref.abs() + mag * (2 * score * reach + 2.0 ** -15 + n * 2.0 ** -24)
    if dtype == F16:
        bound = bound + n * 2.0 ** -40 * float(v.abs().max())
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (256, 32), (32, 4)])
@pytest.mark.parametrize("room", [False, True])
def test_not_a_bit_follows_from_tokens_that_are_not_seen(dtype, d, page, room):
    """Whatever lies past a length, in a hole's stand-in and outside the window: the output is the same to the bit."""
    lens, window, sinks = [5, 40, 333], 70, 3
    want = None
    for bad in (0.0, float("nan"), float("inf"), -3e4):
        q, k, v, table, lengths = make(lens, 4, 2, d, page, dtype, seed=d, stale=bad)
        rows = table.tolist()
        for b, n in enumerate(lens):
            for j in range(sinks, n - window):
                k[rows[b][j // page], :, j % page] = bad
                v[rows[b][j // page], :, j % page] = bad
        got = paged.paged_attention(q, k, v, roomy(table, page) if room else table, lengths, window=window, sinks=sinks,
                                    return_lse=True)
        want = want or got
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), bad
