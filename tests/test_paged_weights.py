"""Softmax weights that are nothing or nearly nothing: what keys of negligible weight add, rows whose keys all have scores of minus
infinity, and infinite values of keys with small weights; in clusters, in shares that are joined, and in every kernel."""

import math

import pytest
import torch

import libcertex_b200 as certex

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# smallest step of a type, halved
TINY = {torch.float32: 2.0**-150, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def one_row(dtype, n, d, scores, values, heads=2):
    """A sequence of n tokens and a row of queries that sees all: token t has score scores[t] exactly (float32 numbers that the
    type holds, times 8 / 8) and values[t] at every coordinate. Returns the answers of both attentions, of one length each."""
    page = 16
    per = -(-n // page)
    keys, flat = torch.zeros((per * page, 1, d), device="cuda"), torch.zeros((per * page, 1, d), device="cuda")
    keys[:n, 0, 0], flat[:n] = scores, values[:, None, None]
    cache = certex.PagedCache(keys=keys.to(dtype).view(per, page, 1, d), values=flat.to(dtype).view(per, page, 1, d))
    q = torch.zeros((1, heads, d), device="cuda").to(dtype)
    q[..., 0] = 8
    order = torch.arange(per, device="cuda", dtype=torch.int32)[None]
    length = torch.tensor([n], device="cuda", dtype=torch.int32)
    whole = cache.attend(q, order, length, scale=0.125, return_lse=True)
    chosen = cache.attend_selected(q, torch.arange(n, device="cuda")[None, None], scale=0.125, return_lse=True)
    return whole, chosen


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", [(500, 64), (2000, 128), (100_000, 64), (131_072, 128), (3000, 40), (100_000, 256), (2000, 200)])
@pytest.mark.parametrize("first", [True, False])
def test_keys_that_weigh_nothing_add_nothing(n, d, first, dtype):
    """One key of score 64 and value 0; the others have score 0, weight e^-64 < 2^-92, and values of 30 000. The answer is n * 30 000 *
    2^-92.3 at most, < 2^-60, which float16 rounds to 0. It may be off by the rounding of that, by its relative error (the sum of n terms,
    n 2^-24 at most, a weight's 2^-16, twice for a quotient), and in float16 by nothing else: weights are kept to 2^-41 of the
    largest, and these round to 0."""
    scores, values = torch.zeros(n, device="cuda"), torch.full((n,), 30_000.0, device="cuda")
    at = 0 if first else n - 1
    scores[at], values[at] = 64, 0
    want = (n - 1) * 29_952.0 * math.exp(-64) if dtype == torch.bfloat16 else (n - 1) * 30_000.0 * math.exp(-64)
    if dtype == torch.float16:
        off = want + TINY[dtype]
    else:
        off = want * (HALF_STEP[dtype] * 1.01 + 2 * (n * 2.0**-24 + 2.0**-16 + 2.0**-21 + 64 * 2.0**-23)) + TINY[dtype]
    for out, lse in one_row(dtype, n, d, scores, values):
        assert float((out.double() - want).abs().max()) <= off, (float(out.double().max()), want)
        assert float((lse.double() - 64).abs().max()) <= 64 * 2.0**-22


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("score", [-16, -21, -24, -26, -27])
def test_small_weights_are_kept_to_a_part_of_the_largest(score, d, dtype):
    """Every sixteenth key has score 0 and value 0, so that every share's largest weight is 1; the others have weights of e^-16 to e^-27 and
    values of 60 000. In float16 each may be off by 2^-41 of the largest (half of the smallest step of float16, 2^-24, where the largest weight
    is 2^16); for the rest see above."""
    n, value = 48_000, 59_904.0  # (a number of all types)
    scores, values = torch.full((n,), float(score), device="cuda"), torch.full((n,), value, device="cuda")
    scores[::16], values[::16] = 0, 0
    weight = 15 * math.exp(score)
    want = value * weight / (1 + weight)
    off = want * (HALF_STEP[dtype] * 1.01 + 2 * (n * 2.0**-24 + 2.0**-16 + 2.0**-21 + 27 * 2.0**-23)) + TINY[dtype]
    if dtype == torch.float16:
        off += 15 * 2.0**-41 * value
    for out, _ in one_row(dtype, n, d, scores, values):
        assert float((out.double() - want).abs().max()) <= off, (float(out.double().max()), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", [(1, 64), (40, 128), (2000, 128), (20_000, 64), (40, 256), (20_000, 256), (500, 24)])
def test_keys_that_are_seen_with_scores_of_minus_infinity(n, d, dtype):
    """Every key is seen and has score minus infinity: the sum of exponentials is 0, its logarithm minus infinity, and the quotient 0 / 0, as in a
    softmax of 64 bits. One key with a finite score is all that counts."""
    scores, values = torch.full((n,), -math.inf, device="cuda"), torch.full((n,), 3.0, device="cuda")
    want = torch.softmax(scores.double(), 0) @ values.double()
    assert bool(torch.isnan(want))
    for out, lse in one_row(dtype, n, d, scores, values):
        assert bool(torch.isnan(out).all()) and bool((lse == -math.inf).all())
    scores[n // 2], values[n // 2] = -7, 5
    for out, lse in one_row(dtype, n, d, scores, values):
        assert bool((out == 5).all()) and float((lse + 7).abs().max()) <= 7 * 2.0**-22


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("bits", [0, 1, 7, 20, 35, 37, 60, 110])
def test_infinite_values_of_small_weights(bits, d, dtype):
    """A key whose weight is 2^-bits of the largest, or that is the largest, has an infinite value: so is the answer, as long as the weight is more
    than nothing (float16: 2^-38 of the largest). No other key's answer becomes NaN."""
    if dtype == torch.float16 and bits > 38:
        pytest.skip("a weight of nothing in float16")
    n = 300
    scores, values = torch.full((n,), -200.0, device="cuda"), torch.ones(n, device="cuda")
    scores[7] = 0
    scores[250] = -bits * math.log(2)
    for value in (math.inf, -math.inf):
        values[250] = value
        for out, lse in one_row(dtype, n, d, scores, values):
            assert bool((out == value).all()) and bool(torch.isfinite(lse).all())
