"""GPU tests of how exact kvc_beam_select's sums are, against 64 bits.

In units of 2^-24, relative to the sum of a row's exponentials: the argument of an
exponential is off by 2.22 |x - max| at most (a difference, a product, the constant's own
0.22; on the way over the maxima of lane, wave and chunk the distances add up to that),
and the mean of max - x under the softmax is at most its entropy, log vocab; each of the
four exponentials is off by 2, the products with two of them by 1; up to 32 terms are
added pairwise, 5, then 64 lanes and 4 waves, 8; the logarithm of the mantissa is the
hardware's, 1; chunks are added in 64 bits.  Together 2.22 log vocab + 24."""
import math

import numpy as np
import pytest

import kvc
from gpu_util import say
from test_gpu_beam import BF16, F32, Case, ctx, noise, scores_of, values  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0**-24


def log_sum_error(vocab):
    return (2.22 * math.log(vocab) + 24) * U


@pytest.mark.parametrize("shape", [(1, 4, 151936), (8, 8, 70001), (4, 8, 151936), (3, 5, 1000), (1, 64, 8192)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [0.01, 1.0, 6.0])
def test_within_the_bound(ctx, shape, dtype, scale):  # noqa: F811
    say(f"beam sums {shape} {dtype} {scale}")
    g, b, v = shape
    n_out = 32
    with Case(noise(shape, 31, scale), dtype, scores_of((g, b), 32), n_out, 0, 1) as c:
        score, beam, token = c.run(ctx)
        val, _ = values(c.logits, c.scores)
    worst = 0.0
    for i in range(g):
        want = -np.sort(-val[i].reshape(-1))[:n_out]
        off = np.abs(score[i] - want) - np.abs(want) * U
        assert (off <= log_sum_error(v)).all(), (i, off.max() / U)
        # between beams: none left out that is better by more than both sums' errors
        assert (want - val[i][beam[i], token[i]] <= 2 * log_sum_error(v)).all()
        worst = max(worst, off.max() / U)
    say(f"  {worst:.1f} of {log_sum_error(v) / U:.1f} units")


def rows_with_small_terms(vocab, dtype):
    """Among the tokens that one lane takes a logit of 0 comes first and all others are
    -17.375, whose exponential is 0.478 units: added to the 1 one by one each is lost."""
    t = np.arange(vocab)
    one = (t % 256 < 64) & (t % (8 if dtype == BF16 else 4) == 0)
    return np.where(one, 0.0, -17.375).astype(np.float32), one


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_small_terms_are_kept(ctx, dtype):  # noqa: F811
    say(f"beam sums of many small terms {dtype}")
    row, one = rows_with_small_terms(151936, dtype)
    x = np.tile(row, (4, 8, 1))
    # scores that leave next to nothing of the result, so that its rounding is nothing
    scores = np.full((4, 8), np.log(one.sum()), np.float32)
    with Case(x, dtype, scores, 16) as c:
        score, beam, token = c.run(ctx)
    want = float(scores[0, 0]) - math.log(one.sum() + (~one).sum() * math.exp(-17.375))
    assert abs(want) < 2.0**-18
    # exponentials of 0 are exact and the others' errors vanish beside them; lanes are alike,
    # so that their sums double exactly: the additions in a lane (4 or 5) and the logarithm
    # are left
    assert (np.abs(score - want) <= (5.1 if dtype == F32 else 6.1) * U).all(), np.abs(score - want).max() / U
    assert (beam == 0).all() and np.array_equal(token[0], np.flatnonzero(one)[:16])


@pytest.mark.parametrize("dtype,less", [(F32, 3.5), (BF16, 8.0)])
def test_close_beams_come_in_the_order_of_their_sums(ctx, dtype, less):  # noqa: F811
    """Beam 1 has the lower score, by `less` units, but not the small terms (7.2 or 14.8
    units of the sum): it is the better one.  (The additions lose 1.2 units of them: 0.48 to
    the 1, then 0.96, while later sums of them round up.  The logarithm may take 1.)"""
    say(f"beam sums of close beams {dtype}")
    row, one = rows_with_small_terms(151936, dtype)
    x = np.tile(row, (16, 2, 1))
    x[:, 1][:, ~one] = -np.inf
    scores = np.tile(np.array([0.0, -less * U], np.float32), (16, 1))
    with Case(x, dtype, scores, 16) as c:
        _, beam, token = c.run(ctx)
    assert (beam == 1).all() and np.array_equal(token[0], np.flatnonzero(one)[:16])
