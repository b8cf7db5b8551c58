"""GPU tests of 8-bit decode with queries of which a channel is far larger than
the others, over keys that are small there (as attention sinks make them): the
other channels decide the scores and must not lose bits to the large one.

The scores' bound is test_gpu_q8.py's, 2^-22 (B + 2) with B the largest sum |q k|
scale log2(e), which takes every product q k as exact.  With A the largest |q| of
the head, a fixed-point q whose last place is A 2^-60 or less is off by that
times sum |k| scale log2(e): here less than 2^-24 (B + 2), which is checked, and
so within what the 16 partial sums leave."""
import numpy as np
import pytest

import _oracle as O
import q8_ref as Q
from gpu_util import D, NKV, NQ, say
from test_gpu_q8 import SCALE, check

pytestmark = pytest.mark.gpu


def small(qb, k, big):
    assert np.abs(Q.f64(qb)).max() * 2.0 ** -60 * np.abs(k).sum(-1).max() * SCALE * Q.LOG2E < 2.0 ** -24 * (big + 2)


@pytest.mark.parametrize("power", [0, 10, 13, 16, 20, 22, 30])
@pytest.mark.parametrize("top", [1.0, 1.3125, 1.9921875])
def test_decode_with_a_large_query_channel(power, top):
    """channel 5 of q is top 2^power; the keys' is 2^-power of their others, or 0"""
    say(f"decode8, q channel of {top} 2^{power}")
    n = 200
    rng = np.random.default_rng(power)
    k, v = rng.normal(size=(n, NKV, D)) * 4, rng.normal(size=(n, NKV, D))
    k[:, :, 5] *= 2.0 ** -power if power < 20 else 0.0
    q = rng.normal(size=(1, NQ, D))
    q[:, :, 5] = top * 2.0 ** power
    q[:, 7, 5] *= -1
    kb, vb, qb = Q.bf16_bits(k), Q.bf16_bits(v), Q.bf16_bits(q)
    with Q.Filled([0], seed=400, extra=n) as f:
        s = f.seqs[0]
        f.add([s], n, rows=[kb, vb])
        f.ctx.kv_quantize([s])
        got = f.run(lambda a, o: f.ctx.decode_attn(0, [s], a, o), (1, NQ, D), np.float32, qb)
    n8 = n // 32 * 32
    k, v = Q.values(kb, n8), Q.values(vb, n8)
    want, mag, big, dig = Q.attend(Q.f64(qb), k, v, SCALE, digits=True)
    small(qb, k, big)
    check(got.astype(np.float64)[0], want[0], mag[0], big, False, False, "large channel", dig[0])


def test_decode_with_heads_of_different_ranges():
    """heads of one kv head whose ranges need more bits beside heads that do not,
    over several blocks per wave, and zeros beside the large channel"""
    say("decode8, mixed heads")
    n = 2000
    rng = np.random.default_rng(9)
    k, v = rng.normal(size=(n, NKV, D)) * 4, rng.normal(size=(n, NKV, D))
    k[:, :, 200] = 0.0
    q = rng.normal(size=(2, NQ, D))
    q[:, 1::3, 200] = 2.0 ** 25
    q[1, 2] = 0.0
    q[1, 2, 200] = 2.0 ** 25
    kb, vb, qb = Q.bf16_bits(k), Q.bf16_bits(v), Q.bf16_bits(q)
    with Q.Filled([0, 0], seed=401, extra=n) as f:
        f.add(f.seqs, n, rows=[kb, vb])
        f.ctx.kv_quantize(f.seqs)
        got = f.run(lambda a, o: f.ctx.decode_attn(0, f.seqs, a, o), (2, NQ, D), np.float32, qb)
    n8 = n // 32 * 32
    k, v = Q.values(kb, n8), Q.values(vb, n8)
    for i in range(2):
        want, mag, big, dig = Q.attend(Q.f64(qb[i:i + 1]), k, v, SCALE, digits=True)
        small(qb, k, big)
        check(got[i].astype(np.float64), want[0], mag[0], big, False, False, f"row {i}", dig[0])
