"""GPU tests of kvc_decode_attn_shared over long caches, against 64 bits: more partials
of a sequence than the fold requests ahead (64) and than it has threads (256), chunks of
one member past the 64 blocks whose ids a wave holds, ending inside a block.  What the
plans of these trees are is tested in test_shared_plan_long.py.

Tolerances are test_gpu_shared.py's and, for the sums over longer chunks and more
partials, (n - 1) 2^-24 of the sum of magnitudes W for n additions one after another, in
the output's numerator and in the sum of weights each: a wave adds 8 tokens of each of a
chunk's `blocks` blocks (one member) or a product of a half block at a time (fewer), the
fold every 4th of `parts` partials and then 4 waves."""
import numpy as np
import pytest

import _oracle as O
import kvc
import q8_ref as Q
from gpu_util import D, NKV, NQ, say
from test_gpu_shared import Forest

pytestmark = pytest.mark.gpu


def check(f, seqs, what, blocks, parts, **k):
    got, want, tol = f.decode(seqs, **k)
    assert np.isfinite(got).all(), what
    mag = np.empty(got.shape)
    for i, s in enumerate(seqs):  # W of an element: within the largest |v| of its dim
        v = np.abs(Q.f64(f.rows[0, s][1])).max(0)
        mag[i] = np.repeat(v, NQ // NKV, axis=0)
    tol = tol + 2 * (8 * blocks + parts / 4 + 4) * 2.0 ** -24 * mag
    worst = (np.abs(got - want) / tol).reshape(len(seqs), -1).max(1)
    assert worst.max() <= 1.0, f"{what}: {worst.max():.2f} times the tolerance at sequence {int(worst.argmax())}"
    say(f"  {what}: {worst.max():.3f} of the tolerance")


@pytest.mark.parametrize("name,prefix,tails,chunk,blocks,parts", [
    ("past 64 partials", 3000, (1, 40, 1000), 1, 2, 100),
    ("past 256 partials", 600, (9000, 3, 100), 1, 2, 300),
    ("past 256 partials, shared and apart", 4000, (7900, 8000), 1, 2, 320),
    ("chunks past 64 and 128 blocks", 1000, (2500, 4500, 30), 1000, 142, 4),
    ("a chunk of 65 blocks", 500, (2080, 1, 64 * 32), 1000, 66, 4),
])
@pytest.mark.parametrize("bf16_out", [True, False])
def test_against_64_bits(name, prefix, tails, chunk, blocks, parts, bf16_out):
    say(f"shared decode: {name} bf16_out={bf16_out}")
    with Forest([(prefix, [(t, 1) for t in tails])], seed=41, decode_chunk_blocks=chunk) as f:
        check(f, f.seqs, "fused, gated", blocks, parts, bf16_out=bf16_out)
        check(f, f.seqs[::-1], "plain", blocks, parts, bf16_out=bf16_out, fused=False, gated=False, seed=30)


@pytest.mark.parametrize("bf16_out", [True, False])
def test_as_the_rule_cuts_it(bf16_out):
    say(f"shared decode of 4 on 65536 bf16_out={bf16_out}")
    with Forest([(65536, [(t, 1) for t in (1, 5, 40, 100)])], seed=42, flags=kvc.FLAG_EXACT_MATH) as f:
        check(f, f.seqs, "fused, gated", 32, 66, bf16_out=bf16_out)


def test_a_refusal_comes_before_the_first_launch():
    """70 sequences are two launches; the last one has no keys: nothing is written"""
    say("shared decode of 70, the last one empty")
    with Forest([(200, 69), (0, 1)], seed=43) as f:
        q = kvc.to_device(O.normal_bf16(70 * NQ * D, 3))
        out = kvc.to_device(np.full(70 * NQ * D, 0x1234, np.uint16))
        with pytest.raises(kvc.KvcError) as e:
            f.ctx.decode_attn_shared(0, f.seqs, q, out, out_dtype=kvc.DTYPE_BF16)
        assert e.value.code == kvc.KVC_ERR_STATE
        f.ctx.sync()
        assert (out.download(np.uint16, 70 * NQ * D) == 0x1234).all()
        q.free()
        out.free()
