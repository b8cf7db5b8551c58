"""GPU tests of fp32 results on a context that has 8-bit blocks, in launches of
which no sequence holds one: sequences too short for a block, or kept in bf16 by
keep_tokens.  They are as exact as those beside an 8-bit neighbour, so the bounds
are test_gpu_q8.py's (weights in fp32, no bf16 rounding of them); without 8-bit
blocks in the context, and in bf16, results stay those of the bf16 kernels, bit
for bit."""
import numpy as np
import pytest

import _oracle as O
import kvc
import q8_ref as Q
from gpu_util import D, NKV, NQ, say
from test_gpu_q8 import SCALE, check, decode_case, prefill_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 2, 7, 16, 30, 31])
@pytest.mark.parametrize("fused", [False, True])
def test_decode_of_sequences_shorter_than_a_block(n, fused):
    say(f"fp32 decode {n} fused {fused}")
    decode_case([n], 0, fused, n % 2 == 1, False, seed=300 + n)


@pytest.mark.parametrize("lens,keep", [([100], 100), ([257, 33], 300), ([3000], 5000), ([900] * 9, 1000),
                                       ([1, 31, 500, 64, 2], 512)])
@pytest.mark.parametrize("fused", [False, True])
def test_decode_with_everything_kept(lens, keep, fused):
    say(f"fp32 decode {lens} keep {keep} fused {fused}")
    decode_case(lens, keep, fused, True, False, seed=310)


@pytest.mark.parametrize("lens,keep,n_q", [([1], 0, 1), ([31], 0, 5), ([20, 7], 0, 33), ([100], 200, 17), ([4001], 5000, 32),
                                           ([0, 300, 31], 512, 48), ([700 + i for i in range(12)], 1000, 130)])
def test_prefill_with_everything_kept(lens, keep, n_q):
    """either kernel: the last case has the rows and keys of prefill_q8_kernel"""
    say(f"fp32 prefill {n_q} over {lens} keep {keep}")
    prefill_case(lens, n_q, keep, True, False, seed=320, check_seqs=[0, len(lens) - 1])


def test_prefill_of_a_first_chunk():
    """nothing cached before the chunk"""
    say("fp32 prefill, first chunk")
    prefill_case([0], 90, 0, False, False, seed=321)


def test_decode_with_and_without_an_8_bit_neighbour():
    """one sequence, alone and beside one that holds 8-bit blocks"""
    say("fp32 decode, neighbours")
    with Q.Filled([90, 400], seed=330) as f:
        f.ctx.kv_quantize(f.seqs[1:])
        f.ctx.kv_quantize(f.seqs[:1], keep_tokens=90)
        q = O.normal_bf16(2 * NQ * D, 331).reshape(2, NQ, D)
        k, v = (Q.f64(f.rows[0, f.seqs[0]][j]) for j in range(2))
        want, mag, big = Q.attend(Q.f64(q[:1]), k, v, SCALE)
        for n in (1, 2):
            got = f.run(lambda a, o: f.ctx.decode_attn(0, f.seqs[:n], a, o), (n, NQ, D), np.float32, q[:n].copy())
            check(got[0].astype(np.float64), want[0], mag[0], big, False, False, f"{n} sequences")


@pytest.mark.parametrize("n_q", [0, 9])
def test_70_sequences_of_which_the_last_hold_none(n_q):
    """two launches, the second without an 8-bit block (n_q 0: decode)"""
    say(f"fp32, 70 sequences, {n_q} rows")
    lens = [int(x) for x in np.random.default_rng(5).integers(40, 200, 64)] + [1, 5, 17, 28, 31, 30]
    if n_q:
        prefill_case(lens, n_q, 0, False, False, seed=340, check_seqs=[0, 63, 64, 66, 69])
    else:
        decode_case(lens, 0, False, False, False, seed=341)


def test_what_keeps_its_bits():
    """fp32 without 8-bit blocks in the context, and bf16 where no sequence of
    the launch holds one: the bf16 kernels' results"""
    say("bits of the bf16 kernels")
    lens, n_q = [500, 31, 2000], 20
    got = {}
    for q8 in (0, 64):
        with Q.Filled(lens, seed=350, extra=n_q, q8_blocks=q8) as f:
            f.add(f.seqs, n_q, commit=False)
            q = O.normal_bf16(3 * n_q * NQ * D, 351).reshape(3, n_q, NQ, D)
            last = q[:, -1].copy()
            bf = dict(out_dtype=kvc.DTYPE_BF16)
            got[q8] = [f.run(lambda a, o: f.ctx.decode_attn(0, f.seqs, a, o, **bf), last.shape, np.uint16, last),
                       f.run(lambda a, o: f.ctx.prefill_attn(0, f.seqs, n_q, a, o, **bf), q.shape, np.uint16, q)]
            if not q8:
                outs = [f.run(lambda a, o: call(0, f.seqs, a, o), last.shape, np.uint32, last)
                        for call in (f.ctx.decode_attn, f.ctx.decode_attn_static)]
                assert np.array_equal(*outs)
    assert all(np.array_equal(a, b) for a, b in zip(got[0], got[64]))
