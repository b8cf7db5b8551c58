"""GPU test of a beam search through the C ABI, its calls together as they are used:
fork, decode over shared blocks, selection, reorder.  Every step's attention and
choice are checked against 64 bits and the recurrent states bit for bit."""
import numpy as np
import pytest

import kvc
from gpu_util import say
from test_gpu_beam import Case, noise
from test_gpu_shared import Forest

pytestmark = pytest.mark.gpu
FLOATS = 32 * 128 * 128 + 3 * 8192  # of a layer's state


@pytest.mark.parametrize("groups,beams,force", [(2, 4, True), (1, 3, True), (5, 5, False)])
def test_search(groups, beams, force):
    say(f"beam search: {groups} prompts of {beams} beams")
    rng = np.random.default_rng(groups * 10 + beams)
    vocab, pad = 1999, 2
    spec = [(150, [(70 + 41 * g, beams) for g in range(groups)])]
    flags = kvc.FLAG_EXACT_MATH | (kvc.FLAG_DECODE_SHARE if force else 0)
    with Forest(spec, seed=31, extra=8, n_ssm_layers=1, flags=flags) as f:
        n = groups * beams
        state = {}

        def buf(s):
            return kvc.DeviceBuffer(kvc.hip(), f.ctx.state_ptrs(s, 0)[0], FLOATS * 4)

        scores = np.full((groups, beams), -np.inf, np.float32)
        scores[:, 0] = 0  # beams of a prompt are alike at first
        for step in range(5):
            f.check(f.seqs, f"step {step}", seed=100 + 10 * step)
            for s in f.seqs:  # stands for the recurrent layers' step
                state[s] = rng.integers(0, 2**32, FLOATS, dtype=np.uint32)
                buf(s).upload(state[s])
            x = noise((groups, beams, vocab), 200 + step)
            with Case(x, kvc.DTYPE_BF16, scores, beams, pad, step % 3) as c:
                scores, chosen, tokens = c.run(f.ctx)
            assert (chosen >= 0).all() and (tokens >= 0).all()
            if step == 0:
                assert (chosen == 0).all()
            parents = (chosen + np.arange(groups)[:, None] * beams).reshape(-1).tolist()
            f.ctx.reorder(f.seqs, parents)
            f.rows = {(0, f.seqs[i]): list(f.rows[0, f.seqs[p]]) for i, p in enumerate(parents)}
            state = {f.seqs[i]: state[f.seqs[p]] for i, p in enumerate(parents)}
            f.ctx.sync()
            for s in f.seqs:
                assert np.array_equal(buf(s).download(np.uint32, FLOATS), state[s]), (step, s)
        f.check(f.seqs, "the end", seed=99)
        assert len(f.seqs) == n
