"""GPU test of a beam search in which prompts run out of choices: kvc_beam_select fills a
group's outputs with -inf, -1, -1, and a slot without a choice goes on as itself, with
the score -inf, from which nothing is chosen.  No prompt gets another one's K/V or state."""
import numpy as np
import pytest

import kvc
from gpu_util import say
from test_gpu_beam import Case, noise
from test_gpu_shared import Forest

pytestmark = pytest.mark.gpu
FLOATS = 32 * 128 * 128 + 3 * 8192  # of a layer's state


def test_groups_with_fewer_choices_than_beams():
    say("beam search of 3 prompts of 4 beams, two of them ending")
    rng = np.random.default_rng(5)
    groups, beams, vocab = 3, 4, 777
    spec = [(150, [(70 + 41 * g, beams) for g in range(groups)])]
    with Forest(spec, seed=51, extra=8, n_ssm_layers=1) as f:
        def buf(s):
            return kvc.DeviceBuffer(kvc.hip(), f.ctx.state_ptrs(s, 0)[0], FLOATS * 4)

        state = {}
        prompt = {s: i // beams for i, s in enumerate(f.seqs)}  # whose state and rows a sequence holds
        scores = (rng.random((groups, beams)) * -5).astype(np.float32)
        for step in range(4):
            f.check(f.seqs, f"step {step}", seed=100 + 10 * step)
            for s in f.seqs:
                state[s] = rng.integers(0, 2**32, FLOATS, dtype=np.uint32)
                buf(s).upload(state[s])
            x = noise((groups, beams, vocab), 200 + step)
            if step >= 1:  # three values in all, of two beams; then of one beam, then none
                keep = np.zeros((beams, vocab), bool)
                if step < 3:
                    keep[0, :2] = True
                    keep[1, 5] = step == 1
                x[1][~keep] = -np.inf
            if step == 2:  # the first prompt: the callers end all of its beams but one
                scores[0, 1:] = -np.inf
            with Case(x, kvc.DTYPE_F32, scores, beams) as c:
                scores, chosen, tokens = c.run(f.ctx)
            live = chosen >= 0
            assert (live == (scores > -np.inf)).all() and (live == (tokens >= 0)).all()
            assert live[2].all() and live[0].all()
            assert live[1].sum() == (4, 3, 2, 0)[step]
            slot = np.arange(beams)[None, :]
            index = (np.where(live, chosen, slot) + np.arange(groups)[:, None] * beams).reshape(-1).tolist()
            f.ctx.reorder(f.seqs, index)
            prompt = {f.seqs[i]: prompt[f.seqs[p]] for i, p in enumerate(index)}
            assert [prompt[s] for s in f.seqs] == [i // beams for i in range(groups * beams)]
            f.rows = {(0, f.seqs[i]): list(f.rows[0, f.seqs[p]]) for i, p in enumerate(index)}
            state = {f.seqs[i]: state[f.seqs[p]] for i, p in enumerate(index)}
            f.ctx.sync()
            for s in f.seqs:
                assert np.array_equal(buf(s).download(np.uint32, FLOATS), state[s]), (step, s)
        f.check(f.seqs, "the end", seed=99)
