"""GPU test of a kvc_seq_commit that lands more sequences on a snapshot boundary
than there are slots: what the slots hold is the first sequences' state and K/V,
bit for bit."""
import numpy as np
import pytest

import kvc
from gpu_util import Mirror, fill_seq, gather, say

pytestmark = pytest.mark.gpu
LAYERS, SSM, IV = 2, 2, 32
FLOATS = SSM * (32 * 128 * 128 + 3 * 8192)  # of one sequence's state


@pytest.mark.parametrize("slots", [1, 3])
def test_more_sequences_than_slots(slots):
    say(f"5 sequences land on a boundary, {slots} slots")
    with kvc.Context(n_attn_layers=LAYERS, n_ssm_layers=SSM, max_seqs=12, max_seq_len=256, pool_blocks=64,
                     snapshot_slots=slots, snapshot_interval=IV, alloc_seed=98) as ctx:
        m = Mirror(LAYERS)
        seqs = [ctx.seq_create() for _ in range(5)]
        tok = np.arange(5 * IV, dtype=np.int32).reshape(5, IV)
        fill_seq(ctx, m, seqs, IV - 1, seed=3, tokens=list(tok[:, :-1]))
        states = []
        for i, s in enumerate(seqs):
            x = np.random.default_rng(i).integers(0, 2**32, FLOATS, dtype=np.uint32)
            kvc.DeviceBuffer(kvc.hip(), ctx.state_ptrs(s, 0)[0], FLOATS * 4).upload(x)
            states.append(x)
        fill_seq(ctx, m, seqs, 1, seed=4, tokens=list(tok[:, -1:]))
        for i, s in enumerate(seqs):
            d = ctx.seq_create()
            n = ctx.prefix_match(d, np.append(tok[i], 9))
            assert n == (IV if i < slots else 0), i
            if n:
                ctx.sync()
                got = kvc.DeviceBuffer(kvc.hip(), ctx.state_ptrs(d, 0)[0], FLOATS * 4).download(np.uint32, FLOATS)
                assert np.array_equal(got, states[i]), i
                for layer in range(LAYERS):
                    (k, v), = gather(ctx, layer, [d], [IV])
                    assert np.array_equal(k, m.get(s, layer)[0]) and np.array_equal(v, m.get(s, layer)[1]), (i, layer)
            ctx.seq_release(d)
