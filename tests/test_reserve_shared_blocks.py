"""CPU tests of the copies that kvc_seq_reserve makes of shared blocks that are not
full: one for every holder but the last.  Contexts are host-only."""
import numpy as np
import pytest

import kvc


def ctx(blocks, **over):
    cfg = dict(device=-1, pool_blocks=blocks, n_ssm_layers=0, max_seqs=12, max_seq_len=2048, snapshot_slots=0)
    cfg.update(over)
    return kvc.Context(**cfg)


def fill(c, n, tokens=None):
    s = c.seq_create()
    c.reserve([s], n)
    c.commit([s], n, tokens)
    return s


def forks(c, s, n):
    d = [c.seq_create() for _ in range(n)]
    c.fork([s] * n, d)
    return d


def refused(c, seqs, n=1):
    free = c.stats().free_blocks
    with pytest.raises(kvc.KvcError) as e:
        c.reserve(seqs, n)
    assert e.value.code == kvc.KVC_ERR_NOMEM and c.stats().free_blocks == free


@pytest.mark.parametrize("together", [True, False])
def test_the_last_holder_keeps_the_block(together):
    """40 tokens, three holders, none besides: two copies, in one call or in three"""
    with ctx(4) as c:
        s = fill(c, 40)
        d = forks(c, s, 3)
        c.seq_release(s)
        assert c.stats().free_blocks == 2
        for part in [d] if together else [[x] for x in d]:
            c.reserve(part, 1)
            c.commit(part, 1)
        assert c.stats().free_blocks == 0
        assert [c.seq_len(x) for x in d] == [41] * 3
        for x in d:
            c.seq_release(x)
        assert c.stats().free_blocks == 4


def test_a_holder_outside_the_call_keeps_it_instead():
    with ctx(4) as c:
        s = fill(c, 40)
        d = forks(c, s, 3)  # s still holds the block
        refused(c, d)
        c.reserve(d[:2], 1)
        c.commit(d[:2], 1)
        assert c.stats().free_blocks == 0
        refused(c, [s])  # shared with d[2] yet
        c.seq_release(d[2])
        c.reserve([s], 1)  # the last one
        c.commit([s], 1)
        assert c.seq_len(s) == 41


def test_the_index_holds_a_block_that_was_cut():
    """A full block that the index holds and that a truncation made partial is
    copied for every holder."""
    with ctx(8) as c:
        s = fill(c, 64, np.arange(64, dtype=np.int32))
        d = forks(c, s, 2)
        c.seq_release(s)
        for x in d:
            c.seq_truncate(x, 50)
        assert c.stats().free_blocks == 6
        c.reserve(d, 1)
        assert c.stats().free_blocks == 4
        c.commit(d, 1, np.array([[900], [901]], np.int32))
        p = c.seq_create()
        assert c.prefix_match(p, np.arange(80, dtype=np.int32)) == 64  # the indexed block is as it was


def test_families_in_one_call():
    """Two families, one with a source outside, a sequence of its own, ends at a block's end."""
    with ctx(32) as c:
        a, b, own, full = fill(c, 33), fill(c, 70), fill(c, 5), fill(c, 64)
        da, db, df = forks(c, a, 3), forks(c, b, 2), forks(c, full, 2)
        c.seq_release(a)
        used = 32 - c.stats().free_blocks
        assert used == 2 + 3 + 1 + 2
        c.reserve([da[0], db[0], own, da[1], df[0], db[1], da[2], df[1]], 1)
        # copies: 2 of 3 (a), 2 of 2 (b holds on); new blocks behind the full ones: 2
        assert c.stats().free_blocks == 32 - used - 2 - 2 - 2


def test_every_step_of_a_beam_search():
    """n beams of one parent: n - 1 copies in each step, in a pool that has no more"""
    n = 4
    with ctx(1 + n) as c:
        beams = [fill(c, 35)]
        beams += forks(c, beams[0], n - 1)
        for step in range(20):
            c.reserve(beams, 1)
            c.commit(beams, 1)
            assert c.stats().free_blocks == 0
            c.reorder(beams, [step % n] * n)
        assert [c.seq_len(x) for x in beams] == [55] * n


def test_a_refused_call_changes_nothing():
    with ctx(5) as c:
        s = fill(c, 40)
        d = forks(c, s, 3)
        c.seq_release(s)
        refused(c, d, 40)  # 2 copies and 3 more blocks: 5 of 3
        c.reserve(d, 24)
        c.commit(d, 24)
        assert c.stats().free_blocks == 5 - 1 - 3
