"""CPU test of the snapshots that one kvc_seq_commit takes of several sequences:
a slot is given to one of them only.  (All copies of a call are one launch.)
Contexts are host-only."""
import numpy as np
import pytest

import kvc

IV = 256


def commit_together(c, n, first):
    """n new sequences of IV tokens each, committed in one call; returns them and their tokens"""
    seqs = [c.seq_create() for _ in range(n)]
    tok = np.arange(n * IV, dtype=np.int32).reshape(n, IV) + first
    c.reserve(seqs, IV)
    c.commit(seqs, IV, tok)
    return seqs, tok


def matched(c, tok):
    s = c.seq_create()
    n = c.prefix_match(s, np.append(tok, 7))
    c.seq_release(s)
    return n


@pytest.mark.parametrize("slots", [1, 3, 5, 8])
def test_a_slot_is_given_out_once(slots):
    with kvc.Context(device=-1, pool_blocks=256, n_ssm_layers=2, max_seqs=12, max_seq_len=1024, snapshot_slots=slots) as c:
        seqs, tok = commit_together(c, 5, 0)
        kept = min(slots, 5)
        assert c.stats().snapshots == kept
        # the first ones have theirs, and the others took no slot from them
        assert [matched(c, t) for t in tok] == [IV] * kept + [0] * (5 - kept)
        for s in seqs:
            c.seq_release(s)
        # a later call evicts them, oldest first
        _, more = commit_together(c, 2, 10000)
        assert [matched(c, t) for t in more] == [IV] * min(slots, 2) + [0] * (2 - min(slots, 2))
        assert c.stats().snapshots == min(slots, 7)


def test_found_again_and_taken_in_one_call():
    """of three sequences the first lands on a snapshot that is there: the others
    do not evict it in the call that counts on it"""
    with kvc.Context(device=-1, pool_blocks=256, n_ssm_layers=2, max_seqs=12, max_seq_len=1024, snapshot_slots=1) as c:
        (s,), (t,) = commit_together(c, 1, 0)
        c.seq_release(s)
        seqs = [c.seq_create() for _ in range(3)]
        c.reserve(seqs, IV)
        c.commit(seqs, IV, np.stack([t, t + 5000, t + 9000]))
        assert [matched(c, x) for x in (t, t + 5000, t + 9000)] == [IV, 0, 0]
