"""CPU tests of eviction beside the prefix index (host-only contexts): fresh
blocks may come from the index, and an eviction that finds too few leaves the
index as it was."""
import numpy as np
import pytest

import kvc
from test_q8_bookkeeping import code, ctx, evict, fill


def prompt(n, seed=0):
    return np.random.default_rng(seed).integers(0, 1000, n).astype(np.int32)


def indexed(c, tokens):
    """A released sequence of these tokens: its blocks stay with the index."""
    s = fill(c, len(tokens), tokens[None])
    c.seq_release(s)


def state(c, s):
    t, i = c.stats(), c.seq_info(s)
    return t.free_blocks, t.cached_blocks, t.indexed_blocks, t.evictions, i.len, i.position, i.q8_tokens


@pytest.mark.parametrize("into_a_copy", [False, True])
def test_too_few_blocks_leave_the_index_alone(into_a_copy):
    with ctx(pool_blocks=20) as c:
        p = prompt(160)
        indexed(c, p)
        s, d = fill(c, 384), c.seq_create()
        assert c.stats().indexed_blocks == 5 and c.stats().free_blocks == 3
        before = state(c, s)
        assert code(evict, c, [s], 383, **(dict(dst=[d]) if into_a_copy else {})) == kvc.KVC_ERR_NOMEM
        assert state(c, s) == before
        e = c.seq_create()
        assert c.prefix_match(e, np.append(p, 7)) == 160


def test_blocks_of_the_index_count_as_free():
    with ctx(pool_blocks=20) as c:
        indexed(c, prompt(160))
        s = fill(c, 384)
        evict(c, [s], 256)  # 8 blocks: 3 free ones and all 5 of the index
        assert c.seq_len(s) == 256 and c.stats().indexed_blocks == 0 and c.stats().free_blocks == 12


def test_only_as_many_as_needed_leave_the_index():
    with ctx(pool_blocks=20) as c:
        p = prompt(160)
        indexed(c, p)
        s = fill(c, 384)
        evict(c, [s], 160)  # 5 blocks: the 2 that are missing are the prompt's last
        assert c.stats().indexed_blocks == 3
        e = c.seq_create()
        assert c.prefix_match(e, p) == 96


def test_blocks_behind_one_in_use_do_not_count():
    """The index gives up a chain from its end only: a block that nobody else
    holds stays while a later one of its chain is in use."""
    with ctx(pool_blocks=16) as c:
        p = prompt(64)
        a = fill(c, 32, p[None, :32])
        b = fill(c, 64, p[None])  # its first block is a second copy, its second one the index's
        c.seq_release(a)
        c.kv_quantize([b], keep_tokens=32)  # gives up its own copy, and its hold on the index's
        s = fill(c, 384)
        t = c.stats()
        assert (t.indexed_blocks, t.cached_blocks, t.free_blocks) == (2, 1, 2)
        before = state(c, s)
        assert code(evict, c, [s], 96) == kvc.KVC_ERR_NOMEM
        assert state(c, s) == before
        evict(c, [s], 64)
        assert c.seq_len(s) == 64 and c.stats().indexed_blocks == 2
        c.seq_release(b)
        f = fill(c, 352)
        evict(c, [f], 96)  # now both count: 14 - 11 + 2 free


def test_a_shared_chain_counts_once_it_is_released():
    with ctx(pool_blocks=12) as c:
        p = prompt(128)
        indexed(c, p)
        m = c.seq_create()
        assert c.prefix_match(m, np.append(p, 1)) == 128
        s = fill(c, 200)
        assert c.stats().free_blocks == 1
        before = state(c, s)
        assert code(evict, c, [s], 64) == kvc.KVC_ERR_NOMEM and state(c, s) == before
        c.seq_release(m)
        evict(c, [s], 64)
        assert c.seq_len(s) == 64
