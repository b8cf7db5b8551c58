"""CPU tests of the bookkeeping behind the 8-bit blocks and eviction: block
accounting, copies and sharing, and every refusal.  Contexts are host-only, so
no kernel runs; kvc_kv_quantize and kvc_evict do their bookkeeping there as the
other sequence calls do."""
import ctypes

import numpy as np
import pytest

import kvc

FAKE = 1 << 20  # a pointer that no host code follows


def ctx(**over):
    cfg = dict(device=-1, pool_blocks=64, q8_blocks=32, n_ssm_layers=0, max_seqs=8, max_seq_len=2048, snapshot_slots=0)
    cfg.update(over)
    return kvc.Context(**cfg)


def fill(c, n, tokens=None):
    s = c.seq_create()
    c.reserve([s], n)
    c.commit([s], n, tokens)
    return s


def code(fn, *a, **k):
    with pytest.raises(kvc.KvcError) as e:
        fn(*a, **k)
    return e.value.code


def evict(c, seqs, budget, **k):
    c.evict(seqs, budget, FAKE, 2048, FAKE + (1 << 30), **k)


def test_config_and_stats():
    with ctx() as c:
        assert c.q8_stats() == (32, 32)
    assert code(ctx, q8_blocks=-1) == kvc.KVC_ERR_INVALID
    with ctx(q8_blocks=0) as c:
        s = fill(c, 40)
        assert code(c.kv_quantize, [s]) == kvc.KVC_ERR_NOMEM
        c.kv_quantize([s], keep_tokens=40)  # nothing to do needs no block


@pytest.mark.parametrize("n,keep,want", [(0, 0, 0), (1, 0, 0), (31, 0, 0), (32, 0, 1), (33, 0, 1), (100, 0, 3),
                                         (100, 4, 3), (100, 5, 2), (100, 100, 0), (100, 10 ** 9, 0), (1024, 0, 32)])
def test_quantize_accounting(n, keep, want):
    with ctx() as c:
        s = c.seq_create()
        if n:
            c.reserve([s], n)
            c.commit([s], n)
        c.kv_quantize([s], keep)
        i = c.seq_info(s)
        assert (i.len, i.pending, i.position, i.q8_tokens) == (n, 0, n, 32 * want)
        assert c.q8_stats() == (32, 32 - want)
        assert c.stats().free_blocks == 64 - ((n + 31) // 32 - want)
        c.kv_quantize([s], keep)  # again: nothing new
        assert c.q8_stats()[1] == 32 - want
        c.seq_release(s)
        assert c.q8_stats()[1] == 32 and c.stats().free_blocks == 64


def test_quantize_in_steps_and_append_after():
    with ctx() as c:
        s = fill(c, 70)
        c.kv_quantize([s])
        assert c.seq_info(s).q8_tokens == 64
        c.reserve([s], 60)
        assert code(c.kv_quantize, [s]) == kvc.KVC_ERR_STATE  # tokens pending
        c.commit([s], 60)
        c.kv_quantize([s], keep_tokens=33)
        assert c.seq_info(s).q8_tokens == 96
        assert c.stats().free_blocks == 64 - 2


def test_quantize_runs_out_without_a_change():
    with ctx(q8_blocks=3) as c:
        a, b = fill(c, 64), fill(c, 64)
        assert code(c.kv_quantize, [a, b]) == kvc.KVC_ERR_NOMEM
        assert c.q8_stats() == (3, 3) and c.seq_info(a).q8_tokens == 0
        c.kv_quantize([a])
        assert c.q8_stats() == (3, 1)


def test_copies_share_blocks_and_release_them():
    with ctx() as c:
        s = fill(c, 100)
        d, e = c.seq_create(), c.seq_create()
        c.kv_quantize([s], dst=[d])
        assert c.seq_info(s).q8_tokens == 0 and c.seq_info(d).q8_tokens == 96 and c.seq_len(d) == 100
        assert c.q8_stats()[1] == 29 and c.stats().free_blocks == 60  # the tail block is shared
        c.kv_quantize([d], dst=[e])  # a copy of the copy shares its 8-bit blocks
        assert c.q8_stats()[1] == 29 and c.seq_info(e).q8_tokens == 96
        c.seq_release(d)
        assert c.q8_stats()[1] == 29
        c.reserve([e], 1)  # into the shared tail: copied before it is written
        assert c.stats().free_blocks == 59
        c.commit([e], 1)
        c.seq_release(s)
        c.seq_release(e)
        assert c.q8_stats()[1] == 32 and c.stats().free_blocks == 64


def test_copy_of_an_empty_sequence():
    with ctx() as c:
        s, d = c.seq_create(), c.seq_create()
        c.kv_quantize([s], dst=[d])
        evict(c, [s], 4, dst=[d])
        assert c.seq_len(d) == 0 and c.seq_info(d).position == 0
        assert c.prefix_match(d, np.arange(40)) == 0  # still an ordinary empty sequence


def test_truncate_of_8_bit_blocks():
    with ctx() as c:
        s = fill(c, 100)
        c.kv_quantize([s])
        assert code(c.seq_truncate, s, 50) == kvc.KVC_ERR_UNSUPPORTED
        assert c.seq_len(s) == 100
        c.seq_truncate(s, 98)
        c.seq_truncate(s, 64)
        assert c.seq_info(s).q8_tokens == 64 and c.q8_stats()[1] == 30
        c.reserve([s], 1)
        c.commit([s], 1)
        c.seq_truncate(s, 0)
        assert c.q8_stats()[1] == 32 and c.stats().free_blocks == 64


def test_quantized_sequence_leaves_the_prefix_index():
    tok = np.arange(100, dtype=np.int32)
    with ctx() as c:
        s = fill(c, 100, tok)
        assert c.stats().indexed_blocks == 3
        c.kv_quantize([s])
        # the indexed bf16 blocks are now only the index's
        assert c.stats().cached_blocks == 3
        c.reserve([s], 60)
        c.commit([s], 60, np.arange(60))
        assert c.stats().indexed_blocks == 3  # and what follows is not indexed
        d = c.seq_create()
        assert c.prefix_match(d, tok) == 96 and c.seq_info(d).q8_tokens == 0


def test_evict_accounting_and_positions():
    with ctx() as c:
        s = fill(c, 200)
        evict(c, [s], 50, n_sink=2, n_recent=10)
        i = c.seq_info(s)
        assert (i.len, i.position, i.q8_tokens) == (50, 200, 0)
        assert c.stats().free_blocks == 62
        c.reserve([s], 20)
        assert c.seq_info(s).pending == 20
        c.commit([s], 20)
        evict(c, [s], 50)
        assert c.seq_info(s).position == 220 and c.seq_len(s) == 50
        c.seq_truncate(s, 40)
        assert c.seq_info(s).position == 210
        evict(c, [s], 40)  # within the budget: as it is
        assert c.stats().free_blocks == 62 and c.seq_info(s).position == 210
        c.seq_truncate(s, 0)
        assert c.seq_info(s).position == 0
        c.seq_reset(s)
        assert c.stats().free_blocks == 64


def test_evict_copy_and_8_bit_source():
    with ctx() as c:
        s = fill(c, 200)
        c.kv_quantize([s])
        d = c.seq_create()
        evict(c, [s], 33, dst=[d])
        assert (c.seq_len(d), c.seq_info(d).q8_tokens, c.seq_info(d).position) == (33, 0, 200)
        assert (c.seq_len(s), c.seq_info(s).q8_tokens) == (200, 192)
        evict(c, [s], 33)
        assert c.q8_stats()[1] == 32 and c.stats().free_blocks == 60


def test_evict_runs_out_without_a_change():
    with ctx(pool_blocks=10) as c:
        s = fill(c, 300)
        assert code(evict, c, [s], 32) == kvc.KVC_ERR_NOMEM
        assert c.seq_len(s) == 300 and c.stats().free_blocks == 0


@pytest.mark.parametrize("budget,sink,recent", [(0, 0, 0), (-1, 0, 0), (4, -1, 0), (4, 0, -1), (4, 3, 2),
                                                (2 ** 31 - 1, 2 ** 31 - 1, 1)])
def test_evict_refuses_budgets(budget, sink, recent):
    with ctx() as c:
        s = fill(c, 10)
        assert code(evict, c, [s], budget, n_sink=sink, n_recent=recent) == kvc.KVC_ERR_INVALID


def test_source_and_destination_refusals():
    L = kvc.lib()
    with ctx() as c:
        s, t, d = fill(c, 40), fill(c, 40), c.seq_create()
        for call in (lambda a, b: c.kv_quantize(a, dst=b), lambda a, b: evict(c, a, 8, dst=b)):
            assert code(call, [s], [s]) == kvc.KVC_ERR_INVALID
            assert code(call, [s], [t]) == kvc.KVC_ERR_STATE  # not empty
            assert code(call, [s, t], [d, d]) == kvc.KVC_ERR_INVALID
            assert code(call, [s, s], [d, t]) == kvc.KVC_ERR_INVALID
            assert code(call, [99], [d]) == kvc.KVC_ERR_INVALID
            assert code(call, [s], [99]) == kvc.KVC_ERR_INVALID
            with pytest.raises(ValueError):
                call([s], [])
        assert code(c.kv_quantize, [s], -1) == kvc.KVC_ERR_INVALID
        assert code(c.evict, [s], 8, None, 64, FAKE) == kvc.KVC_ERR_INVALID
        assert code(c.evict, [s], 8, FAKE, 64, None) == kvc.KVC_ERR_INVALID
        assert code(c.evict, [s], 8, FAKE, 39, FAKE * 2) == kvc.KVC_ERR_RANGE  # stride under the length
        assert code(c.evict, [s], 8, FAKE, 64, FAKE * 2, acc_out=FAKE + 64) == kvc.KVC_ERR_INVALID  # overlap
        assert c.seq_len(s) == 40 and c.q8_stats()[1] == 32
        assert L.kvc_seq_get_info(c.ptr, s, None) == kvc.KVC_ERR_INVALID
        assert L.kvc_seq_get_info(c.ptr, 99, ctypes.byref(kvc.SeqInfo())) == kvc.KVC_ERR_INVALID
        assert L.kvc_q8_stats(c.ptr, None, None) == kvc.KVC_ERR_INVALID
        assert code(c.attn_weights, 0, [s], 1, FAKE, FAKE, 64) == kvc.KVC_ERR_NO_DEVICE


def test_copies_with_recurrent_layers_are_refused():
    with ctx(n_ssm_layers=2) as c:
        s, d = fill(c, 40), c.seq_create()
        assert code(c.kv_quantize, [s], dst=[d]) == kvc.KVC_ERR_UNSUPPORTED
        assert code(evict, c, [s], 8, dst=[d]) == kvc.KVC_ERR_UNSUPPORTED
        c.kv_quantize([s])  # in place the state stays with its sequence
        evict(c, [s], 8)
        assert c.seq_len(s) == 8


def test_random_calls_keep_the_books():
    """Random sequences of calls; the free lists and lengths follow a model."""
    rng = np.random.default_rng(5)
    with ctx(max_seqs=6, pool_blocks=80, q8_blocks=40) as c:
        live = {}
        for _ in range(600):
            op = rng.integers(7)
            s = int(rng.choice(list(live))) if live else None
            try:
                if op == 0 or s is None:
                    live[c.seq_create()] = (0, 0, 0)  # len, n8, evicted
                elif op == 1:
                    n = int(rng.integers(1, 150))
                    c.reserve([s], n)
                    c.commit([s], n)
                    live[s] = (live[s][0] + n, *live[s][1:])
                elif op == 2:
                    k = int(rng.integers(0, 80))
                    c.kv_quantize([s], k)
                    ln, n8, e = live[s]
                    live[s] = (ln, max(n8, max(0, ln - k) // 32), e)
                elif op == 3:
                    b = int(rng.integers(1, 120))
                    evict(c, [s], b)
                    ln, n8, e = live[s]
                    live[s] = (b, 0, e + ln - b) if ln > b else live[s]
                elif op == 4:
                    c.seq_release(s)
                    del live[s]
                elif op == 5:
                    d = c.seq_create()
                    live[d] = (0, 0, 0)
                    if rng.integers(2):
                        c.kv_quantize([s], 10, dst=[d])
                        ln, n8, e = live[s]
                        live[d] = (ln, max(n8, max(0, ln - 10) // 32), e)
                    else:
                        evict(c, [s], 60, dst=[d])
                        ln, n8, e = live[s]
                        live[d] = (min(ln, 60), 0, e + max(0, ln - 60))
                else:
                    n = int(rng.integers(0, live[s][0] + 1))
                    c.seq_truncate(s, n)
                    ln, n8, e = live[s]
                    live[s] = (n, min(n8, (n + 31) // 32), e if n else 0)
            except kvc.KvcError as err:
                assert err.code in (kvc.KVC_ERR_NOMEM, kvc.KVC_ERR_RANGE, kvc.KVC_ERR_UNSUPPORTED)
            for x, (ln, n8, e) in live.items():
                i = c.seq_info(x)
                assert (i.len, i.q8_tokens, i.position) == (ln, 32 * n8, ln + e)
        for x in list(live):
            c.seq_release(x)
        assert c.q8_stats()[1] == 40 and c.stats().free_blocks == 80


def test_evict_refuses_arrays_that_overlap():
    """kept is read back as positions"""
    with ctx(n_attn_layers=2) as c:
        s = fill(c, 100)
        acc_bytes, kept_bytes = 2 * 4 * 128 * 4, 2 * 4 * 10 * 4
        far = FAKE + (1 << 30)

        def call(acc, kept, acc_out=None):
            c.evict([s], 10, acc, 128, kept, acc_out=acc_out)

        for args in ((FAKE, FAKE), (FAKE, FAKE + acc_bytes - 4), (FAKE, FAKE - kept_bytes + 4), (FAKE, far, FAKE),
                     (FAKE, far, FAKE + acc_bytes - 4), (FAKE, far, far), (FAKE, far, far - acc_bytes + 4),
                     (FAKE, far, far + kept_bytes - 4)):
            assert code(call, *args) == kvc.KVC_ERR_INVALID, args
        assert c.seq_info(s).len == 100
        call(FAKE, FAKE + acc_bytes, FAKE + acc_bytes + kept_bytes)  # back to back
        assert c.seq_info(s).len == 10


def test_positions_end_below_31_bits():
    """a sequence that is cut again and again: its positions go on, up to where
    those of the next tokens could pass a 32-bit integer"""
    n = 1 << 23
    with ctx(max_seq_len=n, pool_blocks=n // 32 + 8, max_seqs=1, n_attn_layers=1, q8_blocks=0) as c:
        s = fill(c, n)
        rounds = 0
        while True:
            try:
                c.evict([s], 1, FAKE, n, FAKE + (1 << 40))
            except kvc.KvcError as e:
                assert e.code == kvc.KVC_ERR_RANGE
                break
            rounds += 1
            assert c.seq_info(s).position == n + (rounds - 1) * (n - 1)
            c.reserve([s], n - 1)
            c.commit([s], n - 1)
        i = c.seq_info(s)
        assert i.len == n and 2 ** 31 - 1 - n < i.position <= 2 ** 31 - 1
        c.seq_reset(s)
        assert c.seq_info(s).position == 0
