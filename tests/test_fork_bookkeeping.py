"""CPU tests of the bookkeeping behind kvc_seq_fork and kvc_seq_reorder: block
accounting against a model of shared blocks, the prefix index beside them, and
every refusal.  Contexts are host-only, so no kernel runs."""
import random

import numpy as np
import pytest

import kvc

BT = 32


def ctx(**over):
    cfg = dict(device=-1, pool_blocks=400, q8_blocks=16, n_ssm_layers=0, max_seqs=12, max_seq_len=2048, snapshot_slots=0)
    cfg.update(over)
    return kvc.Context(**cfg)


def fill(c, n, tokens=None):
    s = c.seq_create()
    if n:
        c.reserve([s], n)
        c.commit([s], n, tokens)
    return s


def code(fn, *a, **k):
    with pytest.raises(kvc.KvcError) as e:
        fn(*a, **k)
    return e.value.code


@pytest.mark.parametrize("n_ssm", [0, 2])
@pytest.mark.parametrize("length", [0, 1, 31, 32, 33, 100])
def test_fork_shares_blocks_until_they_are_written(length, n_ssm):
    with ctx(n_ssm_layers=n_ssm) as c:
        s = fill(c, length)
        used = (length + BT - 1) // BT
        d = [c.seq_create() for _ in range(3)]
        c.fork([s] * 3, d)
        assert [c.seq_len(x) for x in d] == [length] * 3
        assert c.stats().free_blocks == 400 - used
        c.reserve(d, 1)  # a shared block that is not full is copied first
        full = length // BT
        assert c.stats().free_blocks == 400 - (used + 3)
        c.commit(d, 1)
        assert c.seq_len(s) == length and [c.seq_len(x) for x in d] == [length + 1] * 3
        c.seq_release(s)
        assert c.stats().free_blocks == 400 - (full + 3)
        for x in d:
            c.seq_release(x)
        assert c.stats().free_blocks == 400


def test_fork_of_8_bit_and_evicted_sequences():
    with ctx() as c:
        s = fill(c, 100)
        c.kv_quantize([s], keep_tokens=40)  # 1 block
        d = c.seq_create()
        c.fork([s], [d])
        i = c.seq_info(d)
        assert (i.len, i.position, i.q8_tokens) == (100, 100, 32)
        assert c.q8_stats() == (16, 15)
        c.seq_release(s)
        assert c.q8_stats() == (16, 15)
        c.kv_quantize([d], keep_tokens=0)
        assert c.seq_info(d).q8_tokens == 96
        c.evict([d], 50, 1 << 20, 2048, 1 << 40)
        e = c.seq_create()
        c.fork([d], [e])
        assert (c.seq_info(e).len, c.seq_info(e).position) == (50, 100)
        c.reorder([d, e], [1, 1])
        c.seq_release(d)
        c.seq_release(e)
        assert c.q8_stats() == (16, 16) and c.stats().free_blocks == 400


def test_forks_feed_the_prefix_index():
    tok = np.arange(200, dtype=np.int32)
    with ctx() as c:
        s = fill(c, 100, tok[:100])
        d = c.seq_create()
        c.fork([s], [d])
        for x, more in ((s, tok[100:140]), (d, tok[150:190])):
            c.reserve([x], 40)
            c.commit([x], 40, more)
        a, b = c.seq_create(), c.seq_create()
        assert c.prefix_match(a, np.concatenate([tok[:140], tok[:30]])) == 128
        assert c.prefix_match(b, np.concatenate([tok[:100], tok[150:190], tok[:30]])) == 128
        for x in (s, d, a, b):
            c.seq_release(x)
        st = c.stats()
        assert st.indexed_blocks == st.cached_blocks == 400 - st.free_blocks == 5


def test_refusals():
    with ctx() as c:
        a, b = fill(c, 40), fill(c, 50)
        d, e = c.seq_create(), c.seq_create()
        L = kvc.lib()
        one = kvc._i32([a])
        assert L.kvc_seq_fork(None, one, one, 1, None) == kvc.KVC_ERR_INVALID
        assert L.kvc_seq_fork(c.ptr, None, one, 1, None) == kvc.KVC_ERR_INVALID
        assert L.kvc_seq_fork(c.ptr, one, None, 1, None) == kvc.KVC_ERR_INVALID
        assert L.kvc_seq_fork(c.ptr, one, kvc._i32([d]), 0, None) == kvc.KVC_ERR_INVALID
        assert L.kvc_seq_reorder(None, one, kvc._i32([0]), 1, None) == kvc.KVC_ERR_INVALID
        assert L.kvc_seq_reorder(c.ptr, one, None, 1, None) == kvc.KVC_ERR_INVALID
        assert code(c.fork, [a, a], [d, d]) == kvc.KVC_ERR_INVALID
        assert code(c.fork, [a, 99], [d, e]) == kvc.KVC_ERR_INVALID
        assert code(c.fork, [a, b], [d, a]) == kvc.KVC_ERR_INVALID  # both source and destination
        assert code(c.fork, [a], [b]) == kvc.KVC_ERR_STATE  # not empty
        assert code(c.reorder, [a, b], [0, 2]) == kvc.KVC_ERR_RANGE
        assert code(c.reorder, [a, b], [-1, 0]) == kvc.KVC_ERR_RANGE
        assert code(c.reorder, [a, a], [0, 0]) == kvc.KVC_ERR_INVALID
        c.reserve([a], 3)
        assert code(c.fork, [a], [d]) == kvc.KVC_ERR_STATE
        assert code(c.reorder, [a, b], [1, 1]) == kvc.KVC_ERR_STATE
        c.commit([a], 3)
        c.reserve([d], 1)
        assert code(c.fork, [a], [d]) == kvc.KVC_ERR_STATE
        with pytest.raises(ValueError):
            c.fork([a], [d, e])
        assert [c.seq_len(x) for x in (a, b)] == [43, 50]


@pytest.mark.parametrize("seed", range(6))
def test_against_a_model_of_shared_blocks(seed):
    """Random forks, reorders, appends, rollbacks and releases: lengths and the
    number of blocks in use follow a model in which a sequence is a list of
    block objects."""
    rng = random.Random(seed)
    with ctx(n_ssm_layers=seed % 2) as c:
        model = {}  # seq -> (len, [block objects])
        fresh = iter(range(10 ** 9))
        model[c.seq_create()] = (0, [])
        for _ in range(300):
            op = rng.choice(["append", "append", "fork", "reorder", "truncate", "release"])
            live = list(model)
            if op == "append":
                n = rng.randint(1, 40)
                seqs = [s for s in rng.sample(live, rng.randint(1, len(live))) if model[s][0] + n <= 400]
                if not seqs:
                    continue
                c.reserve(seqs, n)
                c.commit(seqs, n)
                shared = lambda b: sum(b in bl for _, bl in model.values()) > 1  # noqa: E731
                copied = [s for s in seqs if model[s][0] % BT and shared(model[s][1][model[s][0] // BT])]
                for s in seqs:
                    length, bl = model[s]
                    bl = bl[:]
                    if s in copied:
                        bl[length // BT] = next(fresh)
                    while len(bl) * BT < length + n:
                        bl.append(next(fresh))
                    model[s] = (length + n, bl)
            elif op == "fork":
                k = rng.randint(1, 3)
                if len(live) + k > 12:
                    continue
                src = [rng.choice(live) for _ in range(k)]
                dst = [c.seq_create() for _ in range(k)]
                c.fork(src, dst)
                for a, b in zip(src, dst):
                    model[b] = model[a]
            elif op == "reorder":
                seqs = rng.sample(live, rng.randint(1, len(live)))
                parent = [rng.randrange(len(seqs)) for _ in seqs]
                c.reorder(seqs, parent)
                was = [model[s] for s in seqs]
                for s, p in zip(seqs, parent):
                    model[s] = was[p]
            elif op == "truncate":
                s = rng.choice(live)
                n = rng.randint(0, model[s][0])
                c.seq_truncate(s, n)
                model[s] = (n, model[s][1][:(n + BT - 1) // BT])
            elif len(live) > 1:
                s = rng.choice(live)
                c.seq_release(s)
                del model[s]
            assert all(c.seq_len(s) == n for s, (n, _) in model.items())
            assert c.stats().free_blocks == 400 - len({b for _, bl in model.values() for b in bl})
        for s in model:
            c.seq_release(s)
        assert c.stats().free_blocks == 400


@pytest.mark.parametrize("seed", range(4))
def test_reordered_beams_feed_the_prefix_index(seed):
    """Beams commit tokens between reorders; every full block of every path that
    was ever committed is found again, and only those."""
    def common(a, b):
        return next((i for i, (x, y) in enumerate(zip(a, b)) if x != y), min(len(a), len(b)))

    rng = random.Random(seed)
    with ctx() as c:
        root = fill(c, 70, np.arange(70, dtype=np.int32))
        seqs = [c.seq_create() for _ in range(4)]
        c.fork([root] * 4, seqs)
        path = {s: list(range(70)) for s in seqs}
        seen = {tuple(range(70))}
        for step in range(8):
            n = rng.choice([1, 7, 32, 45])
            new = {s: [1000 * step + 10 * rng.randrange(3) + 7 * i for i in range(n)] for s in seqs}
            c.reserve(seqs, n)
            c.commit(seqs, n, np.array([new[s] for s in seqs], dtype=np.int32))
            for s in seqs:
                path[s] = path[s] + new[s]
                seen.add(tuple(path[s]))
            parent = [rng.randrange(4) for _ in seqs]
            c.reorder(seqs, parent)
            path = {s: path[seqs[p]] for s, p in zip(seqs, parent)}
            assert [c.seq_len(s) for s in seqs] == [len(path[s]) for s in seqs]
        probe = c.seq_create()
        for p in sorted(seen):
            for tail in ([5], [path[seqs[0]][len(p) - 1] + 1]):
                prompt = list(p) + tail
                best = max(common(q, prompt) for q in seen)
                assert c.prefix_match(probe, np.array(prompt, dtype=np.int32)) == min(best, len(prompt) - 1) // BT * BT
                c.seq_reset(probe)
        for s in [root, probe] + seqs:
            c.seq_release(s)
        st = c.stats()
        assert st.indexed_blocks == st.cached_blocks == 400 - st.free_blocks
