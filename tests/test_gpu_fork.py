"""GPU tests of kvc_seq_fork and kvc_seq_reorder.  Both move bytes and block
table entries, so every check is bit-exact: K/V read back through kvc_gather,
the recurrent state through kvc_state_ptrs (random 32-bit patterns, NaN
payloads included)."""
import ctypes

import numpy as np
import pytest

import _oracle as O
import kvc
from gpu_util import ROW, Mirror, fill_seq, gather, say

pytestmark = pytest.mark.gpu

LAYERS, SSM = 2, 2
FLOATS = 32 * 128 * 128 + 3 * 8192  # of one layer's state


def ctx_of(**over):
    cfg = dict(n_attn_layers=LAYERS, n_ssm_layers=SSM, max_seqs=12, max_seq_len=1024, pool_blocks=256,
               snapshot_slots=4, alloc_seed=99)
    cfg.update(over)
    return kvc.Context(**cfg)


def state_buf(ctx, s):
    return kvc.DeviceBuffer(kvc.hip(), ctx.state_ptrs(s, 0)[0], SSM * FLOATS * 4)


def write_state(ctx, s, seed):
    x = np.random.default_rng(seed).integers(0, 2**32, SSM * FLOATS, dtype=np.uint32)
    state_buf(ctx, s).upload(x)
    return x


def read_state(ctx, s):
    ctx.sync()
    return state_buf(ctx, s).download(np.uint32, SSM * FLOATS)


def check_kv(ctx, m, seqs):
    for layer in range(LAYERS):
        lens = [ctx.seq_len(s) for s in seqs]
        for s, (k, v) in zip(seqs, gather(ctx, layer, seqs, lens)):
            assert np.array_equal(k, m.get(s, layer)[0]) and np.array_equal(v, m.get(s, layer)[1]), (s, layer)


@pytest.mark.parametrize("length", [1, 32, 77])
def test_fork_copies_and_then_diverges(length):
    say(f"fork of {length} tokens")
    with ctx_of() as ctx:
        m = Mirror(LAYERS)
        s, t = ctx.seq_create(), ctx.seq_create()
        fill_seq(ctx, m, [s], length, seed=1)
        fill_seq(ctx, m, [t], 40, seed=2)
        states = {x: write_state(ctx, x, 10 + x) for x in (s, t)}
        d = [ctx.seq_create() for _ in range(5)]
        src = [s, t, s, s, t]
        ctx.fork(src, d)
        for a, b in zip(src, d):
            m.copy_seq(a, b, ctx.seq_len(a))
            assert np.array_equal(read_state(ctx, b), states[a])
        check_kv(ctx, m, [s, t] + d)
        fill_seq(ctx, m, d + [s], 3, seed=5)  # each its own rows: shared blocks are copied first
        check_kv(ctx, m, [s, t] + d)
        write_state(ctx, d[0], 77)
        assert np.array_equal(read_state(ctx, s), states[s])
        assert np.array_equal(read_state(ctx, d[2]), states[s])
        ctx.seq_release(s)
        check_kv(ctx, m, [t] + d)


def test_fork_of_sequences_without_state_or_tokens():
    say("fork of a fresh sequence")
    with ctx_of() as ctx:
        old = ctx.seq_create()
        write_state(ctx, old, 3)
        ctx.seq_release(old)
        s, d = ctx.seq_create(), ctx.seq_create()
        write_state(ctx, d, 4)
        ctx.seq_reset(d)
        ctx.fork([s], [d])  # s takes the released slot: its state reads as zero, and so does the copy's
        assert not read_state(ctx, d).any() and not read_state(ctx, s).any()


def test_fork_of_more_than_one_launch():
    say("fork of 130 sequences")
    with ctx_of(n_ssm_layers=SSM, max_seqs=140, pool_blocks=512) as ctx:
        m = Mirror(LAYERS)
        src = [ctx.seq_create() for _ in range(3)]
        for i, s in enumerate(src):
            fill_seq(ctx, m, [s], 50 + i, seed=20 + i)
        states = [write_state(ctx, s, 30 + i) for i, s in enumerate(src)]
        d = [ctx.seq_create() for _ in range(130)]
        who = [int(x) for x in np.random.default_rng(5).integers(0, 3, 130)]
        ctx.fork([src[w] for w in who], d)
        for w, x in zip(who, d):
            m.copy_seq(src[w], x, 50 + w)
        check_kv(ctx, m, d)
        for i in (0, 1, 63, 64, 65, 127, 128, 129):
            assert np.array_equal(read_state(ctx, d[i]), states[who[i]]), i


@pytest.mark.parametrize("parents", [[0, 1, 2, 3, 4, 5], [1, 2, 3, 4, 5, 0], [3, 3, 3, 3, 3, 3], [1, 0, 0, 1, 5, 5],
                                     [5, 4, 3, 2, 1, 0], [2, 2, 1, 1, 0, 0]])
def test_reorder(parents):
    say(f"reorder {parents}")
    with ctx_of() as ctx:
        m = Mirror(LAYERS)
        seqs = [ctx.seq_create() for _ in range(6)]
        fill_seq(ctx, m, seqs[:1], 70, seed=1)
        ctx.fork(seqs[:1] * 5, seqs[1:])
        for s in seqs[1:]:
            m.copy_seq(seqs[0], s, 70)
        for i, s in enumerate(seqs):
            fill_seq(ctx, m, [s], 1 + 9 * i, seed=40 + i)
        states = [write_state(ctx, s, 50 + i) for i, s in enumerate(seqs)]
        for turn in range(3):  # again and again: what moved is the next call's start
            was = {(s, la): m.get(s, la) for s in seqs for la in range(LAYERS)}
            ctx.reorder(seqs, parents)
            states = [states[p] for p in parents]
            for s, p in zip(seqs, parents):
                for la in range(LAYERS):
                    m.k[(s, la)], m.v[(s, la)] = was[(seqs[p], la)]
            for s, x in zip(seqs, states):
                assert np.array_equal(read_state(ctx, s), x), (turn, s)
            check_kv(ctx, m, seqs)
            fill_seq(ctx, m, seqs, 2, seed=60 + turn)
            check_kv(ctx, m, seqs)
        for s in seqs:  # every slot still belongs to one sequence
            ctx.seq_release(s)
        fresh = [ctx.seq_create() for _ in range(12)]
        assert len({ctx.state_ptrs(s, 0)[0] for s in fresh}) == 12
        assert not any(read_state(ctx, s).any() for s in fresh)


def test_step_snapshot_and_reset_follow_a_reorder():
    say("DeltaNet steps, snapshots and resets behind a reorder")
    h = kvc.hip()
    with ctx_of() as ctx:
        m = Mirror(LAYERS)
        a, b, c = (ctx.seq_create() for _ in range(3))
        fill_seq(ctx, m, [a, b, c], 256, seed=3)
        for s in (a, b, c):
            state_buf(ctx, s).upload(np.random.default_rng(s).standard_normal(SSM * FLOATS).astype(np.float32))
        ctx.reorder([a, b, c], [1, 0, 0])
        want = {s: read_state(ctx, s) for s in (a, b, c)}
        ids = ctx.snapshot_save([a, b])
        d = ctx.seq_create()
        ctx.snapshot_restore([d], ids[:1])
        assert np.array_equal(read_state(ctx, d), want[a])
        proj = kvc.to_device(O.normal_bf16(4 * 12352, 7))
        w = [kvc.to_device(np.random.default_rng(8 + i).standard_normal(n).astype(np.float32) * 0.1)
             for i, n in enumerate((4 * 8192, 32, 32, 128))]
        out = h.malloc(4 * 4096 * 4)
        ctx.deltanet_step(0, [a, b, c, d], 1, proj, *w, out)
        x = out.download(np.uint32, (4, 4096))
        y = {s: read_state(ctx, s) for s in (a, b, c, d)}
        # b and c held one state, a and d another: the same row gives the same step
        rows = np.tile(O.normal_bf16(12352, 9), 4)
        ctx.reorder([a, b, c, d], [3, 2, 2, 3])
        proj.upload(rows)
        ctx.deltanet_step(0, [a, b, c, d], 1, proj, *w, out)
        x = out.download(np.uint32, (4, 4096))
        assert np.array_equal(x[0], x[3]) and np.array_equal(x[1], x[2]) and not np.array_equal(x[0], x[1])
        assert not np.array_equal(read_state(ctx, a), y[d])
        ctx.seq_reset(b)
        assert not read_state(ctx, b).any() and np.array_equal(read_state(ctx, a), read_state(ctx, d))
        ctx.reorder([a, b], [1, 1])  # a zeroed state moves on as one
        assert not read_state(ctx, a).any() and not read_state(ctx, b).any()
        for buf in (proj, out, *w):
            buf.free()


def test_own_stream_and_capture():
    say("fork and reorder on a stream of their own, and under capture")
    h = kvc.hip()
    st = h.stream()
    with ctx_of() as ctx:
        m = Mirror(LAYERS)
        a, b, c = (ctx.seq_create() for _ in range(3))
        fill_seq(ctx, m, [a], 50, seed=1)
        x = write_state(ctx, a, 2)
        write_state(ctx, c, 3)
        h.sync()
        ctx.fork([a], [b], stream=st)
        ctx.reorder([a, b, c], [2, 0, 1], stream=st)
        ctx.sync(st)
        h.sync()
        assert np.array_equal(read_state(ctx, b), x) and np.array_equal(read_state(ctx, c), x)
        m.copy_seq(a, b, 50)
        m.copy_seq(a, c, 50)
        check_kv(ctx, m, [b, c])
        d = ctx.seq_create()

        def refused():
            for call in (lambda: ctx.fork([b], [d], stream=st), lambda: ctx.reorder([a, b], [1, 0], stream=st)):
                with pytest.raises(kvc.KvcError) as e:
                    call()
                assert e.value.code == kvc.KVC_ERR_STATE

        ex = ctypes.c_void_p()
        h.ok(h.L.hipStreamBeginCapture(st, 0), "capture")
        refused()
        h.ok(h.L.hipStreamEndCapture(st, ctypes.byref(ex)), "end capture")
        assert ctx.seq_len(d) == 0 and ctx.seq_len(b) == 50
    h.ok(h.L.hipStreamDestroy(st), "hipStreamDestroy")
