"""GPU tests of snapshots beside 8-bit blocks and evicted tokens: saves of a
sequence whose 8-bit blocks end before the segment, the refusals, and restores
over sequences whose 8-bit blocks reach up to, into and past it.  All bit for
bit."""
import numpy as np
import pytest

import _oracle as O
import kvc
import q8_ref as Q
from gpu_util import D, NKV, NQ, say
from test_gpu_q8 import SCALE, check

pytestmark = pytest.mark.gpu
IV, LAYERS = 64, 2


def filled(lens, **over):
    return Q.Filled(lens, layers=LAYERS, seed=600, extra=40, snapshot_slots=3, snapshot_interval=IV, **over)


def counts(f):
    t = f.ctx.stats()
    return t.free_blocks, f.ctx.q8_stats()[1], t.snapshots, t.indexed_blocks


def refused(f, fn):
    before = counts(f), [tuple(getattr(f.ctx.seq_info(s), n) for n in ("len", "pending", "position", "q8_tokens"))
                         for s in f.seqs]
    with pytest.raises(kvc.KvcError) as e:
        fn()
    assert e.value.code == kvc.KVC_ERR_UNSUPPORTED
    assert before == (counts(f), [tuple(getattr(f.ctx.seq_info(s), n) for n in ("len", "pending", "position", "q8_tokens"))
                                  for s in f.seqs])


@pytest.mark.parametrize("n_ssm", [0, 2])
@pytest.mark.parametrize("n8", [0, 1, 3, 4])
def test_save_and_restore_behind_8_bit_blocks(n8, n_ssm):
    """blocks 4 and 5 are the segment; the prefix is in 8 bits up to block n8"""
    say(f"snapshot behind {n8} 8-bit blocks, {n_ssm} recurrent layers")
    with filled([192], n_ssm_layers=n_ssm) as f:
        (s,) = f.seqs
        f.ctx.kv_quantize([s], 192 - 32 * n8)
        (snap,) = f.ctx.snapshot_save([s])
        rows = {k: [x.copy() for x in v] for k, v in f.rows.items()}
        f.add([s], 33)  # goes on, and back
        before = counts(f)
        f.ctx.snapshot_restore([s], [snap])
        i = f.ctx.seq_info(s)
        assert (i.len, i.position, i.q8_tokens) == (192, 192, 32 * n8)
        assert counts(f)[0] == before[0] + 2 and counts(f)[1:] == before[1:]
        for layer in range(LAYERS):
            for got, r in zip(f.gather(layer, s, 192), rows[layer, s]):
                Q.same_bits(got, Q.readback(r, 32 * n8))


@pytest.mark.parametrize("n8", [5, 6])
def test_save_of_an_8_bit_segment_is_refused(n8):
    say(f"snapshot of a segment with {n8 - 4} 8-bit blocks")
    with filled([192, 192]) as f:
        s, other = f.seqs
        f.ctx.kv_quantize([s], 192 - 32 * n8)
        refused(f, lambda: f.ctx.snapshot_save([other, s]))
        assert f.ctx.snapshot_save([other]) is not None


@pytest.mark.parametrize("n,n8", [(128, 0), (128, 4), (150, 3), (192, 4), (192, 5), (192, 6), (256, 8), (225, 7)])
def test_restore_over_8_bit_blocks(n, n8):
    """A segment of blocks 4 and 5 onto a sequence of n tokens, n8 blocks in 8
    bits: those behind block 4 go back to the 8-bit pool.  Decode, an append and a
    reset follow."""
    say(f"restore at 192 over {n} tokens, {n8} 8-bit blocks")
    with filled([192, n]) as f:
        a, b = f.seqs
        (snap,) = f.ctx.snapshot_save([a])
        start = counts(f)
        f.ctx.kv_quantize([b], n - 32 * n8)
        f.ctx.snapshot_restore([b], [snap])
        left = min(n8, 4)
        i = f.ctx.seq_info(b)
        assert (i.len, i.position, i.q8_tokens) == (192, 192, 32 * left)
        assert counts(f)[1] == start[1] - left
        blocks = (n + 31) // 32
        assert counts(f)[0] == start[0] + blocks - (6 - left)
        for layer in range(LAYERS):
            for j in range(2):
                f.rows[layer, b][j] = np.concatenate([f.rows[layer, b][j][:128], f.rows[layer, a][j][128:192]])
                Q.same_bits(f.gather(layer, b, 192)[j], Q.readback(f.rows[layer, b][j], 32 * left))
        f.add([b], 3)
        q = O.normal_bf16(NQ * D, 601).reshape(1, NQ, D)
        got = f.run(lambda x, o: f.ctx.decode_attn(1, [b], x, o), (1, NQ, D), np.float32, q)
        k, v = (Q.values(f.rows[1, b][j], 32 * left) for j in range(2))
        want, mag, big, dig = Q.attend(Q.f64(q), k, v, SCALE, digits=True)
        check(got[0].astype(np.float64), want[0], mag[0], big, False, False, "after the restore", dig[0])
        f.ctx.seq_reset(b)
        assert counts(f)[1] == start[1] and counts(f)[0] == start[0] + blocks


def test_restored_sequences_do_not_feed_the_index():
    """its prefix is not that of its token ids: what is committed after a restore
    over 8-bit blocks is not indexed"""
    say("restore over 8-bit blocks and the index")
    with filled([0, 0], max_seq_len=512, pool_blocks=64, q8_blocks=16) as f:
        c, (a, b) = f.ctx, f.seqs
        tokens = np.arange(1, 193, dtype=np.int32)
        for s in (a, b):
            c.reserve([s], 192)
            c.commit([s], 192, tokens[None])
        (snap,) = c.snapshot_save([a])
        c.kv_quantize([b], 64)
        c.snapshot_restore([b], [snap])
        before = c.stats().indexed_blocks
        c.reserve([b], 64)
        c.commit([b], 64, tokens[None, :64])
        assert c.stats().indexed_blocks == before
        m = c.seq_create()
        assert c.prefix_match(m, np.concatenate([tokens, tokens[:64]])) == 192  # a's


def test_evicted_sequences_are_refused():
    say("snapshots and eviction")
    with filled([192, 192]) as f:
        c, (a, b) = f.ctx, f.seqs
        (snap,) = c.snapshot_save([a])
        acc, kept = f.h.malloc(LAYERS * NKV * 192 * 4).zero(), f.h.malloc(LAYERS * NKV * 128 * 4)
        c.evict([b], 128, acc, 192, kept)
        c.sync()
        refused(f, lambda: c.snapshot_save([b]))
        refused(f, lambda: c.snapshot_restore([b], [snap]))
        refused(f, lambda: c.snapshot_restore([a, b], [snap, snap]))
        c.seq_truncate(b, 0)  # an empty one is an ordinary one again
        f.rows[0, b] = f.rows[1, b] = None
        f.rows = {k: v for k, v in f.rows.items() if v is not None}
        f.add([b], 128)
        c.snapshot_restore([b], [snap])
        for layer in range(LAYERS):
            for j in range(2):
                Q.same_bits(f.gather(layer, b, 192)[j], np.concatenate([f.rows[layer, b][j], f.rows[layer, a][j][128:]]))
        acc.free()
        kept.free()
