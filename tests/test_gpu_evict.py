"""GPU tests of attention weights and eviction against 64-bit results, alone and
in the run they are made for: attend, accumulate, evict, park in 8 bits, go on.

Tolerance of the accumulated weights (derived): a weight's score is within
2^-22 B of the exact one in the log2 domain (B as in test_gpu_q8.py), the
exponential, the row's sum and the division add 2^-21, and the sum over the
rows of a token loses at most 2^-24 of the result per row."""
import numpy as np
import pytest

import _oracle as O
import kvc
import q8_ref as Q
from gpu_util import D, NKV, NQ, say

pytestmark = pytest.mark.gpu
SCALE = 1.0 / 16


def weights_case(lens, n_q, keep, scale=SCALE, seed=90, acc="own", pending=0, stride_more=3):
    with Q.Filled(lens, seed=seed, extra=pending) as f:
        f.ctx.kv_quantize(f.seqs, keep)
        if pending:
            f.add(f.seqs, pending, commit=False)
        n = len(lens)
        total = [x + pending for x in lens]
        stride = max(total) + stride_more
        q = O.normal_bf16(n * n_q * NQ * D, seed + 1).reshape(n, n_q, NQ, D)
        start = np.random.default_rng(seed).random((n, NKV, stride)).astype(np.float32)
        qb, ab, ob = kvc.to_device(q), kvc.to_device(start), kvc.to_device(np.full_like(start, 7.0))
        src = {"own": ab, "none": None, "same": ob}[acc]
        if acc == "same":
            ob.upload(start)
        f.ctx.attn_weights(0, f.seqs, n_q, qb, ob, stride, acc_in=src, scale=scale)
        f.ctx.sync()
        got = ob.download(np.float32, start.shape)
        if acc != "same":  # the same call, the same bits
            f.ctx.attn_weights(0, f.seqs, n_q, qb, ob, stride, acc_in=src, scale=scale)
            f.ctx.sync()
            assert np.array_equal(ob.download(np.uint32, start.shape), got.view(np.uint32))
            assert np.array_equal(ab.download(np.uint32, start.shape), start.view(np.uint32))
        for x in (qb, ab, ob):
            x.free()
        for i, s in enumerate(f.seqs):
            n8 = max(0, lens[i] - keep) // 32 * 32
            k = Q.values(f.rows[0, s][0], n8)
            w = Q.weights(Q.f64(q[i]), k, scale, total[i] - n_q)
            _, _, big = Q.attend(Q.f64(q[i]), k, k, scale, first=total[i] - n_q)
            base = start[i].astype(np.float64) if acc != "none" else np.zeros((NKV, stride))
            want = base[:, :total[i]] + w
            rows = 4 * n_q
            tol = w * (2.0 ** -22 * big + 2.0 ** -21) + want * 2.0 ** -24 * (rows + 1)
            off = np.abs(got[i, :, :total[i]] - want) / np.maximum(tol, 1e-30)
            assert off.max() <= 1.0, (i, lens[i], float(off.max()))
            say(f"  {n_q} rows over {total[i]} ({n8} in 8 bits): {off.max():.3f} of the tolerance")
            rest = start[i, :, total[i]:] if acc == "same" else np.float32(7.0)
            assert (got[i, :, total[i]:] == rest).all()


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 127, 128, 129, 300, 1000, 4100])
@pytest.mark.parametrize("keep", [0, 10 ** 6])
def test_weights_of_one_token(n, keep):
    say(f"weights {n} keep {keep}")
    weights_case([n], 1, keep, seed=91 + n)


@pytest.mark.parametrize("n,n_q", [(2, 2), (33, 33), (40, 3), (64, 16), (300, 5), (300, 32), (511, 100), (700, 256)])
def test_weights_of_several_rows(n, n_q):
    """rows that end inside 8-bit blocks too: the last of them are committed"""
    say(f"weights {n_q} rows of {n}")
    weights_case([n], n_q, 0, seed=92 + n)


@pytest.mark.parametrize("acc", ["own", "none", "same"])
def test_weights_of_a_ragged_batch(acc):
    say(f"weights ragged acc {acc}")
    weights_case([7, 32, 64, 100, 1500, 333, 96, 12], 7, 50, seed=93, acc=acc)


def test_weights_with_pending_rows():
    say("weights pending")
    weights_case([100, 64, 31], 4, 0, seed=94, pending=4, stride_more=0)


@pytest.mark.parametrize("scale", [0.0, -0.25])
def test_weights_scales(scale):
    say(f"weights scale {scale}")
    weights_case([200], 3, 40, scale=scale, seed=95)


def test_weights_in_several_launches():
    """70 sequences, and 12 of 2000 keys with 128 rows each"""
    say("weights 70 sequences")
    weights_case([int(x) for x in np.random.default_rng(1).integers(5, 200, 70)], 3, 20, seed=96)
    say("weights 128 rows")
    weights_case([2000] * 12, 128, 0, seed=97)


@pytest.mark.parametrize("n,n_q", [(20, 4), (40, 256)])
def test_weights_that_fill_the_workspace(n, n_q):
    """stored scores (20 sequences of 30000 keys: 156 MB) and row statistics (40:
    154 MB) take two launches: the bits of calls of one sequence each"""
    say(f"weights, workspace filled by {n_q} queries")
    L = 30000
    with Q.Filled([0], seed=110, max_seqs=n + 1, max_seq_len=L, pool_blocks=n * (L // 32 + 1), q8_blocks=8) as f:
        c, h = f.ctx, f.h
        c.pool_fill_normal(5)
        seqs = [f.seqs[0]] + [c.seq_create() for _ in range(n - 1)]
        c.reserve(seqs, L)
        c.commit(seqs, L)
        q = kvc.to_device(O.normal_bf16(n * n_q * NQ * D, 111))
        per = NKV * L * 4
        a, b = h.malloc(n * per).zero(), h.malloc(n * per).zero()
        h.sync()
        c.attn_weights(0, seqs, n_q, q, a, L)
        for i, s in enumerate(seqs):
            c.attn_weights(0, [s], n_q, q.ptr + i * n_q * NQ * D * 2, b.ptr + i * per, L)
        c.sync()
        x, y = (z.download(np.float32, (n, NKV, L)) for z in (a, b))
        assert np.array_equal(x, y)
        # a row's weights sum to 1 within the scores' 2^-22 sum |q k| scale log2(e), below 64 here
        assert np.abs(x.sum(2, dtype=np.float64) - 4 * n_q).max() <= 4 * n_q * 2.0 ** -16
        for z in (q, a, b):
            z.free()


def test_alignment_refusals():
    say("weights and evict alignment")
    with Q.Filled([100], seed=98) as f:
        c, (a,) = f.ctx, f.seqs
        buf = kvc.hip().malloc(1 << 20).zero()
        P, F = buf.ptr, buf.ptr + (1 << 19)
        for call in (lambda: c.attn_weights(0, [a], 1, P + 8, F, 100), lambda: c.attn_weights(0, [a], 1, P, F + 2, 100),
                     lambda: c.attn_weights(0, [a], 1, P, F, 100, acc_in=F + 4001), lambda: c.evict([a], 50, P + 1, 100, F),
                     lambda: c.evict([a], 50, P, 100, F + 2), lambda: c.evict([a], 50, P, 100, F, acc_out=F + 8003)):
            with pytest.raises(kvc.KvcError) as e:
                call()
            assert e.value.code == kvc.KVC_ERR_INVALID
        c.sync()
        assert not buf.download(np.uint8, (1 << 20,)).any() and c.seq_len(a) == 100
        buf.free()


@pytest.mark.parametrize("lens,n_q", [([200, 31, 900], 4), ([200, 31, 900], 5), ([257, 600], 33)])
def test_weights_around_a_tile_of_rows(lens, n_q):
    """16 rows per kv head are the last whose scores are stored, 128 the last
    that are staged at once; the rows end inside a tile and inside blocks"""
    if min(lens) < n_q:
        lens = [max(x, n_q) for x in lens]
    for keep in (0, 40):
        say(f"weights {lens} {n_q} rows keep {keep}")
        weights_case(lens, n_q, keep, seed=109 + n_q)


def test_weights_refusals():
    say("weights refusals")
    with Q.Filled([100, 40], seed=98) as f:
        c, (a, b) = f.ctx, f.seqs
        buf = kvc.hip().malloc(1 << 20).zero()
        P = buf.ptr
        for code, args in [
            (kvc.KVC_ERR_INVALID, dict(seqs=[a], n_q=0, q=P, acc_out=P, acc_stride=100)),
            (kvc.KVC_ERR_INVALID, dict(seqs=[a], n_q=1, q=None, acc_out=P, acc_stride=100)),
            (kvc.KVC_ERR_INVALID, dict(seqs=[a], n_q=1, q=P, acc_out=None, acc_stride=100)),
            (kvc.KVC_ERR_INVALID, dict(seqs=[a], n_q=1, q=P, acc_out=P, acc_stride=100, scale=float("nan"))),
            (kvc.KVC_ERR_INVALID, dict(seqs=[a, a], n_q=1, q=P, acc_out=P, acc_stride=100)),
            (kvc.KVC_ERR_INVALID, dict(seqs=[a], n_q=1, q=P, acc_out=P, acc_in=P + 400, acc_stride=100)),
            (kvc.KVC_ERR_RANGE, dict(seqs=[b], n_q=257, q=P, acc_out=P, acc_stride=100)),
            (kvc.KVC_ERR_RANGE, dict(seqs=[a], n_q=1, q=P, acc_out=P, acc_stride=99)),
            (kvc.KVC_ERR_STATE, dict(seqs=[a, b], n_q=41, q=P, acc_out=P, acc_stride=100)),
        ]:
            with pytest.raises(kvc.KvcError) as e:
                c.attn_weights(0, **args)
            assert e.value.code == code, args
        with pytest.raises(kvc.KvcError) as e:
            c.attn_weights(1, [a], 1, P, P, 100)
        assert e.value.code == kvc.KVC_ERR_RANGE
        c.sync()
        assert not buf.download(np.uint8, (1 << 20,)).any()
        buf.free()


# ---- eviction -------------------------------------------------------------------


def accumulated(kind, shape, rng):
    a = rng.random(shape).astype(np.float32) ** 6
    if kind == "ties":
        a = np.floor(a * 8).astype(np.float32) / 8
    elif kind == "equal":
        a[:] = 0.25
    elif kind == "special":
        a = rng.normal(size=shape).astype(np.float32)  # negative ones too
        flat = a.reshape(-1)
        pick = rng.permutation(flat.size)
        m = max(1, flat.size // 12)
        for j, x in enumerate((np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-42)):
            flat[pick[j * m:(j + 1) * m]] = x
    return a


def evict_case(lens, budget, sink, recent, kind, copy, keep=10 ** 6, seed=100, layers=2, with_acc_out=True):
    with Q.Filled(lens, layers=layers, seed=seed) as f:
        f.ctx.kv_quantize(f.seqs, keep)
        n, stride = len(lens), max(lens) + 5
        acc = accumulated(kind, (layers, n, NKV, stride), np.random.default_rng(seed))
        ab = kvc.to_device(acc)
        kb = kvc.hip().malloc(layers * n * NKV * budget * 4)
        kb.upload(np.full((layers, n, NKV, budget), -9, np.int32))
        ob = kvc.to_device(np.full_like(acc, 7.0)) if with_acc_out else None
        dst = [f.ctx.seq_create() for _ in lens] if copy else None
        f.ctx.evict(f.seqs, budget, ab, stride, kb, n_sink=sink, n_recent=recent, dst=dst, acc_out=ob)
        f.ctx.sync()
        kept = kb.download(np.int32, (layers, n, NKV, budget))
        out = ob.download(np.float32, acc.shape) if with_acc_out else None
        assert np.array_equal(ab.download(np.uint32, acc.shape), acc.view(np.uint32))
        for i, L in enumerate(lens):
            new = min(L, budget)
            s = dst[i] if copy else f.seqs[i]
            assert f.ctx.seq_len(s) == new and f.ctx.seq_info(s).position == L
            n8 = max(0, L - keep) // 32 * 32
            for layer in range(layers):
                rows = [Q.readback(x, n8) for x in f.rows[layer, f.seqs[i]]]
                got = f.gather(layer, s, new)
                for h in range(NKV):
                    want = Q.keep(acc[layer, i, h, :L], budget, sink, recent)
                    assert np.array_equal(kept[layer, i, h, :new], want), (L, layer, h)
                    assert (kept[layer, i, h, new:] == -1).all()
                    if out is not None:
                        assert np.array_equal(out[layer, i, h, :new].view(np.uint32),
                                              acc[layer, i, h][want].view(np.uint32))
                        assert (out[layer, i, h, new:L] == 0).all() and (out[layer, i, h, L:] == 7).all()
                    for j in range(2):
                        Q.same_bits(got[j][:, h], rows[j][want, h])
                if copy:
                    for j in range(2):
                        Q.same_bits(f.gather(layer, f.seqs[i], L)[j], rows[j])
        for b in (ab, kb, ob):
            if b is not None:
                b.free()


@pytest.mark.parametrize("kind", ["plain", "ties", "equal", "special"])
@pytest.mark.parametrize("copy", [False, True])
def test_evict_choices(kind, copy):
    say(f"evict {kind} copy {copy}")
    evict_case([300, 64, 65, 1, 1100, 200], 64, 3, 20, kind, copy, seed=101)


@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (50, 50, 0), (50, 0, 50), (33, 16, 17),
                                                (199, 0, 0), (200, 4, 4), (500, 1, 1)])
def test_evict_budgets(budget, sink, recent):
    say(f"evict {budget} {sink} {recent}")
    evict_case([200, 33], budget, sink, recent, "ties", False, seed=102, with_acc_out=budget % 2 == 0)


def test_evict_long_rows():
    """rows longer than a workgroup, with ties across its passes"""
    say("evict 5000")
    evict_case([5000, 2048, 1025], 1001, 2, 100, "ties", True, seed=103, layers=1)


@pytest.mark.parametrize("lens", [[8192, 1], [8193, 70, 2049]])
@pytest.mark.parametrize("kind", ["ties", "special"])
def test_evict_longest_rows(lens, kind):
    """the longest rows whose keys stay in registers, and longer ones"""
    say(f"evict {lens} {kind}")
    evict_case(lens, 2500, 3, 77, kind, True, seed=108, layers=1)


@pytest.mark.parametrize("keep", [0, 100])
def test_evict_8_bit_sources(keep):
    say(f"evict 8-bit keep {keep}")
    evict_case([300, 128, 97], 90, 1, 7, "plain", keep == 0, keep=keep, seed=104)


def test_evict_70_sequences():
    say("evict 70")
    evict_case([int(x) for x in np.random.default_rng(9).integers(1, 150, 70)], 40, 2, 5, "plain", False, seed=105, layers=1)


def test_positions_go_on_after_eviction():
    """kvc_qkv_append rotates a new token at its position in the text: the rows
    equal those of a sequence that kept everything; the one-launch steps and the
    snapshots refuse the cut sequence."""
    say("evict positions")
    rng = np.random.default_rng(6)
    with Q.Filled([150, 150, 90], seed=106, extra=4, rope_dim=64, snapshot_slots=2, snapshot_interval=32,
                  max_seq_len=160) as f:
        c, (a, b, d) = f.ctx, f.seqs
        acc = kvc.to_device(rng.random((1, 1, NKV, 150)).astype(np.float32))
        kept = kvc.hip().malloc(NKV * 64 * 4)
        c.evict([a], 64, acc, 150, kept)
        row = NQ * 2 * D + 2 * NKV * D
        qkv = kvc.to_device(O.normal_bf16(3 * row, 5))
        w = kvc.to_device((rng.random(D) + 0.5).astype(np.float32))
        for s, n in ((a, 64), (b, 150)):
            c.reserve([s], 3)
            qo = kvc.hip().malloc(3 * NQ * D * 2)
            c.qkv_append(0, [s], 3, qkv, w, w, q_out=qo)
            c.commit([s], 3)
            c.sync()
            got = f.gather(0, s, 3, n) + [qo.download(np.uint16, (3, NQ, D))]
            if s == a:
                want = got
            for x, y in zip(got, want):
                assert np.array_equal(x, y)
        assert c.seq_info(a).position == 153 and c.seq_len(a) == 67
        # a batch of sequences with different shifts
        c.reserve([a, d], 1)
        c.qkv_append(0, [d, a], 1, qkv, w, w)
        un = kvc.KVC_ERR_UNSUPPORTED
        for call in (lambda: c.decode_step(0, [a], qkv, w, w, qo), lambda: c.prefill_step(0, [a], 1, qkv, w, w, qo)):
            with pytest.raises(kvc.KvcError) as e:
                call()
            assert e.value.code == un
        c.commit([a, d], 1)
        c.seq_truncate(a, 64)
        for call in (lambda: c.snapshot_save([a]),):
            with pytest.raises(kvc.KvcError) as e:
                call()
            assert e.value.code == un
        c.reserve([a], 11)  # position 150 + 11 is past max_seq_len 160
        with pytest.raises(kvc.KvcError) as e:
            c.qkv_append(0, [a], 11, qkv, w, w)
        assert e.value.code == kvc.KVC_ERR_RANGE


def test_the_run_they_are_made_for():
    """Two sessions: a prompt, its window's weights, a cut, the rest in 8 bits,
    then decode steps that go on accumulating, another cut and a new chunk."""
    say("evict + 8 bits run")
    n_q, budget, layers = 16, 96, 2
    rng = np.random.default_rng(8)
    with Q.Filled([400, 250], layers=layers, seed=107, extra=400) as f:
        c, seqs = f.ctx, f.seqs
        stride = 512
        acc = [kvc.hip().malloc(layers * 2 * NKV * stride * 4).zero() for _ in range(2)]
        per = 2 * NKV * stride * 4
        model = {}  # (layer, i) -> [k, v] values, and accumulated weights
        for layer in range(layers):
            for i, s in enumerate(seqs):
                model[layer, i] = [[Q.f64(x) for x in f.rows[layer, s]], np.zeros((NKV, len(f.rows[layer, s][0])))]

        def accumulate(n_q):
            for layer in range(layers):
                q = O.normal_bf16(2 * n_q * NQ * D, int(rng.integers(1 << 30))).reshape(2, n_q, NQ, D)
                qb = kvc.to_device(q)
                at = acc[0].ptr + layer * per
                c.attn_weights(layer, seqs, n_q, qb, at, stride, acc_in=at)
                c.sync()
                qb.free()
                for i in range(2):
                    (k, _), w = model[layer, i]
                    w += Q.weights(Q.f64(q[i]), k, SCALE, len(k) - n_q)
            got = acc[0].download(np.float32, (layers, 2, NKV, stride))
            for layer in range(layers):
                for i in range(2):
                    w = model[layer, i][1]
                    assert np.abs(got[layer, i, :, :w.shape[1]] - w).max() <= 2.0 ** -16 * max(1.0, w.max())

        def cut():
            kept = kvc.hip().malloc(layers * 2 * NKV * budget * 4)
            c.evict(seqs, budget, acc[0], stride, kept, n_sink=2, n_recent=12, acc_out=acc[1])
            c.sync()
            acc.reverse()
            got = kept.download(np.int32, (layers, 2, NKV, budget))
            kept.free()
            for layer in range(layers):
                for i in range(2):
                    kv, w = model[layer, i]
                    idx = got[layer, i]
                    # the choice is the one of the device's own sums: held to
                    # the model's where no two of its values are near
                    for h in range(NKV):
                        want = Q.keep(w[h], budget, 2, 12)
                        assert len(np.setdiff1d(want, idx[h])) <= 1
                    model[layer, i] = [[np.stack([x[idx[h], h] for h in range(NKV)], 1) for x in kv],
                                       np.stack([w[h][idx[h]] for h in range(NKV)])]

        def park(keep):
            c.kv_quantize(seqs, keep)
            for layer in range(layers):
                for i in range(2):
                    kv, _ = model[layer, i]
                    n8 = c.seq_info(seqs[i]).q8_tokens
                    model[layer, i][0] = [np.concatenate([Q.values(Q.bf16_bits(x[:n8]), n8), x[n8:]]) for x in kv]

        def step():
            c.reserve(seqs, 1)
            for layer in range(layers):
                q, k, v = (O.normal_bf16(2 * w * D, int(rng.integers(1 << 30))).reshape(2, w, D) for w in (NQ, NKV, NKV))
                got = f.run(lambda a, b, d, o: c.decode_attn(layer, seqs, a, o, k_new=b, v_new=d), (2, NQ, D), np.float32,
                            q, k, v)
                for i in range(2):
                    kv, w = model[layer, i]
                    kv = [np.concatenate([x, Q.f64(y[i])[None]]) for x, y in zip(kv, (k, v))]
                    model[layer, i] = [kv, np.concatenate([w, np.zeros((NKV, 1))], 1)]
                    want, mag, big, dig = Q.attend(Q.f64(q[i])[None], *kv, SCALE, digits=True)
                    tol = mag * 2.0 ** -22 * (big + 2) + np.abs(want) * 2.0 ** -22 + 2.0 ** -30 * dig
                    assert (np.abs(got[i] - want[0]) <= tol[0]).all()
            c.commit(seqs, 1)

        accumulate(n_q)
        cut()
        park(20)
        assert c.seq_info(seqs[0]).q8_tokens == 64
        for _ in range(5):
            step()
        # weights over the mixed cache, then a cut that reads 8-bit rows
        for layer in range(layers):
            q = O.normal_bf16(2 * NQ * D, 77 + layer).reshape(2, 1, NQ, D)
            qb = kvc.to_device(q)
            at = acc[0].ptr + layer * per
            c.attn_weights(layer, seqs, 1, qb, at, stride, acc_in=at)
            c.sync()
            qb.free()
            for i in range(2):
                (k, _), w = model[layer, i]
                w += Q.weights(Q.f64(q[i]), k, SCALE, len(k) - 1)
        cut()
        for layer in range(layers):
            for i in range(2):
                n = len(model[layer, i][0][0])
                for got, x in zip(f.gather(layer, seqs[i], n), model[layer, i][0]):
                    Q.same_bits(got, Q.bf16_bits(x))
                model[layer, i][0] = [Q.f64(Q.bf16_bits(x)) for x in model[layer, i][0]]
        park(20)
        step()
        assert c.seq_info(seqs[0]).position == 400 + 6 and c.seq_len(seqs[0]) == budget + 1


def test_calls_in_a_row_on_a_stream():
    """weights, a cut, 8 bits, a chunk's rows, its attention and a decode step,
    queued on a stream of their own with nothing waited for: the bits of the
    same calls made one after the other"""
    say("a run on a stream")
    h = kvc.hip()
    layers, n_q, budget, stride = 2, 16, 700, 1500
    rng = np.random.default_rng(14)
    rows = [O.normal_bf16(3 * n_q * NKV * D, 140 + i).reshape(3, n_q, NKV, D) for i in range(2)]
    q = O.normal_bf16(3 * n_q * NQ * D, 142)
    start = rng.random((layers, 3, NKV, stride)).astype(np.float32)

    def run(stream, sync):
        with Q.Filled([1400, 333, 900], layers=layers, seed=143, extra=n_q) as f:
            c, seqs = f.ctx, f.seqs
            qb, kb, vb = kvc.to_device(q), kvc.to_device(rows[0]), kvc.to_device(rows[1])
            acc = kvc.to_device(start)
            acc2 = kvc.to_device(np.full_like(start, 7.0))
            kept = h.malloc(layers * 3 * NKV * budget * 4)
            outs = [h.malloc(3 * n_q * NQ * D * 4) for _ in range(layers)] + [h.malloc(3 * NQ * D * 4) for _ in range(layers)]
            h.sync()
            per = 3 * NKV * stride * 4
            steps = [lambda l=l: c.attn_weights(l, seqs, n_q, qb, acc.ptr + l * per, stride, acc_in=acc.ptr + l * per,
                                                stream=stream) for l in range(layers)]
            steps += [lambda: c.evict(seqs, budget, acc, stride, kept, n_sink=4, n_recent=64, acc_out=acc2, stream=stream),
                      lambda: c.kv_quantize(seqs, 30, stream=stream), lambda: c.reserve(seqs, n_q, stream=stream)]
            for l in range(layers):
                steps += [lambda l=l: c.append(l, seqs, n_q, kb, vb, stream=stream),
                          lambda l=l: c.prefill_attn(l, seqs, n_q, qb, outs[l], stream=stream)]
            steps += [lambda: c.commit(seqs, n_q, stream=stream)]
            steps += [lambda l=l: c.decode_attn(l, seqs, qb, outs[layers + l], stream=stream) for l in range(layers)]
            for s in steps:
                s()
                if sync:
                    h.sync()
            h.sync()
            assert [c.seq_info(s).position for s in seqs] == [1416, 349, 916]
            assert [c.seq_len(s) for s in seqs] == [716, 349, 716]
            got = [acc.download(np.uint32, start.shape), acc2.download(np.uint32, start.shape),
                   kept.download(np.int32, (layers, 3, NKV, budget))]
            return got + [o.download(np.uint32, (3, (n_q if i < layers else 1) * NQ * D)) for i, o in enumerate(outs)]

    st = h.stream()
    for a, b in zip(run(None, True), run(st, False)):
        assert np.array_equal(a, b)


def test_blocks_past_4_gib():
    """pools of which a layer's K or V is over 4 GiB, bf16 and 8-bit: block ids
    on either side"""
    say("blocks past 4 GiB")
    big = 66000  # blocks; 32 KiB each in 8 bits, 64 KiB in bf16
    with Q.Filled([0], seed=150, max_seqs=4, max_seq_len=big * 32, pool_blocks=2 * big + 2000, q8_blocks=2 * big + 100) as f:
        c = f.ctx
        c.pool_fill_normal(3)
        fill = [f.seqs[0], c.seq_create()]
        for s in fill:  # the 8-bit ids below 4 GiB
            c.reserve([s], big * 32)
            c.commit([s], big * 32)
            c.kv_quantize([s])
            assert c.seq_info(s).q8_tokens == big * 32
        c.sync()
        a = c.seq_create()
        n = 2000
        f.add([a], n)
        c.kv_quantize([a], 900)  # 34 8-bit blocks, 29 bf16 ones spread over their pool
        rows = f.rows[0, a]
        for got, x in zip(f.gather(0, a, n), rows):
            Q.same_bits(got, Q.readback(x, 1088))
        for n_q in (1, 8, 600):  # decode, and either prefill
            if n_q > 1:
                f.add([a], n_q, commit=False)
                n += n_q
            k, v = (Q.values(x, 1088) for x in f.rows[0, a])
            q = O.normal_bf16(n_q * NQ * D, 151 + n_q).reshape(1, n_q, NQ, D)
            if n_q == 1:
                got = f.run(lambda x, o: c.decode_attn(0, [a], x, o, scale=SCALE), (1, NQ, D), np.float32, q)
            else:
                got = f.run(lambda x, o: c.prefill_attn(0, [a], n_q, x, o, scale=SCALE), (n_q, NQ, D), np.float32, q)
            want, mag, big_qk, dig = Q.attend(Q.f64(q[0]), k, v, SCALE, first=n - n_q, digits=True)
            tol = mag * 2.0 ** -22 * (big_qk + 2) + np.abs(want) * 2.0 ** -22 + 2.0 ** -30 * dig
            assert (np.abs(got - want) <= tol).all(), n_q
            if n_q <= 8:
                w = f.run(lambda x, o: c.attn_weights(0, [a], n_q, x, o, n, scale=SCALE), (1, NKV, n), np.float32, q)
                assert np.abs(w[0] - Q.weights(Q.f64(q[0]), k, SCALE, n - n_q)).max() <= 2.0 ** -16
            if n_q > 1:
                c.commit([a], n_q)
        acc = np.random.default_rng(152).random((1, 1, NKV, n)).astype(np.float32)
        ab, kept = kvc.to_device(acc), kvc.hip().malloc(NKV * 500 * 4)
        c.evict([a], 500, ab, n, kept, n_sink=2, n_recent=9)
        back = [Q.readback(x, 1088) for x in f.rows[0, a]]
        got = f.gather(0, a, 500)
        for h in range(NKV):
            want = Q.keep(acc[0, 0, h], 500, 2, 9)
            for j in range(2):
                Q.same_bits(got[j][:, h], back[j][want, h])


def test_calls_that_change_tables_are_not_captured():
    say("quantize and evict refuse capture")
    h = kvc.hip()
    with Q.Filled([200, 100], seed=160) as f:
        c, seqs = f.ctx, f.seqs
        st = h.stream()
        acc, kept = h.malloc(2 * NKV * 200 * 4).zero(), h.malloc(2 * NKV * 50 * 4).zero()
        out = h.malloc(2 * NKV * 200 * 4).zero()
        q = kvc.to_device(O.normal_bf16(2 * NQ * D, 161))
        h.sync()
        codes = []

        def body():
            for call in (lambda: c.kv_quantize(seqs, stream=st), lambda: c.evict(seqs, 50, acc, 200, kept, stream=st)):
                try:
                    call()
                    codes.append(0)
                except kvc.KvcError as e:
                    codes.append(e.code)
            c.attn_weights(0, seqs, 1, q, out, 200, stream=st)

        g = h.capture(st, body)
        assert codes == [kvc.KVC_ERR_STATE] * 2
        h.graph_launch(g, st)
        h.stream_sync(st)
        assert [c.seq_len(s) for s in seqs] == [200, 100] and c.seq_info(seqs[0]).q8_tokens == 0
        assert not kept.download(np.uint32, (2 * NKV * 50,)).any()
        got = out.download(np.float32, (2, NKV, 200))
        assert np.abs(got[0].sum(1) - 4).max() < 1e-4 and np.abs(got[1].sum(1) - 4).max() < 1e-4
        h.graph_destroy(g)
