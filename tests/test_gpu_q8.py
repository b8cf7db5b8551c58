"""GPU tests of the 8-bit blocks: quantize and read back bit for bit, decode and
prefill attention over sequences that start with 8-bit blocks against 64-bit
results.

Tolerances (derived, per element; W = sum w |v| of the element, B = the largest
sum |q k| scale log2(e) over a key):
  scores   fp32 sums of exact products: within 2^-22 B in the log2 domain (16
           partial sums of 2^-24 each), times ln 2 on a weight, plus 2^-22 for
           the exponential and the sums of weights: below 2^-22 (B + 2)
  decode   W 2^-22 (B + 2).  A weight over an 8-bit block is cut to
           30 bits below the block's largest weight of the head, so it is less
           than 2^-30 of that off, however small it is itself: another
           2^-30 sum over keys of |v| (largest weight of the key's block).
           That is what remains where the heavy keys' v is 0: with one key of
           weight 1 and 31 light ones, 2^-30 * 31 |v| beside W near 0
  prefill  fp32 out: the same (weights in three bf16 parts, 2^-26); bf16 out:
           weights as one bf16 part, 2^-8 each
  bf16 output: half a step more, 2^-8 of the value
and 2^-22 of the value for the division and the gate."""
import numpy as np
import pytest

import _oracle as O
import kvc
import q8_ref as Q
from gpu_util import D, NKV, NQ, say

pytestmark = pytest.mark.gpu
SCALE = 1.0 / 16


def check(got, want, mag, big, rounded_weights, bf16_out, what, dig=0.0):
    tol = mag * (2.0 ** -22 * (big + 2) + (2.0 ** -8 if rounded_weights else 0.0)) + np.abs(want) * 2.0 ** -22
    tol = tol + 2.0 ** -30 * dig
    if bf16_out:
        tol = tol * (1 + 2.0 ** -8) + np.abs(want) * 2.0 ** -8
    off = np.abs(got - want)
    assert np.isfinite(got).all(), what
    worst = float((off / np.maximum(tol, 1e-30)).max())
    assert worst <= 1.0, f"{what}: {worst:.2f} times the tolerance, max|diff| {off.max():.3e}"
    say(f"  {what}: {worst:.3f} of the tolerance")


def load_out(raw, bf16_out):
    return Q.f64(raw) if bf16_out else raw.astype(np.float64)


# ---- quantize and read back ---------------------------------------------------


@pytest.mark.parametrize("lens,keep", [([1, 31, 32, 33], 0), ([64, 95, 96, 257], 0), ([100, 300], 40), ([70], 200)])
def test_quantize_reads_back_the_formula(lens, keep):
    say(f"quantize {lens} keep {keep}")
    with Q.Filled(lens, layers=2, seed=31) as f:
        f.ctx.kv_quantize(f.seqs, keep)
        for n, s in zip(lens, f.seqs):
            n8 = max(0, n - keep) // 32 * 32
            assert f.ctx.seq_info(s).q8_tokens == n8
            for layer in range(2):
                for got, rows in zip(f.gather(layer, s, n), f.rows[layer, s]):
                    Q.same_bits(got, Q.readback(rows, n8))
                lo = min(n - 1, 17)  # a range that starts and ends inside blocks
                for got, rows in zip(f.gather(layer, s, n - lo - n // 5, lo), f.rows[layer, s]):
                    Q.same_bits(got, Q.readback(rows, n8)[lo:n - n // 5])


def test_quantize_of_special_units():
    """zeros, values under the floor, a lone large value, exact ties, infinities
    and NaN; each stays in its own unit"""
    say("quantize special units")
    rows = [np.zeros((224, NKV, D), np.uint16) for _ in range(2)]
    x = Q.f64(O.normal_bf16(224 * NKV * D, 5)).reshape(224, NKV, D)
    x[0:32] = 0.0
    x[32:64] *= 2.0 ** -110  # under 2^-100
    x[64:96] *= 2.0 ** -96
    x[96, 1, 7] = 3.0e38
    x[128:160] = np.round(x[128:160]) + 0.5  # many ties of i
    x[128, :, 0] = 127.0
    for r, bad in zip(rows, (np.inf, np.nan)):
        y = x.copy()
        y[170, 2, 200] = bad
        r[:] = Q.bf16_bits(y)
    with Q.Filled([0], seed=32, extra=224) as f:
        s = f.seqs[0]
        f.add([s], 224, rows=rows)
        f.ctx.kv_quantize([s])
        for got, r in zip(f.gather(0, s, 224), rows):
            want = Q.readback(r, 224)
            assert np.isnan(O.bf16_to_f32(want[160:192, 2])).all() and not np.isnan(O.bf16_to_f32(want[160:192, 1])).any()
            Q.same_bits(got, want)


def test_copy_leaves_its_source():
    say("quantize into a copy")
    with Q.Filled([100, 64, 7], layers=2, seed=33, extra=35) as f:
        dst = [f.ctx.seq_create() for _ in f.seqs]
        f.ctx.kv_quantize(f.seqs, 0, dst=dst)
        f.add(f.seqs, 30)  # into blocks that the copies share
        f.add(dst[:1], 5)
        for s, d, n in zip(f.seqs, dst, (100, 64, 7)):
            for layer in range(2):
                for i in range(2):
                    Q.same_bits(f.gather(layer, s, n + 30)[i], f.rows[layer, s][i])
                    Q.same_bits(f.gather(layer, d, n)[i], Q.readback(f.rows[layer, s][i][:n], n // 32 * 32))
        for i in range(2):
            Q.same_bits(f.gather(1, dst[0], 5, 100)[i], f.rows[1, dst[0]][i])


def test_many_sequences_in_one_call():
    """more than a launch's 64, more table updates than one launch takes"""
    say("quantize 70 sequences")
    lens = [int(x) for x in np.random.default_rng(2).integers(1, 400, 70)]
    with Q.Filled(lens, seed=34) as f:
        f.ctx.kv_quantize(f.seqs, 20)
        for i in (0, 1, 33, 63, 64, 69):
            n8 = max(0, lens[i] - 20) // 32 * 32
            Q.same_bits(f.gather(0, f.seqs[i], lens[i])[0], Q.readback(f.rows[0, f.seqs[i]][0], n8))
        q = O.normal_bf16(70 * NQ * D, 77).reshape(70, NQ, D)
        out = f.run(lambda qb, ob: f.ctx.decode_attn(0, f.seqs, qb, ob), (70, NQ, D), np.float32, q)
        for i in range(0, 70, 9):
            n8 = max(0, lens[i] - 20) // 32 * 32
            k, v = (Q.values(f.rows[0, f.seqs[i]][j], n8) for j in range(2))
            want, mag, big, dig = Q.attend(Q.f64(q[i])[None], k, v, SCALE, digits=True)
            check(out[i].astype(np.float64), want[0], mag[0], big, False, False, f"seq {i} of {lens[i]}", dig[0])


# ---- decode ---------------------------------------------------------------------


def decode_case(lens, keep, fused, gated, bf16_out, scale=SCALE, seed=40, n8s=None, q_scale=1.0, **over):
    with Q.Filled(lens, seed=seed, extra=1, **over) as f:
        f.ctx.kv_quantize(f.seqs, keep)
        n = len(lens)
        q = Q.bf16_bits(Q.f64(O.normal_bf16(n * NQ * D, seed + 1)).reshape(n, NQ, D) * q_scale)
        gate = O.normal_bf16(n * NQ * D, seed + 2).reshape(n, NQ, D) if gated else None
        kn = vn = None
        if fused:
            kn, vn = (O.normal_bf16(n * NKV * D, seed + j).reshape(n, NKV, D) for j in (3, 4))
            f.ctx.reserve(f.seqs, 1)
        args = dict(out_dtype=kvc.DTYPE_BF16 if bf16_out else kvc.DTYPE_F32, scale=scale)
        outs = [f.run(lambda qb, gb, kb, vb, ob: f.ctx.decode_attn(0, f.seqs, qb, ob, k_new=kb, v_new=vb, gate=gb, **args),
                      (n, NQ, D), np.uint16 if bf16_out else np.float32, q, gate, kn, vn) for _ in range(2)]
        assert np.array_equal(outs[0], outs[1], equal_nan=not bf16_out)  # no atomics in the sums
        got = load_out(outs[0], bf16_out)
        if fused:
            f.ctx.commit(f.seqs, 1)
        for i, s in enumerate(f.seqs):
            n8 = max(0, lens[i] - keep) // 32 * 32
            k, v = (Q.values(f.rows[0, s][j], n8) if (0, s) in f.rows else np.zeros((0, NKV, D)) for j in range(2))
            if fused:
                k, v = np.concatenate([k, Q.f64(kn[i])[None]]), np.concatenate([v, Q.f64(vn[i])[None]])
                Q.same_bits(f.gather(0, s, 1, lens[i])[0], kn[i][None])
                Q.same_bits(f.gather(0, s, 1, lens[i])[1], vn[i][None])
            want, mag, big, dig = Q.attend(Q.f64(q[i])[None], k, v, scale, gate=Q.f64(gate[i])[None] if gated else None,
                                           digits=True)
            check(got[i], want[0], mag[0], big, False, bf16_out, f"len {lens[i]} ({n8} in 8 bits)", dig[0])


@pytest.mark.parametrize("n", [32, 33, 63, 64, 65, 96, 127, 160, 255, 300, 1000, 4133])
@pytest.mark.parametrize("fused", [False, True])
def test_decode_one_sequence(n, fused):
    say(f"decode8 {n} fused {fused}")
    decode_case([n], 0, fused, True, n % 2 == 1, seed=41 + n)


@pytest.mark.parametrize("keep", [0, 1, 32, 77, 500])
def test_decode_bf16_tails(keep):
    say(f"decode8 keep {keep}")
    decode_case([700, 129], keep, True, False, False, seed=43)


def test_decode_ragged_batch_with_and_without_8_bit_blocks():
    say("decode8 ragged")
    decode_case([1, 20, 31, 32, 40, 64, 777, 2000, 3001, 5, 96], 30, False, True, False, seed=44)
    decode_case([0, 20, 31, 32, 40, 64, 777, 2000, 3001, 5, 96], 30, True, True, True, seed=45)


@pytest.mark.parametrize("scale", [0.0, -1.0 / 16, 0.5])
def test_decode_scales(scale):
    say(f"decode8 scale {scale}")
    decode_case([500], 40, True, False, False, scale=scale, seed=46)


@pytest.mark.parametrize("q_scale", [0.0, 2.0 ** -60, 2.0 ** 20])
def test_decode_query_magnitudes(q_scale):
    """all-zero, tiny and large queries: digits follow the row's largest value.
    Large ones make one key take all the weight; the tolerance follows B."""
    say(f"decode8 q {q_scale}")
    decode_case([300], 0, False, False, False, scale=2.0 ** -24 if q_scale > 1 else SCALE, q_scale=q_scale, seed=47)


def test_decode_one_heavy_key_among_many_light_ones():
    """A sink that takes about half of the weight, the rest spread over 20000
    keys: light weights must not be lost in the digits of heavy ones."""
    say("decode8 sink")
    n = 20000
    k = np.zeros((n, NKV, D))
    k[:, :, 0] = np.random.default_rng(3).normal(size=(n, NKV)) * 0.1
    k[0, :, 0] = 10.0
    v = np.random.default_rng(4).normal(size=(n, NKV, D)) + 1.0
    with Q.Filled([0], seed=48, extra=n) as f:
        s = f.seqs[0]
        f.add([s], n, rows=[Q.bf16_bits(k), Q.bf16_bits(v)])
        f.ctx.kv_quantize([s])
        q = np.zeros((1, NQ, D))
        q[:, :, 0] = 1.0
        qb = Q.bf16_bits(q)
        got = f.run(lambda a, o: f.ctx.decode_attn(0, [s], a, o, scale=1.0), (1, NQ, D), np.float32, qb)
        want, mag, big, dig = Q.attend(Q.f64(qb), Q.values(Q.bf16_bits(k), n // 32 * 32), Q.values(Q.bf16_bits(v), n // 32 * 32),
                                       1.0, digits=True)
        check(got.astype(np.float64)[0], want[0], mag[0], big, False, False, "sink", dig[0])


def test_decode_non_finite_units_and_queries():
    """A NaN or infinity in a unit, or in q, gives NaN where it takes part and
    nowhere else."""
    say("decode8 NaN")
    with Q.Filled([0, 200], seed=49, extra=200) as f:
        a, b = f.seqs
        k = O.normal_bf16(200 * NKV * D, 7).reshape(200, NKV, D)
        v = O.normal_bf16(200 * NKV * D, 8).reshape(200, NKV, D)
        k[40, 1, 3] = 0x7F80  # infinity
        v[70, 2, 9] = 0x7FC0  # NaN
        f.add([a], 200, rows=[k, v])
        f.ctx.kv_quantize(f.seqs)
        q = O.normal_bf16(2 * NQ * D, 9).reshape(2, NQ, D)
        q[1, 5, 100] = 0xFF80
        got = f.run(lambda x, o: f.ctx.decode_attn(0, f.seqs, x, o), (2, NQ, D), np.float32, q)
        nan = np.isnan(got).all(axis=2)
        assert np.array_equal(np.isnan(got).any(axis=2), nan)
        assert nan[0].tolist() == [h // 4 in (1, 2) for h in range(NQ)]
        assert nan[1].tolist() == [h == 5 for h in range(NQ)]


def test_decode_in_a_graph():
    """captured with its fused append, replayed between eager calls"""
    say("decode8 graph")
    h = kvc.hip()
    with Q.Filled([500, 70, 1201], seed=50, extra=1) as f:
        f.ctx.kv_quantize(f.seqs, 16)
        f.ctx.reserve(f.seqs, 1)
        st = h.stream()
        q, kn, vn = (kvc.to_device(O.normal_bf16(3 * w * D, 60 + w)) for w in (NQ, NKV, NKV))
        o1, o2 = h.malloc(3 * NQ * D * 4), h.malloc(3 * NQ * D * 4)
        call = lambda o, st: f.ctx.decode_attn(0, f.seqs, q, o, k_new=kn, v_new=vn, stream=st)
        call(o1, st)
        h.stream_sync(st)
        want = o1.download(np.uint32, (3, NQ, D))
        g = h.capture(st, lambda: call(o2, st))
        for i in range(4):
            o2.zero()
            h.sync()
            h.graph_launch(g, st)
            h.stream_sync(st)
            assert np.array_equal(o2.download(np.uint32, (3, NQ, D)), want), i
            call(o1, st)
            h.stream_sync(st)
            assert np.array_equal(o1.download(np.uint32, (3, NQ, D)), want), i
        h.graph_destroy(g)


# ---- prefill --------------------------------------------------------------------


def prefill_case(lens, n_q, keep, gated, bf16_out, scale=SCALE, seed=70, check_seqs=None):
    with Q.Filled(lens, seed=seed, extra=n_q) as f:
        f.ctx.kv_quantize(f.seqs, keep)
        f.add(f.seqs, n_q, commit=False)
        n = len(lens)
        q = O.normal_bf16(n * n_q * NQ * D, seed + 1).reshape(n, n_q, NQ, D)
        gate = O.normal_bf16(n * n_q * NQ * D, seed + 2).reshape(n, n_q, NQ, D) if gated else None
        args = dict(out_dtype=kvc.DTYPE_BF16 if bf16_out else kvc.DTYPE_F32, scale=scale)
        raw = f.run(lambda qb, gb, ob: f.ctx.prefill_attn(0, f.seqs, n_q, qb, ob, gate=gb, **args), (n, n_q, NQ, D),
                    np.uint16 if bf16_out else np.float32, q, gate)
        got = load_out(raw, bf16_out)
        for i in (range(n) if check_seqs is None else check_seqs):
            s, n8 = f.seqs[i], max(0, lens[i] - keep) // 32 * 32
            k, v = (Q.values(f.rows[0, s][j], n8) for j in range(2))
            want, mag, big = Q.attend(Q.f64(q[i]), k, v, scale, first=lens[i], gate=Q.f64(gate[i]) if gated else None)
            check(got[i], want, mag, big, bf16_out, bf16_out, f"{n_q} rows over {lens[i]} ({n8} in 8 bits)")


@pytest.mark.parametrize("n,n_q", [(32, 1), (32, 2), (64, 5), (96, 16), (96, 33), (100, 31), (33, 64), (160, 17),
                                   (1000, 40), (300, 130)])
@pytest.mark.parametrize("bf16_out", [False, True])
def test_prefill_one_sequence(n, n_q, bf16_out):
    say(f"prefill8 {n_q} over {n} bf16 {bf16_out}")
    prefill_case([n], n_q, 0, True, bf16_out, seed=71 + n)


@pytest.mark.parametrize("bf16_out", [False, True])
def test_prefill_short_chunk_over_a_long_prefix(bf16_out):
    """split over the keys"""
    say("prefill8 32 over 4001")
    prefill_case([4001], 32, 50, False, bf16_out, seed=72)


@pytest.mark.parametrize("bf16_out", [False, True])
def test_prefill_ragged_batch(bf16_out):
    say("prefill8 ragged")
    prefill_case([0, 5, 32, 64, 95, 200, 1111, 640, 31, 800, 96, 1500], 48, 40, True, bf16_out, seed=73)


def test_prefill_unsplit_large_launch():
    """enough workgroups that no group is split"""
    say("prefill8 24 x 700")
    prefill_case([64 * (i % 5) + 33 * (i % 2) + 32 for i in range(24)], 700, 0, False, True, seed=74, check_seqs=[0, 11, 23])


@pytest.mark.parametrize("gated,bf16_out", [(True, False), (False, False), (True, True), (False, True)])
def test_prefill_ragged_runs(gated, bf16_out):
    """enough rows and keys for prefill_q8_kernel: sequences of no 8-bit block,
    of one, of an odd and an even number; row blocks of 64, 64 and 2 rows"""
    say(f"prefill8 ragged runs gated {gated} bf16 {bf16_out}")
    prefill_case([0, 5, 32, 64, 95, 200, 1111, 640, 31, 800, 96, 2500], 130, 40, gated, bf16_out, seed=76)


@pytest.mark.parametrize("n,keep", [(8100, 0), (8100, 300), (8100, 7000)])
@pytest.mark.parametrize("bf16_out", [False, True])
def test_prefill_items_cut_into_many_runs(n, keep, bf16_out):
    """few items, each over tens of workgroups, with tails of 4, 13 and 222 bf16
    blocks, and a short sequence beside them"""
    say(f"prefill8 cut items {n} keep {keep}")
    prefill_case([n, 64], 100, keep, True, bf16_out, seed=77 + keep % 7, check_seqs=[0, 1])


def test_prefill_70_sequences():
    """two launches, the second one small"""
    say("prefill8 70 sequences")
    lens = [int(x) for x in np.random.default_rng(12).integers(60, 400, 70)]
    prefill_case(lens, 65, 33, False, False, seed=79, check_seqs=[0, 1, 31, 63, 64, 69])


def test_prefill_many_short_sequences_of_few_blocks():
    """the 32-row variant, not split"""
    say("prefill8 64 x 40 rows")
    lens = [int(x) for x in np.random.default_rng(13).integers(20, 130, 64)]
    prefill_case(lens, 40, 0, True, True, seed=80, check_seqs=[0, 7, 40, 63])


@pytest.mark.parametrize("scale", [0.0, -1.0 / 16])
def test_prefill_scales_of_a_large_launch(scale):
    say(f"prefill8 scale {scale}, large")
    prefill_case([4500], 129, 64, False, False, scale=scale, seed=81)


@pytest.mark.parametrize("n_q", [3, 130])
def test_prefill_in_a_graph(n_q):
    """either prefill, weights and decode captured as one run, replayed between
    eager calls of them"""
    say(f"prefill8 graph {n_q}")
    h = kvc.hip()
    lens = [3000, 70, 1201]
    with Q.Filled(lens, seed=82, extra=n_q) as f:
        f.ctx.kv_quantize(f.seqs, 16)
        f.add(f.seqs, n_q, commit=False)
        st = h.stream()
        q = kvc.to_device(O.normal_bf16(3 * n_q * NQ * D, 60))
        shape, ashape = (3, n_q, NQ, D), (3, NKV, 3200)
        bufs = [[h.malloc(int(np.prod(shape)) * 4), h.malloc(int(np.prod(ashape)) * 4), h.malloc(3 * NQ * D * 4)]
                for _ in range(2)]

        def call(b):
            f.ctx.prefill_attn(0, f.seqs, n_q, q, b[0], stream=st)
            f.ctx.attn_weights(0, f.seqs, n_q, q, b[1], 3200, stream=st)
            f.ctx.decode_attn(0, f.seqs, q, b[2], stream=st)

        def read(b):
            return [b[0].download(np.uint32, shape), b[1].download(np.uint32, ashape), b[2].download(np.uint32, (3, NQ, D))]

        for b in bufs:
            for x in b:
                x.zero()
        h.sync()
        call(bufs[0])
        h.stream_sync(st)
        want = read(bufs[0])
        assert all(w.any() for w in want)
        g = h.capture(st, lambda: call(bufs[1]))
        for i in range(4):
            for x in bufs[1]:
                x.zero()
            h.sync()
            h.graph_launch(g, st)
            h.stream_sync(st)
            assert all(np.array_equal(a, b) for a, b in zip(read(bufs[1]), want)), i
            call(bufs[0])
            h.stream_sync(st)
            assert all(np.array_equal(a, b) for a, b in zip(read(bufs[0]), want)), i
        h.graph_destroy(g)


@pytest.mark.parametrize("n_q,lens", [(5, [75, 200, 33]), (130, [2500, 75, 200, 33, 1500, 1000])])
def test_rows_behind_the_last_token_hold_nan(n_q, lens):
    """Blocks that another sequence filled with NaN, taken again: slots past a
    sequence's end take part in nothing, and stay as they are."""
    say(f"stale NaN rows, {n_q} queries over {lens}")
    blocks = sum((x + n_q) // 32 + 1 for x in lens) + len(lens)
    bad = [np.full((blocks * 32, NKV, D), 0x7FC0, np.uint16)] * 2
    with Q.Filled([0], seed=83, extra=blocks * 32, pool_blocks=blocks, q8_blocks=blocks, max_seqs=len(lens) + 1) as f:
        c, p = f.ctx, f.seqs[0]
        f.add([p], blocks * 32, rows=bad)
        c.seq_reset(p)
        del f.rows[0, p]
        seqs = [c.seq_create() for _ in lens]
        for s, x in zip(seqs, lens):
            f.add([s], x)
        c.kv_quantize(seqs, 20)
        f.add(seqs, n_q, commit=False)
        n = len(lens)
        q = O.normal_bf16(n * n_q * NQ * D, 84).reshape(n, n_q, NQ, D)
        stride = max(lens) + n_q
        got = [f.run(lambda qb, ob: c.prefill_attn(0, seqs, n_q, qb, ob, scale=SCALE), q.shape, np.float32, q),
               f.run(lambda qb, ob: c.prefill_attn(0, seqs, n_q, qb, ob, scale=SCALE, out_dtype=kvc.DTYPE_BF16), q.shape,
                     np.uint16, q),
               f.run(lambda qb, ob: c.decode_attn(0, seqs, qb, ob, scale=SCALE), (n, NQ, D), np.float32, q[:, -1].copy()),
               f.run(lambda qb, ob: c.attn_weights(0, seqs, n_q, qb, ob, stride, scale=SCALE), (n, NKV, stride), np.float32,
                     q, fill=0)]
        for i, s in enumerate(seqs):
            n8 = max(0, lens[i] - 20) // 32 * 32
            k, v = (Q.values(f.rows[0, s][j], n8) for j in range(2))
            want, mag, big, dig = Q.attend(Q.f64(q[i]), k, v, SCALE, first=lens[i], digits=True)
            check(got[0][i].astype(np.float64), want, mag, big, False, False, f"fp32, {lens[i]}", dig)
            check(load_out(got[1][i], True), want, mag, big, True, True, f"bf16, {lens[i]}", dig)
            check(got[2][i].astype(np.float64), want[-1], mag[-1], big, False, False, f"decode, {lens[i]}", dig[-1])
            w = Q.weights(Q.f64(q[i]), k, SCALE, lens[i])
            assert np.abs(got[3][i, :, :lens[i] + n_q] - w).max() <= 2.0 ** -16 * max(1.0, w.max())


@pytest.mark.parametrize("scale", [0.0, -1.0 / 16])
def test_prefill_scales(scale):
    say(f"prefill8 scale {scale}")
    prefill_case([200], 20, 0, False, False, scale=scale, seed=75)


# ---- refusals -------------------------------------------------------------------


def test_calls_that_do_not_read_8_bit_blocks_refuse():
    say("8-bit refusals")
    un = kvc.KVC_ERR_UNSUPPORTED
    with Q.Filled([100, 50], seed=80, extra=8, rope_dim=64) as f:
        c, (a, b) = f.ctx, f.seqs
        c.kv_quantize([a])
        c.reserve([a, b], 1)
        buf = kvc.hip().malloc(1 << 20).zero()
        for what, call in [
            ("decode_step", lambda: c.decode_step(0, [b, a], buf, buf, buf, buf)),
            ("prefill_step", lambda: c.prefill_step(0, [b, a], 1, buf, buf, buf, buf)),
            ("static", lambda: c.decode_attn_static(0, [a], buf, buf)),
            ("checksum", lambda: c.kv_checksum(0, [a], buf)),
        ]:
            with pytest.raises(kvc.KvcError) as e:
                call()
            assert e.value.code == un, what
        c.sync()
        assert not buf.download(np.uint8, (1 << 20,)).any()
        c.decode_step(0, [b], buf, buf, buf, buf)  # the other sequence is an ordinary one
        c.sync()
        buf.free()
