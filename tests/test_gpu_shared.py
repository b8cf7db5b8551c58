"""GPU tests of kvc_decode_attn_shared: decode over sequences that share blocks,
against 64-bit results.

Tolerances (derived, per element; W = sum w |v| of the element, B = the largest
sum |q k| scale log2(e) over a key):
  scores   fp32 sums of exact products: within 2^-22 B in the log2 domain (16
           partial sums of 2^-24 each), times ln 2 on a weight, plus 2^-22 for
           the exponential, the sums of weights and the fold: 2^-22 (B + 2)
  weights  bf16 output: rounded to bf16, 2^-8 each; fp32 output: three bf16
           parts, 24 bits, within the 2^-22 above
  output   2^-22 of the value for the division and the gate; bf16: half a step
           more, 2^-8 of the value"""
import ctypes

import numpy as np
import pytest

import _oracle as O
import kvc
import q8_ref as Q
from gpu_util import D, NKV, NQ, say

pytestmark = pytest.mark.gpu
SCALE = 1.0 / 16


def tolerance(want, mag, big, bf16_out):
    tol = mag * (2.0 ** -22 * (big + 2) + (2.0 ** -8 if bf16_out else 0.0)) + np.abs(want) * 2.0 ** -22
    return tol * (1 + 2.0 ** -8) + np.abs(want) * 2.0 ** -8 if bf16_out else tol


class Forest(Q.Filled):
    """Sequences that share prefixes: spec is a tree [(tokens, children), ...],
    a leaf's children the number of sequences that end there."""

    def __init__(self, spec, layers=1, seed=1, extra=1, **over):
        def count(nodes):
            return sum(n if isinstance(n, int) else count(n) for _, n in nodes)

        def deepest(nodes):
            return max(t + (0 if isinstance(n, int) else deepest(n)) for t, n in nodes)

        def tokens(nodes):
            return sum(t + 64 + (0 if isinstance(n, int) else tokens(n)) for t, n in nodes)

        n = count(spec)
        cfg = dict(max_seqs=2 * n + 4, max_seq_len=deepest(spec) + extra + 32,
                   pool_blocks=tokens(spec) // 32 + n * (extra // 32 + 3) + 8, q8_blocks=0,
                   flags=kvc.FLAG_EXACT_MATH | kvc.FLAG_DECODE_SHARE)  # however little is shared
        super().__init__([0], layers=layers, seed=seed, **{**cfg, **over})
        self.ctx.seq_release(self.seqs.pop())

        def grow(nodes, parent):
            for t, rest in nodes:
                s = self.fork(parent) if parent is not None else self.ctx.seq_create()
                if t:
                    self.add([s], t)
                if isinstance(rest, int):
                    self.seqs += [s] + [self.fork(s) for _ in range(rest - 1)]
                else:
                    grow(rest, s)
                    self.ctx.seq_release(s)

        grow(spec, None)

    def fork(self, s):
        d = self.ctx.seq_create()
        self.ctx.fork([s], [d])
        for layer in range(self.layers):
            self.rows.pop((layer, d), None)
            if (layer, s) in self.rows:
                self.rows[layer, d] = list(self.rows[layer, s])
        return d

    def decode(self, seqs, fused=True, gated=True, bf16_out=True, scale=SCALE, seed=7, layer=0, stream=None, q_scale=1.0,
               spread=None):
        """One token of every sequence; returns (outputs float64, what they should be, their tolerance)"""
        n = len(seqs)
        q = Q.bf16_bits(Q.f64(O.normal_bf16(n * NQ * D, seed + 1)).reshape(n, NQ, D) * q_scale)
        gate = O.normal_bf16(n * NQ * D, seed + 2).reshape(n, NQ, D) if gated else None
        kn = vn = None
        if fused:
            kn, vn = (O.normal_bf16(n * NKV * D, seed + j).reshape(n, NKV, D) for j in (3, 4))
            self.ctx.reserve(seqs, 1)
            for i, s in enumerate(seqs):
                for la in range(self.layers):
                    old = self.rows.get((la, s), [np.zeros((0, NKV, D), np.uint16)] * 2)
                    self.rows[la, s] = [np.concatenate([old[j], (kn, vn)[j][i:i + 1]]) for j in range(2)]
        got = self.run(lambda qb, kb, vb, gb, ob: self.ctx.decode_attn_shared(
            layer, seqs, qb, ob, k_new=kb, v_new=vb, gate=gb, scale=scale, stream=stream,
            out_dtype=kvc.DTYPE_BF16 if bf16_out else kvc.DTYPE_F32),
            (n, NQ, D), np.uint16 if bf16_out else np.float32, q, kn, vn, gate, fill=0x7FC1 if bf16_out else np.nan)
        if fused:
            self.ctx.commit(seqs, 1)
        got = Q.f64(got) if bf16_out else got.astype(np.float64)
        want, tol = np.empty(got.shape), np.empty(got.shape)
        for i, s in enumerate(seqs):
            k, v = (Q.f64(x) for x in self.rows[layer, s])
            w, mag, big = Q.attend(Q.f64(q[i])[None], k, v, scale, gate=None if gate is None else Q.f64(gate[i])[None])
            want[i], tol[i] = w[0], tolerance(w[0], mag[0], big, bf16_out)
        return got, want, tol

    def check(self, seqs, what, **k):
        got, want, tol = self.decode(seqs, **k)
        assert np.isfinite(got).all(), what
        worst = (np.abs(got - want) / np.maximum(tol, 1e-30)).reshape(len(seqs), -1).max(1)
        assert worst.max() <= 1.0, f"{what}: {worst.max():.2f} times the tolerance at sequence {int(worst.argmax())}"
        say(f"  {what}: {worst.max():.3f} of the tolerance")


# every kind of node: few blocks, split keys, tiles for all waves, several groups
SPECS = {
    "pair": [(520, [(0, 1), (0, 1)])],
    "two_ends": [(513, [(1, 1), (40, 1)])],
    "four": [(1100, [(3, 1), (64, 1), (31, 1), (0, 1)])],
    "five": [(700, [(3, 1), (64, 1), (31, 1), (0, 1), (300, 1)])],
    "sixteen": [(260, 16)],
    "seventeen": [(333, 17)],
    "forty": [(97, [(200, 20), (1, 20)])],
    "sixty_four": [(160, [(5, 33), (500, 31)])],
    "tree": [(100, [(300, [(20, 3), (0, 2), (333, 2)]), (64, [(64, 6), (1, 1)])])],
    "apart": [(400, 6), (300, 2), (33, 1), (1, 1)],
    "wide": [(6600, [(5, 9), (40, 9)])],  # work for groups of two tiles
    "long": [(5000, [(1, 2), (700, 1)])],
}


@pytest.mark.parametrize("name", list(SPECS))
@pytest.mark.parametrize("bf16_out", [True, False])
def test_against_64_bits(name, bf16_out):
    say(f"shared decode {name} bf16_out={bf16_out}")
    with Forest(SPECS[name], seed=11) as f:
        order = [f.seqs[i] for i in np.random.default_rng(3).permutation(len(f.seqs))]
        f.check(order, "fused, gated", bf16_out=bf16_out)
        f.check(order, "again, ends moved on", bf16_out=bf16_out, seed=20)
        f.check(order[::-1], "plain", bf16_out=bf16_out, fused=False, gated=False, seed=30)


@pytest.mark.parametrize("chunk", [1, 2, 3, 5, 64, 1000])
def test_chunk_lengths(chunk):
    say(f"shared decode, chunks of {chunk} blocks")
    with Forest([(1000, [(40, 5), (300, [(1, 18)])])], seed=12, decode_chunk_blocks=chunk) as f:
        f.check(f.seqs, "bf16")
        f.check(f.seqs, "fp32", bf16_out=False, seed=9)


@pytest.mark.parametrize("chunk", [20, 128])
@pytest.mark.parametrize("bf16_out", [True, False])
def test_two_tiles(chunk, bf16_out):
    say(f"shared decode of two tiles, chunks of {chunk}")
    with Forest(SPECS["wide"], seed=33, decode_chunk_blocks=chunk) as f:
        f.check(f.seqs, f"chunk {chunk}", bf16_out=bf16_out)


def test_more_than_one_launch_and_layers():
    say("shared decode of 70 sequences, second layer")
    with Forest([(300, [(7, 30), (90, 40)])], seed=13, layers=2) as f:
        f.check(f.seqs, "layer 1", layer=1)


@pytest.mark.parametrize("scale", [-1.0 / 16, 0.0, 1.0])
def test_scales(scale):
    say(f"shared decode, scale {scale}")
    with Forest([(600, 6)], seed=14) as f:
        f.check(f.seqs, "bf16", scale=scale)
        f.check(f.seqs, "fp32", scale=scale, bf16_out=False, seed=9)


@pytest.mark.parametrize("name", ["pair", "sixty_four"])
@pytest.mark.parametrize("bf16_out", [True, False])
def test_where_the_rule_decides(name, bf16_out):
    """without the flag: too little in common for one, enough for the other"""
    say(f"shared decode {name} by the rule")
    with Forest(SPECS[name], seed=26, flags=kvc.FLAG_EXACT_MATH) as f:
        f.check(f.seqs, "fused, gated", bf16_out=bf16_out)


def test_reference_gate():
    """the default gate: the reference's sigmoid, within its own error of the exact one"""
    say("shared decode with the reference's gate")
    with Forest([(600, 6)], seed=27, flags=kvc.FLAG_DECODE_SHARE) as f:
        gate = O.normal_bf16(6 * NQ * D, 5).reshape(6, NQ, D)
        q = O.normal_bf16(6 * NQ * D, 6).reshape(6, NQ, D)
        outs = [f.run(lambda qb, gb, ob: f.ctx.decode_attn_shared(0, f.seqs, qb, ob, gate=gb), (6, NQ, D), np.float32, q, g)
                for g in (gate, None)]
        # out = plain * sigma(gate), sigma bit for bit the reference's (the model tests/_oracle.py holds)
        sig = np.array([O.sigmoid_ref_model(float(x)) for x in Q.f64(gate).reshape(-1)], np.float32).reshape(gate.shape)
        want = outs[1].astype(np.float64) * sig
        assert (np.abs(outs[0] - want) <= np.abs(want) * 2.0 ** -23).all()


def test_large_scores():
    """weights that span many powers of two, and running maxima that rise"""
    say("shared decode, queries of 30 times the size")
    with Forest([(900, [(3, 5), (200, 3)])], seed=15) as f:
        f.check(f.seqs, "bf16", q_scale=30.0)
        f.check(f.seqs, "fp32", q_scale=30.0, bf16_out=False, seed=9)


def test_the_new_rows_are_in_the_cache():
    say("shared decode appends")
    with Forest([(129, [(30, 3), (95, 4)])], seed=16, layers=2) as f:
        f.ctx.reserve(f.seqs, 1)
        n = len(f.seqs)
        kn, vn = (O.normal_bf16(n * NKV * D, 60 + j).reshape(n, NKV, D) for j in range(2))
        q = O.normal_bf16(n * NQ * D, 70).reshape(n, NQ, D)
        f.run(lambda qb, kb, vb, ob: f.ctx.decode_attn_shared(1, f.seqs, qb, ob, k_new=kb, v_new=vb), (n, NQ, D), np.float32, q, kn, vn)
        f.ctx.commit(f.seqs, 1)
        for i, s in enumerate(f.seqs):
            m = f.ctx.seq_len(s)
            for got, new, old in zip(f.gather(1, s, m), (kn, vn), f.rows[1, s]):
                assert np.array_equal(got[:m - 1], old) and np.array_equal(got[m - 1], new[i])


def test_rows_behind_the_last_key_may_hold_anything():
    """NaN and infinities in the slots of a partial block that hold no token, and
    in rows of other sequences' tokens"""
    say("shared decode beside NaN rows")
    with Forest([(200, [(10, 2), (50, 5)])], seed=17, extra=64) as f:
        bad = np.full((40, NKV, D), 0x7FC0, np.uint16)
        bad[::2] = 0xFF80
        for s in f.seqs:  # written behind the sequence, then dropped
            n = f.ctx.seq_len(s)
            kept = {la: list(f.rows[la, s]) for la in range(f.layers)}
            f.add([s], 40, rows=(bad, bad))
            f.ctx.seq_truncate(s, n)
            for la in kept:
                f.rows[la, s] = kept[la]
        f.check(f.seqs, "bf16")
        f.check(f.seqs, "plain", fused=False, seed=9)
        f.check(f.seqs, "fp32", bf16_out=False, seed=19)


def test_infinite_values_stay_with_their_sequences():
    """An infinite value reaches the elements that it enters and no others.  With
    bf16 output those are infinite.  With fp32 output they are NaN: a weight is
    the sum of three bf16 parts, of which the later ones are negative or, as for
    a weight of 1, zero, and infinity times zero, or minus infinity, is NaN."""
    say("shared decode, one sequence with an infinite value")
    for bf16_out in (True, False):
        with Forest([(300, 5)], seed=18, extra=8) as f:
            rows = [O.normal_bf16(NKV * D, 5 + j).reshape(1, NKV, D) for j in range(2)]
            rows[1][0, 2, 17] = 0x7F80
            f.add(f.seqs[:1], 1, rows=rows)
            f.add(f.seqs[1:], 2)
            got, want, tol = f.decode(f.seqs, fused=False, gated=False, bf16_out=bf16_out)
            fine = np.isfinite(want)
            assert (~fine).sum() == 4 and (want[0, 8:12, 17] == np.inf).all()
            assert (np.abs(got - want)[fine] <= tol[fine]).all()
            assert (got[~fine] == np.inf).all() if bf16_out else not np.isfinite(got[~fine]).any()


def test_a_truncated_fork_sees_only_its_own_keys():
    say("shared decode of rolled-back forks")
    with Forest([(500, 7)], seed=19) as f:
        for i, s in enumerate(f.seqs[1:]):
            n = (499, 480, 479, 257, 32, 1)[i]
            f.ctx.seq_truncate(s, n)
            f.rows[0, s] = [x[:n] for x in f.rows[0, s]]
        f.check(f.seqs, "plain", fused=False)
        f.check(f.seqs, "fused", seed=9)


def test_a_first_token():
    """sequences whose only key is the new one, alone and beside others"""
    say("shared decode of first tokens")
    with Forest([(700, 6), (0, 1), (0, 1)], seed=20) as f:
        f.check(f.seqs, "bf16")
        f.check(f.seqs[-2:], "alone", seed=9)
    with Forest([(0, 1), (0, 1)], seed=21) as f:
        f.check(f.seqs, "bf16")


def test_prefixes_from_the_index():
    """sequences that share blocks through kvc_prefix_match"""
    say("shared decode over matched prefixes")
    tok = np.arange(400, dtype=np.int32)
    with Forest([(0, 1)], seed=22, max_seqs=8, max_seq_len=600, pool_blocks=64) as f:
        s = f.seqs[0]
        f.add([s], 320, commit=False)
        f.ctx.commit([s], 320, tok[:320])
        seqs = [s]
        for i in range(5):
            d = f.ctx.seq_create()
            assert f.ctx.prefix_match(d, np.concatenate([tok[:320], tok[:5 + i]])) == 320
            f.rows[0, d] = [x[:320] for x in f.rows[0, s]]
            f.add([d], 3 * i + 1)
            seqs.append(d)
        f.check(seqs, "bf16")


def test_8_bit_blocks_run_the_unshared_kernels():
    say("shared decode over 8-bit blocks")
    with Forest([(300, 3)], seed=23, q8_blocks=32) as f:
        f.ctx.kv_quantize(f.seqs[:1])
        want = {s: Q.values(f.rows[0, s][0], 288 if s == f.seqs[0] else 0) for s in f.seqs}
        v = {s: Q.values(f.rows[0, s][1], 288 if s == f.seqs[0] else 0) for s in f.seqs}
        q = O.normal_bf16(3 * NQ * D, 3).reshape(3, NQ, D)
        got = f.run(lambda qb, ob: f.ctx.decode_attn_shared(0, f.seqs, qb, ob), (3, NQ, D), np.float32, q)
        for i, s in enumerate(f.seqs):
            w, mag, big, dig = Q.attend(Q.f64(q[i])[None], want[s], v[s], SCALE, digits=True)
            assert (np.abs(got[i] - w[0]) <= tolerance(w[0], mag[0], big, False) + 2.0 ** -30 * dig[0]).all()


def test_same_bits_again_on_a_stream_and_in_a_graph():
    say("shared decode: repeated, on its own stream, captured and replayed")
    h = kvc.hip()
    st = h.stream()
    with Forest([(1000, [(10, 9), (200, 3)])], seed=24) as f:
        n = len(f.seqs)
        f.ctx.reserve(f.seqs, 1)
        q = kvc.to_device(O.normal_bf16(n * NQ * D, 3))
        kn, vn = (kvc.to_device(O.normal_bf16(n * NKV * D, 4 + j)) for j in range(2))
        outs = [h.malloc(n * NQ * D * 2) for _ in range(3)]
        call = lambda o, stream: f.ctx.decode_attn_shared(0, f.seqs, q, o, k_new=kn, v_new=vn, out_dtype=kvc.DTYPE_BF16, stream=stream)  # noqa: E731
        call(outs[0], None)
        h.sync()
        want = outs[0].download(np.uint16, n * NQ * D)
        call(outs[1], st)
        h.stream_sync(st)
        assert np.array_equal(outs[1].download(np.uint16, n * NQ * D), want)
        ex = h.capture(st, lambda: call(outs[2], st))
        for i in range(4):
            outs[2].zero()
            h.sync()
            call(outs[1], st)  # eager work between the replays
            h.graph_launch(ex, st)
            h.stream_sync(st)
            assert np.array_equal(outs[2].download(np.uint16, n * NQ * D), want), i
            if i == 1:  # other queries in the same arrays
                q.upload(O.normal_bf16(n * NQ * D, 99))
                call(outs[0], None)
                h.sync()
                want = outs[0].download(np.uint16, n * NQ * D)
        h.graph_destroy(ex)
        for b in (q, kn, vn, *outs):
            b.free()
    h.ok(h.L.hipStreamDestroy(st), "hipStreamDestroy")


def test_refusals():
    say("shared decode refusals")
    h = kvc.hip()
    with Forest([(100, 3)], seed=25) as f:
        c, s = f.ctx, f.seqs
        buf = h.malloc(1 << 20)
        p, o = buf.ptr, buf.ptr + (1 << 19)

        def code(*a, **k):
            with pytest.raises(kvc.KvcError) as e:
                c.decode_attn_shared(*a, **k)
            return e.value.code

        assert code(1, s, p, o) == kvc.KVC_ERR_RANGE
        assert code(0, s + s[:1], p, o) == kvc.KVC_ERR_INVALID
        assert code(0, [], p, o) == kvc.KVC_ERR_INVALID
        assert code(0, s, None, o) == kvc.KVC_ERR_INVALID
        assert code(0, s, p, None) == kvc.KVC_ERR_INVALID
        assert code(0, s, p, o, k_new=p) == kvc.KVC_ERR_INVALID
        assert code(0, s, p, o, k_new=p, v_new=p) == kvc.KVC_ERR_STATE  # nothing reserved
        assert code(0, s, p, o, out_dtype=2) == kvc.KVC_ERR_INVALID
        assert code(0, s, p, o, scale=float("nan")) == kvc.KVC_ERR_INVALID
        assert code(0, s, p + 2, o) == kvc.KVC_ERR_INVALID
        assert code(0, s, p, o + 8) == kvc.KVC_ERR_INVALID
        assert code(0, s, p, p) == kvc.KVC_ERR_INVALID
        assert code(0, s, p, o, gate=o + 32) == kvc.KVC_ERR_INVALID
        d = c.seq_create()
        assert code(0, [d], p, o) == kvc.KVC_ERR_STATE  # no keys
        buf.free()
    with kvc.Context(device=-1, pool_blocks=8, n_ssm_layers=0, max_seqs=2, snapshot_slots=0) as c:
        s = c.seq_create()
        c.reserve([s], 1)
        with pytest.raises(kvc.KvcError) as e:
            c.decode_attn_shared(0, [s], 16, 32)
        assert e.value.code == kvc.KVC_ERR_NO_DEVICE
    assert kvc.lib().kvc_decode_attn_shared(None, 0, (ctypes.c_int32 * 1)(0), 1, None, None, None, None, None, 0, 1.0, None) == kvc.KVC_ERR_INVALID
