"""GPU tests of kvc_beam_select against the same choice in 64 bits.

Tokens are checked exactly within a beam, where their order is that of the logits;
between beams they follow sums whose log sum of exponentials is taken in 32 bits.
Its relative error, in units of 2^-24: 1.5 |x - max| for the argument of the
exponential (a product and a constant, both rounded; |x - max| <= 88, beyond which
terms vanish), which sums to the same through the rescalings; 2 for each of at most
4 exponentials and 1 for each product with one; 52 additions one after another; 2 for
the logarithm of the mantissa.  That is 132 + 12 + 52 + 2 < 200, so log sum is off by at most 200 x 2^-24, and a
score by that and half a step of fp32, |score| 2^-24."""
import numpy as np
import pytest

import _oracle as O
import kvc
from gpu_util import say

pytestmark = pytest.mark.gpu

LOG_SUM = 200 * 2.0**-24
LOWEST_BF16 = 0xFF7F
F32, BF16 = kvc.DTYPE_F32, kvc.DTYPE_BF16


@pytest.fixture(scope="module")
def ctx():
    with kvc.Context(n_attn_layers=1, n_ssm_layers=0, max_seqs=1, max_seq_len=32, pool_blocks=1, snapshot_slots=0) as c:
        yield c


def values(logits, scores):
    """[groups][beams][vocab] in 64 bits; -inf for what can't be chosen."""
    x = logits.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    m = x.max(axis=2, keepdims=True)
    ok = np.isfinite(m[..., 0]) & np.isfinite(scores)
    with np.errstate(all="ignore"):
        v = scores[..., None].astype(np.float64) - np.log(np.exp(x - m).sum(axis=2, keepdims=True)) + (x - m)
    return np.where(ok[..., None], v, -np.inf), x


def check(logits, scores, n_out, got):
    """logits [g][b][v] as fp32, scores [g][b]; got: scores, beams, tokens [g][n_out]."""
    val, x = values(logits, scores)
    for g in range(len(val)):
        v = val[g].reshape(-1)
        n = min(n_out, int((v > -np.inf).sum()))
        gs, gb, gt = (a[g] for a in got)
        assert (gs[n:] == -np.inf).all() and (gb[n:] == -1).all() and (gt[n:] == -1).all(), g
        assert (gb[:n] >= 0).all() and (gt[:n] >= 0).all(), g
        want = -np.sort(-v)[:n]
        tol = LOG_SUM + np.abs(want) * 2.0**-24
        assert (np.abs(gs[:n] - want) <= tol).all(), (g, np.abs(gs[:n] - want).max())
        mine = val[g][gb[:n], gt[:n]]
        assert (np.abs(mine - want) <= 2 * LOG_SUM).all(), g  # between beams: no better one left out
        assert (np.diff(gs[:n]) <= 0).all()
        for b in range(x.shape[1]):  # within a beam: exact
            t = gt[:n][gb[:n] == b]
            assert np.array_equal(t, np.lexsort((np.arange(x.shape[2]), -x[g, b]))[: len(t)]), (g, b)


def as_f32(bits_or_f32, dtype):
    return O.bf16_to_f32(bits_or_f32.reshape(-1)).reshape(bits_or_f32.shape) if dtype == BF16 else bits_or_f32


class Case:
    """Logits of a case on the device, rows `pad` elements longer, the first one `at` elements in."""

    def __init__(self, logits, dtype, scores, n_out, pad=0, at=0):
        self.dtype, self.scores, self.n_out = dtype, scores, n_out
        g, b, v = logits.shape
        bits = O.f32_to_bf16(logits.reshape(-1).astype(np.float32)).reshape(g, b, v) if dtype == BF16 and logits.dtype != np.uint16 else logits
        fill = np.uint16(0x7F80) if dtype == BF16 else np.float32(np.inf)  # +inf between rows: never read
        flat = np.full(at + g * b * (v + pad) + 8, fill, bits.dtype)
        flat[at : at + g * b * (v + pad)].reshape(g, b, v + pad)[..., :v] = bits
        self.logits = as_f32(bits, dtype)
        self.esz = 2 if dtype == BF16 else 4
        self.shape, self.stride, self.at = (g, b, v), v + pad, at
        self.x = kvc.to_device(flat)
        self.s = None if scores is None else kvc.to_device(scores.astype(np.float32))
        self.outs = [kvc.hip().malloc(g * n_out * 4) for _ in range(3)]

    def call(self, ctx, stream=None):
        ctx.beam_select(self.x.ptr + self.at * self.esz, *self.shape, self.n_out, *self.outs, scores=self.s,
                        row_stride=self.stride, dtype=self.dtype, stream=stream)

    def read(self):
        kvc.hip().sync()
        n = (self.shape[0], self.n_out)
        return [b.download(t, n) for b, t in zip(self.outs, (np.float32, np.int32, np.int32))]

    def run(self, ctx):
        for b in self.outs:
            b.upload(np.full(b.nbytes // 4, 0x7FC12345, np.int32))
        self.call(ctx)
        got = self.read()
        g, b, _ = self.shape
        check(self.logits, np.zeros((g, b), np.float32) if self.scores is None else self.scores.astype(np.float32),
              self.n_out, got)
        return got

    def __enter__(self):
        return self

    def __exit__(self, *a):
        for b in (self.x, self.s, *self.outs):
            if b is not None:
                b.free()


def noise(shape, seed, scale=3.0):
    return (np.random.default_rng(seed).standard_normal(shape) * scale).astype(np.float32)


def scores_of(shape, seed):
    return (np.random.default_rng(seed).random(shape) * -20).astype(np.float32)


SHAPES = {  # groups, beams, vocab, n_out, pad, at
    "one": (1, 1, 1, 1, 0, 0),
    "fewer_than_asked": (2, 1, 2, 4, 0, 1),
    "below_a_segment": (3, 4, 255, 8, 1, 1),
    "a_segment": (3, 4, 256, 8, 0, 0),
    "above_a_segment": (3, 4, 257, 8, 0, 3),
    "all_of_a_row": (1, 1, 128, 128, 5, 1),
    "one_of_many": (2, 3, 5000, 1, 7, 0),
    "odd": (2, 5, 1023, 128, 0, 5),
    "a_chunk_and_one": (1, 32, 2049, 100, 0, 0),
    "most_beams": (1, 64, 8192, 128, 0, 0),
    "long_chunks": (8, 8, 70001, 16, 0, 1),
    "vocabulary": (2, 3, 151936, 16, 64, 0),
    "many_segments": (1, 48, 60000, 7, 0, 0),
    "fewer_segments_than_asked": (3, 4, 400, 30, 5, 0),  # values are counted again,
    "more_values_than_held": (2, 17, 2622, 120, 71, 1),  # from the logits
    "some_values": (2, 10, 66, 13, 0, 0),
    "many_groups": (70000, 1, 2, 1, 0, 0),
}


@pytest.mark.parametrize("name", list(SHAPES))
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_against_64_bits(ctx, name, dtype):
    say(f"beam select {name} {dtype}")
    g, b, v, n_out, pad, at = SHAPES[name]
    with Case(noise((g, b, v), 1), dtype, scores_of((g, b), 2), n_out, pad, at) as c:
        c.run(ctx)
    with Case(noise((g, b, v), 3), dtype, None, n_out, pad, at) as c:
        c.run(ctx)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("levels", [1, 2, 7])
def test_equal_logits(ctx, dtype, levels):
    """Lower tokens first within a beam; beams of equal rows and scores in turn."""
    say(f"beam select of {levels} levels")
    x = (np.random.default_rng(5).integers(0, levels, (2, 4, 5003)) * 0.5).astype(np.float32)
    with Case(x, dtype, scores_of((2, 4), 6), 128, 0, 1) as c:
        c.run(ctx)
    x[:, :] = x[:1, :1]
    with Case(x, dtype, np.full((2, 4), -1.5, np.float32), 100, 0, 1) as c:  # rows at every alignment
        s, b, t = c.run(ctx)
        order = np.lexsort((np.arange(5003), -x[0, 0].astype(np.float64)))
        flat = [(bb, tt) for lv in np.unique(x)[::-1] for bb in range(4) for tt in order[x[0, 0][order] == lv]][:100]
        for g in range(2):
            assert [(int(i), int(j)) for i, j in zip(b[g], t[g])] == flat


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("levels", [1, 3])
def test_more_equal_segments_than_are_listed(ctx, dtype, levels):
    say(f"beam select of {levels} levels in thousands of segments")
    x = (np.random.default_rng(21).integers(0, levels, (1, 48, 60000)) * 0.5).astype(np.float32)
    with Case(x, dtype, np.zeros((1, 48), np.float32), 128) as c:
        _, b, t = c.run(ctx)
        if levels == 1:  # equal sums everywhere
            assert (b == 0).all() and t[0].tolist() == list(range(128))


def test_more_close_values_than_are_sorted(ctx):
    """Above the least chosen maximum stand more values than the last step sorts."""
    say("beam select of a crowded top")
    x = noise((1, 3, 60000), 7, 0.01)
    for b in range(3):
        for j in range(40):  # whole segments of high values, their maxima all but equal
            x[0, b, 1024 * j : 1024 * j + 256] = 5 + 1e-4 * np.random.default_rng(j).random(256)
    with Case(x, F32, np.zeros((1, 3), np.float32), 128) as c:
        c.run(ctx)
    with Case(x, BF16, np.zeros((1, 3), np.float32), 128) as c:
        c.run(ctx)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masks_and_special_values(ctx, dtype):
    say("beam select of masked rows")
    rng = np.random.default_rng(8)
    lowest = float(O.bf16_to_f32(np.array([LOWEST_BF16], np.uint16))[0])
    x = noise((6, 5, 1700), 9)
    s = scores_of((6, 5), 10)
    x[0][rng.random((5, 1700)) < 0.9] = -np.inf
    x[0, 3] = -np.inf  # a row without tokens
    x[1][rng.random((5, 1700)) < 0.99] = lowest  # masked by the lowest value: still tokens
    x[1, 2] = lowest
    x[2][rng.random((5, 1700)) < 0.3] = np.nan
    x[2, 0] = np.nan
    x[2, 1, 77] = np.inf  # no finite maximum
    s[3] = [-np.inf, np.nan, np.inf, -1.0, -3.0]
    x[3, 4, 5:] = -np.inf
    s[4] = -np.inf  # nothing at all
    x[5] = -np.inf
    x[5, 1, 3] = -0.0
    x[5, 1, 2] = 0.0
    x[5, 1, 1] = -0.0
    s[5] = 0.0
    with Case(x, dtype, s, 24, 3, 1) as c:
        _, b, t = c.run(ctx)
        assert (b[4] == -1).all()
        assert t[5, :4].tolist() == [1, 2, 3, -1] and b[5, :4].tolist() == [1, 1, 1, -1]
        assert set(b[3].tolist()) <= {3, 4}


def test_large_magnitudes(ctx):
    say("beam select of large logits and scores")
    x = noise((2, 3, 999), 11, 1e4)
    x[1] *= 1e30
    with Case(x, F32, np.array([[-1e6, 0, 5], [3, 3, 1e6]], np.float32), 9) as c:
        c.run(ctx)


def test_scores_in_place(ctx):
    say("beam select with its scores replaced")
    x = noise((3, 6, 901), 12)
    s = scores_of((3, 6), 13)
    with Case(x, BF16, s, 6) as c:
        want = c.run(ctx)
        c.outs[0].free()
        c.outs[0] = c.s
        c.call(ctx)
        got = c.read()
        c.s = None
        for a, b in zip(got, want):
            assert np.array_equal(a, b)


def test_same_bits_again_on_a_stream_and_in_a_graph(ctx):
    say("beam select: repeated, on its own stream, captured and replayed")
    h = kvc.hip()
    st = h.stream()
    with Case(noise((3, 4, 20001), 14), BF16, scores_of((3, 4), 15), 12, 0, 1) as c:
        want = c.run(ctx)
        c.call(ctx, st)
        h.stream_sync(st)
        assert all(np.array_equal(a, b) for a, b in zip(c.read(), want))
        ex = h.capture(st, lambda: c.call(ctx, st))
        for i in range(4):
            for b in c.outs:
                b.zero()
            h.sync()
            h.graph_launch(ex, st)
            h.stream_sync(st)
            assert all(np.array_equal(a, b) for a, b in zip(c.read(), want)), i
            if i == 1:  # other scores in the same array, and eager work in between
                c.scores = scores_of((3, 4), 16)
                c.s.upload(c.scores)
            want = c.run(ctx)
        h.graph_destroy(ex)
    h.ok(h.L.hipStreamDestroy(st), "hipStreamDestroy")
