"""Plain 64-bit forms of the 8-bit blocks, of attention over them, of attention
weights and of eviction (numpy, no library code), and a helper that fills a
context and keeps what it put in.

Layouts follow the library's: rows are [token][kv head][256], q heads 4 h ..
4 h + 3 belong to kv head h."""
import numpy as np

import _oracle as O
import kvc
from gpu_util import D, NKV, NQ, ROW

BT = 32
GROUP = NQ // NKV
LOG2E = 1.4426950408889634


def f64(bits):
    """bf16 bits -> float64"""
    return O.bf16_to_f32(np.asarray(bits, np.uint16)).astype(np.float64)


def bf16_bits(x):
    """float -> bf16 bits (RNE), through the fp32 value"""
    x = np.ascontiguousarray(x, np.float32)
    return O.f32_to_bf16(x).reshape(x.shape)


def quantize(rows):
    """[32 b tokens][4][256] bf16 bits -> (int8 integers as float32 [same shape],
    scales fp32 [b][4]).  One fp32 rounding per operation of the formula."""
    x = O.bf16_to_f32(rows).reshape(-1, BT, NKV, D)
    bad = ~np.isfinite(x).all(axis=(1, 3))
    with np.errstate(all="ignore"):
        a = np.maximum(np.abs(x).max(axis=(1, 3)), np.float32(2.0 ** -100))
        a = np.where(bad, np.float32(1), a).astype(np.float32)
        s = (a / np.float32(127)).astype(np.float32)
        inv = (np.float32(127) / a).astype(np.float32)
        i = np.clip(np.rint((x * inv[:, None, :, None]).astype(np.float32)), -127, 127).astype(np.float32)
    s = np.where(bad, np.float32(np.nan), s).astype(np.float32)
    i = np.where(bad[:, None, :, None], np.float32(0), i)
    return i.reshape(rows.shape[0], NKV, D) + np.float32(0), s  # an integer has no -0


def values(rows, n8):
    """float64 values of [tokens][4][256] bf16 bits, the first n8 tokens in 8 bits"""
    y = f64(rows)
    if n8:
        i, s = quantize(rows[:n8])
        y[:n8] = (i.astype(np.float64).reshape(-1, BT, NKV, D) * s.astype(np.float64)[:, None, :, None]).reshape(n8, NKV, D)
    return y


def readback(rows, n8):
    """What kvc_gather returns for them: bf16 bits (NaN as a quiet NaN)."""
    out = np.array(rows, np.uint16)
    if n8:
        i, s = quantize(rows[:n8])
        with np.errstate(all="ignore"):
            y = (i.reshape(-1, BT, NKV, D) * s[:, None, :, None]).astype(np.float32).reshape(n8, NKV, D)
        out[:n8] = bf16_bits(y)
    return out


def same_bits(got, want):
    """Equal bf16 bits, any NaN for a NaN."""
    got, want = np.asarray(got, np.uint16), np.asarray(want, np.uint16)
    nan = np.isnan(O.bf16_to_f32(want))
    assert np.array_equal(np.isnan(O.bf16_to_f32(got)), nan)
    assert np.array_equal(got[~nan], want[~nan])


def attend(q, k, v, scale, first=None, gate=None, digits=False):
    """q [rows][16][256], k / v [keys][4][256] (float64); row i sees keys up to
    first + i (all, if None).  Returns the output, sum w |v| per element and the
    largest sum |q k| scale log2(e) of a seen key (the bounds of rounding
    errors are built from these), and with `digits` the sum over keys of |v|
    times the largest weight of the key's 32-token block."""
    n = q.shape[0]
    out, mag, dig = np.empty(q.shape), np.empty(q.shape), np.zeros(q.shape)
    begin = np.arange(0, len(k), BT)
    big = 0.0
    for h in range(NQ):
        kh, vh = k[:, h // GROUP], v[:, h // GROUP]
        s = q[:, h] @ kh.T * scale
        t = np.abs(q[:, h]) @ np.abs(kh).T * abs(scale) * LOG2E
        if first is not None:
            hide = np.arange(len(k))[None, :] > first + np.arange(n)[:, None]
            s[hide] = -np.inf
            t[hide] = 0.0
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        out[:, h], mag[:, h] = w @ vh, w @ np.abs(vh)
        if digits:
            top = np.maximum.reduceat(w, begin, axis=1)
            dig[:, h] = top @ np.add.reduceat(np.abs(vh), begin, axis=0)
        big = max(big, float(t.max()))
    if gate is not None:
        sg = 1.0 / (1.0 + np.exp(-gate))
        out, mag, dig = out * sg, mag * sg, dig * sg
    return (out, mag, big, dig) if digits else (out, mag, big)


def weights(q, k, scale, first):
    """[4][keys]: the weights of q's rows [rows][16][256], summed per kv head."""
    out = np.zeros((NKV, len(k)))
    for h in range(NQ):
        s = q[:, h] @ k[:, h // GROUP].T * scale
        s[np.arange(len(k))[None, :] > first + np.arange(len(q))[:, None]] = -np.inf
        w = np.exp(s - s.max(1, keepdims=True))
        out[h // GROUP] += (w / w.sum(1, keepdims=True)).sum(0)
    return out


def keep(acc, budget, sink, recent):
    """Indices that stay of one row of accumulated weights."""
    n = len(acc)
    if n <= budget:
        return np.arange(n)
    mid = np.arange(sink, n - recent)
    a = np.where(np.isnan(acc[mid]), -np.inf, acc[mid].astype(np.float64))
    nan = np.isnan(acc[mid])
    order = np.lexsort((mid, nan, -a))  # greatest first; NaN behind -infinity; then the position
    return np.sort(np.concatenate([np.arange(sink), mid[order[:budget - sink - recent]], np.arange(n - recent, n)]))


class Filled:
    """A context whose sequences were filled with known rows (all layers alike
    in shape, different in content)."""

    def __init__(self, lens, layers=1, seed=1, extra=0, gain=True, **over):
        self.h = kvc.hip()
        self.layers = layers
        most = max(lens) + extra + BT
        cfg = dict(n_attn_layers=layers, n_ssm_layers=0, max_seqs=3 * len(lens) + 1, max_seq_len=most,
                   pool_blocks=3 * sum((n + extra) // BT + 2 for n in lens), q8_blocks=2 * sum((n + extra) // BT + 1 for n in lens),
                   snapshot_slots=0, alloc_seed=seed + 11, rope_dim=0, flags=kvc.FLAG_EXACT_MATH)
        cfg.update(over)
        self.ctx = kvc.Context(**cfg)
        self.rows = {}  # (layer, seq) -> [k, v] bits [tokens][4][256]
        self.seqs = []
        self.seed = seed
        # a few large channels, as trained keys have, so that scales differ
        rng = np.random.default_rng(seed)
        self.gain = np.where(rng.random((NKV, D)) < 0.02, 3.0, 1.0) if gain else np.ones((NKV, D))
        for n in lens:
            s = self.ctx.seq_create()
            self.seqs.append(s)
            if n:
                self.add([s], n)

    def draw(self, n):
        self.seed += 1
        return O.normal_bf16(n * ROW, self.seed).reshape(n, NKV, D)

    def add(self, seqs, n, commit=True, rows=None):
        """n new tokens for every sequence, on every layer"""
        self.ctx.reserve(seqs, n)
        for layer in range(self.layers):
            k = np.stack([bf16_bits(f64(self.draw(n)) * self.gain) for _ in seqs])
            v = np.stack([self.draw(n) for _ in seqs])
            if rows is not None:
                k, v = np.stack([rows[0]] * len(seqs)), np.stack([rows[1]] * len(seqs))
            kb, vb = kvc.to_device(k), kvc.to_device(v)
            self.ctx.append(layer, seqs, n, kb, vb)
            self.ctx.sync()
            kb.free()
            vb.free()
            for i, s in enumerate(seqs):
                old = self.rows.get((layer, s))
                self.rows[layer, s] = [k[i], v[i]] if old is None else [np.concatenate([old[0], k[i]]),
                                                                       np.concatenate([old[1], v[i]])]
        if commit:
            self.ctx.commit(seqs, n)

    def gather(self, layer, s, n, tok0=0):
        kb, vb = (self.h.malloc(max(n, 1) * ROW * 2) for _ in range(2))
        self.ctx.gather(layer, [s], tok0, [n], kb, vb)
        self.ctx.sync()
        out = [b.download(np.uint16, (n, NKV, D)) for b in (kb, vb)]
        kb.free()
        vb.free()
        return out

    def run(self, fn, shape, dtype, *arrays, fill=None):
        """fn(device buffers of arrays..., out buffer); the out buffer's content"""
        bufs = [kvc.to_device(a) if a is not None else None for a in arrays]
        isz = np.dtype(dtype).itemsize
        out = self.h.malloc(int(np.prod(shape)) * isz)
        if fill is not None:
            out.upload(np.full(shape, fill, dtype))
        fn(*bufs, out)
        self.ctx.sync()
        got = out.download(dtype, shape)
        for b in bufs + [out]:
            if b is not None:
                b.free()
        return got

    def close(self):
        self.ctx.close()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()
