"""The operators that keep long sessions in less memory, as measurable cases.

  park     a batch of sessions is copied into 8 bits, the originals kept for
           reuse (kvc_kv_quantize), and the copies are read back (kvc_gather)
  decode   one token per sequence attends over a cache whose cold blocks are in
           8 bits (kvc_decode_attn with the fused append and the gate)
  prefill  a chunk per sequence attends over such a cache (kvc_prefill_attn)
  weights  the attention weight that the last queries give every cached token,
           added to an accumulator (kvc_attn_weights)
  evict    every (layer, kv head) of a batch of sessions keeps the tokens of
           greatest accumulated weight, in copies (kvc_evict), and the kept rows
           are read back (kvc_gather)

A unit of the 8-bit cache is 32 tokens of one kv head, K or V: values i * s
with s = max(a, 2^-100) / 127, i = rne(x * (127 / max(a, 2^-100))), a = max |x|.
Shapes are the ones the library is built for: 16 q / 4 kv heads of 256 dims,
blocks of 32 tokens, up to 8 attention layers.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

HQ, HKV, D, BT = 16, 4, 256, 32
GROUP = HQ // HKV
SCALE = 1.0 / 16
TINY = 2.0 ** -100
TORCH_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one session branched into a parked copy
        {"name": "park_1x4096", "kind": "park", "n": 1, "len": 4096, "keep": 0, "layers": 8},
        # a batch of sessions of no round size whose last 100 tokens stay in bf16
        {"name": "park_16x1000", "kind": "park", "n": 16, "len": 1000, "keep": 100, "layers": 2},
        # the first answer tokens of a chat: one sequence, a short context, latency counts
        {"name": "decode8_1x300", "kind": "decode", "n": 1, "lo": 300, "hi": 300, "keep": 0, "layers": 8, "out": "bf16"},
        # one longer conversation
        {"name": "decode8_1x4096", "kind": "decode", "n": 1, "lo": 4096, "hi": 4096, "keep": 0, "layers": 8,
         "out": "bf16"},
        # a few conversations served together, their latest tokens in bf16
        {"name": "decode8_8_ragged", "kind": "decode", "n": 8, "lo": 777, "hi": 6001, "keep": 200, "layers": 8,
         "out": "f32"},
        # a full batch of ragged sequences: the throughput end
        {"name": "decode8_64_ragged", "kind": "decode", "n": 64, "lo": 512, "hi": 16384, "keep": 0, "layers": 1,
         "out": "bf16"},
        # a short chunk in the middle of a parked conversation
        {"name": "prefill8_1x32", "kind": "prefill", "n": 1, "lo": 4001, "hi": 4001, "n_q": 32, "keep": 0, "layers": 8,
         "out": "bf16"},
        # a batch of new turns over parked prefixes
        {"name": "prefill8_16x128", "kind": "prefill", "n": 16, "lo": 256, "hi": 6000, "n_q": 128, "keep": 64,
         "layers": 1, "out": "bf16"},
        # the weights of one decode token, every layer
        {"name": "weights_1x4096", "kind": "weights", "n": 1, "lo": 4096, "hi": 4096, "n_q": 1, "keep": 4096,
         "layers": 8},
        # the last 32 prompt tokens score the whole prompt, in 8 bits
        {"name": "weights_16x32", "kind": "weights", "n": 16, "lo": 500, "hi": 6000, "n_q": 32, "keep": 0, "layers": 1},
        # one session cut to a quarter, every layer and kv head its own tokens
        {"name": "evict_1x4096", "kind": "evict", "n": 1, "len": 4096, "budget": 1024, "sink": 4, "recent": 128,
         "layers": 8},
        # a batch cut to an odd budget
        {"name": "evict_16x5000", "kind": "evict", "n": 16, "len": 5000, "budget": 1501, "sink": 1, "recent": 200,
         "layers": 1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["park", "decode", "decode", "prefill", "prefill", "weights", "weights", "evict"])
    n = _log(rng, 1, 64)
    if kind == "park":
        length = _log(rng, 1, min(16384, 60000 // n))
        return {"kind": kind, "n": n, "len": length, "keep": rng.choice([0, 0, rng.randint(1, length)]),
                "layers": 8 if n * length <= 6000 else 1}
    if kind == "evict":
        length = _log(rng, 2, min(20000, 80000 // n))
        budget = rng.randint(1, length)
        sink = rng.randint(0, min(8, budget))
        return {"kind": kind, "n": n, "len": length, "budget": budget, "sink": sink,
                "recent": rng.randint(0, budget - sink), "layers": 8 if n * length <= 6000 else 1}
    hi = min(_log(rng, 33, 16384), 400000 // n)
    lo = rng.randint(max(1, hi // 32), hi)
    keep = rng.choice([0, 0, rng.randint(1, 300)])
    if kind == "decode":
        return {"kind": kind, "n": n, "lo": lo, "hi": hi, "keep": keep, "layers": 8 if n * hi <= 50000 else 1,
                "out": rng.choice(["bf16", "bf16", "f32"])}
    if kind == "weights":
        hi = min(hi, 90000 // n)
        lo = min(lo, hi)
        n_q = _log(rng, 1, max(1, min(64, 3000000 // (n * hi))))
        return {"kind": kind, "n": n, "lo": lo, "hi": hi, "n_q": min(n_q, lo),
                "keep": rng.choice([0, keep, hi]), "layers": 8 if n * hi * n_q <= 50000 else 1}
    n_q = _log(rng, 2, max(2, min(512, 4096 // n)))
    hi = max(1, min(hi, 12000000 // (n * n_q)))
    lo = min(lo, hi)
    return {"kind": kind, "n": n, "lo": lo, "hi": hi, "n_q": n_q, "keep": keep,
            "layers": 8 if n * n_q * (hi + n_q) <= 400000 else 1, "out": rng.choice(["bf16", "bf16", "f32"])}


# ---------------------------------------------------------------------------
# inputs, made from the seed alone


def _lengths(case):
    """Ragged lengths in [lo, hi], fixed by the case: tokens cached before the
    chunk (prefill), attended keys in all (decode, weights)."""
    rng = random.Random(case["n"] * 1000003 + case["lo"] * 8191 + case["hi"])
    return [rng.randint(case["lo"], case["hi"]) for _ in range(case["n"])]


def _cached(case):
    """Tokens of each sequence in the cache and not part of the call."""
    return [x - 1 for x in _lengths(case)] if case["kind"] == "decode" else _lengths(case)


def _parked(case, cached):
    """Leading tokens held in 8 bits: full blocks before the last `keep` tokens."""
    return [max(0, x - case["keep"]) // BT * BT for x in cached]


def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 4099 + salt)


def _normal(g, shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _inputs(case, seed):
    """What a case's call is given, as tensors.  k, v: [layers][n][len][4][256]
    with the cached tokens first in each row; keys carry a few large channels,
    as trained ones do, so that block scales differ."""
    layers, n = case["layers"], case["n"]
    g = _gen(seed, 17)
    length = case["len"] if "len" in case else max(_cached(case)) + (case.get("n_q", 0) if case["kind"] == "prefill" else 0)
    inp = {"k": torch.empty((layers, n, length, HKV, D), device="cuda", dtype=torch.bfloat16)}
    inp["v"] = torch.empty_like(inp["k"])
    gain = torch.where(torch.rand((HKV, D), generator=g, device="cuda") < 0.02, 3.0, 1.0)
    for layer in range(layers):
        inp["k"][layer] = torch.randn((n, length, HKV, D), generator=g, device="cuda") * gain
        inp["v"][layer] = torch.randn((n, length, HKV, D), generator=g, device="cuda")
    if case["kind"] == "decode":
        for name, heads in (("q", HQ), ("gate", HQ), ("k_new", HKV), ("v_new", HKV)):
            inp[name] = _normal(g, (layers, n, heads, D))
    elif case["kind"] == "prefill":
        inp["q"], inp["gate"] = (_normal(g, (layers, n, case["n_q"], HQ, D)) for _ in range(2))
    elif case["kind"] == "weights":
        inp["q"] = _normal(g, (layers, n, case["n_q"], HQ, D))
        inp["acc"] = torch.rand((layers, n, HKV, length), generator=g, device="cuda") * 0.1
    elif case["kind"] == "evict":
        # accumulated weights: mostly small, a few heavy tokens; a tenth of them
        # on a coarse grid, so that equal ones meet at the border
        a = torch.rand((layers, n, HKV, length), generator=g, device="cuda").pow_(8)
        tie = torch.rand((layers, n, HKV, length), generator=g, device="cuda") < 0.1
        inp["acc"] = torch.where(tie, (a * 16).ceil() / 16, a)
    return inp


def _units(x):
    """[..., tokens, 4, 256] of whole blocks -> [..., blocks, 32, 4, 256]."""
    return x.reshape(*x.shape[:-3], x.shape[-3] // BT, BT, HKV, D)


def _quantize(x):
    """Whole blocks in 8 bits: integers [..., tokens, 4, 256] and scales
    [..., blocks, 4]."""
    u = _units(x).float()
    a = u.abs().amax(dim=(-3, -1)).clamp_min(TINY)
    hundred27 = torch.full_like(a, 127.0)
    i = torch.round(u * (hundred27 / a)[..., None, :, None]).clamp_(-127, 127)
    return i.to(torch.int8).reshape(x.shape), a / hundred27


def _dequantize(i, scale):
    return (_units(i).float() * scale[..., None, :, None]).reshape(i.shape)


# ---------------------------------------------------------------------------
# what a user's program holds before the call


class _State:
    pass


def _library():
    package = os.path.join(os.getcwd(), "qwen3.5-9b-bfp8b-1xn300_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import kvc

    return kvc


def _context(case, seed, max_len, max_parked):
    """A context that fits the case, copies included: the cache handle that a
    program keeps."""
    kvc = _library()

    class Ctx(kvc.Context):
        def __del__(self):
            if getattr(self, "ptr", None):
                self.close()

    per = (max_len + case.get("budget", 0)) // BT + 2
    blocks = case["n"] * per
    return Ctx(n_attn_layers=case["layers"], n_ssm_layers=0, max_seqs=2 * case["n"], max_seq_len=max_len + BT,
               pool_blocks=blocks + 8, q8_blocks=max(1, case["n"] * max_parked // BT), snapshot_slots=0,
               alloc_seed=seed % 1000003 + 1, rope_dim=0, flags=kvc.FLAG_EXACT_MATH)


def _fill(st, case, seed, cached, extra):
    """The context with every sequence's cached tokens."""
    st.ctx = ctx = _context(case, seed, max(cached) + extra, max(cached))
    st.seqs = _library()._i32([ctx.seq_create() for _ in cached])
    for i, (s, length) in enumerate(zip(st.seqs, cached)):
        if length == 0:
            continue
        ctx.reserve([s], length)
        for layer in range(case["layers"]):
            k, v = (st.inp[x][layer, i, :length].contiguous() for x in ("k", "v"))
            ctx.append(layer, [s], length, k.data_ptr(), v.data_ptr())
        ctx.commit([s], length)
        ctx.sync()


def _split_cache(st, case, cached):
    """The same cache for the plain form: 8-bit prefix with its scales, bf16
    tail, both padded to the longest, and which of their slots hold a key."""
    parked = _parked(case, cached)
    n8 = max(parked)
    extra = case["n_q"] if case["kind"] == "prefill" else 0
    tail = [c + extra - p for c, p in zip(cached, parked)]
    nt = max(max(tail), 1)
    at = torch.tensor(parked, device="cuda")[:, None] + torch.arange(nt, device="cuda")
    at = at.clamp_(max=st.inp["k"].shape[2] - 1)[None, :, :, None, None].expand(case["layers"], -1, -1, HKV, D)
    st.parked, st.tail = torch.tensor(parked, device="cuda"), torch.tensor(tail, device="cuda")
    for x in ("k", "v"):
        full = st.inp[x]
        i, s = _quantize(full[:, :, :n8])
        setattr(st, x + "8", i)
        setattr(st, x + "s", s)
        setattr(st, x + "t", torch.gather(full, 2, at))


def prepare(case, seed):
    st = _State()
    st.case, st.inp = case, _inputs(case, seed)
    kind, n, layers = case["kind"], case["n"], case["layers"]
    if kind in ("park", "evict"):
        rows = case["len"] if kind == "park" else min(case["budget"], case["len"])
        if own:
            _fill(st, case, seed, [case["len"]] * n, 0)
            st.copies = _library()._i32([st.ctx.seq_create() for _ in range(n)])
            st.k, st.v = (torch.empty((layers, n, rows, HKV, D), device="cuda", dtype=torch.bfloat16) for _ in range(2))
        if own and kind == "evict":
            st.kept = torch.empty((layers, n, HKV, case["budget"]), device="cuda", dtype=torch.int32)
            st.acc_out = torch.zeros_like(st.inp["acc"])
        return st
    cached = _cached(case)
    extra = {"decode": 1, "prefill": case.get("n_q"), "weights": 0}[kind]
    if own:
        _fill(st, case, seed, cached, extra)
        st.ctx.kv_quantize(st.seqs, case["keep"])
        if extra:
            st.ctx.reserve(st.seqs, extra)
        if kind == "prefill":  # the chunk's K/V are in the cache before its attention
            for layer in range(layers):
                k, v = (torch.stack([st.inp[x][layer, i, c:c + extra] for i, c in enumerate(cached)]) for x in ("k", "v"))
                st.ctx.append(layer, st.seqs, extra, k.data_ptr(), v.data_ptr())
                st.ctx.sync()
        if kind == "weights":
            st.out = torch.zeros_like(st.inp["acc"])
        else:
            st.out = torch.empty(st.inp["q"].shape, device="cuda", dtype=TORCH_DTYPE[case["out"]])
        st.ctx.sync()
    _split_cache(st, case, cached)
    del st.inp["k"], st.inp["v"]
    return st


# ---------------------------------------------------------------------------
# one pass of the framework's operators


def _run_own(st):
    case, ctx, inp = st.case, st.ctx, st.inp
    kind, layers, n = case["kind"], case["layers"], case["n"]
    if kind in ("park", "evict"):
        for s in st.copies:  # the last pass's
            ctx.seq_reset(s)
        rows = st.k.shape[2]
        if kind == "park":
            ctx.kv_quantize(st.seqs, case["keep"], dst=st.copies)
        else:
            ctx.evict(st.seqs, case["budget"], inp["acc"].data_ptr(), case["len"], st.kept.data_ptr(), dst=st.copies,
                      n_sink=case["sink"], n_recent=case["recent"], acc_out=st.acc_out.data_ptr())
        for layer in range(layers):
            ctx.gather(layer, st.copies, 0, [rows] * n, st.k[layer].data_ptr(), st.v[layer].data_ptr())
        out = {"k": st.k, "v": st.v}
        return out if kind == "park" else {**out, "kept": st.kept, "acc": st.acc_out}
    odt = 1 if case.get("out") == "bf16" else 0
    for layer in range(layers):
        q = inp["q"][layer].data_ptr()
        if kind == "weights":
            ctx.attn_weights(layer, st.seqs, case["n_q"], q, st.out[layer].data_ptr(), st.out.shape[-1],
                             acc_in=inp["acc"][layer].data_ptr(), scale=SCALE)
        elif kind == "decode":
            ctx.decode_attn(layer, st.seqs, q, st.out[layer].data_ptr(), k_new=inp["k_new"][layer].data_ptr(),
                            v_new=inp["v_new"][layer].data_ptr(), gate=inp["gate"][layer].data_ptr(), out_dtype=odt,
                            scale=SCALE)
        else:
            ctx.prefill_attn(layer, st.seqs, case["n_q"], q, st.out[layer].data_ptr(),
                             gate=inp["gate"][layer].data_ptr(), out_dtype=odt, scale=SCALE)
    return {"out": st.out}


# ---------------------------------------------------------------------------
# one pass of their plain forms, in 32 bits


def _plain_park(st):
    case, out = st.case, {}
    m = max(0, case["len"] - case["keep"]) // BT * BT
    for x in ("k", "v"):
        full = st.inp[x]
        out[x] = torch.cat([_dequantize(*_quantize(full[:, :, :m])).to(torch.bfloat16), full[:, :, m:]], dim=2)
    return out


def _plain_evict(st):
    case, acc = st.case, st.inp["acc"]
    length, budget = case["len"], case["budget"]
    j = torch.arange(length, device="cuda")
    forced = (j < case["sink"]) | (j >= length - case["recent"])
    score = torch.where(forced, math.inf, acc)
    kept = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :budget].sort(dim=-1).values
    kept_acc = torch.zeros_like(acc)
    kept_acc[..., :budget] = torch.gather(acc, -1, kept)
    at = kept.transpose(2, 3)[..., None].expand(-1, -1, -1, -1, D)  # [layers][n][budget][4][256]
    return {"k": torch.gather(st.inp["k"], 2, at), "v": torch.gather(st.inp["v"], 2, at), "kept": kept.int(),
            "acc": kept_acc}


def _heads(x):
    """[layers][n][tokens][4][256] -> [layers][n][4][tokens][256], in fp32."""
    return x.float().transpose(2, 3)


def _scores(st, q, n_new):
    """Softmax numerators [layers][n][4][rows][keys] of q [layers][n][n_new][16][256]
    over the 8-bit prefix, then the tail (then a new token's key), their
    values, and the row sums."""
    case = st.case
    layers, n, t = q.shape[0], q.shape[1], q.shape[2]
    qh = q.float().reshape(layers, n, t, HKV, GROUP, D).permute(0, 1, 3, 2, 4, 5).reshape(layers, n, HKV, t * GROUP, D)
    k = [_heads(_dequantize(st.k8, st.ks)), _heads(st.kt)]
    v = [_heads(_dequantize(st.v8, st.vs)), _heads(st.vt)]
    n8, nt = k[0].shape[3], k[1].shape[3]
    row = torch.arange(t, device="cuda").repeat_interleave(GROUP)
    # keys of the tail that a row sees: those up to its own position
    seen = st.tail[:, None] - (t - 1 - row if n_new else 0 * row)
    at8, att = torch.arange(n8, device="cuda"), torch.arange(nt, device="cuda")
    own8 = st.parked[:, None] + torch.clamp(seen, max=0)  # rows inside the prefix see less of it
    hide = [(at8 >= own8[..., None])[None, :, None], (att >= seen[..., None])[None, :, None]]
    if case["kind"] == "decode":
        k.append(st.inp["k_new"].float()[:, :, :, None])
        v.append(st.inp["v_new"].float()[:, :, :, None])
        hide.append(torch.zeros((1, 1, 1, 1, 1), dtype=torch.bool, device="cuda"))
    s = torch.cat([torch.matmul(qh, x.transpose(3, 4)).mul_(SCALE).masked_fill_(y, -math.inf) for x, y in zip(k, hide)], -1)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return p, p.sum(-1, keepdim=True), v


def _attend(st, q, gate, n_new):
    p, total, v = _scores(st, q, n_new)
    o, at = 0.0, 0
    for x in v:
        o = o + torch.matmul(p[..., at:at + x.shape[3]], x)
        at += x.shape[3]
    layers, n, t = q.shape[0], q.shape[1], q.shape[2]
    o = (o / total).reshape(layers, n, HKV, t, GROUP, D).permute(0, 1, 3, 2, 4, 5).reshape(q.shape)
    return (o / (1.0 + torch.exp(-gate.float()))).to(TORCH_DTYPE[st.case["out"]])


def _plain_weights(st):
    p, total, _ = _scores(st, st.inp["q"], True)
    w = (p / total).sum(3)  # over the rows of a kv head
    n8 = st.k8.shape[2]
    acc = st.inp["acc"]
    length = acc.shape[-1]
    # key slots back to positions: prefix, then the tail from where it ends
    j = torch.arange(length, device="cuda")
    slot = torch.where(j < st.parked[:, None], j, n8 + j - st.parked[:, None]).clamp_(max=w.shape[-1] - 1)
    cached = j < (st.parked + st.tail)[:, None]
    got = torch.gather(w, -1, slot[None, :, None].expand(w.shape[0], -1, HKV, -1))
    return torch.where(cached[None, :, None], acc + got, 0.0)


def run(st):
    if own:
        return _run_own(st)
    kind, inp = st.case["kind"], st.inp
    if kind == "park":
        return _plain_park(st)
    if kind == "evict":
        return _plain_evict(st)
    if kind == "weights":
        return {"out": _plain_weights(st)}
    if kind == "decode":
        return {"out": _attend(st, inp["q"][:, :, None], inp["gate"][:, :, None], False)[:, :, 0]}
    return {"out": _attend(st, inp["q"], inp["gate"], True)}


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    n, layers = case["n"], case["layers"]
    row = HKV * D
    if case["kind"] == "park":
        t8 = max(0, case["len"] - case["keep"]) // BT * BT
        tail = case["len"] - t8
        # rows in, 8 bits and scales out and in again, rows out
        return {"bytes": layers * n * 2 * (t8 * (row * 6 + 2 * HKV * 4 // BT) + tail * row * 4), "flops": 0}
    if case["kind"] == "evict":
        kept = case["budget"]
        return {"bytes": layers * n * (HKV * (4 * case["len"] + 8 * kept) + kept * 2 * row * 4), "flops": 0}
    cached = _cached(case)
    parked = _parked(case, cached)
    sides = 1 if case["kind"] == "weights" else 2  # K alone, or K and V
    keys = sum(p * (row + 4 * HKV / BT) + (c - p) * row * 2 for p, c in zip(parked, cached)) * sides
    esz = {"f32": 4, "bf16": 2}.get(case.get("out"))
    if case["kind"] == "decode":
        return {"bytes": layers * (keys + n * (HQ * D * (4 + esz) + 2 * row * 2)), "flops": layers * sum(cached) * HQ * D * 4}
    t = case["n_q"]
    if case["kind"] == "weights":
        pairs = sum(t * c - t * (t - 1) // 2 for c in cached)
        return {"bytes": layers * (keys + n * t * HQ * D * 2 + sum(cached) * HKV * 8), "flops": layers * pairs * HQ * D * 2}
    pairs = sum(t * c + t * (t + 1) // 2 for c in cached)
    return {"bytes": layers * (keys + n * t * (HQ * D * (4 + esz) + 2 * row * 2)), "flops": layers * pairs * HQ * D * 4}


# ---------------------------------------------------------------------------
# the same results in 64 bits, sequence by sequence


def _exact_values(x, parked):
    """fp64 values of one sequence's rows [tokens][4][256], the first `parked`
    of them through 8 bits."""
    y = x.double()
    if parked:
        u = y[:parked].view(parked // BT, BT, HKV, D)
        a = torch.maximum(u.abs().amax(3).amax(1), torch.tensor(TINY, device="cuda", dtype=torch.float64))
        inv = (127.0 / a).float().double()[:, None, :, None]  # a quotient of 53 bits, rounded to fp32
        s = (a / 127.0).float().double()[:, None, :, None]
        y = torch.cat([((u * inv).float().double().round() * s).view(parked, HKV, D), y[parked:]])
    return y


def _exact_softmax(q, k, h, first):
    """Weights of q head h's rows [rows][256] over k [keys][4][256]; row i sees
    keys up to first + i."""
    s = q @ k[:, h // GROUP].t().contiguous() * SCALE
    s.masked_fill_(torch.arange(len(k), device="cuda") > first + torch.arange(len(q), device="cuda")[:, None], -math.inf)
    return torch.softmax(s, -1)


def exact(case, seed):
    inp = _inputs(case, seed)
    kind, n, layers = case["kind"], case["n"], case["layers"]
    if kind == "park":
        t8 = max(0, case["len"] - case["keep"]) // BT * BT
        return {x: torch.stack([torch.stack([_exact_values(inp[x][l, i], t8) for i in range(n)]) for l in range(layers)])
                for x in ("k", "v")}
    if kind == "evict":
        acc = inp["acc"].double().cpu().numpy()
        length, budget, sink, recent = case["len"], case["budget"], case["sink"], case["recent"]
        mid = np.arange(sink, length - recent)
        kept = np.empty((layers, n, HKV, budget), np.int64)
        for at in np.ndindex(layers, n, HKV):
            heavy = mid[np.argsort(-acc[at][mid], kind="stable")[:budget - sink - recent]]
            kept[at] = np.concatenate([np.arange(sink), np.sort(heavy), np.arange(length - recent, length)])
        out = np.zeros_like(acc)
        out[..., :budget] = np.take_along_axis(acc, kept, -1)
        t = torch.from_numpy(kept).cuda()
        heads = torch.arange(HKV, device="cuda")
        rows = {x: torch.stack([torch.stack([inp[x][l, i][t[l, i].t(), heads].double() for i in range(n)])
                                for l in range(layers)]) for x in ("k", "v")}
        return {**rows, "kept": t.int(), "acc": torch.from_numpy(out).cuda()}
    cached = _cached(case)
    parked = _parked(case, cached)
    t = case.get("n_q", 1)
    result = torch.zeros(inp["acc"].shape if kind == "weights" else inp["q"].shape, device="cuda", dtype=torch.float64)
    for l in range(layers):
        for i, (c, p) in enumerate(zip(cached, parked)):
            total = c + t if kind == "prefill" else c
            k = _exact_values(inp["k"][l, i, :total], p)
            q = inp["q"][l, i].double().reshape(t, HQ, D)
            if kind == "weights":
                result[l, i, :, :c] = inp["acc"][l, i, :, :c].double()
                for h in range(HQ):
                    result[l, i, h // GROUP, :c] += _exact_softmax(q[:, h], k, h, c - t).sum(0)
                continue
            v = _exact_values(inp["v"][l, i, :total], p)
            if kind == "decode":
                k = torch.cat([k, inp["k_new"][l, i][None].double()])
                v = torch.cat([v, inp["v_new"][l, i][None].double()])
            o = torch.stack([_exact_softmax(q[:, h], k, h, len(k) - t) @ v[:, h // GROUP] for h in range(HQ)], 1)
            result[l, i] = (o * torch.sigmoid(inp["gate"][l, i].double().reshape(t, HQ, D))).reshape(result[l, i].shape)
    return {"out": result}
