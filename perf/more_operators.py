"""The operators that continue one prompt in several ways, as measurable cases.

  fork     sequences become copies of others: K/V blocks shared, the recurrent
           state copied (kvc_seq_fork); the copies' state and, through
           kvc_gather, their K/V are what comes back
  reorder  every beam of a batch goes on from the beam it descends from, in
           place (kvc_seq_reorder); state and K/V come back likewise.  The
           batch moves on with each pass, as it does in use
  shared   one decode token per sequence over a cache whose sequences share
           prefixes, each shared block read once (kvc_decode_attn_shared with
           the fused append and the gate)
  select   beam search's choice: the n_out greatest of score + log_softmax over
           all beams and tokens of a prompt, in order (kvc_beam_select)

Sequences of a `shared` case stand in a tree: `p0` tokens common to all (a
system prompt), then `groups` prompts of `p1` tokens, then `n` / `groups`
continuations of each with tails of their own.  Shapes are the ones the library
is built for: 16 q / 4 kv heads of 256 dims, 24 recurrent layers with 32 states
of 128 x 128 and a window of 3 x 8192.
"""
import math
import os
import random
import sys

import torch

own = False

HQ, HKV, D = 16, 4, 256
GROUP = HQ // HKV
ROW = HKV * D
ATTN_LAYERS, SSM_LAYERS = 8, 24
STATE = SSM_LAYERS * (32 * 128 * 128 + 3 * 8192)  # floats of one sequence's recurrent state
VOCAB = 151936
SCALE = 1.0 / 16
TORCH_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # four samples of one short prompt, about to start
        {"name": "fork_1to4", "kind": "fork", "src": 1, "n": 4, "len": 300},
        # a few conversations branched unevenly
        {"name": "fork_5to13", "kind": "fork", "src": 5, "n": 13, "len": 77},
        # a beam search of four beams after its first tokens
        {"name": "reorder_4", "kind": "reorder", "n": 4, "len": 300, "tail": 20},
        # the beams of a batch
        {"name": "reorder_16", "kind": "reorder", "n": 16, "len": 150, "tail": 70},
        # four beams over a short prompt: latency counts
        {"name": "shared_4x300", "kind": "shared", "p0": 300, "groups": 1, "p1": 0, "n": 4, "lo": 1, "hi": 40,
         "layers": 8, "out": "bf16"},
        # eight samples of a longer prompt
        {"name": "shared_8x4096", "kind": "shared", "p0": 4096, "groups": 1, "p1": 0, "n": 8, "lo": 1, "hi": 200,
         "layers": 8, "out": "bf16"},
        # beams of several prompts behind one system prompt, of no round size, compared in fp32
        {"name": "shared_6x5_tree", "kind": "shared", "p0": 777, "groups": 6, "p1": 2001, "n": 30, "lo": 3, "hi": 100,
         "layers": 4, "out": "f32"},
        # a full batch of conversations behind one long system prompt
        {"name": "shared_64x8192", "kind": "shared", "p0": 8192, "groups": 1, "p1": 0, "n": 64, "lo": 20, "hi": 1500,
         "layers": 1, "out": "bf16"},
        # groups of samples of long prompts that have nothing in common
        {"name": "shared_4x16_apart", "kind": "shared", "p0": 0, "groups": 4, "p1": 16000, "n": 64, "lo": 1, "hi": 300,
         "layers": 1, "out": "bf16"},
        # the choice of one prompt's four beams
        {"name": "select_1x4", "kind": "select", "groups": 1, "beams": 4, "vocab": VOCAB, "pad": 0, "n_out": 8,
         "dtype": "bf16", "masked": 0.0, "dead": 0.0},
        # an odd vocabulary, some tokens forbidden, some beams at an end
        {"name": "select_7x5", "kind": "select", "groups": 7, "beams": 5, "vocab": 32001, "pad": 0, "n_out": 10,
         "dtype": "f32", "masked": 0.3, "dead": 0.2},
        # a full batch
        {"name": "select_32x8", "kind": "select", "groups": 32, "beams": 8, "vocab": VOCAB, "pad": 64, "n_out": 16,
         "dtype": "bf16", "masked": 0.0, "dead": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["fork", "reorder", "shared", "shared", "shared", "select", "select", "select"])
    if kind == "fork":
        n = _log(rng, 1, 13)
        return {"kind": kind, "src": rng.randint(1, min(n, 5)), "n": n, "len": _log(rng, 1, 300)}
    if kind == "reorder":
        return {"kind": kind, "n": _log(rng, 1, 16), "len": _log(rng, 1, 150), "tail": _log(rng, 1, 70)}
    if kind == "select":
        beams = _log(rng, 1, 32)
        vocab = _log(rng, 2, 200000)
        groups = _log(rng, 1, max(1, min(64, 32 * 8 * VOCAB // (beams * vocab))))
        return {"kind": kind, "groups": groups, "beams": beams, "vocab": vocab, "pad": rng.choice([0, 0, rng.randint(1, 99)]),
                "n_out": min(_log(rng, 1, 128), 2 * beams * vocab), "dtype": rng.choice(["bf16", "bf16", "f32"]),
                "masked": rng.choice([0.0, 0.0, round(rng.random(), 3)]), "dead": rng.choice([0.0, 0.0, 0.3])}
    per, groups = _log(rng, 1, 64), 1
    if rng.random() < 0.5:
        groups = _log(rng, 1, 64 // per)
    n = per * groups
    p0 = rng.choice([0, _log(rng, 1, 16384)])
    p1 = _log(rng, 1, max(1, min(16384, 64000 // groups))) if p0 == 0 or rng.random() < 0.5 else 0
    hi = _log(rng, 1, max(1, min(1500, 64000 // n)))
    lo = rng.randint(1, hi)
    return {"kind": kind, "p0": p0, "groups": groups, "p1": p1, "n": n, "lo": lo, "hi": hi,
            "layers": 8 if p0 + groups * p1 + n * hi <= 8000 else 1, "out": rng.choice(["bf16", "bf16", "f32"])}


# ---------------------------------------------------------------------------
# inputs, made from the seed alone


def _tails(case):
    """Cached tokens of each sequence behind its prompts, the new one not
    among them: ragged in [lo, hi] - 1, fixed by the case."""
    rng = random.Random(case["n"] * 1000003 + case["lo"] * 8191 + case["hi"])
    return [rng.randint(case["lo"], case["hi"]) - 1 for _ in range(case["n"])]


def _parents(case, seed):
    """Which source each copy comes from: all of them somewhere for a fork; for
    a beam search a few of the beams have most children, in no order."""
    rng = random.Random(seed * 7 + case["n"])
    if case["kind"] == "fork":
        p = list(range(case["src"])) + [rng.randrange(case["src"]) for _ in range(case["n"] - case["src"])]
        rng.shuffle(p)
        return p
    return [min(int(rng.expovariate(1.0) * case["n"] / 3), case["n"] - 1) for _ in range(case["n"])]


def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 4099 + salt)


def _normal(g, shape, dtype=torch.bfloat16):
    x = torch.empty(shape, device="cuda", dtype=dtype)
    for part in x.view(-1).split(1 << 28):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
    return x


def _inputs(case, seed):
    kind = case["kind"]
    g = _gen(seed, 29)
    if kind in ("fork", "reorder"):
        n = case["src"] if kind == "fork" else case["n"]
        length = case["len"] + case.get("tail", 0)
        inp = {"state": _normal(g, (n, STATE), torch.float32)}
        for x in ("k", "v"):
            inp[x] = _normal(g, (ATTN_LAYERS, n, length, HKV, D))
            if kind == "reorder":  # beams of one prompt
                inp[x][:, :, :case["len"]] = inp[x][:, :1, :case["len"]]
        return inp
    if kind == "shared":
        layers, n = case["layers"], case["n"]
        inp = {x: _normal(g, (layers, n, h, D)) for x, h in (("q", HQ), ("gate", HQ), ("k_new", HKV), ("v_new", HKV))}
        gain = torch.where(torch.rand((HKV, D), generator=g, device="cuda") < 0.02, 3.0, 1.0)
        for level, (m, length) in enumerate(((1, case["p0"]), (case["groups"], case["p1"]), (n, max(_tails(case))))):
            inp["k%d" % level] = (_normal(g, (layers, m, length, HKV, D), torch.float32) * gain).to(torch.bfloat16)
            inp["v%d" % level] = _normal(g, (layers, m, length, HKV, D))
        return inp
    # select: logits as a language model gives them, mostly low, a few tokens
    # that stand out and near ties among them; sums of log probabilities
    rows = (case["groups"], case["beams"])
    x = torch.empty((*rows, case["vocab"] + case["pad"]), device="cuda", dtype=TORCH_DTYPE[case["dtype"]])
    for part in x:
        v = torch.randn(part.shape, generator=g, device="cuda") * 2
        v += torch.rand(part.shape, generator=g, device="cuda").pow_(200) * 14
        if case["masked"]:
            v.masked_fill_(torch.rand(part.shape, generator=g, device="cuda") < case["masked"], -math.inf)
        part.copy_(v)
    score = torch.rand(rows, generator=g, device="cuda") * -20
    score.masked_fill_(torch.rand(rows, generator=g, device="cuda") < case["dead"], -math.inf)
    return {"logits": x, "score": score}


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


def _context(**config):
    kvc = _library()

    class Ctx(kvc.Context):
        def __del__(self):
            if getattr(self, "ptr", None):
                self.close()

    return Ctx(snapshot_slots=0, rope_dim=0, flags=kvc.FLAG_EXACT_MATH, **config)


class _Device:
    """Device memory of a context as an array, which keeps the context."""

    def __init__(self, ctx, ptr, n):
        self.ctx = ctx
        self.__cuda_array_interface__ = {"shape": (n,), "typestr": "<f4", "data": (ptr, False), "version": 2}


def _add(ctx, layers, seqs, k, v, stay):
    """The rows k, v [layers][seqs][tokens][4][256] behind what seqs hold."""
    n_tok = k.shape[2]
    if n_tok == 0:
        return
    ctx.reserve(seqs, n_tok)
    for layer in range(layers):
        rows = [x[layer].contiguous() for x in (k, v)]
        ctx.append(layer, seqs, n_tok, rows[0].data_ptr(), rows[1].data_ptr())
        stay.append(rows)
    ctx.commit(seqs, n_tok)


def _state_at(st, seq):
    """The recurrent state of a sequence: where the library has it now."""
    at = st.ctx.state_ptrs(seq, 0)[0]
    if at not in st.views:
        st.views[at] = torch.as_tensor(_Device(st.ctx, at, STATE), device="cuda")
    return st.views[at]


def _prepare_copies(st, case, seed):
    kind, n, inp = case["kind"], case["n"], st.inp
    st.parents = _parents(case, seed)
    if not own:
        st.index = torch.tensor(st.parents, device="cuda")
        return
    length = inp["k"].shape[2]
    n_src = inp["k"].shape[1]
    total = n_src + n if kind == "fork" else n
    st.ctx = ctx = _context(n_attn_layers=ATTN_LAYERS, n_ssm_layers=SSM_LAYERS, max_seqs=total, max_seq_len=length + 32,
                            pool_blocks=(total + 1) * (length // 32 + 3), alloc_seed=seed % 1000003 + 1)
    st.views, stay = {}, []
    st.seqs = [ctx.seq_create() for _ in range(n_src)]
    if kind == "reorder":
        head = case["len"]
        _add(ctx, ATTN_LAYERS, st.seqs[:1], inp["k"][:, :1, :head], inp["v"][:, :1, :head], stay)
        if n > 1:
            ctx.fork(st.seqs[:1] * (n - 1), st.seqs[1:])
        _add(ctx, ATTN_LAYERS, st.seqs, inp["k"][:, :, head:], inp["v"][:, :, head:], stay)
    else:
        _add(ctx, ATTN_LAYERS, st.seqs, inp["k"], inp["v"], stay)
    ctx.sync()
    for i, s in enumerate(st.seqs):
        _state_at(st, s).copy_(inp["state"][i])
    st.result = st.seqs
    if kind == "fork":
        st.result = [ctx.seq_create() for _ in range(n)]
        st.source = _library()._i32([st.seqs[p] for p in st.parents])
    st.result, st.parents = _library()._i32(st.result), _library()._i32(st.parents)
    st.lengths = _library()._i32([length] * n)
    st.k, st.v = (torch.empty((ATTN_LAYERS, n, length, HKV, D), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    torch.cuda.synchronize()
    st.inp = None


def _prepare_shared(st, case, seed):
    inp, layers, n, groups = st.inp, case["layers"], case["n"], case["groups"]
    tails = _tails(case)
    if not own:
        st.seen = torch.arange(max(tails), device="cuda") < torch.tensor(tails, device="cuda")[:, None]
        return
    most = case["p0"] + case["p1"] + max(tails) + 1
    blocks = (case["p0"] + groups * case["p1"] + sum(tails)) // 32 + 3 * (n + groups) + 8
    st.ctx = ctx = _context(n_attn_layers=layers, n_ssm_layers=0, max_seqs=n + groups + 1, max_seq_len=most,
                            pool_blocks=blocks, alloc_seed=seed % 1000003 + 1)
    stay = []
    root = ctx.seq_create()
    _add(ctx, layers, [root], inp["k0"], inp["v0"], stay)
    prompts = [ctx.seq_create() for _ in range(groups)]
    ctx.fork([root] * groups, prompts)
    _add(ctx, layers, prompts, inp["k1"], inp["v1"], stay)
    st.seqs = [ctx.seq_create() for _ in range(n)]
    ctx.fork([prompts[i * groups // n] for i in range(n)], st.seqs)
    for s in [root] + prompts:
        ctx.seq_release(s)
    for i, (s, t) in enumerate(zip(st.seqs, tails)):
        _add(ctx, layers, [s], inp["k2"][:, i:i + 1, :t], inp["v2"][:, i:i + 1, :t], stay)
    ctx.reserve(st.seqs, 1)
    ctx.sync()
    st.seqs = _library()._i32(st.seqs)
    st.out = torch.empty(inp["q"].shape, device="cuda", dtype=TORCH_DTYPE[case["out"]])
    for x in ("k0", "v0", "k1", "v1", "k2", "v2"):
        del inp[x]


def prepare(case, seed):
    st = _State()
    st.case, st.inp = case, _inputs(case, seed)
    if case["kind"] in ("fork", "reorder"):
        _prepare_copies(st, case, seed)
    elif case["kind"] == "shared":
        _prepare_shared(st, case, seed)
    elif own:
        st.ctx = _context(n_attn_layers=1, n_ssm_layers=0, max_seqs=1, max_seq_len=32, pool_blocks=1)
        shape = (case["groups"], case["n_out"])
        st.score = torch.empty(shape, device="cuda", dtype=torch.float32)
        st.beam, st.token = (torch.empty(shape, device="cuda", dtype=torch.int32) for _ in range(2))
    return st


# ---------------------------------------------------------------------------
# one pass of the framework's operators


def _run_own(st):
    case, ctx, inp = st.case, st.ctx, st.inp
    kind = case["kind"]
    if kind in ("fork", "reorder"):
        if kind == "fork":
            for s in st.result:  # the last pass's
                ctx.seq_reset(s)
            ctx.fork(st.source, st.result)
        else:
            ctx.reorder(st.result, st.parents)
        for layer in range(ATTN_LAYERS):
            ctx.gather(layer, st.result, 0, st.lengths, st.k[layer].data_ptr(), st.v[layer].data_ptr())
        return {"state": [_state_at(st, s) for s in st.result], "k": st.k, "v": st.v}
    if kind == "select":
        x = inp["logits"]
        ctx.beam_select(x.data_ptr(), case["groups"], case["beams"], case["vocab"], case["n_out"], st.score.data_ptr(),
                        st.beam.data_ptr(), st.token.data_ptr(), scores=inp["score"].data_ptr(), row_stride=x.shape[2],
                        dtype=1 if case["dtype"] == "bf16" else 0)
        return {"score": st.score, "beam": st.beam, "token": st.token}
    for layer in range(case["layers"]):
        ctx.decode_attn_shared(layer, st.seqs, inp["q"][layer].data_ptr(), st.out[layer].data_ptr(),
                               k_new=inp["k_new"][layer].data_ptr(), v_new=inp["v_new"][layer].data_ptr(),
                               gate=inp["gate"][layer].data_ptr(), out_dtype=1 if case["out"] == "bf16" else 0,
                               scale=SCALE)
    return {"out": st.out}


# ---------------------------------------------------------------------------
# one pass of their plain forms


def _plain_copies(st):
    inp = st.inp
    state, k, v = inp["state"][st.index], inp["k"][:, st.index], inp["v"][:, st.index]
    if st.case["kind"] == "reorder":
        st.inp = {"state": state, "k": k, "v": v}
    return {"state": list(state.unbind(0)), "k": k, "v": v}


def _plain_shared(st):
    """In 32 bits: the scores over each level of the tree, one product for all
    sequences under a node, then one softmax over all of them."""
    case, inp = st.case, st.inp
    layers, n = case["layers"], case["n"]
    q = inp["q"].float().reshape(layers, n, HKV, GROUP, D) * SCALE

    def under(x, m):  # [layers][n][4][4][..] -> [layers][m][4][rows of a node][..]
        return x.reshape(layers, m, n // m, HKV, GROUP, -1).transpose(2, 3).reshape(layers, m, HKV, n // m * GROUP, -1)

    def back(x, m):
        return x.reshape(layers, m, HKV, n // m, GROUP, -1).transpose(2, 3).reshape(layers, n, HKV, GROUP, -1)

    levels = [(1, inp["k0"], inp["v0"]), (case["groups"], inp["k1"], inp["v1"]), (n, inp["k2"], inp["v2"])]
    s = [back(torch.matmul(under(q, m), k.float().permute(0, 1, 3, 4, 2).contiguous()), m) for m, k, _ in levels]
    s[2] = s[2].masked_fill(~st.seen[None, :, None, None], -math.inf)
    s.append((q * inp["k_new"].float()[:, :, :, None]).sum(-1, keepdim=True))
    s = torch.cat(s, -1)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    part = p.split([k.shape[2] for _, k, _ in levels] + [1], -1)
    o = part[3] * inp["v_new"].float()[:, :, :, None]
    for (m, _, v), x in zip(levels, part):
        o = o + back(torch.matmul(under(x, m), v.float().transpose(2, 3).contiguous()), m)
    o = (o / p.sum(-1, keepdim=True)).reshape(layers, n, HQ, D)
    return {"out": (o / (1.0 + torch.exp(-inp["gate"].float()))).to(TORCH_DTYPE[case["out"]])}


def _plain_select(st):
    """A beam's tokens in the order of their logits (ties: the lower token),
    its first ones against the other beams' by their sums in 64 bits (ties:
    the lower beam)."""
    case, score = st.case, st.inp["score"].double()
    groups, beams, vocab, n_out = case["groups"], case["beams"], case["vocab"], case["n_out"]
    x = st.inp["logits"][..., :vocab].float()
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.amax(-1, keepdim=True)
    alive = top[..., 0].isfinite() & score.isfinite()
    y = x.double().sub_(torch.where(top.isfinite(), top, 0.0))
    offset = torch.where(alive, score - torch.log(y.exp_().sum(-1)) - top[..., 0].double(), 0.0)
    x, token = torch.sort(x, dim=-1, descending=True, stable=True)
    kept = min(n_out, vocab)
    value = torch.where(alive[..., None], x[..., :kept].double() + offset[..., None], -math.inf).reshape(groups, -1)
    value, at = torch.sort(value, dim=-1, descending=True, stable=True)
    value, at = value[:, :n_out], at[:, :n_out]
    token = torch.gather(token[..., :kept].reshape(groups, -1), 1, at)
    real = value > -math.inf
    out = {"score": (value.float(), -math.inf), "beam": (torch.where(real, at // kept, -1).int(), -1),
           "token": (torch.where(real, token, -1).int(), -1)}
    return {name: torch.nn.functional.pad(t, (0, n_out - t.shape[1]), value=fill) for name, (t, fill) in out.items()}


def run(st):
    if own:
        return _run_own(st)
    return {"fork": _plain_copies, "reorder": _plain_copies, "shared": _plain_shared, "select": _plain_select}[
        st.case["kind"]](st)


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    kind, n = case["kind"], case["n"] if "n" in case else 0
    if kind == "fork":
        per = STATE * 4 + ATTN_LAYERS * case["len"] * ROW * 4
        return {"bytes": (case["src"] + n) * per, "flops": 0}
    if kind == "reorder":
        # a beam with one child goes on where it is; the seeds' mean share of
        # copies is that of the first seeds
        kept = sum(len(set(_parents(case, seed))) for seed in range(1, 9)) / 8
        rows = ATTN_LAYERS * ROW * 4
        return {"bytes": (2 * (n - kept)) * STATE * 4 + rows * (case["len"] + kept * case["tail"] + n * (case["len"] + case["tail"])),
                "flops": 0}
    if kind == "select":
        esz = 2 if case["dtype"] == "bf16" else 4
        size = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": size * esz + case["groups"] * (case["beams"] * 4 + case["n_out"] * 12), "flops": size * 4}
    tails = sum(_tails(case))
    keys = case["p0"] + case["groups"] * case["p1"] + tails + n
    pairs = n * (case["p0"] + case["p1"] + 1) + tails
    esz = 2 if case["out"] == "bf16" else 4
    return {"bytes": case["layers"] * (keys * ROW * 4 + n * (HQ * D * (4 + esz) + ROW * 4)),
            "flops": case["layers"] * pairs * HQ * D * 4}


# ---------------------------------------------------------------------------
# the same results in 64 bits, one sequence or prompt at a time


def _exact_select(case, inp):
    groups, vocab, n_out = case["groups"], case["vocab"], case["n_out"]
    out = {"score": torch.full((groups, n_out), -math.inf, dtype=torch.float64, device="cuda"),
           "beam": torch.full((groups, n_out), -1, dtype=torch.int32, device="cuda")}
    out["token"] = out["beam"].clone()
    for i in range(groups):
        x = inp["logits"][i, :, :vocab].double()
        v = inp["score"][i].double()[:, None] + torch.log_softmax(x, -1)
        v = torch.where(v.isnan(), -math.inf, v).reshape(-1)
        v, at = torch.sort(v, descending=True, stable=True)
        m = min(n_out, int((v > -math.inf).sum()))
        out["score"][i, :m] = v[:m]
        out["beam"][i, :m] = (at[:m] // vocab).int()
        out["token"][i, :m] = (at[:m] % vocab).int()
    return out


def exact(case, seed):
    inp = _inputs(case, seed)
    kind, n = case["kind"], case["n"] if "n" in case else 0
    if kind in ("fork", "reorder"):
        parents = _parents(case, seed)
        return {"state": [inp["state"][p].double() for p in parents],
                **{x: torch.stack([inp[x][:, p].double() for p in parents], 1) for x in ("k", "v")}}
    if kind == "select":
        return _exact_select(case, inp)
    out = torch.empty(inp["q"].shape, device="cuda", dtype=torch.float64)
    for layer in range(case["layers"]):
        for i, t in enumerate(_tails(case)):
            j = i * case["groups"] // n
            k, v = (torch.cat([inp[x + "0"][layer, 0], inp[x + "1"][layer, j], inp[x + "2"][layer, i, :t],
                               inp[x + "_new"][layer, i][None]]).double().transpose(0, 1).contiguous() for x in ("k", "v"))
            q = inp["q"][layer, i].double().view(HKV, GROUP, D)
            p = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) * SCALE, -1)
            out[layer, i] = torch.matmul(p, v).view(HQ, D) * torch.sigmoid(inp["gate"][layer, i].double())
    return {"out": out}
