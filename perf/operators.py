"""Timed cases of the 8-bit KV-cache operators and the log-probability operator.

Four operators of a decoder that serves from a quantised cache:

- ``write``: a step's or a prompt's keys and values quantised into the cache
  (head norm and rotary on the keys first) and read back as the values the
  codes stand for;
- ``attend``: grouped-query attention over that cache, the call's own tokens
  appended first: one token per sequence, a chunk of a prompt, a whole prompt;
- ``tree``: the same attention for a tree of drafted tokens per sequence, then
  the rows of the accepted path moved to the front of the drafted rows;
- ``logprobs``: log probabilities of given tokens, entropy and the k likeliest
  alternatives of rows of logits.

Where ``own`` is true, ``run`` makes the calls a user makes through the C ABI
binding; otherwise it computes the plain form.
"""
import math

import torch

own = False  # set by the program that times the cases


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # The append of one decode step: 64 sequences, the decoder's 8 kv heads of 128.
        dict(name="write-step-b64", op="write", kv="int8", b=64, s=1, past=500, ragged=True, cap=1024, kvh=8, d=128,
             rot=128, inter=False, norm=True),
        # Prompts being admitted behind cached prefixes, an odd number of tokens each.
        dict(name="write-prompt-b8-s2047", op="write", kv="e4m3", b=8, s=2047, past=512, ragged=True, cap=2560, kvh=8,
             d=128, rot=128, inter=False, norm=True),
        # The smallest call: one sequence's decode step, where latency counts.
        dict(name="attend-step-b1-511", op="attend", kv="int8", b=1, s=1, past=511, ragged=False, cap=1024, h=16,
             kvh=8, d=128, rot=128, inter=False, norm=True, out="f32"),
        # A full serving batch late in its generation: the cache is read once, everything else is small.
        dict(name="attend-step-b64-8191", op="attend", kv="int8", b=64, s=1, past=8191, ragged=True, cap=8256, h=16,
             kvh=8, d=128, rot=128, inter=False, norm=True, out="f16"),
        # Three long documents, eight query heads on each kv head.
        dict(name="attend-step-b3-40000", op="attend", kv="e4m3", b=3, s=1, past=40000, ragged=True, cap=40960, h=32,
             kvh=4, d=128, rot=128, inter=False, norm=False, out="f32"),
        # Heads of 64, three query heads on each kv head, interleaved rotary on part of the head.
        dict(name="attend-step-b17-1001", op="attend", kv="int8", b=17, s=1, past=1001, ragged=True, cap=1100, h=12,
             kvh=4, d=64, rot=32, inter=True, norm=False, out="f32"),
        # Whole prompts from an empty cache.
        dict(name="attend-prompt-b4-s2048", op="attend", kv="int8", b=4, s=2048, past=0, ragged=False, cap=2176, h=16,
             kvh=8, d=128, rot=128, inter=False, norm=True, out="f16"),
        # A chunk of a longer prompt behind what is cached, with fp32 rows out.
        dict(name="attend-chunk-b2-s777", op="attend", kv="e4m3", b=2, s=777, past=3001, ragged=True, cap=4096, h=32,
             kvh=8, d=128, rot=128, inter=False, norm=False, out="f32"),
        # Eight drafted tokens for each sequence of a batch.
        dict(name="tree-b32-n8-1500", op="tree", kv="int8", b=32, s=8, past=1500, ragged=True, cap=2048, h=16, kvh=8,
             d=128, rot=128, inter=False, norm=True, out="f16"),
        # The widest tree, on two long sequences.
        dict(name="tree-b2-n64-6000", op="tree", kv="e4m3", b=2, s=64, past=6000, ragged=True, cap=6144, h=16, kvh=8,
             d=128, rot=128, inter=False, norm=True, out="f32"),
        # One generated token's report.
        dict(name="logprobs-r1", op="logprobs", rows=1, v=151936, ld=151936, k=5, banned=False),
        # Scoring a batch of prompts, a chunk of positions at a time, some tokens banned.
        dict(name="logprobs-r1024", op="logprobs", rows=1024, v=151936, ld=151936, k=20, banned=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("write", "attend", "attend", "tree", "logprobs"))
    if op == "logprobs":
        rows = _log_int(rng, 1, 1024)
        v = min(_log_int(rng, 1000, 151936), 151936)
        return dict(op=op, rows=rows, v=v, ld=v + rng.choice((0, 0, 3, 64)), k=rng.choice((0, 1, 5, 20, 32)),
                    banned=rng.random() < 0.5)
    d = rng.choice((32, 64, 80, 96, 128, 128, 128, 256))
    kvh = rng.choice((1, 2, 4, 8))
    c = dict(op=op, kv=rng.choice(("int8", "e4m3")), ragged=rng.random() < 0.7, kvh=kvh, d=d,
             rot=rng.choice((0, d // 2, d)), inter=rng.random() < 0.3, norm=rng.random() < 0.5)
    if op == "write":
        b = _log_int(rng, 1, 64)
        s = _log_int(rng, 1, max(1, 8 * 2047 * 8 * 128 // (b * kvh * d)))
        s = min(s, 2047)
        past = rng.randrange(0, 1000)
        return dict(c, b=b, s=s, past=past, cap=past + s + rng.randrange(0, 200))
    c["h"] = kvh * rng.choice((1, 2, 3, 4, 8))
    c["out"] = rng.choice(("f32", "f16"))
    if op == "tree":
        b, s = _log_int(rng, 1, 32), rng.randrange(2, 65)
        past = _log_int(rng, 1, max(2, min(8000, 64 * 8000 * 8 * 128 // (4 * b * kvh * d))))
    elif rng.random() < 0.6:  # one token
        b, s = _log_int(rng, 1, 64), 1
        past = _log_int(rng, 1, max(2, min(40000, 64 * 6000 * 8 * 128 // (b * kvh * d))))
    else:  # a prompt, or a chunk of one
        b, s = _log_int(rng, 1, 8), _log_int(rng, 2, 2048)
        past = rng.choice((0, rng.randrange(0, 2000)))
        while b * c["h"] * d * s * (past + s) > 4 * 16 * 128 * 2048 * 2048:
            b, s, past = max(1, b // 2), max(2, s * 3 // 4), past // 2
    return dict(c, b=b, s=s, past=past, cap=past + s + rng.randrange(0, 100))


def _pasts(c):
    """Cached positions of each sequence: all the same, or from `past` down to half of it."""
    return [c["past"] - ((i * c["past"]) // (2 * c["b"]) if c["ragged"] else 0) for i in range(c["b"])]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _random_cache(gen, c):
    """Codes and scales of a cache as earlier calls left it: rows of normal values, some channels larger."""
    b, kvh, cap, d = c["b"], c["kvh"], c["cap"], c["d"]
    codes, scales = [], []
    for _ in range(2):
        chan = 0.5 + torch.rand((kvh, 1, d), generator=gen, device="cuda")
        q = torch.empty((b, kvh, cap, d), device="cuda", dtype=torch.int8 if c["kv"] == "int8" else torch.uint8)
        s = torch.empty((b, kvh, cap), device="cuda")
        for i in range(b):
            x = torch.randn((kvh, cap, d), generator=gen, device="cuda") * chan
            a = x.abs().amax(-1, keepdim=True)
            if c["kv"] == "int8":
                t = a / 127.0
                q[i] = torch.round(x / t).clamp(-127, 127).to(torch.int8)
            else:
                t = a / 448.0
                q[i] = (x / t).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
            s[i] = t[..., 0]
        codes.append(q)
        scales.append(s)
    return codes[0], codes[1], scales[0], scales[1]


def _random_tree(c, seed):
    """A drafted tree per sequence: parents, ancestor bits (the node itself included), depths, an accepted path."""
    import random

    rng = random.Random(seed)
    n = c["s"]
    bits, depths, paths, counts = [], [], [], []
    for _ in range(c["b"]):
        parent = [-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, n)]
        bit, dep = [], []
        for i, p in enumerate(parent):
            bit.append((1 << i) | (bit[p] if p >= 0 else 0))
            dep.append(dep[p] + 1 if p >= 0 else 0)
        leaf = rng.randrange(n)
        path = [i for i in range(n) if bit[leaf] >> i & 1]
        bits.append([x - (1 << 64) if x >> 63 else x for x in bit])
        depths.append(dep)
        paths.append(path + [0] * (n - len(path)))
        counts.append(len(path))
    dev = dict(device="cuda")
    return (torch.tensor(bits, dtype=torch.int64, **dev), torch.tensor(depths, dtype=torch.int32, **dev),
            torch.tensor(paths, dtype=torch.int32, **dev), torch.tensor(counts, dtype=torch.int32, **dev))


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st = {"case": c}
    f32 = dict(device="cuda", dtype=torch.float32)
    if c["op"] == "logprobs":
        rows, v, k = c["rows"], c["v"], c["k"]
        x = torch.randn((rows, c["ld"]), generator=gen, device="cuda") * 2.5
        # a few likely tokens a row, as a trained model gives
        hot = torch.randint(0, v, (rows, 8), generator=gen, device="cuda")
        x.scatter_add_(1, hot, 12 * torch.rand((rows, 8), generator=gen, device="cuda"))
        if c["banned"]:
            ban = torch.randperm(v, generator=gen, device="cuda")[: v // 64]
            x[:, ban] = -math.inf
        pick = torch.randint(0, v, (rows,), generator=gen, device="cuda")
        likely = torch.rand((rows,), generator=gen, device="cuda") < 0.7
        st.update(x=x, ids=torch.where(likely, hot[:, 0], pick), lp=torch.empty(rows, **f32),
                  ent=torch.empty(rows, **f32), top=torch.empty((rows, k), device="cuda", dtype=torch.int64),
                  top_lp=torch.empty((rows, k), **f32))
    else:
        b, s, kvh, d, cap = c["b"], c["s"], c["kvh"], c["d"], c["cap"]
        h = c.get("h", 0)
        # one packed q | k | v projection row per token
        st["rows"] = torch.randn((b * s, (h + 2 * kvh) * d), generator=gen, device="cuda") * 1.5
        st["codes"] = _random_cache(gen, c)
        st["past"] = torch.tensor(_pasts(c), dtype=torch.int32, device="cuda")
        st["gain"] = (1.0 + 0.2 * torch.randn((h + kvh, d), generator=gen, device="cuda")) if c["norm"] else None
        if c["rot"]:
            half = c["rot"] // 2
            inv = 1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
            ang = torch.arange(cap, device="cuda", dtype=torch.float64)[:, None] * inv
            st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        if c["op"] == "tree":
            st["bits"], st["depth"], st["path"], st["count"] = _random_tree(c, seed)
        if h:
            st["out"] = torch.empty((b, s, h * d), device="cuda",
                                    dtype=torch.float32 if c["out"] == "f32" else torch.float16)
        st["k_val"], st["v_val"] = torch.empty((b, kvh, s, d), **f32), torch.empty((b, kvh, s, d), **f32)
    if own:
        _bind(st)
    return st


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------
_CTX = []


def _bind(st):
    """The context and the argument lists a user's program keeps for its buffers."""
    import ctypes

    import onnx_runtime_dart_b200 as b2m
    from onnx_runtime_dart_b200 import _native as N

    if not _CTX:
        _CTX.append(b2m.Context(torch.cuda.current_device()))
    ctx, c = _CTX[0], st["case"]
    lib, hd = ctx.lib, ctx.handle

    def p(t, off=0):
        return None if t is None else ctypes.c_void_p(t.data_ptr() + off)

    st["calls"] = calls = []
    st["ctx"] = ctx
    if c["op"] == "logprobs":
        k = c["k"]
        calls.append((lib.b2m_logprobs_dev,
                      (hd, p(st["x"]), c["ld"], p(st["ids"]), c["rows"], c["v"], p(st["lp"]), p(st["ent"]), k,
                       p(st["top"]) if k else None, p(st["top_lp"]) if k else None)))
        return
    b, s, kvh, d, h = c["b"], c["s"], c["kvh"], c["d"], c.get("h", 0)
    kc, vc, ks, vs = st["codes"]
    cache = N.Kv8Cache(kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(),
                       N.B2M_INT8 if c["kv"] == "int8" else N.B2M_FLOAT8E4M3FN, b, kvh, c["cap"], d)
    st["cache"] = cache
    cr = ctypes.byref(cache)
    rs = (h + 2 * kvh) * d
    q, k, v = p(st["rows"]), p(st["rows"], 4 * h * d), p(st["rows"], 4 * (h + kvh) * d)
    eps = ctypes.c_double(1e-6)
    rotary = (p(st["cos"]), p(st["sin"]), c["rot"] // 2, c["rot"], int(c["inter"])) if c["rot"] else \
        (None, None, 0, 0, 0)
    past = p(st["past"])
    if c["op"] == "write":
        calls.append((lib.b2m_kv8_append_dev, (hd, cr, k, v, rs, p(st["gain"]), eps, past, None, *rotary, s)))
    else:
        tree = (p(st["bits"]), p(st["depth"])) if c["op"] == "tree" else (None, None)
        outs = (p(st["out"]), None) if c["out"] == "f32" else (None, p(st["out"]))
        calls.append((lib.b2m_gqa_kv8_dev, (hd, cr, q, k, v, rs, rs, p(st["gain"]), eps, past, *tree, *rotary, *outs,
                                            s, h, ctypes.c_float(0.0))))
        if c["op"] == "tree":
            calls.append((lib.b2m_kv8_keep_dev, (hd, cr, 1, past, p(st["path"]), p(st["count"]), s)))
    calls.append((lib.b2m_kv8_read_dev, (hd, cr, past, s, p(st["k_val"]), p(st["v_val"]))))


def _run_own(st):
    from onnx_runtime_dart_b200 import _native as N
    from onnx_runtime_dart_b200.runtime import use_torch_stream

    use_torch_stream(st["ctx"])
    for fn, args in st["calls"]:
        N.check(fn(*args))
    if st["case"]["op"] == "logprobs":
        return {"logprob": st["lp"], "entropy": st["ent"], "top_ids": st["top"], "top_logprobs": st["top_lp"]}
    r = {"k": st["k_val"], "v": st["v_val"]}
    if "out" in st:
        r["out"] = st["out"]
    return r


# ---------------------------------------------------------------------------
# Plain form
# ---------------------------------------------------------------------------
def _rotate(x, cos, sin, rot, inter):
    """Rotary of the first `rot` values of x[..., d]; cos / sin broadcast to x[..., :rot / 2]."""
    if not rot:
        return x
    y = x.clone()
    if inter:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2] = a * cos - b * sin
        y[..., 1:rot:2] = b * cos + a * sin
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2:rot]
        y[..., : rot // 2] = a * cos - b * sin
        y[..., rot // 2:rot] = b * cos + a * sin
    return y


def _head_norm(x, gain):
    return x if gain is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * gain


def _round_e4m3(x):
    """Nearest e4m3 value, ties to even, of float64 values with |x| <= 448."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), torch.clamp(e - 4, min=-9))
    return torch.round(x / step) * step


def _quantise(x, kv):
    """Codes (as stored) and scales of float64 rows."""
    top = 127.0 if kv == "int8" else 448.0
    scale = (x.abs().amax(-1, keepdim=True) / top).float()
    t = (x / scale.double()).clamp(-top, top)
    t = torch.where(scale == 0, torch.zeros_like(t), t)
    if kv == "int8":
        return torch.round(t).to(torch.int8), scale[..., 0]
    return _round_e4m3(t).to(torch.float8_e4m3fn).view(torch.uint8), scale[..., 0]


def _values(codes, scale, kv):
    x = codes.float() if kv == "int8" else codes.view(torch.float8_e4m3fn).float()
    return x * scale[..., None]


def _positions(st):
    """Cache slot and rotary position of every new token, [b][s]."""
    c = st["case"]
    t = torch.arange(c["s"], device="cuda")
    past = st["past"].long()[:, None]
    return past + t, past + (st["depth"].long() if c["op"] == "tree" else t)


def _append(st):
    """Quantises the call's keys and values into the cache; float64, so that a value next to a border rounds rightly."""
    c = st["case"]
    b, s, kvh, d, h = c["b"], c["s"], c["kvh"], c["d"], c.get("h", 0)
    rows = st["rows"].view(b, s, h + 2 * kvh, d)
    slot, pos = _positions(st)
    k = _head_norm(rows[:, :, h:h + kvh].double(), None if st["gain"] is None else st["gain"][h:].double())
    if c["rot"]:
        k = _rotate(k, st["cos"].double()[pos][:, :, None], st["sin"].double()[pos][:, :, None], c["rot"], c["inter"])
    at = torch.arange(b, device="cuda")[:, None]
    for x, codes, scale in ((k, st["codes"][0], st["codes"][2]), (rows[:, :, h + kvh:].double(), st["codes"][1],
                                                                   st["codes"][3])):
        q, sc = _quantise(x, c["kv"])
        codes[at, :, slot] = q
        scale[at, :, slot] = sc


def _read(st):
    kc, vc, ks, vs = st["codes"]
    at = torch.arange(st["case"]["b"], device="cuda")[:, None]
    slot, _ = _positions(st)
    kv = st["case"]["kv"]
    return {"k": _values(kc[at, :, slot], ks[at, :, slot], kv).transpose(1, 2).contiguous(),
            "v": _values(vc[at, :, slot], vs[at, :, slot], kv).transpose(1, 2).contiguous()}


def _visible(st, total):
    """[b][s][total]: which keys each new token sees."""
    c = st["case"]
    j = torch.arange(total, device="cuda")
    past = st["past"].long()[:, None, None]
    if c["op"] != "tree":
        return j <= past + torch.arange(c["s"], device="cuda")[:, None]
    node = (j - past).clamp(0, c["s"] - 1)
    bit = (st["bits"][:, :, None] >> node) & 1
    return (j < past) | ((j < past + c["s"]) & (bit == 1))


def _attend(st):
    c = st["case"]
    b, s, kvh, d, h = c["b"], c["s"], c["kvh"], c["d"], c["h"]
    g = h // kvh
    total = c["past"] + s
    kc, vc, ks, vs = st["codes"]
    keys = _values(kc[:, :, :total], ks[:, :, :total], c["kv"])
    vals = _values(vc[:, :, :total], vs[:, :, :total], c["kv"])
    q = _head_norm(st["rows"].view(b, s, h + 2 * kvh, d)[:, :, :h], None if st["gain"] is None else st["gain"][:h])
    if c["rot"]:
        pos = _positions(st)[1]
        q = _rotate(q, st["cos"][pos][:, :, None], st["sin"][pos][:, :, None], c["rot"], c["inter"])
    q = q.view(b, s, kvh, g, d).permute(0, 2, 3, 1, 4).reshape(b, kvh, g * s, d)
    x = (q @ keys.transpose(2, 3)) * d ** -0.5
    seen = _visible(st, total)[:, None, None]
    x = x.view(b, kvh, g, s, total).masked_fill_(~seen, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    norm = x.sum(-1, keepdim=True)
    o = (x.view(b, kvh, g * s, total) @ vals).view(b, kvh, g, s, d) / norm
    return o.permute(0, 3, 1, 2, 4).reshape(b, s, h * d).to(st["out"].dtype)


def _keep(st):
    """Rows past + path[j] move to past + j for j < count."""
    c = st["case"]
    past = st["past"].long()[:, None]
    j = torch.arange(c["s"], device="cuda")[None]
    src = past + torch.where(j < st["count"].long()[:, None], st["path"].long(), j)
    at = torch.arange(c["b"], device="cuda")[:, None]
    for t in st["codes"]:
        t[at, :, past + j] = t[at, :, src]


def _logprobs(st):
    c = st["case"]
    x = st["x"][:, : c["v"]]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    # ln of the sum as log1p of what stands beside the maximum, which a confident row would lose in 1 + z
    z = torch.log1p(e.double().sum(-1, keepdim=True) - 1.0).float()
    lp = (x - m) - z
    p = torch.exp(lp)
    ent = torch.where(p > 0, -p * lp, torch.zeros_like(p)).sum(-1)
    top_ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, : c["k"]]
    return {"logprob": lp.gather(1, st["ids"][:, None])[:, 0], "entropy": ent, "top_ids": top_ids,
            "top_logprobs": lp.gather(1, top_ids)}


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "logprobs":
        return _logprobs(state)
    _append(state)
    r = {}
    if op != "write":
        r["out"] = _attend(state)
    if op == "tree":
        _keep(state)
    return dict(r, **_read(state))


# ---------------------------------------------------------------------------
# Work and the 64-bit values
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "logprobs":
        n = c["rows"] * c["v"]
        return {"bytes": 4 * n + c["rows"] * (16 + 12 * c["k"]), "flops": 6 * n}
    new = c["b"] * c["s"] * c["kvh"]  # rows of keys, and as many of values
    rows = 2 * new * (4 * c["d"] + c["d"] + 4)  # read in fp32, written as codes and scales
    back = 2 * new * (c["d"] + 4 + 4 * c["d"])
    if c["op"] == "write":
        return {"bytes": rows + back, "flops": 2 * new * 10 * c["d"]}
    pasts = _pasts(c)
    cached = sum(pasts) * c["kvh"] * 2 * (c["d"] + 4)
    qo = c["b"] * c["s"] * c["h"] * c["d"] * (4 + (4 if c["out"] == "f32" else 2))
    seen = sum(c["s"] * p + (c["s"] * (c["s"] + 1)) // 2 for p in pasts)
    moved = 2 * 2 * new * (c["d"] + 4) if c["op"] == "tree" else 0
    return {"bytes": cached + rows + back + qo + moved, "flops": 4 * c["h"] * c["d"] * seen}


def _exact_codes(x, kv):
    """The values that the codes of float64 rows stand for, and the code values and fp32 scales."""
    top = {"int8": 127.0, "e4m3": 448.0}[kv]
    scale = (torch.max(torch.abs(x), -1)[0] / top).to(torch.float32).to(torch.float64)[..., None]
    y = torch.where(scale > 0, x / torch.where(scale > 0, scale, torch.ones_like(scale)), torch.zeros_like(x))
    y = torch.clamp(y, -top, top)
    if kv == "int8":
        code = torch.round(y)
    else:  # three bits behind the leading one, steps of 2^-9 below 2^-6
        mag = torch.abs(y)
        expo = torch.floor(torch.log2(torch.clamp(mag, min=2.0 ** -20)))
        expo = torch.where(torch.pow(2.0, expo + 1) <= mag, expo + 1, torch.where(torch.pow(2.0, expo) > mag, expo - 1,
                                                                                 expo))
        quantum = torch.pow(torch.full_like(mag, 2.0), torch.clamp(expo, min=-6.0) - 3.0)
        code = torch.sign(y) * quantum * torch.round(mag / quantum)
    return code * scale


def _exact_rope(x, pos, st):
    """x[s][heads][d] rotated by the angles of positions pos[s] (tables as given), pair by pair."""
    rot, inter = st["case"]["rot"], st["case"]["inter"]
    if rot == 0:
        return x
    half = rot // 2
    lo = torch.arange(half, device=x.device)
    i0, i1 = (2 * lo, 2 * lo + 1) if inter else (lo, lo + half)
    co, si = st["cos"][pos].double()[:, None, :], st["sin"][pos].double()[:, None, :]
    y = x.clone()
    y[..., i0] = co * x[..., i0] - si * x[..., i1]
    y[..., i1] = si * x[..., i0] + co * x[..., i1]
    return y


def _exact_norm(x, gain):
    if gain is None:
        return x
    rms = torch.sqrt(torch.sum(x * x, -1, keepdim=True) / x.shape[-1] + 1e-6)
    return x / rms * gain.double()


def _exact_logprobs(st):
    c = st["case"]
    parts = []
    for r in range(0, c["rows"], 64):
        x = st["x"][r:r + 64, : c["v"]].double()
        lse = torch.logsumexp(x, 1, keepdim=True)
        lp = x - lse
        ent = -(torch.exp(lp) * torch.where(torch.isinf(lp), torch.zeros_like(lp), lp)).sum(1)
        # descending by value, then ascending by index: the k largest of (value, -index)
        idx = torch.argsort(-x, dim=1, stable=True)[:, : c["k"]]
        parts.append((torch.take_along_dim(lp, st["ids"][r:r + 64, None], 1)[:, 0], ent, idx,
                      torch.take_along_dim(lp, idx, 1)))
    return {n: torch.cat([p[i] for p in parts]) for i, n in enumerate(("logprob", "entropy", "top_ids",
                                                                       "top_logprobs"))}


def exact(case, seed):
    st = prepare(case, seed)
    c = st["case"]
    if c["op"] == "logprobs":
        return _exact_logprobs(st)
    b, s, kvh, d, h = c["b"], c["s"], c["kvh"], c["d"], c.get("h", 0)
    if c["op"] != "write" and 4 * h * d * b * s * (c["past"] + s) > 4e12:
        return None
    kc, vc, ks, vs = st["codes"]
    outs, kk, vv = [], [], []
    for i in range(b):
        past = int(st["past"][i])
        rows = st["rows"][i * s:(i + 1) * s].double().view(s, h + 2 * kvh, d)
        pos = past + (st["depth"][i].long() if c["op"] == "tree" else torch.arange(s, device="cuda"))
        gq, gk = (None, None) if st["gain"] is None else (st["gain"][:h], st["gain"][h:])
        nk = _exact_codes(_exact_rope(_exact_norm(rows[:, h:h + kvh], gk), pos, st), c["kv"]).transpose(0, 1)
        nv = _exact_codes(rows[:, h + kvh:], c["kv"]).transpose(0, 1)
        if h:
            q = _exact_rope(_exact_norm(rows[:, :h], gq), pos, st)

            def old(codes, scale):
                t = codes[i, :, :past]
                t = t.double() if c["kv"] == "int8" else t.view(torch.float8_e4m3fn).double()
                return t * scale[i, :, :past].double()[..., None]

            keys, vals = torch.cat([old(kc, ks), nk], 1), torch.cat([old(vc, vs), nv], 1)
            if c["op"] == "tree":
                own_rows = torch.stack([(st["bits"][i] >> j) & 1 for j in range(s)], 1) == 1
            else:
                own_rows = torch.ones((s, s), dtype=torch.bool, device="cuda").tril()
            hide = torch.cat([torch.zeros((s, past), dtype=torch.bool, device="cuda"), ~own_rows], 1)
            o = torch.empty((s, h, d), dtype=torch.float64, device="cuda")
            for n in range(h):
                a = q[:, n] @ keys[n // (h // kvh)].T / math.sqrt(d)
                o[:, n] = torch.softmax(a.masked_fill(hide, -math.inf), 1) @ vals[n // (h // kvh)]
            outs.append(o.view(s, h * d))
        if c["op"] == "tree":
            n = int(st["count"][i])
            src = torch.cat([st["path"][i, :n].long(), torch.arange(n, s, device="cuda")])
            nk, nv = nk[:, src], nv[:, src]
        kk.append(nk)
        vv.append(nv)
    r = {"k": torch.stack(kk), "v": torch.stack(vv)}
    if outs:
        r["out"] = torch.stack(outs)
    return r
