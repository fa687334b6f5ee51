"""GPU tests of the 8-bit KV cache: quantised append and read-back, attention
over the cache (single tokens, chunks, prompts, drafted trees) and the move of
accepted rows, each against a plain implementation in 64 bits.

Tolerances are worked out from the formats (a rounding is off by at most half
a step: 2^-24 in fp32, 2^-11 in f16) in `_bound`, from each case's own sizes
and inputs. Codes and scales are held to equality."""
import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import onnx_runtime_dart_b200 as b2m  # noqa: E402
from onnx_runtime_dart_b200 import _native as N  # noqa: E402
from onnx_runtime_dart_b200.runtime import use_torch_stream  # noqa: E402

TYPES = {"int8": N.B2M_INT8, "e4m3": N.B2M_FLOAT8E4M3FN}
TOP = {"int8": 127.0, "e4m3": 448.0}


@pytest.fixture(scope="module")
def ctx():
    c = b2m.Context(0)
    use_torch_stream(c)
    yield c
    c.close()


def _p(t, off=0):
    return None if t is None else ctypes.c_void_p(t.data_ptr() + off)


def _round_e4m3(x):
    """Nearest e4m3 value of float64 |x| <= 448, ties to even."""
    _, e = torch.frexp(x)
    q = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return torch.round(x / q) * q


def _codes_of(x, kv):
    """(value of each code before its scale, fp32 scale) of float64 rows."""
    s = (x.abs().amax(-1) / TOP[kv]).float()
    t = torch.where(s[..., None] > 0, x / s[..., None].double(), torch.zeros_like(x)).clamp(-TOP[kv], TOP[kv])
    return (torch.round(t) if kv == "int8" else _round_e4m3(t)), s


def _decode(codes, kv):
    return codes.view(torch.int8).double() if kv == "int8" else codes.view(torch.float8_e4m3fn).double()


def _rope64(x, pos, cos, sin, rot, inter):
    """x [..., tokens, heads, d] float64 at positions pos [..., tokens]."""
    if not rot:
        return x
    y = x.clone()
    pos = pos.clamp(0, cos.shape[0] - 1)  # tokens that are refused anyway
    c, s = cos.double()[pos][..., None, : rot // 2], sin.double()[pos][..., None, : rot // 2]
    i = torch.arange(rot // 2, device=x.device)
    i0, i1 = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i1] * c + x[..., i0] * s
    return y


def _norm64(x, gain, eps=1e-6):
    return x if gain is None else x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * gain.double()


class Problem:
    """Random inputs of one call, the cache before it, and the 64-bit answer."""

    def __init__(self, kv, b, s, h, kvh, d, cap, pasts, rot=0, inter=False, norm=False, tree=None, half=None, seed=0,
                 pad=0, scale=0.0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed * 7919 + b * 31 + s * 7 + d)
        rnd = lambda *sh: torch.randn(sh, generator=g, device="cuda")  # noqa: E731
        self.kv, self.b, self.s, self.h, self.kvh, self.d, self.cap = kv, b, s, h, kvh, d, cap
        self.rot, self.inter, self.scale = rot, inter, scale
        self.rs = (h + 2 * kvh) * d + pad
        self.rows = rnd(b * s, self.rs) * 1.5
        self.past = torch.tensor(pasts, dtype=torch.int32, device="cuda")
        self.gain = 1 + 0.2 * rnd(h + kvh, d) if norm else None
        self.half = half or max(1, rot // 2)
        ang = torch.arange(cap, device="cuda", dtype=torch.float64)[:, None] * 1e4 ** (
            -torch.arange(self.half, device="cuda", dtype=torch.float64) / self.half)
        self.cos, self.sin = ang.cos().float(), ang.sin().float()
        # positions past the sequence hold noise: any byte, NaN scales
        self.codes = [torch.randint(0, 256, (b, kvh, cap, d), generator=g, device="cuda", dtype=torch.uint8)
                      for _ in range(2)]
        self.scales = [torch.full((b, kvh, cap), float("nan"), device="cuda") for _ in range(2)]
        for side in range(2):
            for i, p in enumerate(pasts):
                x = rnd(kvh, max(0, min(p, cap)), d) * (0.5 + torch.rand((kvh, 1, d), generator=g, device="cuda"))
                q, sc = _codes_of(x.double(), kv)
                self.codes[side][i, :, : x.shape[1]] = (q.to(torch.int8) if kv == "int8" else
                                                         q.to(torch.float8_e4m3fn)).view(torch.uint8)
                self.scales[side][i, :, : x.shape[1]] = sc
        self.tree = self.depth = None
        if tree is not None:
            bits, depth = tree
            self.bits = bits
            self.tree = torch.tensor([[x - (1 << 64) if x >> 63 else x for x in r] for r in bits], dtype=torch.int64,
                                     device="cuda")
            self.depth = torch.tensor(depth, dtype=torch.int32, device="cuda")
        self.cache = N.Kv8Cache(self.codes[0].data_ptr(), self.codes[1].data_ptr(), self.scales[0].data_ptr(),
                                self.scales[1].data_ptr(), TYPES[kv], b, kvh, cap, d)

    def rotary(self):
        return (_p(self.cos), _p(self.sin), self.half, self.rot, int(self.inter)) if self.rot else \
            (None, None, 0, 0, 0)

    def append(self, ctx):
        o = 4 * self.h * self.d
        gain = None if self.gain is None else _p(self.gain, o)
        N.check(ctx.lib.b2m_kv8_append_dev(ctx.handle, ctypes.byref(self.cache), _p(self.rows, o),
                                           _p(self.rows, o + 4 * self.kvh * self.d), self.rs, gain, 1e-6,
                                           _p(self.past), _p(self.depth), *self.rotary(), self.s))

    def attend(self, ctx, out=True, out16=False):
        o = 4 * self.h * self.d
        n = self.h * self.d
        self.out = torch.full((self.b, self.s, n), 7.0, device="cuda") if out else None
        self.out16 = torch.full((self.b, self.s, n), 7.0, device="cuda", dtype=torch.float16) if out16 else None
        N.check(ctx.lib.b2m_gqa_kv8_dev(ctx.handle, ctypes.byref(self.cache), _p(self.rows), _p(self.rows, o),
                                        _p(self.rows, o + 4 * self.kvh * self.d), self.rs, self.rs, _p(self.gain), 1e-6,
                                        _p(self.past), _p(self.tree), _p(self.depth), *self.rotary(), _p(self.out),
                                        _p(self.out16), self.s, self.h, ctypes.c_float(self.scale)))

    def read(self, ctx, start, n):
        k = torch.full((self.b, self.kvh, n, self.d), 7.0, device="cuda")
        v = k.clone()
        N.check(ctx.lib.b2m_kv8_read_dev(ctx.handle, ctypes.byref(self.cache), _p(start), n, _p(k), _p(v)))
        return k, v

    def positions(self):
        t = torch.arange(self.s, device="cuda")
        return self.past.long()[:, None] + (self.depth.long() if self.depth is not None else t)

    def split(self):
        r = self.rows[:, : (self.h + 2 * self.kvh) * self.d].double().view(self.b, self.s, self.h + 2 * self.kvh, self.d)
        return r[:, :, : self.h], r[:, :, self.h: self.h + self.kvh], r[:, :, self.h + self.kvh:]

    def new_rows(self):
        """Code values and scales [b][kvh][s] of the call's keys and values."""
        _, k, v = self.split()
        k = _rope64(_norm64(k, None if self.gain is None else self.gain[self.h:]), self.positions(), self.cos, self.sin,
                    self.rot, self.inter)
        return [tuple(t.transpose(1, 2) for t in _codes_of(x, self.kv)) for x in (k, v)]

    def answer(self):
        """64-bit attention over what the cache holds now, and a bound per output on the error of fp32 rows."""
        q = _rope64(_norm64(self.split()[0], None if self.gain is None else self.gain[: self.h]), self.positions(),
                    self.cos, self.sin, self.rot, self.inter)
        scale = self.scale if self.scale > 0 else 1 / math.sqrt(self.d)
        want = torch.zeros((self.b, self.s, self.h, self.d), dtype=torch.float64, device="cuda")
        mass, spread = want.clone(), want.clone()
        for i in range(self.b):
            n = min(self.cap, int(self.past[i]) + self.s)
            ks, vs = (_decode(self.codes[x][i, :, :n], self.kv) * self.scales[x][i, :, :n].double()[..., None]
                      for x in range(2))
            j = torch.arange(n, device="cuda")
            t = torch.arange(self.s, device="cuda")[:, None]
            if self.tree is None:
                seen = j <= int(self.past[i]) + t
            else:
                node = (j - int(self.past[i])).clamp(0, 63)
                seen = (j < int(self.past[i])) | (((self.tree[i][:, None] >> node) & 1) == 1)
            for hh in range(self.h):
                kk, vv = ks[hh // (self.h // self.kvh)], vs[hh // (self.h // self.kvh)]
                x = (q[i, :, hh] @ kk.T * scale).masked_fill(~seen, -math.inf)
                w = torch.softmax(x, -1)
                w = torch.where(seen.any(-1, keepdim=True), w, torch.zeros_like(w))
                vis = torch.where(seen.any(0)[:, None], vv, torch.zeros_like(vv))
                want[i, :, hh] = w @ vis
                mass[i, :, hh] = w @ vis.abs()
                kabs = torch.where(seen.any(0)[:, None], kk, torch.zeros_like(kk)).abs()
                spread[i, :, hh] = (q[i, :, hh].abs() @ kabs.T * scale).amax(-1, keepdim=True)
        # Score error ds: 64 roundings of at most 2^-24 of the score's mass (norm, rotary, scales and up to
        # 2 * 256 / 16 tensor-core additions, or 8 + 5 additions on the CUDA cores; operands split in two f16 terms
        # are off by 2^-22). A weight e^(x - m) is then off by 2 ds, the exponential by 2^-22 plus 2^-23 |x - m| with
        # |x - m| <= 24 where the weight matters (2^-18 together), the sums over n keys by (n / 4 + 64) 2^-24.
        f32 = mass * (2 * spread * 64 * 2.0 ** -24 + 2.0 ** -18 + (self.cap / 4 + 64) * 2.0 ** -24)
        # f16-only output: q and the weights rounded once (2^-11 each), and the output itself.
        f16 = f32 + mass * (2 * spread * 2.0 ** -11 + 2 * 2.0 ** -11) + want.abs() * 2.0 ** -11 + 2.0 ** -25
        shape = (self.b, self.s, self.h * self.d)
        return want.view(shape), f32.view(shape) + 1e-30, f16.view(shape)


def _check(p, ctx, f16_too=True):
    p.attend(ctx, out=True, out16=False)
    want, tol, tol16 = p.answer()
    err = (p.out.double() - want).abs()
    assert bool((err <= tol).all()), f"fp32 rows: {float((err / tol).max()):.2f} of the bound"
    if f16_too and p.h * p.d % 8 == 0:
        full = p.out.clone()
        p.attend(ctx, out=False, out16=True)
        err = (p.out16.double() - want).abs()
        assert bool((err <= tol16).all()), f"f16 rows: {float((err / tol16).max()):.2f} of the bound"
        p.attend(ctx, out=True, out16=True)
        assert torch.equal(p.out, full)
        assert torch.equal(p.out16, p.out.half())


def _ragged(b, hi, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [hi if i == 0 else int(torch.randint(0, hi + 1, (1,), generator=g)) for i in range(b)]


# ---------------------------------------------------------------------------
# Append and read-back
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("b,s,kvh,d,rot,inter,norm,pad", [
    (1, 1, 1, 128, 128, False, True, 0),
    (3, 5, 8, 128, 128, False, False, 0),
    (2, 33, 4, 64, 32, True, True, 4),
    (2, 7, 2, 256, 256, False, True, 0),
    (2, 3, 3, 80, 40, False, False, 3),   # rows that are not 16-byte aligned
    (1, 4, 2, 96, 0, False, True, 0),
    (2, 2, 1, 7, 2, True, False, 1),      # a head of seven: codes byte by byte
    (1, 300, 8, 128, 64, True, False, 0),
    (2, 9, 2, 32, 32, False, True, 0),
])
def test_append_and_read(ctx, kv, b, s, kvh, d, rot, inter, norm, pad):
    """Codes, scales and read-back values equal to the 64-bit definition; every other row as it was."""
    p = Problem(kv, b, s, 2 * kvh, kvh, d, 340, _ragged(b, 340 - s, d), rot, inter, norm, half=max(1, d // 2), pad=pad)
    before = [t.clone() for t in p.codes + p.scales]
    p.append(ctx)
    for side, (val, sc) in enumerate(p.new_rows()):
        for i in range(b):
            lo = int(p.past[i])
            assert torch.equal(p.scales[side][i, :, lo:lo + s], sc[i])
            assert torch.equal(_decode(p.codes[side][i, :, lo:lo + s], kv), val[i])
            for now, was in ((p.codes[side], before[side]), (p.scales[side], before[2 + side])):
                now, was = now.view(torch.uint8), was.view(torch.uint8)  # bytes: the noise holds NaN
                w = now.shape[-1] // (1 if now.dim() == 4 else 340)
                now, was = now.view(b, kvh, 340, w), was.view(b, kvh, 340, w)
                assert torch.equal(now[i, :, :lo], was[i, :, :lo]) and torch.equal(now[i, :, lo + s:], was[i, :, lo + s:])
    k, v = p.read(ctx, p.past, s)
    for got, (val, sc) in zip((k, v), p.new_rows()):
        assert torch.equal(got, (val * sc.double()[..., None]).float())
    k0, _ = p.read(ctx, None, 2)  # start NULL: from position 0
    want = (_decode(p.codes[0][:, :, :2], kv) * p.scales[0][:, :, :2].double()[..., None]).float()
    assert torch.equal(torch.nan_to_num(k0), torch.nan_to_num(want))


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
def test_append_borders(ctx, kv):
    """Rows whose values lie on rounding borders (ties to even), all zeros, one huge value among tiny ones, the
    smallest subnormals, and rows with NaN or infinity."""
    d = 64
    p = Problem(kv, 1, 8, 1, 1, d, 16, [0])
    r = p.rows.view(8, 3, d)
    ties = torch.arange(d, device="cuda") - 31.5
    r[0, 1:] = torch.where(ties.abs() > 31, torch.full_like(ties, TOP[kv]), ties)  # scale 1: halves are ties
    r[1, 1:] = 0
    r[2, 1:] = 1e-30
    r[2, 1:, 5] = 3e38
    r[3, 1:] = 1.4e-45
    r[4, 1, 3] = float("nan")
    r[5, 2, 60] = -math.inf
    r[6, 1:] = torch.where(ties.abs() > 31, torch.full_like(ties, 3 * TOP[kv]), ties * 3)  # scale 3
    r[7, 1:] = -0.0
    p.append(ctx)
    k, v = p.read(ctx, None, 8)
    want = p.new_rows()
    for side, got in ((0, k), (1, v)):
        for t in range(8):
            if (t, side) in ((4, 0), (5, 1)):
                assert bool(got[0, 0, t].isnan().all()) and bool(p.scales[side][0, 0, t].isnan())
                assert not bool(p.codes[side][0, 0, t].any())
                continue
            val, sc = want[side][0][0, 0, t], want[side][1][0, 0, t]
            assert torch.equal(p.scales[side][0, 0, t], sc), (side, t)
            assert torch.equal(_decode(p.codes[side][0, 0, t], kv), val), (side, t)
            assert torch.equal(got[0, 0, t], (val * sc.double()).float()), (side, t)


def test_append_capacity_and_positions(ctx):
    """A full sequence, a negative past and a bad depth: an error each, nothing written where it must not be."""
    p = Problem("int8", 3, 4, 2, 2, 32, 16, [14, 3, 0], rot=32, half=16)
    before = [t.clone() for t in p.codes]
    p.append(ctx)
    with pytest.raises(N.ArgumentError, match="capacity"):
        ctx.synchronize()
    val, _ = p.new_rows()[1]
    assert torch.equal(_decode(p.codes[1][0, :, 14:16], "int8"), val[0][:, :2])  # the two that fit
    assert torch.equal(_decode(p.codes[1][1, :, 3:7], "int8"), val[1])
    ctx.synchronize()
    p.past[1] = -1
    p.codes[0].copy_(before[0])
    p.append(ctx)
    with pytest.raises(N.ArgumentError):
        ctx.synchronize()
    assert torch.equal(p.codes[0][1], before[0][1])
    p.past[:] = 2
    p.depth = torch.tensor([[0, 1, 2, 4]] * 3, dtype=torch.int32, device="cuda")
    p.codes[0].copy_(before[0])
    p.append(ctx)
    with pytest.raises(N.ArgumentError, match="index"):
        ctx.synchronize()
    assert torch.equal(p.codes[0][:, :, 5], before[0][:, :, 5])
    assert not torch.equal(p.codes[0][:, :, 4], before[0][:, :, 4])


def test_read_outside(ctx):
    p = Problem("e4m3", 2, 1, 1, 1, 64, 8, [8, 8])
    start = torch.tensor([6, -1], dtype=torch.int32, device="cuda")
    k, _ = p.read(ctx, start, 3)
    with pytest.raises(N.ArgumentError, match="index"):
        ctx.synchronize()
    assert bool((k[0, :, 2] == 7).all()) and bool((k[1, :, 0] == 7).all())
    assert not bool((k[0, :, :2] == 7).any())


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
STEPS = [  # b, h, kvh, d, cap, past, rot, inter, norm
    (1, 1, 1, 128, 8, 0, 0, False, False),          # one key: the token itself
    (1, 16, 8, 128, 700, 511, 128, False, True),
    (5, 16, 8, 128, 1100, 1040, 128, False, True),
    (64, 16, 8, 128, 130, 129, 128, False, False),
    (3, 32, 4, 128, 2100, 2050, 0, False, False),   # eight query heads a kv head
    (2, 12, 4, 64, 333, 301, 32, True, True),
    (2, 6, 2, 64, 90, 31, 64, False, False),
    (3, 5, 1, 32, 65, 63, 32, False, True),         # five query heads on one
    (2, 4, 4, 96, 80, 77, 96, False, False),
    (2, 8, 2, 256, 300, 290, 128, False, True),
    (2, 9, 3, 80, 120, 100, 40, False, True),
    (2, 24, 2, 128, 260, 255, 128, False, False),   # twelve query heads a kv head
    (2, 2, 2, 20, 40, 17, 20, True, False),         # a head dim of twenty
    (1, 3, 1, 7, 70, 64, 0, False, False),
]


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("b,h,kvh,d,cap,past,rot,inter,norm", STEPS)
def test_single_token(ctx, kv, b, h, kvh, d, cap, past, rot, inter, norm):
    _check(Problem(kv, b, 1, h, kvh, d, cap, _ragged(b, past, past), rot, inter, norm), ctx)


CHUNKS = [  # b, s, h, kvh, d, cap, past, rot, inter, norm
    (2, 2, 4, 2, 128, 40, 3, 128, False, False),
    (2, 8, 16, 8, 128, 300, 200, 128, False, True),
    (3, 5, 8, 2, 64, 100, 90, 64, True, True),
    (2, 16, 4, 4, 128, 64, 0, 0, False, False),      # from an empty cache
    (1, 65, 16, 8, 128, 200, 65, 128, False, True),  # one past a tile of 64 tokens
    (2, 129, 4, 2, 64, 140, 11, 64, False, False),
    (1, 300, 8, 4, 128, 700, 333, 128, False, True),
    (2, 64, 2, 2, 128, 64, 0, 128, False, False),    # fills the cache
    (2, 70, 6, 2, 128, 150, 60, 0, False, False),    # three query heads on each
    (1, 40, 8, 1, 96, 90, 13, 96, False, True),
    (1, 33, 4, 2, 256, 70, 20, 256, False, False),
    (1, 21, 4, 2, 80, 50, 9, 80, False, True),
    (1, 200, 12, 1, 128, 260, 50, 128, False, False),
    (1, 9, 3, 1, 32, 20, 2, 0, False, False),
    (25, 20, 8, 4, 64, 80, 50, 64, False, True),     # 40 rows of many kv heads
]


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("b,s,h,kvh,d,cap,past,rot,inter,norm", CHUNKS)
def test_chunk(ctx, kv, b, s, h, kvh, d, cap, past, rot, inter, norm):
    _check(Problem(kv, b, s, h, kvh, d, cap, _ragged(b, past, s), rot, inter, norm), ctx)


def _random_tree(b, n, seed, orphan=False):
    g = torch.Generator().manual_seed(seed)
    bits, depth = [], []
    for _ in range(b):
        bit, dep = [], []
        for i in range(n):
            par = -1 if i == 0 else int(torch.randint(max(0, i - 5), i, (1,), generator=g))
            bit.append((1 << i) | (bit[par] if par >= 0 else 0))
            dep.append(dep[par] + 1 if par >= 0 else 0)
        if orphan:
            bit[n // 2] = 0  # a token that sees no new token
        bits.append(bit)
        depth.append(dep)
    return bits, depth


TREES = [  # b, n, h, kvh, d, cap, past, rot, norm, orphan
    (2, 2, 16, 8, 128, 100, 50, 128, True, False),
    (3, 8, 16, 8, 128, 700, 600, 128, True, False),
    (2, 17, 8, 2, 64, 100, 70, 64, False, True),
    (2, 64, 16, 8, 128, 400, 300, 128, True, False),
    (1, 64, 4, 4, 128, 64, 0, 128, False, True),     # an empty cache: the orphan sees nothing
    (2, 33, 6, 2, 80, 60, 20, 80, False, False),
    (1, 40, 8, 1, 256, 100, 31, 0, False, True),
    (2, 5, 3, 1, 32, 12, 7, 32, False, False),
    (2, 12, 12, 4, 96, 90, 64, 96, True, True),
    (13, 24, 16, 8, 128, 100, 70, 128, True, True),  # 48 rows of many kv heads
]


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("b,n,h,kvh,d,cap,past,rot,norm,orphan", TREES)
def test_tree(ctx, kv, b, n, h, kvh, d, cap, past, rot, norm, orphan):
    pasts = [past] + [0 if orphan else past // 2] * (b - 1)
    p = Problem(kv, b, n, h, kvh, d, cap, pasts, rot, False, norm, tree=_random_tree(b, n, n, orphan))
    _check(p, ctx)
    if orphan:
        for i in range(b):
            if int(p.past[i]) == 0:
                assert not bool(p.out[i, n // 2].any())


def test_chain_tree_is_causal(ctx):
    """A tree that is a chain gives the causal call's rows."""
    n = 9
    bits = [[(1 << (i + 1)) - 1 for i in range(n)]] * 2
    args = ("int8", 2, n, 16, 8, 128, 300, [200, 7], 128, False, True)
    a, c = Problem(*args), Problem(*args, tree=(bits, [list(range(n))] * 2))
    a.attend(ctx)
    c.attend(ctx)
    assert torch.equal(a.out, c.out)
    for x, y in zip(a.codes + a.scales, c.codes + c.scales):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("s", [1, 6, 80])
def test_poisoned_row_only_reaches_who_sees_it(ctx, s):
    """A NaN key or value poisons exactly the tokens that see it; noise behind the sequence poisons nobody."""
    p = Problem("e4m3", 2, s, 4, 2, 128, 300, [150, 90])
    if s > 1:
        p.rows[s // 2, 4 * 128 + 3] = float("nan")  # kv head 0's key of token s // 2 of sequence 0
    else:
        p.scales[1][0, 0, 10] = float("nan")
    p.attend(ctx)
    o = p.out.view(2, s, 2, 2 * 128)
    first = s // 2 if s > 1 else 0
    assert bool(o[0, first:, 0].isnan().all())
    assert not bool(o[0, :first].isnan().any()) and not bool(o[0, :, 1].isnan().any()) and not bool(o[1].isnan().any())


def test_large_and_small_values(ctx):
    """Rows of very different magnitude (scales from 2^-60 to 2^60) keep their accuracy."""
    for e in (-60, -12, 12, 60):
        p = Problem("int8", 2, 1, 4, 2, 128, 200, [150, 33])
        p.scales[1].mul_(2.0 ** e)
        p.rows[:, (4 + 2) * 128:] *= 2.0 ** e
        _check(p, ctx, f16_too=abs(e) < 13)
    # one loud value row among quiet ones, queries large and keys small
    p = Problem("e4m3", 2, 3, 4, 2, 128, 200, [150, 33])
    p.scales[1][:, :, 20] *= 2.0 ** 20
    p.rows[:, : 4 * 128] *= 2.0 ** 30
    p.rows[:, 4 * 128: 6 * 128] *= 2.0 ** -30
    p.scales[0].mul_(2.0 ** -30)
    _check(p, ctx, f16_too=False)


def test_long_flat_row(ctx):
    """40,000 keys of nearly equal, small weight beside one dominant key: sums of tiny weights keep their share."""
    p = Problem("int8", 1, 1, 2, 1, 128, 40001, [40000])
    p.rows[0, : 2 * 128] = 0.02
    p.codes[0].fill_(0)
    p.codes[0][0, 0, 77] = 100
    p.scales[0].fill_(1.0)
    q = p.rows[0, :128].double()
    x = float((q * 100).sum()) / math.sqrt(128)
    p.scales[0][0, 0, 77] = 14.0 / x  # e^14 against 40,000 keys of e^0
    p.rows[0, 2 * 128: 3 * 128] = 0
    _check(p, ctx)


def test_exact_mode(ctx):
    """EXACT attention: fp32 kernel, and a sequence's rows do not depend on the batch around it."""
    ctx.set_attention_mode(N.MODE_EXACT)
    try:
        p = Problem("int8", 4, 1, 16, 8, 128, 300, [200, 7, 0, 150], 128, False, True)
        _check(p, ctx, f16_too=False)
        whole = p.out.clone()
        one = Problem("int8", 1, 1, 16, 8, 128, 300, [200], 128, False, True)
        one.rows.copy_(p.rows[:1])
        one.gain.copy_(p.gain)
        for x, y in zip(one.codes + one.scales, p.codes + p.scales):
            x.copy_(y[:1])
        one.attend(ctx)
        assert torch.equal(one.out[0], whole[0])
    finally:
        ctx.set_attention_mode(N.MODE_FAST)


def test_attend_capacity(ctx):
    """A token past the capacity raises the error; the others' rows are right."""
    p = Problem("int8", 2, 1, 4, 2, 128, 64, [64, 20])
    p.attend(ctx)
    with pytest.raises(N.ArgumentError, match="capacity"):
        ctx.synchronize()
    want, tol, _ = p.answer()
    assert bool(((p.out.double() - want).abs() <= tol)[1].all())
    ctx.synchronize()


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("s,d", [(1, 128), (5, 64), (40, 128)])
def test_keys_at_odd_strides(ctx, kv, s, d):
    """Keys and values in buffers of their own, unaligned and with an odd row stride: the packed rows' answers."""
    p = Problem(kv, 2, s, 8, 2, d, 160, [70, 33], d, False, True)
    nk = p.kvh * d
    bufs = []
    for side in range(2):
        o = (p.h + side * p.kvh) * d
        t = torch.full((2 * s * (nk + 3) + 1,), float("nan"), device="cuda")
        t[1:].view(2 * s, nk + 3)[:, :nk] = p.rows[:, o: o + nk]
        bufs.append(t)
    p.out = torch.full((2, s, 8 * d), 7.0, device="cuda")
    N.check(ctx.lib.b2m_gqa_kv8_dev(ctx.handle, ctypes.byref(p.cache), _p(p.rows), _p(bufs[0], 4), _p(bufs[1], 4), p.rs,
                                    nk + 3, _p(p.gain), 1e-6, _p(p.past), None, None, *p.rotary(), _p(p.out), None, s,
                                    p.h, ctypes.c_float(0.0)))
    ctx.synchronize()
    want, tol, _ = p.answer()
    assert bool(((p.out.double() - want).abs() <= tol).all())
    new = p.new_rows()
    for side in range(2):
        for i in range(2):
            at = int(p.past[i])
            assert torch.equal(_decode(p.codes[side][i, :, at: at + s], kv), new[side][0][i])
            assert torch.equal(p.scales[side][i, :, at: at + s], new[side][1][i].float())


@pytest.mark.parametrize("s,d,tree", [(1, 128, False), (6, 64, False), (40, 128, False), (40, 64, True), (3, 36, False)])
def test_positions_at_the_ends_of_int32(ctx, s, d, tree):
    """Positions far outside the cache: the error, no row written, the other sequence's rows right."""
    p = Problem("e4m3", 3, s, 4, 2, d, 128, [20, 20, 20], rot=32, half=16)
    if tree:
        p.depth = torch.arange(s, dtype=torch.int32, device="cuda").repeat(3, 1)
        p.tree = torch.full((3, s), 1, dtype=torch.int64, device="cuda")
    for bad, what in ((2**31 - 1, "capacity"), (-(2**31), "index")):
        p.past[:] = torch.tensor([20, bad, 20], dtype=torch.int32)
        was = [t[1].clone() for t in p.codes + p.scales]
        p.attend(ctx)
        with pytest.raises(N.ArgumentError, match=what):
            ctx.synchronize()
        assert all(torch.equal(t[1].view(torch.uint8), w.view(torch.uint8)) for t, w in zip(p.codes + p.scales, was))
        p.past[1] = 20
        want, tol, _ = p.answer()
        assert bool(((p.out.double() - want).abs() <= tol)[[0, 2]].all())


@pytest.mark.parametrize("b,s,h,kvh,d", [(3, 1, 16, 8, 128), (2, 12, 8, 2, 64), (1, 150, 4, 2, 128)])
def test_graph_replay_and_other_stream(ctx, b, s, h, kvh, d):
    """Captured on a side stream and replayed with new inputs and positions: the same bits as eager calls."""
    p = Problem("int8", b, s, h, kvh, d, 700, [100] * b, d, False, True)
    p.attend(ctx)  # eager, on the default stream
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    try:
        with torch.cuda.stream(side):
            use_torch_stream(ctx)
            p.attend(ctx, out=True, out16=True)
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                use_torch_stream(ctx)
                p.attend(ctx, out=True, out16=True)
        for step in range(3):
            p.rows.normal_()
            p.past += s
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            got, got16 = p.out.clone(), p.out16.clone()
            keep = p.out, p.out16
            use_torch_stream(ctx)
            p.attend(ctx, out=True, out16=True)
            torch.cuda.synchronize()
            assert torch.equal(got, p.out) and torch.equal(got16, p.out16)
            p.out, p.out16 = keep
    finally:
        use_torch_stream(ctx)


# ---------------------------------------------------------------------------
# Keep
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("layers,b,kvh,d,n", [(1, 2, 2, 128, 8), (3, 4, 8, 64, 64), (2, 3, 1, 80, 5), (2, 2, 2, 7, 33)])
def test_keep(ctx, layers, b, kvh, d, n):
    g = torch.Generator(device="cuda").manual_seed(n)
    cap = 100
    codes = [torch.randint(0, 256, (layers, b, kvh, cap, d), generator=g, device="cuda", dtype=torch.uint8)
             for _ in range(2)]
    scales = [torch.rand((layers, b, kvh, cap), generator=g, device="cuda") for _ in range(2)]
    was = [t.clone() for t in codes + scales]
    cpu = torch.Generator().manual_seed(n)
    past = [int(torch.randint(0, cap - n + 1, (1,), generator=cpu)) for _ in range(b)]
    counts = [0, n, 1, max(1, n // 2)][:b]
    paths = [sorted(torch.randperm(n, generator=cpu)[:c].tolist()) for c in counts]
    dev = dict(dtype=torch.int32, device="cuda")
    path = torch.tensor([p + [-5] * (n - len(p)) for p in paths], **dev)
    pa, co = torch.tensor(past, **dev), torch.tensor(counts, **dev)
    cache = N.Kv8Cache(codes[0].data_ptr(), codes[1].data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(),
                       N.B2M_INT8, b, kvh, cap, d)
    N.check(ctx.lib.b2m_kv8_keep_dev(ctx.handle, ctypes.byref(cache), layers, _p(pa), _p(path), _p(co), n))
    ctx.synchronize()
    for now, old in zip(codes + scales, was):
        for i in range(b):
            want = old[:, i].clone()
            for j, src in enumerate(paths[i]):
                want[:, :, past[i] + j] = old[:, i, :, past[i] + src]
            assert torch.equal(now[:, i], want)


def test_keep_refuses_bad_paths(ctx):
    """Not increasing, below its place, outside the drafted rows, a bad count: that sequence stays as it is."""
    d, cap, n = 64, 32, 4
    codes = [torch.arange(6 * cap * d, device="cuda").view(6, 1, cap, d).to(torch.uint8) for _ in range(2)]
    scales = [torch.rand((6, 1, cap), device="cuda") for _ in range(2)]
    was = [t.clone() for t in codes + scales]
    dev = dict(dtype=torch.int32, device="cuda")
    path = torch.tensor([[1, 1, 2, 3], [0, 0, 3, 3], [1, 4, 0, 0], [1, 2, 3, 0], [1, 3, 0, 0], [3, 0, 0, 0]], **dev)
    count = torch.tensor([2, 2, 2, 5, 2, 1], **dev)
    past = torch.tensor([0, 0, 0, 0, 5, 29], **dev)  # the last: row 32 is past the capacity
    cache = N.Kv8Cache(codes[0].data_ptr(), codes[1].data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(),
                       N.B2M_INT8, 6, 1, cap, d)
    N.check(ctx.lib.b2m_kv8_keep_dev(ctx.handle, ctypes.byref(cache), 1, _p(past), _p(path), _p(count), n))
    with pytest.raises(N.ArgumentError, match="index"):
        ctx.synchronize()
    for now, old in zip(codes + scales, was):
        for i in (0, 1, 2, 3, 5):
            assert torch.equal(now[i], old[i])
        assert torch.equal(now[4, :, 5], old[4, :, 6]) and torch.equal(now[4, :, 6], old[4, :, 8])


def test_empty_calls(ctx):
    """No sequences, no tokens, no layers: nothing to do, no error."""
    p = Problem("int8", 1, 1, 1, 1, 32, 8, [0])
    c = N.Kv8Cache(None, None, None, None, N.B2M_INT8, 0, 1, 8, 32)
    lib, h = ctx.lib, ctx.handle
    N.check(lib.b2m_kv8_append_dev(h, ctypes.byref(c), None, None, 32, None, 0.0, None, None, None, None, 0, 0, 0, 3))
    N.check(lib.b2m_kv8_append_dev(h, ctypes.byref(p.cache), None, None, 32, None, 0.0, None, None, None, None, 0, 0, 0, 0))
    N.check(lib.b2m_kv8_read_dev(h, ctypes.byref(p.cache), None, 0, None, None))
    N.check(lib.b2m_gqa_kv8_dev(h, ctypes.byref(c), None, None, None, 32, 32, None, 0.0, None, None, None, None, None,
                                0, 0, 0, None, None, 1, 1, ctypes.c_float(0)))
    N.check(lib.b2m_kv8_keep_dev(h, ctypes.byref(p.cache), 0, None, None, None, 4))
    ctx.synchronize()
