"""GPU tests of attention over the 8-bit KV cache where the magnitudes in one
sequence differ: value rows that a token does not see, or hardly weighs, must
not cost the others' digits. Each against 64 bits, and rows that do not see a
loud value row also against the same call without it."""
import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import onnx_runtime_dart_b200 as b2m  # noqa: E402
from onnx_runtime_dart_b200 import _native as N  # noqa: E402
from onnx_runtime_dart_b200.runtime import use_torch_stream  # noqa: E402
from test_gpu_kv8 import Problem, _decode, _norm64, _p, _random_tree, _rope64  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    c = b2m.Context(0)
    use_torch_stream(c)
    yield c
    c.close()


def _mass(p):
    """[b][s][h][d]: sum of weight times |value| over the keys each row sees, in 64 bits."""
    q = _rope64(_norm64(p.split()[0], None if p.gain is None else p.gain[: p.h]), p.positions(), p.cos, p.sin, p.rot,
                p.inter)
    out = torch.zeros((p.b, p.s, p.h, p.d), dtype=torch.float64, device="cuda")
    for i in range(p.b):
        past = int(p.past[i])
        n = past + p.s
        k, v = (_decode(p.codes[x][i, :, :n], p.kv) * p.scales[x][i, :, :n].double()[..., None] for x in range(2))
        seen = _seen(p, i)
        for hh in range(p.h):
            x = (q[i, :, hh] @ k[hh // (p.h // p.kvh)].T / math.sqrt(p.d)).masked_fill(~seen, -math.inf)
            w = torch.where(seen.any(-1, keepdim=True), torch.softmax(x, -1), torch.zeros_like(x))
            out[i, :, hh] = w @ v[hh // (p.h // p.kvh)].abs()
    return out


def _seen(p, i):
    past = int(p.past[i])
    j, t = torch.arange(past + p.s, device="cuda"), torch.arange(p.s, device="cuda")[:, None]
    if p.tree is None:
        return j <= past + t
    return (j < past) | (((p.tree[i][:, None] >> (j - past).clamp(0, 63)) & 1) == 1)


def _row_tol(p, tol):
    """The elements' bound of Problem.answer and what a row of very different values adds: a weight times its V scale is
    held to 2^-25 beside a largest one of 2^2 or more, 2^-27 of that, for each of n keys. (An int8 row has code 0 in some
    dimensions: there only the quiet keys count, but the loud row's weight sets the digits. The largest weight times V
    scale times the largest code is at most the row's largest mass.)"""
    mass = _mass(p).amax(-1, keepdim=True).expand(p.b, p.s, p.h, p.d).reshape(tol.shape)
    return tol + (int(p.past.max()) + p.s) * 2.0 ** -27 * mass


HIDDEN = [  # b, s, h, kvh, d, cap, past, tree
    (2, 3, 4, 2, 128, 80, 40, False),
    (1, 6, 4, 2, 128, 1100, 1000, False),    # key splits over a cluster
    (2, 7, 4, 1, 64, 100, 70, False),
    (1, 6, 6, 2, 96, 60, 30, False),
    (1, 5, 2, 1, 256, 60, 30, False),
    (1, 90, 4, 2, 128, 1200, 1000, False),   # many rows, key splits
    (2, 150, 4, 2, 64, 160, 5, False),
    (20, 100, 8, 8, 128, 120, 10, False),    # many rows, one CTA for all keys
    (3, 4, 4, 2, 80, 60, 30, False),         # fp32 kernel
    (2, 12, 4, 2, 128, 100, 70, True),
    (2, 64, 4, 2, 128, 400, 300, True),
    (1, 60, 8, 2, 64, 64, 0, True),
]


@pytest.mark.parametrize("kv,loud", [("int8", 12), ("e4m3", 20), ("int8", 20), ("int8", 40), ("e4m3", 80)])
@pytest.mark.parametrize("b,s,h,kvh,d,cap,past,tree", HIDDEN)
def test_a_hidden_loud_value_changes_nothing(ctx, kv, loud, b, s, h, kvh, d, cap, past, tree):
    """One new token's values 2^loud larger: rows that do not see it stay, all rows hold their bound.

    Bound of the first: two calls whose weights are taken against other references. A weight's exponent is rounded once
    at a magnitude below 2^7 (2^-18 ln 2), its exponential is off by 2^-22, its two f16 terms by 2^-22: twice these
    are below 2^-17.2. Sums over up to 1200 keys: 76 products' additions, cut off at 2^-23 each, in either call, and
    the weights' sum by 2^-18: below 2^-16.4 together. In all 2^-15.7 of the row's mass; an f16 row alone rounds the
    weights to 2^-11 and the result to 2^-11 in each call."""
    args = (kv, b, s, h, kvh, d, cap, [past] * b, 0, False, False)
    kw = dict(tree=_random_tree(b, s, 5)) if tree else {}
    quiet, p = Problem(*args, **kw), Problem(*args, **kw)
    t = s // 2
    for i in range(b):
        p.rows[i * s + t, (h + kvh) * d:] *= 2.0 ** loud
    outs = []
    for prob in (quiet, p):
        prob.attend(ctx, out=False, out16=True)
        f16 = prob.out16.double().view(b, s, h, d)
        prob.attend(ctx)
        outs.append((prob.out.double().view(b, s, h, d), f16))
    want, tol, _ = p.answer()
    assert bool(((p.out.double() - want).abs() <= _row_tol(p, tol)).all())
    mass = _mass(quiet)
    for i in range(b):
        blind = ~_seen(p, i)[:, past + t]
        assert bool(blind.any())
        m = mass[i, blind]
        (a, a16), (c, c16) = ((x[i, blind] for x in o) for o in outs)
        assert bool(((a - c).abs() <= m * 2.0 ** -15.7).all())
        assert bool(((a16 - c16).abs() <= m * (2.0 ** -15.7 + 2 * 2.0 ** -11) + (a16.abs() + c16.abs()) * 2.0 ** -11
                     + 2.0 ** -24).all())


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("b,s,h,kvh,d,past", [(1, 1, 2, 1, 128, 1000), (2, 1, 8, 1, 64, 60), (1, 3, 2, 1, 128, 300),
                                              (1, 2, 2, 1, 256, 40), (1, 90, 2, 2, 128, 700), (1, 70, 4, 2, 64, 30),
                                              (1, 2, 2, 1, 80, 50)])
@pytest.mark.parametrize("score,loud", [(-40.0, 24), (-40.0, 45), (-40.0, 58), (-40.0, 70), (40.0, -20), (40.0, -45),
                                        (40.0, -70), (40.0, None)])
def test_a_loud_value_of_no_weight(ctx, kv, b, s, h, kvh, d, past, score, loud):
    """One cached key that every row sees, e^score times the weight of the others and with values 2^loud times as large
    (None: zeros): against 64 bits with a bound from the weights that count."""
    p = Problem(kv, b, s, h, kvh, d, past + s, [past] * b)
    p.rows[:, : h * d] = 0.02
    p.rows[:, h * d: (h + kvh) * d] = 0
    p.codes[0].zero_()
    p.scales[0][:, :, :past] = 1.0
    j = past // 3
    p.codes[0][:, :, j] = 0x40  # 64 as int8, 2 as e4m3
    x = 0.02 * (64 if kv == "int8" else 2) * d / math.sqrt(d)
    p.scales[0][:, :, j] = abs(score) / x
    if score < 0:
        p.rows[:, : h * d] *= -1
    if loud is None:
        p.scales[1][:, :, j] = 0
    else:
        p.scales[1][:, :, j] *= 2.0 ** loud
    p.attend(ctx)
    want, tol, _ = p.answer()
    err, tol = (p.out.double() - want).abs(), _row_tol(p, tol)
    assert bool((err <= tol).all()), f"{float((err / tol).max()):.2f} of the bound"
    assert bool((p.out != 0).any())


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("b,s,h,kvh,d,cap,past", [(2, 1, 4, 2, 128, 700, 600), (1, 1, 16, 1, 64, 90, 50),
                                                  (2, 5, 4, 2, 96, 60, 30), (1, 3, 2, 2, 256, 40, 20),
                                                  (2, 1, 3, 1, 32, 300, 290), (2, 90, 4, 2, 128, 400, 300),
                                                  (8, 64, 32, 8, 64, 80, 10), (1, 4, 4, 2, 80, 40, 9)])
def test_f16_rows_are_the_fp32_rows_rounded(ctx, kv, b, s, h, kvh, d, cap, past):
    """An f16 output alone is computed as the fp32 rows are: the same bits as rounding those."""
    p = Problem(kv, b, s, h, kvh, d, cap, [past] * b, d, False, True)
    p.attend(ctx)
    full = p.out.clone()
    p.attend(ctx, out=False, out16=True)
    assert torch.equal(p.out16, full.half())


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("b,s,h,kvh,d,n", [
    (19, 64, 16, 8, 128, 16384),  # one CTA for all keys of 128 query rows
    (19, 64, 16, 8, 64, 16000),
    (28, 1, 16, 8, 128, 32768),   # one CTA, four warps, for all keys of a few rows
    (28, 1, 16, 8, 64, 32760),
    (28, 6, 16, 8, 64, 16384)])
def test_sums_do_not_drift(ctx, kv, b, s, h, kvh, d, n):
    """Equal scores and equal values: each output is the value itself, however many keys there are.

    All weights are 2^10 and their sum is exact. What the tensor cores cut off an addition is below 2^-23 of the sum so
    far: over a window of 64 additions (eight tiles, four steps, two terms) 32 * 2^-23 of the window, less where a window
    has 16. At most 64 windows are added up, each rounded to 2^-24 of the sum so far: 32 * 2^-24. The weights' two terms
    are off by 2^-22, the warps' or CTAs' merge, the division and its product by eight roundings of 2^-24."""
    p = Problem(kv, b, s, h, kvh, d, n, [0] * b)
    p.past[:] = n - s
    third = torch.tensor(1 / 3, device="cuda")
    top = 127 if kv == "int8" else 448
    p.rows[:, : h * d] = 1.0
    p.rows[:, h * d: (h + kvh) * d] = 0
    p.rows[:, (h + kvh) * d:] = third * top
    p.codes[0].zero_()
    p.scales[0].fill_(1.0)
    p.codes[1].fill_(127 if kv == "int8" else 0x7e)
    p.scales[1].fill_(third)
    p.attend(ctx)
    want = float(third) * top
    bound = 32 * 2.0 ** -23 + 32 * 2.0 ** -24 + 2.0 ** -22 + 8 * 2.0 ** -24
    assert float((p.out.double() / want - 1).abs().max()) <= bound


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("s,d", [(3, 128), (60, 128), (64, 64), (5, 80)])
@pytest.mark.parametrize("scale", [1.0, 1e-3, 1e-6, 1e-20, 1e-37])
def test_zero_queries_under_a_small_scale(ctx, s, d, scale, tree):
    """Rows of zeros among the queries weigh all they see alike, whatever the scale; hidden keys stay hidden."""
    p = Problem("int8", 2, s, 4, 2, d, 200, [90, 0], scale=scale, tree=_random_tree(2, s, 3) if tree else None)
    p.rows[::2, : 4 * d] = 0
    p.rows[1::2, : 4 * d] *= 1e-38  # subnormal and nearly so
    p.attend(ctx)
    want, tol, _ = p.answer()
    assert bool(((p.out.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("e", [62, 70, 120, -60, -100])
@pytest.mark.parametrize("s,d,rot,inter", [(1, 128, 128, False), (3, 64, 32, False), (2, 96, 96, True), (70, 128, 64, False),
                                           (90, 64, 64, False), (2, 80, 80, False), (1, 256, 0, False)])
def test_head_norm_of_large_and_small_queries(ctx, s, d, rot, inter, e):
    """Queries whose squares leave fp32's range are normalised all the same (one row in three stays as it is)."""
    p = Problem("int8", 2, s, 4, 2, d, 200, [90, 7], rot, inter, True, half=d // 2)
    r = p.rows.view(2 * s, 8, d)
    r[:, [0, 1, 3]] *= 2.0 ** e
    p.attend(ctx)
    want, tol, _ = p.answer()
    assert bool(((p.out.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("seed", range(12))
def test_values_of_any_size(ctx, kv, seed):
    """Value rows of random magnitudes, 2^-20 .. 2^20 from one key to the next and some of zeros, over random shapes."""
    g = torch.Generator().manual_seed(seed)

    def pick(*xs):
        return xs[int(torch.randint(0, len(xs), (1,), generator=g))]

    d, kvh = pick(32, 64, 64, 96, 128, 128, 256, 80), pick(1, 2, 4)
    h, s = kvh * pick(1, 2, 3, 8), pick(1, 1, 2, 7, 30, 64, 200)
    b, past = pick(1, 2, 5), pick(0, 5, 63, 300, 1500)
    tree = _random_tree(b, s, seed, orphan=True) if s <= 64 and pick(True, False) else None
    p = Problem(kv, b, s, h, kvh, d, past + s + pick(0, 9), [past] + [past // 2] * (b - 1), pick(0, d), False,
                pick(True, False), tree=tree)
    e = torch.randint(-20, 21, (b, kvh, past), generator=g).float()
    e[torch.rand(e.shape, generator=g) < 0.1] = -math.inf
    p.scales[1][:, :, :past] *= (2.0 ** e).cuda()
    p.rows.view(b * s, -1, d)[:, h + kvh:] *= (2.0 ** torch.randint(-20, 21, (b * s, kvh, 1), generator=g).float()).cuda()
    p.attend(ctx)
    want, tol, _ = p.answer()
    err, tol = (p.out.double() - want).abs(), _row_tol(p, tol)
    assert bool((err <= tol).all()), f"{float((err / tol).max()):.2f} of the bound"


@pytest.mark.parametrize("s,past", [(1, 300), (90, 1000), (1, 524000), (5, 524000), (150, 524000)])
def test_offsets_beyond_32_bits(ctx, s, past):
    """A cache of more than 2^32 bytes, the last sequence behind that border, with few and with many keys."""
    b, kvh, d, cap = 9, 8, 128, 1 << 19
    p = Problem("int8", b, s, kvh, kvh, d, 4, [0] * b)  # (its small cache is replaced)
    free, _ = torch.cuda.mem_get_info()
    if free < 20 << 30:
        pytest.skip("needs 20 GB of device memory")
    p.cap = cap
    p.codes = [torch.zeros((b, kvh, cap, d), device="cuda", dtype=torch.uint8) for _ in range(2)]
    p.scales = [torch.zeros((b, kvh, cap), device="cuda") for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(s)
    for side in range(2):
        p.codes[side][-1, :, :past] = torch.randint(0, 255, (kvh, past, d), generator=g, device="cuda",
                                                    dtype=torch.uint8) + 129  # -127 .. 127
        p.scales[side][-1, :, :past] = 0.01 + 0.01 * torch.rand((kvh, past), generator=g, device="cuda")
    p.past[-1] = past
    p.cache = N.Kv8Cache(p.codes[0].data_ptr(), p.codes[1].data_ptr(), p.scales[0].data_ptr(), p.scales[1].data_ptr(),
                         N.B2M_INT8, b, kvh, cap, d)
    p.attend(ctx)
    new = p.new_rows()
    for side in range(2):
        assert torch.equal(_decode(p.codes[side][-1, :, past: past + s], "int8"), new[side][0][-1])
    out = p.out
    p.out = None
    last = Problem("int8", 1, s, kvh, kvh, d, 4, [0])
    last.rows, last.cap, last.past = p.rows[-s:], past + s, p.past[-1:]
    last.codes = [t[-1:, :, : past + s] for t in p.codes]
    last.scales = [t[-1:, :, : past + s] for t in p.scales]
    want, tol, _ = last.answer()
    assert bool(((out[-1:].double() - want).abs() <= tol).all())
