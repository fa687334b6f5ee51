"""GPU tests of b2m_logprobs_dev against the definition in 64 bits."""
import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import onnx_runtime_dart_b200 as b2m  # noqa: E402
from onnx_runtime_dart_b200 import _native as N  # noqa: E402
from onnx_runtime_dart_b200.runtime import use_torch_stream  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    c = b2m.Context(0)
    use_torch_stream(c)
    yield c
    c.close()


def _p(t, off=0):
    return None if t is None else ctypes.c_void_p(t.data_ptr() + off)


def _call(ctx, x, v, ids, k, off=0, entropy=True, top_lp=True):
    """x: [rows][ld] fp32; off: floats to skip at its start (alignment)."""
    rows, ld = x.shape
    lp = torch.full((rows,), 7.0, device="cuda") if ids is not None else None
    ent = torch.full((rows,), 7.0, device="cuda") if entropy else None
    top = torch.full((rows, k), -7, device="cuda", dtype=torch.int64) if k else None
    tlp = torch.full((rows, k), 7.0, device="cuda") if k and top_lp else None
    N.check(ctx.lib.b2m_logprobs_dev(ctx.handle, _p(x, 4 * off), ld, _p(ids), rows, v, _p(lp), _p(ent), k, _p(top),
                                     _p(tlp)))
    return lp, ent, top, tlp


def _want(x, k):
    x = x.double()
    x = x - x.amax(1, keepdim=True)  # beside -3.4e38 the logarithm of the sum is below 2^-53
    lp = x - torch.logsumexp(x, 1, keepdim=True)
    ent = -(lp.exp() * torch.where(lp.isinf(), torch.zeros_like(lp), lp)).sum(1)
    ids = torch.argsort(-x, dim=1, stable=True)[:, :k]
    return lp, ent, ids


def _check(ctx, x, v, k, off=0):
    rows = x.shape[0]
    xv = x.reshape(-1)[off:].as_strided((rows, v), (x.shape[1], 1)) if off else x[:, :v]
    g = torch.Generator(device="cuda").manual_seed(v)
    ids = torch.randint(0, v, (rows,), generator=g, device="cuda")
    ids[0] = int(xv[0].argmax())
    lp, ent, top, tlp = _call(ctx, x, v, ids, k, off)
    wlp, went, wtop = _want(xv, k)
    # ln of the sum: each term is off by 2^-22 (exponential) and 2^-24 * (|x - m| log2 e + 1) with |x - m| <= 24 where
    # it counts, sums of n / 256 + 64 terms by as many 2^-24: rel; then x - m, minus the ln: two roundings.
    rel = 2.0 ** -22 + 36 * 2.0 ** -24 + (v / 256 + 64) * 2.0 ** -24
    want = wlp.gather(1, ids[:, None])[:, 0]
    fin = want.isfinite()
    assert torch.equal(lp.isfinite(), fin) and bool((lp[~fin] == -math.inf).all())
    tol = rel * torch.expm1(-wlp.amax(1)).clamp(max=1.0) + 2 * 2.0 ** -24 * want.abs() + 1e-37
    assert bool(((lp.double() - want).abs() <= tol)[fin].all())
    # entropy: the same relative error on the ln and on each (x - m) p, whose sum is at most (entropy + |ln p_max|)
    assert bool(((ent.double() - went).abs() <= 2 * rel * (went + wlp.amax(1).abs()) + 1e-37).all())
    if k:
        assert torch.equal(top, wtop)
        wt = wlp.gather(1, wtop)
        tf = wt.isfinite()
        tol = (rel * torch.expm1(-wlp.amax(1)).clamp(max=1.0))[:, None] + 2 * 2.0 ** -24 * wt.abs() + 1e-37
        assert bool(((tlp.double() - wt).abs() <= tol)[tf].all()) and bool((tlp[~tf] == -math.inf).all())


@pytest.mark.parametrize("rows,v,ld,k,off", [
    (1, 1, 1, 1, 0), (3, 2, 2, 2, 0), (1, 33, 40, 32, 1), (5, 50, 53, 20, 2), (2, 1000, 1003, 5, 3),
    (1, 32001, 32001, 20, 0), (7, 32001, 32001, 32, 1), (1, 151936, 151936, 5, 0), (40, 20011, 20012, 20, 0),
    (300, 4097, 4097, 8, 0), (700, 1025, 1030, 1, 0), (2, 151936, 151936, 0, 0), (3, 9, 9, 0, 0)])
def test_normal_rows(ctx, rows, v, ld, k, off):
    g = torch.Generator(device="cuda").manual_seed(rows + v)
    x = torch.randn((rows + (1 if off else 0), ld), generator=g, device="cuda") * 3
    x = x[:rows] if not off else x
    if off:
        x = x.reshape(-1)[: rows * ld + off]
        full = torch.empty(rows * ld + ld, device="cuda")
        full[: x.numel()] = x
        _check(ctx, full[: rows * ld].view(rows, ld), v if off + v <= ld else ld - off, min(k, ld - off), off)
    else:
        _check(ctx, x, v, k)


@pytest.mark.parametrize("v", [40, 5000, 40003])
def test_ties_go_to_the_lowest_id(ctx, v):
    g = torch.Generator(device="cuda").manual_seed(v)
    x = torch.randint(-3, 4, (6, v), generator=g, device="cuda").float()
    x[1] = 2.5          # every logit equal
    x[2] = torch.where(x[2] > 0, torch.zeros_like(x[2]), -torch.zeros_like(x[2]))  # +0 and -0 are equal
    x[3] = torch.arange(v, device="cuda").float() % 7
    x[4] = -torch.arange(v, device="cuda").float() / 64   # descending
    x[5] = torch.arange(v, device="cuda").float() / 4096  # ascending: every entry beats those before it
    _check(ctx, x, v, 32)


def test_masked_rows(ctx):
    """-inf logits: some, all but three, all but one; the type's lowest value as a mask."""
    v = 30000
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((5, v), generator=g, device="cuda")
    x[0, ::3] = -math.inf
    keep = [17, 12345, 29999]
    x[1, [i for i in range(v) if i not in keep]] = -math.inf
    y = torch.full((v,), -math.inf, device="cuda")
    y[2222] = -5.0
    x[2] = y
    x[3, 5:] = torch.finfo(torch.float32).min
    x[4] = torch.finfo(torch.float32).min
    _check(ctx, x, v, 20)
    ids = torch.tensor([0, 17, 2222, 0, 9], device="cuda")
    lp, ent, top, tlp = _call(ctx, x, v, ids, 5)
    assert float(lp[0]) == -math.inf and float(lp[2]) == 0.0 and float(ent[2]) == 0.0
    assert top[1].tolist()[3:] == [0, 1]  # equal -inf logits: lowest ids
    assert abs(float(lp[4]) + math.log(v)) < 1e-5


def test_confident_rows(ctx):
    """Log probabilities far below 2^-24 keep their digits."""
    x = torch.zeros((4, 2000), device="cuda")
    for r, gap in enumerate((10.0, 20.0, 25.0, 60.0)):
        x[r, 700] = gap
    ids = torch.full((4,), 700, device="cuda")
    lp, ent, _, _ = _call(ctx, x, 2000, ids, 1)
    for r, gap in enumerate((10.0, 20.0, 25.0, 60.0)):
        rest = 1999 * math.exp(-gap)
        assert abs(float(lp[r]) + math.log1p(rest)) <= 2e-5 * rest
        want = math.log1p(rest) + gap * rest / (1 + rest)
        assert abs(float(ent[r]) - want) <= 2e-5 * want


def test_rows_without_a_distribution(ctx):
    x = torch.randn((4, 5000), device="cuda")
    x[0, 4321] = float("nan")
    x[1, 3] = math.inf
    x[2] = -math.inf
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    lp, ent, top, tlp = _call(ctx, x, 5000, ids, 3)
    assert lp[:3].isnan().all() and ent[:3].isnan().all() and tlp[:3].isnan().all()
    assert bool(lp[3].isfinite()) and bool(ent[3].isfinite())
    assert top[2].tolist() == [0, 1, 2] and int(top[1, 0]) == 3
    assert torch.equal(top[0], torch.argsort(-torch.nan_to_num(x[0], nan=-math.inf), stable=True)[:3])
    x = torch.full((1, 6), float("nan"), device="cuda")
    x[0, 4] = -math.inf
    assert _call(ctx, x, 6, None, 6)[2][0].tolist() == [4, 0, 1, 2, 3, 5]


def test_optional_outputs_and_bad_ids(ctx):
    x = torch.randn((3, 777), device="cuda")
    ids = torch.tensor([0, 777, -1], device="cuda")
    lp, ent, _, _ = _call(ctx, x, 777, ids, 0)
    with pytest.raises(N.ArgumentError, match="index"):
        ctx.synchronize()
    assert bool(lp[0].isfinite()) and lp[1:].isnan().all() and ent.isfinite().all()
    top = _call(ctx, x, 777, None, 4, entropy=False, top_lp=False)[2]
    assert torch.equal(top, _want(x, 4)[2])
    ctx.synchronize()
    N.check(ctx.lib.b2m_logprobs_dev(ctx.handle, None, 5, None, 0, 5, None, None, 0, None, None))


def test_graph_replay(ctx):
    x = torch.randn((2, 60000), device="cuda")
    ids = torch.tensor([5, 59999], device="cuda")
    lp, top = torch.empty(2, device="cuda"), torch.empty((2, 7), device="cuda", dtype=torch.int64)
    tlp = torch.empty((2, 7), device="cuda")

    def call():
        use_torch_stream(ctx)
        N.check(ctx.lib.b2m_logprobs_dev(ctx.handle, _p(x), 60000, _p(ids), 2, 60000, _p(lp), None, 7, _p(top), _p(tlp)))

    side = torch.cuda.Stream()
    try:
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            call()
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                call()
        for _ in range(3):
            x.normal_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            got = lp.clone(), top.clone(), tlp.clone()
            call()
            torch.cuda.synchronize()
            assert torch.equal(got[0], lp) and torch.equal(got[1], top) and torch.equal(got[2], tlp)
            assert torch.equal(top, _want(x, 7)[2])
    finally:
        use_torch_stream(ctx)
