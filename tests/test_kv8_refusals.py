"""CPU tests: every refusal of the 8-bit KV cache and log-probability entry
points. They check their arguments before the context, so a call that passes
them ends at the null context here and never reaches a device."""
import ctypes

import pytest

from onnx_runtime_dart_b200 import _native as N
from onnx_runtime_dart_b200 import build


@pytest.fixture(scope="module")
def lib():
    import os

    if not os.path.exists(build.LIB):
        build.build()
    return N.load()


P = 4096  # a pointer value that no refused call reads


def _cache(**over):
    f = dict(k=P, v=P, k_scale=P, v_scale=P, type=N.B2M_INT8, b=2, kvh=2, cap=32, head_dim=64)
    f.update(over)
    return N.Kv8Cache(*(f[n] for n, _ in N.Kv8Cache._fields_))


def _append(lib, cache=None, k=P, v=P, kv_rs=128, gain=None, eps=0.0, past=P, depth=None, cos=None, sin=None, half=0,
            rot=0, s=1):
    c = _cache() if cache is None else cache
    N.check(lib.b2m_kv8_append_dev(None, ctypes.byref(c), k, v, kv_rs, gain, eps, past, depth, cos, sin, half, rot, 0, s))


def _gqa(lib, cache=None, q=P, k=P, v=P, q_rs=256, kv_rs=128, gain=None, eps=0.0, past=P, tree=None, depth=None,
         cos=None, sin=None, half=0, rot=0, out=P, out16=None, s=1, h=4):
    c = _cache() if cache is None else cache
    N.check(lib.b2m_gqa_kv8_dev(None, ctypes.byref(c), q, k, v, q_rs, kv_rs, gain, eps, past, tree, depth, cos, sin,
                                half, rot, 0, out, out16, s, h, 0.0))


BAD_CACHES = [(dict(type=N.B2M_FLOAT), N.UnsupportedError, "cache type"),
              (dict(type=N.B2M_UINT8), N.UnsupportedError, "cache type"),
              (dict(head_dim=257), N.ArgumentError, "cache shape"), (dict(head_dim=0), N.ArgumentError, "cache shape"),
              (dict(cap=0), N.ArgumentError, "cache shape"), (dict(kvh=0), N.ArgumentError, "cache shape"),
              (dict(cap=(1 << 30) + 1), N.ArgumentError, "cache shape"),
              (dict(b=-1), N.ArgumentError, "cache shape"), (dict(k=0), N.ArgumentError, "null cache"),
              (dict(v_scale=0), N.ArgumentError, "null cache"), (dict(k=P + 2), N.ArgumentError, "4-byte"),
              (dict(v=P + 1), N.ArgumentError, "4-byte")]


@pytest.mark.parametrize("over,exc,msg", BAD_CACHES)
def test_bad_caches(lib, over, exc, msg):
    with pytest.raises(exc, match=msg):
        _append(lib, cache=_cache(**over))
    with pytest.raises(exc, match=msg):
        _gqa(lib, cache=_cache(**over))
    c = _cache(**over)
    with pytest.raises(exc, match=msg):
        N.check(lib.b2m_kv8_read_dev(None, ctypes.byref(c), None, 1, P, P))
    with pytest.raises(exc, match=msg):
        N.check(lib.b2m_kv8_keep_dev(None, ctypes.byref(c), 1, P, P, P, 2))


def test_null_cache(lib):
    for st in (lib.b2m_kv8_append_dev(None, None, P, P, 128, None, 0.0, P, None, None, None, 0, 0, 0, 1),
               lib.b2m_kv8_read_dev(None, None, None, 1, P, P),
               lib.b2m_gqa_kv8_dev(None, None, P, P, P, 256, 128, None, 0.0, P, None, None, None, None, 0, 0, 0, P,
                                   None, 1, 4, 0.0),
               lib.b2m_kv8_keep_dev(None, None, 1, P, P, P, 2)):
        assert st == N.B2M_ERR_INVALID_ARGUMENT
        assert b"cache is null" in lib.b2m_last_error()


ROTARY = [dict(cos=P), dict(cos=P, sin=P, half=32, rot=0), dict(cos=P, sin=P, half=32, rot=66),
          dict(cos=P, sin=P, half=32, rot=31), dict(cos=P, sin=P, half=8, rot=32), dict(cos=P, sin=P, half=0, rot=32)]


@pytest.mark.parametrize("rotary", ROTARY)
def test_bad_rotary(lib, rotary):
    with pytest.raises(N.ArgumentError, match="rotary"):
        _append(lib, **rotary)
    with pytest.raises(N.ArgumentError, match="rotary"):
        _gqa(lib, **rotary)


@pytest.mark.parametrize("kw,msg", [(dict(k=None), "null"), (dict(v=None), "null"), (dict(past=None), "null"),
                                    (dict(kv_rs=127), "row stride"), (dict(s=-1), "token count"),
                                    (dict(gain=P, eps=-1.0), "eps"), (dict(gain=P, eps=float("nan")), "eps")])
def test_append_refusals(lib, kw, msg):
    with pytest.raises(N.ArgumentError, match=msg):
        _append(lib, **kw)


@pytest.mark.parametrize("kw,exc,msg", [
    (dict(q=None), N.ArgumentError, "null"), (dict(k=None), N.ArgumentError, "null"),
    (dict(past=None), N.ArgumentError, "null"), (dict(out=None), N.ArgumentError, "null"),
    (dict(q_rs=255), N.ArgumentError, "strides"), (dict(kv_rs=100), N.ArgumentError, "strides"),
    (dict(h=3), N.ArgumentError, "shape"), (dict(h=0), N.ArgumentError, "shape"), (dict(s=-2), N.ArgumentError, "shape"),
    (dict(tree=P), N.ArgumentError, "go together"), (dict(depth=P), N.ArgumentError, "go together"),
    (dict(tree=P, depth=P, s=65), N.UnsupportedError, "at most 64"), (dict(gain=P, eps=-1e-6), N.ArgumentError, "eps"),
    (dict(cache=None, out16=P, h=2, q_rs=128), None, None),
])
def test_gqa_refusals(lib, kw, exc, msg):
    if exc is None:  # a call that is right ends at the null context
        exc, msg = N.ArgumentError, "null context"
    with pytest.raises(exc, match=msg):
        _gqa(lib, **kw)


def test_gqa_f16_width(lib):
    c = _cache(kvh=1, head_dim=6)
    with pytest.raises(N.ArgumentError, match="multiple of 8"):
        _gqa(lib, cache=c, out16=P, h=2)


def test_read_and_keep_refusals(lib):
    c = _cache()
    with pytest.raises(N.ArgumentError, match="n must lie"):
        N.check(lib.b2m_kv8_read_dev(None, ctypes.byref(c), None, 33, P, P))
    with pytest.raises(N.ArgumentError, match="n must lie"):
        N.check(lib.b2m_kv8_read_dev(None, ctypes.byref(c), None, -1, P, P))
    with pytest.raises(N.ArgumentError, match="null pointer"):
        N.check(lib.b2m_kv8_keep_dev(None, ctypes.byref(c), 1, P, None, P, 2))
    with pytest.raises(N.ArgumentError, match="negative"):
        N.check(lib.b2m_kv8_keep_dev(None, ctypes.byref(c), -1, P, P, P, 2))


@pytest.mark.parametrize("kw,msg", [
    (dict(x=None), "bad arguments"), (dict(v=0), "bad arguments"), (dict(ld=99), "bad arguments"),
    (dict(rows=-1), "bad arguments"), (dict(v=1 << 31, ld=1 << 31), "bad arguments"),
    (dict(ids=None), "go together"), (dict(lp=None), "go together"), (dict(k=33), "k must"), (dict(k=-1), "k must"),
    (dict(v=10, k=11), "k must"), (dict(top=None), "top_ids is null"),
])
def test_logprobs_refusals(lib, kw, msg):
    a = dict(x=P, ld=100, ids=P, rows=2, v=100, lp=P, ent=P, k=4, top=P, tlp=P)
    a.update(kw)
    with pytest.raises(N.ArgumentError, match=msg):
        N.check(lib.b2m_logprobs_dev(None, a["x"], a["ld"], a["ids"], a["rows"], a["v"], a["lp"], a["ent"], a["k"],
                                     a["top"], a["tlp"]))


def test_right_calls_reach_the_context(lib):
    for call in (lambda: _append(lib), lambda: _gqa(lib), lambda: _gqa(lib, tree=P, depth=P, s=64)):
        with pytest.raises(N.ArgumentError, match="null context"):
            call()
