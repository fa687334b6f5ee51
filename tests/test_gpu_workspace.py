"""GPU tests of the context's workspace and CUDA graphs: a graph keeps the
workspace it was captured on, and one that a capture has to enlarge serves the
calls outside the graph as well."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import onnx_runtime_dart_b200 as b2m  # noqa: E402
from onnx_runtime_dart_b200 import _native as N  # noqa: E402
from onnx_runtime_dart_b200.decoder import DecoderConfig, Int4Decoder, random_nbits  # noqa: E402
from onnx_runtime_dart_b200.runtime import use_torch_stream  # noqa: E402

K, COLS = 1024, 256


class Gemm:
    """A MatMulNBits call whose workspace holds its m rows in f16: 2 m K bytes, and never less than 1 MiB."""

    def __init__(self, seed=0):
        self.ctx = b2m.Context(0)
        bq, sc, zp = random_nbits(np.random.default_rng(seed), K, COLS, 32)
        self.w = self.ctx.prepack_nbits(bq, sc, zp, K, COLS, 4, 32)

    def __call__(self, x, y):
        use_torch_stream(self.ctx)
        N.check(self.ctx.lib.b2m_matmul_nbits_dev(self.ctx.handle, ctypes.c_void_p(x.data_ptr()), x.shape[0],
                                                  self.w.handle, None, N.MODE_FAST, ctypes.c_void_p(y.data_ptr())))

    def close(self):
        torch.cuda.synchronize()
        use_torch_stream(self.ctx)
        self.w.free()
        self.ctx.close()


def _rows(m, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((m, K), generator=g, device="cuda"), torch.zeros((m, COLS), device="cuda")


def _capture(call):
    torch.cuda.synchronize()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            call()
    torch.cuda.synchronize()
    return g


def test_a_graph_keeps_a_workspace_that_was_replaced():
    """Captured on a workspace of 1 MiB, which a call of 4 MiB then replaces: replays give the same rows and write into
    nobody's memory (what the pool handed out since keeps its bytes)."""
    op, other = Gemm(), b2m.Context(0)
    x, y = _rows(256, 1)
    op(x, y)
    torch.cuda.synchronize()
    want = y.clone()
    g = _capture(lambda: op(x, y))
    big, big_y = _rows(2048, 2)
    op(big, big_y)
    torch.cuda.synchronize()
    junk = [other.upload(np.full(1 << 18, 3.0 + i, np.float32)) for i in range(8)]  # 1 MiB each
    for _ in range(3):
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    for i, t in enumerate(junk):
        assert bool((t.numpy() == 3.0 + i).all())
        t.free()
    del g
    op.close()
    other.close()


def test_a_capture_enlarges_the_workspace():
    """The first call of a context, and a larger one later, under a capture: the same rows as an uncaptured call's, from
    the graphs in any order and from calls outside them."""
    plain, op = Gemm(), Gemm()
    small, large, huge = _rows(300, 3), _rows(1500, 4), _rows(5000, 5)
    want = []
    for x, y in (small, large, huge):
        plain(x, y)
        torch.cuda.synchronize()
        want.append(y.clone())
    g0 = _capture(lambda: op(*small))
    op(*small)                       # outside the graph, before it ever ran
    torch.cuda.synchronize()
    assert torch.equal(small[1], want[0])
    g1 = _capture(lambda: op(*large))
    graphs = {0: g0, 1: g1}
    for k in (1, 0, 1, 0, 0, 1):
        y = (small, large)[k][1]
        y.zero_()
        graphs[k].replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[k])
        op(*(small, large)[1 - k])
        torch.cuda.synchronize()
        assert torch.equal((small, large)[1 - k][1], want[1 - k])
    op(*huge)                        # and one that replaces what the second graph holds
    torch.cuda.synchronize()
    assert torch.equal(huge[1], want[2])
    for k in (0, 1):
        y = (small, large)[k][1]
        y.zero_()
        graphs[k].replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[k])
    del g0, g1, graphs
    op.close()
    plain.close()


def test_a_wide_verify_between_replays_of_the_decode_step():
    """Int4Decoder: a speculative step whose workspace is larger than the captured decode step's, drafts all wrong on
    purpose, leaves the greedy tokens as plain decoding gives them."""
    cfg = DecoderConfig.tiny()
    cfg.inter = 4096
    ctxs = [b2m.Context(0), b2m.Context(0)]
    a, b = (Int4Decoder(c, cfg, batch=3, cap=160, max_prefill=64, seed=5, kv_type="int8", producer_f16=False)
            for c in ctxs)
    p = torch.from_numpy(np.random.default_rng(7).integers(0, cfg.vocab, (3, 5)))
    for d in (a, b):
        d.prefill(p)
    want = a.decode(8).cpu()
    got = [b.decode(2).cpu()]
    n = 50  # 150 rows: the down projection's f16 operand, 150 x 4096 x 2 bytes, is over 1 MiB
    route = ctypes.c_int32(-1)
    N.check(b.lib.b2m_matmul_nbits_route(ctxs[1].handle, b.layers[0]["down"].handle, 3 * n, N.MODE_FAST,
                                         ctypes.byref(route)))
    assert route.value == N.ROUTE_TC_F16
    drafts = torch.empty((3, n), dtype=torch.int64)
    for i in range(3):
        wrong = [v for v in range(cfg.vocab) if v not in want[:, i].tolist()]
        drafts[i] = torch.tensor(wrong[:n])
    drafts[:, 0] = b.next_ids.cpu()
    new = b.verify(drafts, [-1] + [0] * (n - 1))
    assert [len(r) for r in new] == [1, 1, 1]
    got += [torch.tensor([[r[0] for r in new]]), b.decode(5).cpu()]
    assert torch.equal(torch.cat(got), want)
    del a, b
    for c in ctxs:
        c.close()
