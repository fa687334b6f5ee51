"""GPU tests of the decoder on an 8-bit KV cache: prefill, greedy decode (as a
CUDA graph and step by step), token scores, and speculative steps with drafted
trees, run together as a serving loop runs them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import onnx_runtime_dart_b200 as b2m  # noqa: E402
from onnx_runtime_dart_b200 import _native as N  # noqa: E402
from onnx_runtime_dart_b200.decoder import DecoderConfig, Int4Decoder  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    c = b2m.Context(0)
    yield c
    c.close()


def _prompt(cfg, b, s, seed=3):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, cfg.vocab, (b, s)))


def _decoder(ctx, kv_type, batch=3, cap=160, max_prefill=40, **kw):
    return Int4Decoder(ctx, DecoderConfig.tiny(), batch=batch, cap=cap, max_prefill=max_prefill, seed=5,
                       kv_type=kv_type, **kw)


def test_kv_type_is_checked(ctx):
    with pytest.raises(N.ArgumentError, match="kv_type"):
        _decoder(ctx, "int4")
    dec = _decoder(ctx, None)
    with pytest.raises(N.UnsupportedError, match="8-bit"):
        dec.verify([[1]] * 3, [-1])


@pytest.mark.parametrize("kv_type", ["int8", "e4m3"])
def test_caches_hold_the_fp32_cache_quantised(ctx, kv_type):
    """Layer 0's keys and values see the same inputs with either cache: an 8-bit row's values are within half a step
    of the fp32 cache's (int8: scale / 2; e4m3: 2^-4 of the value, or half of the smallest step, 2^-10 of the scale),
    and 2^-19 of the row's largest for the fp32 norm and rotary of the fp32 cache."""
    dec, ref = _decoder(ctx, kv_type), _decoder(ctx, None)
    p = _prompt(dec.cfg, 3, 33)
    dec.prefill(p)
    ref.prefill(p)
    torch.cuda.synchronize()
    for codes, scale, full in ((dec.kcache, dec.kscale, ref.kcache), (dec.vcache, dec.vscale, ref.vcache)):
        sc = scale[0, :, :, :33].double()[..., None]
        q = codes[0, :, :, :33]
        val = (q.view(torch.int8) if kv_type == "int8" else q.view(torch.float8_e4m3fn)).double() * sc
        want = full[0, :, :, :33].double()
        top = want.abs().amax(-1, keepdim=True)
        step = sc / 2 if kv_type == "int8" else torch.maximum(val.abs() * 2.0 ** -4, sc * 2.0 ** -10)
        assert bool(((val - want).abs() <= step + top * 2.0 ** -19).all())


@pytest.mark.parametrize("kv_type", ["int8", "e4m3"])
@pytest.mark.parametrize("mode", [N.MODE_FAST, N.MODE_EXACT])
def test_graph_decode_equals_steps(ctx, kv_type, mode):
    a, b = _decoder(ctx, kv_type, mode=mode), _decoder(ctx, kv_type, mode=mode)
    p = _prompt(a.cfg, 3, 21)
    a.prefill(p)
    b.prefill(p)
    ta, tb = a.decode(6), b.decode(6, use_graph=False)
    torch.cuda.synchronize()
    assert torch.equal(ta, tb)
    assert torch.equal(a.logits, b.logits)
    for x, y in ((a.kcache, b.kcache), (a.vcache, b.vcache), (a.kscale, b.kscale), (a.past, b.past)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("kv_type", [None, "int8", "e4m3"])
def test_reports_match_the_logits(ctx, kv_type):
    """decode(top_logprobs=) and score: held to the definition in 64 bits on the decoder's own logits (2e-5: sums of
    1000 exponentials and a logarithm in fp32 around values below 16)."""
    dec = _decoder(ctx, kv_type)
    p = _prompt(dec.cfg, 3, 12)
    dec.prefill(p)
    plain = _decoder(ctx, kv_type)
    plain.prefill(p)
    ids, rep = dec.decode(1, top_logprobs=4)
    torch.cuda.synchronize()
    assert torch.equal(ids, plain.decode(1))
    lp = torch.log_softmax(dec.logits.double(), -1)
    assert torch.equal(rep["top_ids"][0], torch.argsort(-dec.logits, dim=-1, stable=True)[:, :4])
    assert torch.equal(rep["top_ids"][0, :, 0], ids[0])
    assert bool(((rep["top_logprobs"][0].double() - lp.gather(1, rep["top_ids"][0])).abs() < 2e-5).all())
    assert torch.equal(rep["logprob"][0], rep["top_logprobs"][0, :, 0])
    ent = -(lp.exp() * lp).sum(-1)
    assert bool(((rep["entropy"][0].double() - ent).abs() < 2e-5).all())
    more, rep2 = dec.decode(2, top_logprobs=0)
    assert rep2["top_ids"].shape == (2, 3, 0) and bool(rep2["logprob"].isfinite().all())
    assert torch.equal(more, plain.decode(2))

    lps, ents = dec.score(p)
    torch.cuda.synchronize()
    assert lps.shape == ents.shape == (3, 11)
    # each position's logits, one row of every sequence at a time
    for t in (0, 5, 10):
        dec._head(torch.arange(3, device="cuda") * 12 + t, 36)
        ctx.synchronize()
        want = torch.log_softmax(dec.logits.double(), -1)
        got = want.gather(1, p[:, t + 1].cuda()[:, None])[:, 0]
        assert bool(((lps[:, t].double() - got).abs() < 2e-5).all())
        assert bool(((ents[:, t].double() + (want.exp() * want).sum(-1)).abs() < 2e-5).all())
    # scoring leaves the decoder as prefill does
    plain.prefill(p)
    assert torch.equal(dec.next_ids, plain.next_ids) and torch.equal(dec.past, plain.past)


@pytest.mark.parametrize("kv_type", ["int8", "e4m3"])
def test_speculative_steps_generate_the_greedy_tokens(ctx, kv_type):
    """Trees that hold the greedy continuation, part of it, or none of it: the generated tokens are those of plain
    greedy decoding, and the cache behind them serves the next steps (graph decode included)."""
    plain = _decoder(ctx, kv_type)
    p = _prompt(plain.cfg, 3, 17)
    plain.prefill(p)
    first = plain.next_ids.clone()
    want = torch.cat([first[None], plain.decode(24)]).cpu().T.tolist()  # [B][25]
    dec = _decoder(ctx, kv_type)
    dec.prefill(p)
    dec.decode(0)
    got = [[int(x)] for x in dec.next_ids]
    g = torch.Generator().manual_seed(1)
    # (good draft tokens, parents): a chain, a bushy tree, a wrong tree, one node
    for good, parents in ((3, [-1, 0, 1, 2]), (2, [-1, 0, 0, 1, 1, 2, 4, 4, 3]), (0, [-1, 0, 0, 2]), (0, [-1])):
        n = len(parents)
        tokens = torch.randint(0, dec.cfg.vocab, (3, n), generator=g)
        path, node = [0], 0
        for _ in range(good):  # the last child of each node, so that paths skip nodes
            node = max(i for i in range(n) if parents[i] == node)
            path.append(node)
        for b in range(3):
            at = len(got[b]) - 1
            for d, node in enumerate(path):
                tokens[b, node] = want[b][at + d]
            # no other child may hold the right token by chance
            for i in range(1, n):
                if i not in path and int(tokens[b, i]) in want[b][at:at + n + 1]:
                    tokens[b, i] = next(v for v in range(dec.cfg.vocab) if v not in want[b])
        for b, new in enumerate(dec.verify(tokens, parents)):
            assert len(new) == good + 1
            got[b] += new
    assert [r[: len(w)] for r, w in zip(want, got)] == got
    tail = dec.decode(3).cpu().T.tolist()
    for b in range(3):
        assert want[b][len(got[b]): len(got[b]) + 3] == tail[b]


def test_verify_after_a_captured_decode(ctx):
    """A wider step between replays of the captured decode step (whose workspace the graph still uses) changes none
    of its results."""
    a, b = _decoder(ctx, "int8", max_prefill=64), _decoder(ctx, "int8", max_prefill=64)
    p = _prompt(a.cfg, 3, 5)
    a.prefill(p)
    b.prefill(p)
    ta = torch.cat([a.decode(2), a.decode(4)])
    tb = [b.decode(2)]
    other = b2m.Context(0)  # takes what the pool has free
    n = 40
    new = b.verify(torch.cat([b.next_ids.cpu()[:, None], torch.full((3, n - 1), 7)], 1), [-1] + [0] * (n - 1))
    junk = [other.upload(np.full(1 << 20, 3.0, np.float32)) for _ in range(4)]
    tb.append(torch.tensor([[r[0] for r in new]], device="cuda")[: 1])
    tb.append(b.decode(3))
    torch.cuda.synchronize()
    if all(len(r) == 1 for r in new):
        assert torch.equal(ta, torch.cat(tb))
    del junk
    other.close()


def test_verify_refuses(ctx):
    dec = _decoder(ctx, "int8", max_prefill=8)
    dec.prefill(_prompt(dec.cfg, 3, 4))
    for tokens, parents in (([[1, 2]] * 2, [-1, 0]), ([[1, 2]] * 3, [-1]), ([[1, 2]] * 3, [-1, 1]),
                            ([[1, dec.cfg.vocab]] * 3, [-1, 0]), ([[1] * 9] * 3, [-1] + [0] * 8)):
        with pytest.raises((N.ArgumentError, RuntimeError)):
            dec.verify(tokens, parents)
    with pytest.raises(N.ArgumentError, match="top_logprobs"):
        dec.decode(1, top_logprobs=33)
    with pytest.raises(N.ArgumentError, match="score"):
        dec.score([[1] * 9] * 3)


def test_full_cache_is_reported(ctx):
    dec = _decoder(ctx, "int8", cap=24, max_prefill=24)
    dec.prefill(_prompt(dec.cfg, 3, 22))
    torch.cuda.synchronize()
    with pytest.raises(N.ArgumentError, match="capacity"):
        dec.verify([[1, 2, 3]] * 3, [-1, 0, 1])


@pytest.mark.parametrize("kv_type", ["int8", "e4m3"])
def test_projection_shapes_of_the_decoder(ctx, kv_type):
    """Head dim 128, 64 sequences, two layers: tensor-core projections with f16 operands, the flash and the
    single-token kernels with f16 output only. Graph replays equal eager steps, and exactly the
    positions that were fed are written."""
    cfg = DecoderConfig.qwen3_0_6b()
    cfg.layers, cfg.vocab = 2, 4000
    B, S = 64, 40
    p = torch.from_numpy(np.random.default_rng(2).integers(0, cfg.vocab, (B, S)))
    dec = [Int4Decoder(ctx, cfg, batch=B, cap=S + 16, max_prefill=S, seed=9, kv_type=kv_type) for _ in range(2)]
    toks = []
    for d, graph in zip(dec, (True, False)):
        d.prefill(p)
        toks.append(d.decode(4, use_graph=graph))
    torch.cuda.synchronize()
    assert torch.equal(toks[0], toks[1]) and torch.equal(dec[0].logits, dec[1].logits)
    assert bool(dec[0].logits.isfinite().all())
    for x, y in ((dec[0].kcache, dec[1].kcache), (dec[0].vscale, dec[1].vscale)):
        assert torch.equal(x, y)
    assert bool((dec[0].kscale[:, :, :, : S + 4] > 0).all()) and not bool(dec[0].kscale[:, :, :, S + 4:].any())
    assert dec[0].past.tolist() == [S + 4] * B
