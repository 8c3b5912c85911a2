"""GPU tests of the attention over a quantised cache where a head is spread over
several clusters of CTAs, whose parts meet in global memory: both widths, full
parts, other head sizes, graph replays, two contexts at once."""
import numpy as np
import pytest

from test_gpu_kv_quant import QuantizedKvCache, check_attention, dev, host, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("tokens,heads,dim", [(33000, 2, 128), (20011, 3, 64), (30000, 1, 256), (16000, 5, 80), (40000, 1, 17),
                                              (9000, 10, 128), (12345, 7, 160)])
def test_full_parts(ctx, bits, tokens, heads, dim):
    rng = np.random.default_rng(tokens + bits)
    kv, q, out = run_attention(ctx, rng, (tokens,), heads, dim, bits, 64, 70)
    check_attention(kv, q, out, heads, dim, bits)
    for _ in range(3):
        assert np.array_equal(host(kv.attention(dev(q))), out)
    kv.free()


@pytest.mark.parametrize("bits", [4, 8])
def test_two_sequences_of_different_lengths(ctx, bits):
    """One fills its parts, the other leaves most of them empty."""
    rng = np.random.default_rng(bits)
    kv, q, out = run_attention(ctx, rng, (25000, 33), 2, 96, bits, 3, 2)
    check_attention(kv, q, out, 2, 96, bits)
    kv.free()


@pytest.mark.parametrize("bits", [4, 8])
def test_captured_and_replayed(ctx, bits):
    """A replaced prompt, a pushed token and the attention in one graph, replayed with
    other rows: the tickets are as they were after every launch."""
    import torch
    rng = np.random.default_rng(bits)
    heads, dim, tokens = 2, 128, 20000
    width = heads * dim
    k, v = (torch.zeros((tokens, width), device="cuda") for _ in range(2))
    q, out = (torch.zeros((1, width), device="cuda") for _ in range(2))
    plain, captured = (QuantizedKvCache(ctx, 1, heads, dim, 4, tokens, bits) for _ in range(2))
    rows = torch.zeros((2, 33, width), device="cuda")
    side, back = torch.cuda.Stream(), torch.cuda.current_stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    ctx.set_stream(side)
    try:
        with torch.cuda.graph(graph, stream=side):
            captured.reset(0)
            captured.prefill(0, k, v)
            for _ in range(2):
                captured.push(q, q)
                captured.attention(q, out)
            captured.read(0, tokens - 31, 33, rows[0], rows[1])
        for i in range(3):
            for t in (k, v, q):
                t.copy_(torch.from_numpy(rng.standard_normal(t.shape).astype(np.float32)))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got, held = host(out), host(rows)
            ctx.set_stream(back)
            plain.reset(0)
            plain.prefill(0, k, v)
            for _ in range(2):
                plain.push(q, q)
                want = host(plain.attention(q))
            assert np.array_equal(got, want)
            for x, y in zip(held, plain.read(0, tokens - 31, 33)):
                assert np.array_equal(x, host(y))
            ctx.sync()
            assert captured.state(0) == plain.state(0) == (tokens + 2, tokens + 2)
    finally:
        ctx.set_stream(back)
        del graph
    check_attention(captured, host(q), got, heads, dim, bits)
    plain.free()
    captured.free()


def test_two_contexts_at_once():
    """Two caches, each with several clusters per head, served on streams of their own."""
    import torch
    import uocr_q8
    rng = np.random.default_rng(3)
    heads, dim, tokens = 3, 128, 24000
    width = heads * dim
    made = []
    for bits in (4, 8):
        c = uocr_q8.GpuContext(0)
        c.set_stream(torch.cuda.Stream())
        kv = QuantizedKvCache(c, 1, heads, dim, 4, tokens, bits)
        x = dev(rng.standard_normal((2, tokens, width)).astype(np.float32))
        q = dev(rng.standard_normal((1, width)).astype(np.float32))
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        kv.prefill(0, x[0], x[1])
        kv.attention(q, out)
        c.sync()
        made.append((c, kv, x, q, out, host(out)))
        check_attention(kv, host(q), host(out), heads, dim, bits)
    for _ in range(20):
        for c, kv, x, q, out, want in made:
            for _ in range(4):
                kv.attention(q, out)
        for c, kv, x, q, out, want in made:
            c.sync()
            assert np.array_equal(host(out), want)
            out.zero_()
        torch.cuda.synchronize()
    for c, kv, *_ in made:
        kv.free()
        c.close()
