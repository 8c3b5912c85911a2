"""GPU tests of the quantised cache at the largest counts of sequences and heads
that it takes, and of calls that leave an argument out."""
import numpy as np
import pytest

from test_gpu_kv_quant import QuantizedKvCache, check_attention, dev, held, host

import oracle

pytestmark = pytest.mark.gpu


def test_most_sequences(ctx):
    """65,535 sequences of one token and a pushed one: the result is between the two."""
    rng = np.random.default_rng(1)
    batch, dim = 65535, 8
    kv = QuantizedKvCache(ctx, batch, 1, dim, 2, 1, 8)
    x = rng.standard_normal((4, batch, dim)).astype(np.float32)
    rows = dev(x)
    for b in range(batch):
        kv.prefill(b, rows[0, b:b + 1], rows[1, b:b + 1])
    kv.push(rows[2], rows[3])
    q = rng.standard_normal((batch, dim)).astype(np.float32)
    out = host(kv.attention(dev(q)))
    ctx.sync()
    some = [0, 1, 777, 32768, 65533, 65534]
    for b in some:
        got = kv.read(b, 0, 2)
        for t, pair in zip(got, ((0, 2), (1, 3))):
            assert np.array_equal(host(t), held(x[list(pair), b][:, None], 8)[0][:, 0].astype(np.float32))
    k, v = (np.stack([held(x[i], 8)[0] for i in pair], 1) for pair in ((0, 2), (1, 3)))
    scores = np.einsum("btd,bd->bt", k, q.astype(np.float64)) / np.sqrt(dim)
    p = np.exp(scores - scores.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    # FP32 rounding of eight-dim scores and of two values: far below 2^-16 of their sizes
    assert np.max(np.abs(out - np.einsum("bt,btd->bd", p, v))) <= 2.0 ** -16 * np.max(np.abs(x))
    kv.free()


@pytest.mark.parametrize("bits", [4, 8])
def test_most_heads(ctx, bits):
    """65,535 heads of one dim."""
    rng = np.random.default_rng(bits)
    heads, tokens = 65535, 35
    kv = QuantizedKvCache(ctx, 1, heads, 1, 2, tokens, bits)
    k, v = (rng.standard_normal((tokens + 1, heads)).astype(np.float32) for _ in range(2))
    kv.prefill(0, dev(k[:tokens]), dev(v[:tokens]))
    kv.push(dev(k[tokens:]), dev(v[tokens:]))
    q = rng.standard_normal((1, heads)).astype(np.float32)
    out = host(kv.attention(dev(q)))
    for x, got in zip((k, v), kv.export(0)):
        assert np.array_equal(host(got), held(x[..., None], bits)[0][..., 0].astype(np.float32))
    check_attention(kv, q, out, heads, 1, bits)
    kv.free()


def test_rotation_of_queries_alone(ctx):
    """rope without k, as of the FP32 cache."""
    from uocr_q8.attention import Rope
    rng = np.random.default_rng(2)
    heads, dim = 2, 64
    rope = Rope(ctx, dim, 10000.0, 300)
    kv = QuantizedKvCache(ctx, 2, heads, dim, 2, 20, 4)
    x = dev(rng.standard_normal((20, heads * dim)).astype(np.float32))
    kv.prefill(0, x, x)
    kv.prefill(1, x[:3], x[:3])
    q = rng.standard_normal((2, heads * dim)).astype(np.float32)
    t = dev(q)
    kv.rope(rope, t, None)
    ctx.sync()
    for b, n in enumerate((20, 3)):
        assert np.array_equal(host(t)[b], oracle.rope(q[b], dim, n))
    assert kv.state(0) == (20, 20)
    kv.free()
    rope.free()
