"""Calls on the quantised cache and the token log probabilities that follow each
other with nothing between, each reading what the one in front has written, give
the bits that they give one at a time (their kernels overlap at start and end)."""
import numpy as np
import pytest

from test_gpu_kv_quant import QuantizedKvCache, dev, host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 8])
def test_read_push_read(ctx, bits):
    """Every pushed token is in the read behind its push, and in no earlier one."""
    import torch
    rng = np.random.default_rng(bits)
    heads, dim, tokens, rounds = 10, 128, 40, 12
    width = heads * dim
    rows = dev(rng.standard_normal((rounds, 1, width)).astype(np.float32))
    first = dev(rng.standard_normal((tokens, width)).astype(np.float32))
    outs = []
    for one_at_a_time in (True, False):
        kv = QuantizedKvCache(ctx, 1, heads, dim, 5, tokens, bits)
        kv.prefill(0, first, first)
        for _ in range(5):
            kv.push(first[:1], first[:1])
        got = torch.zeros((rounds + 1, 2, tokens + 5, width), device="cuda")
        torch.cuda.synchronize()
        for i in range(rounds + 1):
            kv.read(0, 0, tokens + 5, got[i, 0], got[i, 1])
            if one_at_a_time:
                ctx.sync()
            if i < rounds:
                kv.push(rows[i], rows[i])
            if one_at_a_time:
                ctx.sync()
        ctx.sync()
        outs.append(host(got))
        kv.free()
    assert np.array_equal(*outs)
    assert not np.array_equal(outs[0][0], outs[0][1])


@pytest.mark.parametrize("bits", [4, 8])
def test_what_the_call_in_front_has_written(ctx, bits):
    """A prompt of rows that a cache has just read back, queries that attention has
    just given, logits that have just been written."""
    import torch
    from uocr_q8.decoder import token_logprobs_device
    rng = np.random.default_rng(bits)
    heads, dim, tokens, rounds = 4, 128, 3000, 6
    width = heads * dim
    x = dev(rng.standard_normal((rounds, tokens, width)).astype(np.float32))
    q = dev(rng.standard_normal((1, width)).astype(np.float32))
    at = dev(rng.integers(0, width, tokens))
    outs = []
    for one_at_a_time in (True, False):
        a, b = (QuantizedKvCache(ctx, 1, heads, dim, 4, tokens, bits) for _ in range(2))
        rows = torch.zeros((2, tokens, width), device="cuda")
        qs = torch.zeros((rounds + 1, 1, width), device="cuda")
        qs[0] = q
        scores = []
        torch.cuda.synchronize()
        for i in range(rounds):
            for call in (lambda: a.reset(0), lambda: a.prefill(0, x[i], x[rounds - 1 - i]),
                         lambda: a.read(0, 0, tokens, rows[0], rows[1]),
                         lambda: scores.append(token_logprobs_device(ctx, rows[0], at, 5)),
                         lambda: b.reset(0), lambda: b.prefill(0, rows[1], rows[0]),
                         lambda: b.attention(qs[i], qs[i + 1])):
                call()
                if one_at_a_time:
                    ctx.sync()
        ctx.sync()
        outs.append([host(qs)] + [host(t) for s in scores for t in s])
        a.free()
        b.free()
    assert all(np.array_equal(s, t) for s, t in zip(*outs))
    assert len({host_row.tobytes() for host_row in outs[0][0]}) == rounds + 1
