"""Failure detection on the GPU without a GPU fault: waits for bulk copies that
run out (uocr_ctx_hold_copies makes every barrier wait for an arrival that never
comes, with a short uocr_ctx_set_wait_limit).  The launches return, the outputs
are NaN (ids -1) and the next synchronising call reports Timeout; after it the
same calls give the bits they gave before."""
import numpy as np
import pytest

from test_gpu_kv_quant import QuantizedKvCache, dev, host, raises

pytestmark = pytest.mark.gpu


def held_between(ctx, call, lost):
    before = [host(t) for t in call()]
    ctx.sync()
    ctx.set_wait_limit(0.002)
    ctx.hold_copies(True)
    got = call()
    raises("Timeout", ctx.sync)
    lost([host(t) for t in got])
    ctx.hold_copies(False)
    ctx.set_wait_limit(0)
    after = [host(t) for t in call()]
    ctx.sync()
    assert all(np.array_equal(x, y) for x, y in zip(before, after))


# rows of one CTA and of clusters; fewer copies than ring slots, and many
@pytest.mark.parametrize("rows,vocab", [(1, 2000), (2, 129280), (400, 9001)])
@pytest.mark.parametrize("top", [0, 20])
def test_logits_that_do_not_arrive(rows, vocab, top):
    import uocr_q8
    from uocr_q8.decoder import token_logprobs_device
    ctx = uocr_q8.GpuContext(0)
    rng = np.random.default_rng(vocab)
    x = dev(rng.standard_normal((rows, vocab)).astype(np.float32))
    tokens = dev(rng.integers(0, vocab, rows))

    def lost(got):
        logprob, entropy, ids, logprobs = got
        assert np.all(np.isnan(logprob)) and np.all(np.isnan(entropy)) and np.all(np.isnan(logprobs))
        assert np.all(ids == -1)
    held_between(ctx, lambda: token_logprobs_device(ctx, x, tokens, top), lost)
    ctx.close()


@pytest.mark.parametrize("batch,tokens,dim,bits", [(1, 40, 32, 4), (1, 9000, 128, 4), (100, 300, 64, 8)])
def test_tiles_that_do_not_arrive(batch, tokens, dim, bits):
    import uocr_q8
    ctx = uocr_q8.GpuContext(0)
    rng = np.random.default_rng(tokens)
    kv = QuantizedKvCache(ctx, batch, 4, dim, 1, tokens, bits)
    x = dev(rng.standard_normal((tokens, 4 * dim)).astype(np.float32))
    for b in range(batch):
        kv.prefill(b, x, x)
    q = dev(rng.standard_normal((batch, 4 * dim)).astype(np.float32))
    held_between(ctx, lambda: [kv.attention(q)], lambda got: np.testing.assert_(np.all(np.isnan(got[0]))))
    kv.free()
    ctx.close()
