"""The quantised cache, the attention over it and the token log probabilities
as a decoder uses them: a prompt, then teacher-forced steps whose next tokens
are scored.  The steps are compared with the same device operations around an
attention computed in float64 from what the cache reads back, and the scores
with float64 log probabilities of the step's own logits."""
import numpy as np
import pytest

from test_gpu_decoder import small_config
from test_gpu_kv_quant import attention_ref, held
from test_gpu_logprobs import check

pytestmark = pytest.mark.gpu


def host(t):
    return t.detach().cpu().numpy()


def step_in_parts(dec, state, tokens_t, mode, heads, dim):
    """decode_step with the cache's attention in float64 (numpy)."""
    import torch
    from uocr_q8 import QuantizationMode as M
    from uocr_q8.attention import add_rms_norm_device, rms_norm_device
    from uocr_q8.decoder import feed_forward_device, linear_bf16_device
    ctx, cfg = dec.ctx, dec.cfg
    dyn = mode != M.WEIGHTS_ONLY
    mode = M.DYNAMIC_ROWWISE if dyn else M.WEIGHTS_ONLY
    x = dec.embedding.index_select(0, tokens_t).float()
    y = None
    for layer, cache in zip(dec.layers, state.caches):
        n = (rms_norm_device(ctx, x, layer.input_norm, cfg.eps) if y is None
             else add_rms_norm_device(ctx, x, y, layer.input_norm, cfg.eps, sum_t=x))
        q = cache.rope_push_qkv(state.rope, layer.qkv.linear_device(n, dynamic=dyn))
        a = []
        for b in range(len(tokens_t)):
            k, v = (host(t).reshape(-1, heads, dim) for t in cache.export(b))
            (k, v) = ((t.astype(np.float64), *held(t, cache.bits)[1:]) for t in (k, v))
            a.append(attention_ref(host(q[b]), k, v, heads)[0])
        a = torch.from_numpy(np.stack(a).astype(np.float32)).cuda()
        r = layer.o.linear_device(a, dynamic=dyn)
        n = add_rms_norm_device(ctx, r, x, layer.post_norm, cfg.eps, sum_t=r)
        if layer.moe is not None:
            y = layer.moe.forward_device(n, linear_bf16_device(ctx, layer.router, n), mode)
        else:
            y = feed_forward_device(ctx, *layer.dense, n, mode)
        x = r
    h = add_rms_norm_device(ctx, x, y, dec.final_norm, cfg.eps, sum_t=x)
    return dec.lm_head.linear_device(h, dynamic=dyn)


@pytest.mark.parametrize("bits", [4, 8])
def test_scored_steps(ctx, bits):
    import torch
    from uocr_q8.decoder import DecodeState, Decoder, decode_step, prefill, score_step
    cfg = small_config()
    dec = Decoder.random(ctx, cfg, seed=1)
    batch, steps, lengths = 2, cfg.window + 3, (5, 40)
    rng = np.random.default_rng(bits)
    states = [DecodeState(dec, batch, 40, kv_bits=bits) for _ in range(2)]
    full = DecodeState(dec, batch, 40)
    for b, n in enumerate(lengths):
        emb = torch.from_numpy(rng.standard_normal((n, cfg.hidden)).astype(np.float32)).cuda()
        first = [host(prefill(dec, s, emb, 0, b)) for s in (*states, full)]
        # a prompt attends to its own FP32 rows: its logits do not depend on the cache
        assert np.array_equal(first[0], first[1])
        assert np.max(np.abs(first[0] - first[2])) <= 1e-5 * np.max(np.abs(first[2]))
    tokens = rng.integers(0, cfg.vocab, (steps + 1, batch))
    far = []
    for i in range(steps):
        now, nxt = (torch.from_numpy(t).cuda() for t in tokens[i:i + 2])
        logits = torch.empty((batch, cfg.vocab), device="cuda")
        got = score_step(dec, states[0], now, nxt, 0, 7, logits)
        ctx.sync()
        want = host(step_in_parts(dec, states[1], now, 0, cfg.heads, cfg.head_dim))
        # FP32 projections of rows that differ in the last bits of the attention
        assert np.max(np.abs(host(logits) - want)) <= 2e-4 * np.max(np.abs(want)), i
        check(ctx, host(logits), tokens[i + 1], 7, got)
        plain = host(decode_step(dec, full, now, 0))
        far.append(np.linalg.norm(host(logits) - plain) / np.linalg.norm(plain))
    assert states[0].caches[0].state(1) == (40 + cfg.window, 40 + steps)
    assert max(far) > 0  # the cache is not the FP32 one
    for s in (*states, full):
        s.free()
