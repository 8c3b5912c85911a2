"""GPU tests of the token log probabilities of rows with one token that is nearly
certain: the relative precision of what is left."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


@pytest.mark.parametrize("vocab", [2, 3, 17, 1000, 40000])
@pytest.mark.parametrize("scale", [1.0, 1e-3, 1e4])
def test_what_is_left(ctx, vocab, scale):
    """Logits of any size, the second largest 4 to 85 below the largest.  A term e^z is
    off by 2.25 |z| + 4 steps of 2^-24 (z rounded: |z|; z log2 e rounded twice: 1.25 |z|
    at most; exp2: 4), sums and joins by 64 + 16, log1p and the last product by 8.  The
    entropy is log1p(S') + w, w = sum e^z |z| / (1 + S'): the same steps of w, and 2 of
    each product."""
    import torch
    from uocr_q8.decoder import token_logprobs_device
    rng = np.random.default_rng(vocab + int(scale))
    rows = 200
    x = rng.standard_normal((rows, vocab)) * scale
    gap = rng.uniform(4, 85, rows)
    x = x - x.max(-1, keepdims=True) - gap[:, None]
    at = rng.integers(0, vocab, rows)
    x[np.arange(rows), at] = 0.0
    x = (x + rng.standard_normal((rows, 1)) * scale).astype(np.float32)
    at = x.argmax(-1)
    got = token_logprobs_device(ctx, torch.from_numpy(x).cuda(), torch.from_numpy(at).cuda(), min(2, vocab))
    ctx.sync()
    z = x.astype(np.float64) - x.max(-1, keepdims=True)
    e = np.exp(z)
    e[np.arange(rows), at] = 0
    far = (e * (2.25 * -z + 4)).sum(-1), (e * -z * (2.25 * -z + 4)).sum(-1)
    s = e.sum(-1)
    w = (e * -z).sum(-1)
    # (terms below the smallest normal float may be lost)
    lost = 2.0 ** -126 * vocab
    tol = EPS * (far[0] + 88 * s) + lost
    assert np.all(np.abs(got.logprob.double().cpu().numpy() + np.log1p(s)) <= tol)
    tol_h = tol + EPS * (far[1] + 92 * w) + w * tol + 100 * lost
    assert np.all(np.abs(got.entropy.double().cpu().numpy() - np.log1p(s) - w / (1 + s)) <= tol_h)
    assert np.array_equal(got.top_ids.cpu().numpy(), np.argsort(-x, -1, kind="stable")[:, :min(2, vocab)])
