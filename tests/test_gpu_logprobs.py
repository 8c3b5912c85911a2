"""GPU tests of the token log probabilities, against float64 (numpy).

Tolerances count roundings of 2^-24: z = x - M is rounded once (2 |z| with the
final sum's), log1p and the differences are good to 2 steps of their result
(4 lse); S' is a sum of exponentials that are each off by at most 4 steps of
exp and by |z| steps of its argument (|z| e^z <= 0.37 of the largest term),
and whose tree of sums adds a handful: 32 steps of S', which move the log by at
most 32 min(1, S') of them.  The entropy's second term is a sum of the same
exponentials times |z|: 32 steps of it.  A walk over a vocabulary of V terms
in partial sums of V / 256 serial ones adds sqrt(V) / 16 steps.  Terms below the
smallest normal float may be lost: at most V 2^-126 (1 + 88) < 1e-30 in all.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def logprobs(ctx, logits, tokens=None, top=0):
    import torch
    from uocr_q8.decoder import token_logprobs_device
    t = logits if isinstance(logits, torch.Tensor) else torch.from_numpy(
        np.ascontiguousarray(logits, np.float32)).cuda()
    k = None if tokens is None else torch.from_numpy(np.asarray(tokens, np.int64)).cuda()
    return token_logprobs_device(ctx, t, k, top)


def host(t):
    return t.detach().cpu().numpy()


def reference(x):
    """(log p, entropy, tolerance of log p, tolerance of the entropy), float64."""
    x = x.astype(np.float64)
    z = x - x.max(-1, keepdims=True)
    first = x.argmax(-1)
    e = np.exp(z)
    e[np.arange(len(x)), first] = 0.0
    s = e.sum(-1, keepdims=True)
    lse = np.log1p(s)
    w = -(e * np.maximum(z, -1e3)).sum(-1, keepdims=True) / (1 + s)
    walk = np.sqrt(x.shape[-1]) / 16
    tol = (4 * lse + (32 + walk) * np.minimum(1, s)) * EPS + 1e-30
    return (z - lse, (lse + w)[:, 0], tol + 2 * EPS * np.where(np.isfinite(z), -z, 0),
            (tol + (32 + walk) * w * EPS)[:, 0])


def check(ctx, x, tokens, top, got=None):
    x = np.asarray(x, np.float32)
    rows, vocab = x.shape
    got = got or logprobs(ctx, x, tokens, top)
    ctx.sync()
    logp, entropy, tol, tol_h = reference(x)
    assert np.all(np.abs(host(got.entropy) - entropy) <= tol_h), np.max(np.abs(host(got.entropy) - entropy) / tol_h)
    if tokens is not None:
        at = np.arange(rows), np.maximum(tokens, 0)
        want, lp = logp[at], host(got.logprob)
        none = np.asarray(tokens) < 0
        assert np.all(lp[none] == 0)
        banned = ~none & ~np.isfinite(want)
        assert np.all(lp[banned] == -np.inf)
        live = ~none & ~banned
        assert np.all(np.abs(lp[live] - want[live]) <= tol[at][live])
    order = np.argsort(-x, axis=-1, kind="stable")[:, :top]
    assert np.array_equal(host(got.top_ids), order)
    for r in range(rows):
        want, lp = logp[r, order[r]], host(got.top_logprobs)[r]
        fine = np.isfinite(want)
        assert np.array_equal(fine, np.isfinite(lp)) and np.all(lp[~fine] == -np.inf)
        assert np.all(np.abs(lp[fine] - want[fine]) <= tol[r, order[r]][fine])


@pytest.mark.parametrize("top", [0, 1, 5, 32])
@pytest.mark.parametrize("rows,vocab", [(1, 33), (3, 255), (2, 4096), (5, 4097), (70, 1000), (1, 129280),
                                        (9, 50021), (300, 2047), (1, 300001), (2, 1048577)])
def test_random_rows(ctx, rows, vocab, top):
    rng = np.random.default_rng(rows + vocab + top)
    x = 3 * rng.standard_normal((rows, vocab))
    check(ctx, x, rng.integers(0, vocab, rows), top)


@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 32])
def test_small_vocabularies(ctx, vocab):
    """Every logit among the alternatives; one token is certain."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((4, vocab))
    check(ctx, x, rng.integers(0, vocab, 4), vocab)


@pytest.mark.parametrize("vocab", [50, 5000, 129280])
@pytest.mark.parametrize("kind", ["ties", "equal", "up", "down", "one stripe", "zeros of both signs"])
def test_orders_and_ties(ctx, vocab, kind):
    """Equal logits go to the lower id, in any arrangement."""
    rng = np.random.default_rng(vocab)
    x = np.round(rng.standard_normal((2, vocab)) * 2) / 2
    if kind == "equal":
        x[:] = 1.5
    elif kind == "up":
        x = np.sort(rng.standard_normal((2, vocab)), -1)
    elif kind == "down":
        x = -np.sort(rng.standard_normal((2, vocab)), -1)
    elif kind == "one stripe":  # the largest lie 256 apart, those of one thread in many layouts
        x[:, 3::256] += 50
    elif kind == "zeros of both signs":
        x = np.where(rng.random((2, vocab)) < 0.5, -0.0, 0.0)
    check(ctx, x, rng.integers(0, vocab, 2), 32)


@pytest.mark.parametrize("share", [0.5, 0.99])
def test_banned_tokens(ctx, share):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, 9000))
    x[rng.random(x.shape) < share] = -np.inf
    x[:, 17] = 0.25
    x[4] = -np.inf
    x[4, 8999] = -3.0  # a single token is left
    check(ctx, x, rng.integers(0, 9000, 6), 32)


def test_banned_runs(ctx):
    """Whole stretches of a row banned, its lowest finite value among the rest."""
    x = np.full((3, 40000), -np.inf)
    x[0, :100] = np.arange(100)
    x[1, 39900:] = -np.arange(100)
    x[2, 20000:20007] = np.finfo(np.float32).min
    check(ctx, x, [3, 39950, 20003], 32)


def test_nearly_certain(ctx):
    """log p near 0 and an entropy near 0 keep their relative precision."""
    x = np.zeros((4, 1000))
    x[:, 500] = [5.0, 20.0, 40.0, 80.0]
    got = logprobs(ctx, x, [500] * 4, 2)
    check(ctx, x, [500] * 4, 2, got)
    s = 999 * np.exp(-x[:, 500])
    assert np.all(np.abs(host(got.logprob) + np.log1p(s)) <= 2.0 ** -18 * s)
    assert np.all(np.abs(host(got.entropy) / (np.log1p(s) + s * x[:, 500] / (1 + s)) - 1) <= 2.0 ** -18)


@pytest.mark.parametrize("shift", [-3e4, 3e4, 3e38])
def test_large_logits(ctx, shift):
    rng = np.random.default_rng(2)
    x = (shift + np.abs(shift) / 64 * rng.standard_normal((2, 3000))).clip(-3.4e38, 3.4e38)
    x[0, :4] = x[0].max()
    check(ctx, x, [0, 5], 8)


def test_rows_apart_and_without_tokens(ctx):
    import torch
    rng = np.random.default_rng(3)
    for pad, first in ((0, 0), (1, 0), (3, 1), (8, 5)):
        wide = torch.from_numpy(rng.standard_normal((7, 5000 + pad + first)).astype(np.float32)).cuda()
        x = wide[:, first:first + 5000]
        tokens = np.array([0, 4999, -1, 17, -1, -9, 2500])
        check(ctx, host(x), tokens, 4, logprobs(ctx, x, tokens, 4))
        check(ctx, host(x), None, 3, logprobs(ctx, x, None, 3))
    none = logprobs(ctx, torch.empty((0, 100), device="cuda"), [], 3)
    assert none.top_ids.shape == (0, 3)


@pytest.mark.parametrize("bad", [np.nan, np.inf, None])
@pytest.mark.parametrize("vocab", [100, 20000])
def test_rows_that_say_nothing(ctx, bad, vocab):
    import uocr_q8
    rng = np.random.default_rng(4)
    x = rng.standard_normal((5, vocab)).astype(np.float32)
    if bad is None:
        x[2] = -np.inf
    else:
        x[2, vocab * 2 // 3] = bad
    got = logprobs(ctx, x, [1] * 5, 6)
    with pytest.raises(uocr_q8.OcrError) as e:
        ctx.sync()
    assert e.value.kind == "Numerical"
    assert all(np.isnan(host(t)[2]).all() for t in (got.logprob, got.entropy, got.top_logprobs))
    assert np.all(host(got.top_ids)[2] == -1)
    rest = [0, 1, 3, 4]
    check(ctx, x[rest], [1] * 4, 6, type(got)(*(t[rest] for t in got)))


def test_refusals(ctx):
    import torch
    import uocr_q8
    x = torch.zeros((2, 50), device="cuda")
    t = torch.zeros(2, dtype=torch.int64, device="cuda")

    def kind(*a):
        from uocr_q8.decoder import token_logprobs_device
        with pytest.raises(uocr_q8.OcrError) as e:
            token_logprobs_device(ctx, *a)
        return e.value.kind
    assert kind(x, t, 33) == "Unsupported"
    assert kind(x[:, :20], t, 21) == "Shape"
    assert kind(x, t, -1) == "Shape"
    assert kind(x[:, :0], t, 0) == "Shape"
    for bad in (x.half(), x.cpu(), x[0], x.t().contiguous().t(), x[:, ::2]):
        assert kind(bad, t, 1) == "Shape"
    for bad in (t.int(), t[:1], t.cpu(), torch.zeros(4, dtype=torch.int64, device="cuda")[::2]):
        assert kind(x, bad, 1) == "Shape"
    got = logprobs(ctx, host(x), [50, 1], 2)
    with pytest.raises(uocr_q8.OcrError) as e:
        ctx.sync()
    assert e.value.kind == "Shape"
    assert np.isnan(host(got.logprob)[0]) and abs(host(got.logprob)[1] + np.log(50)) < 1e-5


def test_captured(ctx):
    """Captured once, replayed on other logits."""
    import torch
    rng = np.random.default_rng(5)
    x = torch.zeros((3, 30000), device="cuda")
    tokens = torch.zeros(3, dtype=torch.int64, device="cuda")
    from uocr_q8.decoder import token_logprobs_device
    back, side, graph = torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    ctx.set_stream(side)
    try:
        with torch.cuda.graph(graph, stream=side):
            got = token_logprobs_device(ctx, x, tokens, 9)
        for _ in range(3):
            new, at = rng.standard_normal((3, 30000)).astype(np.float32), rng.integers(0, 30000, 3)
            x.copy_(torch.from_numpy(new))
            tokens.copy_(torch.from_numpy(at))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            check(ctx, new, at, 9, got)
    finally:
        ctx.set_stream(back)
        del graph


def test_repeatable(ctx):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((20, 129280)).astype(np.float32)
    first = [host(t) for t in logprobs(ctx, x, [5] * 20, 20)]
    for _ in range(3):
        assert all(np.array_equal(a, host(b)) for a, b in zip(first, logprobs(ctx, x, [5] * 20, 20)))
