"""GPU tests of the token log probabilities of rows whose terms are all alike:
running FP32 sums lose the same way at every step there, so that they show how
many terms are summed one after the other."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


@pytest.mark.parametrize("rows,vocab", [(1, 129280), (300, 129280), (1, 1 << 20), (300, (1 << 20) + 3), (1, (1 << 26) + 1),
                                        (1, 1 << 30)])
@pytest.mark.parametrize("below", [0.3, 1.1, 2.3, 4.5])
def test_flat_rows(ctx, rows, vocab, below):
    """One logit of 0, the others `below` it: S' = (V - 1) e^-below.  128 equal terms
    one after the other, each step rounded to 2^-24 of the sum so far, lose 64 steps of
    2^-24 of S' at most, in either of the sums; exp's argument is rounded twice and exp
    is good to 4 steps (2 below + 4), the joins of lanes, warps and CTAs are 16; the
    result's own roundings are 4 of it.  Of S' in log1p, and of the entropy's second
    term, w = S' below / (1 + S')."""
    import torch
    from uocr_q8.decoder import token_logprobs_device
    x = torch.full((rows, vocab), -below, device="cuda")
    top = (vocab * 5 // 7 + torch.arange(rows, device="cuda") * 1013) % vocab
    x[torch.arange(rows, device="cuda"), top] = 0.0
    got = token_logprobs_device(ctx, x, top, 2)
    ctx.sync()
    z = float(np.float32(below))
    s = (vocab - 1) * np.exp(-z)
    lse, w = np.log1p(s), s * z / (1 + s)
    steps = 64 + 2 * below + 4 + 16
    assert np.all(np.abs(got.logprob.double().cpu().numpy() + lse) <= EPS * (steps * min(1, s) + 4 * lse))
    # (w's numerator and 1 + S' err on their own)
    tol = EPS * (steps * min(1, s) + 2 * steps * w + 4 * (lse + w))
    assert np.all(np.abs(got.entropy.double().cpu().numpy() - lse - w) <= tol)
    ids = got.top_ids.cpu().numpy()
    assert np.array_equal(ids[:, 0], top.cpu().numpy())
    assert np.array_equal(ids[:, 1], np.where(ids[:, 0] == 0, 1, 0))


@pytest.mark.parametrize("rows,vocab", [(1, (1 << 24) + 5), (2, 3000001), (240, 600011)])
@pytest.mark.parametrize("kind", ["rising", "falling", "banned ends", "random"])
@pytest.mark.parametrize("top", [0, 5])
def test_long_rows(ctx, rows, vocab, kind, top):
    """Rows of many turns, whose running maximum moves at every one of them, late, or
    early.  Steps of 2^-24 of S': 64 serial ones, the terms' own 8, the joins' 16, and
    3 sqrt(turns) 4 for a factor good to 4 steps at every turn (at most vocab / 4096
    of them, an eighth of that where a row is spread over eight CTAs)."""
    import torch
    from uocr_q8.decoder import token_logprobs_device
    g = torch.Generator(device="cuda")
    g.manual_seed(vocab + len(kind))
    if kind in ("rising", "falling"):
        x = torch.linspace(-20, 0, vocab, device="cuda").repeat(rows, 1)
        if kind == "falling":
            x = x.flip(-1).contiguous()
    else:
        x = 2 * torch.randn((rows, vocab), generator=g, device="cuda")
        if kind == "banned ends":
            x[:, :vocab * 2 // 5] = x[:, vocab * 4 // 5:] = -np.inf
    at = torch.randint(vocab // 2, vocab * 3 // 4, (rows,), generator=g, device="cuda")
    got = token_logprobs_device(ctx, x, at, top)
    ctx.sync()
    for r in (0, rows - 1):
        y = x[r].double()
        z = y - y.max()
        e = z.exp()
        s = float(e.sum()) - 1
        w = float(-(e * z.clamp_min(-1e3)).sum()) / (1 + s)
        lse = np.log1p(s)
        steps = 64 + 8 + 16 + 12 * np.sqrt(vocab / 4096 / (8 if rows < 50 else 1))
        tol = EPS * (steps * min(1, s) + 4 * lse)
        assert abs(float(got.logprob[r]) - (float(z[at[r]]) - lse)) <= tol + 2 * EPS * -float(z[at[r]])
        assert abs(float(got.entropy[r]) - (lse + w)) <= tol + EPS * (2 * steps + 4) * w
        best = torch.sort(x[r], descending=True, stable=True)
        assert torch.equal(got.top_ids[r], best.indices[:top])
        assert np.all(np.abs(got.top_logprobs[r].double().cpu().numpy() - (best.values[:top].double() - y.max()).cpu().numpy()
                             + lse) <= tol + 2 * EPS * 25)


def test_long_rows_that_say_nothing(ctx):
    """NaN far from either end of a long row; nothing but -inf."""
    import torch
    import uocr_q8
    from uocr_q8.decoder import token_logprobs_device
    x = torch.zeros((3, 5000001), device="cuda")
    x[0, 2345678] = np.nan
    x[1] = -np.inf
    got = token_logprobs_device(ctx, x, torch.zeros(3, dtype=torch.int64, device="cuda"), 2)
    with pytest.raises(uocr_q8.OcrError) as e:
        ctx.sync()
    assert e.value.kind == "Numerical"
    assert torch.isnan(got.logprob[:2]).all() and torch.isnan(got.entropy[:2]).all()
    assert (got.top_ids[:2] == -1).all() and got.top_ids[2].tolist() == [0, 1]
    assert abs(float(got.logprob[2]) + np.log(5000001)) <= 1e-5
