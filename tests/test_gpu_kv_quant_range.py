"""GPU tests of the attention over a quantised cache where tokens, scores and
values are of very different sizes, against the definition in 64 bits (numpy)."""
import numpy as np
import pytest

from test_gpu_kv_quant import QuantizedKvCache, check_attention, dev, held, host, run_attention

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def reference(q, k, v):
    """softmax(q K^T / sqrt(d)) V in float64 of one query [heads, dim] over what the
    cache holds (`held`'s triples), and its tolerance.

    A score that is off by e_t moves the result by p_t e_t (v_t - out).  e_t: some 48
    roundings of parts of |q| (s code + |m|) (A_t) that add up like a walk, 3 sigma =
    12 steps of A_t; the argument of exp, R below the maximum, is rounded twice (2 R);
    exp, the products and the joins are 16 steps and the sums walk, 3 sqrt(T).  All in
    steps of 2^-24 and weighed by the token's own p_t: a token of no weight adds
    nothing, whatever its values are.  Weights, and the factors that join parts, below
    the smallest normal float, 2^-126, are lost; they stand to a maximum that is
    passed by 2^2 at most: 2^-124 of the values' sizes."""
    (kv, ks, km), (vv, vs, vm) = k, v
    tokens, _, dim = kv.shape
    q = q.astype(np.float64)
    scores = np.einsum("thd,hd->ht", kv, q) / np.sqrt(dim)
    gap = scores.max(-1, keepdims=True) - scores
    p = np.exp(-gap)
    p /= p.sum(-1, keepdims=True)
    size = np.einsum("thd,hd->ht", (kv - km) + np.abs(km), np.abs(q)) / np.sqrt(dim)
    out = np.einsum("ht,thd->hd", p, vv)
    e = EPS * (12 * size + 2 * gap + 16 + 3 * np.sqrt(tokens))
    terms = (vv - vm) + np.abs(vm)
    tol = np.einsum("ht,thd->hd", p * e, terms) + (p * e).sum(-1)[:, None] * np.abs(out)
    tol += 2.0 ** -124 * terms.sum(0)
    return out, tol


def with_low_scores(rng, heads, dim, tokens, low, depth):
    """A query and keys whose tokens `low` score `depth` below zero, the others
    around it."""
    q = rng.standard_normal((heads, dim)).astype(np.float32)
    k = (0.5 * rng.standard_normal((tokens, heads, dim))).astype(np.float32)
    k[low] = -q * (depth * np.sqrt(dim) / (q * q).sum(-1, keepdims=True))
    return q, k


def check(kv, seq, q, out, heads, dim, bits):
    k, v = (host(t).reshape(-1, heads, dim) for t in kv.export(seq))
    k, v = ((x.astype(np.float64), *held(x, bits)[1:]) for x in (k, v))
    ref, tol = reference(q, k, v)
    off = np.abs(out.reshape(heads, dim) - ref)
    assert np.all(off <= tol), (seq, np.max(off / tol), np.max(off) / np.max(np.abs(ref)))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("ratio,depth", [(1e4, 45), (1e6, 45), (1e12, 60), (1e25, 110)])
@pytest.mark.parametrize("where", ["first", "middle", "last", "pushed", "every tile"])
def test_large_values_of_no_weight(ctx, bits, ratio, depth, where):
    """Tokens whose values are far larger than the others', and whose weight is
    nothing, leave the others' results as they are."""
    rng = np.random.default_rng(int(depth) + bits + len(where))
    heads, dim, tokens, pushes = 3, 96, 500, 4
    low = {"first": [3], "middle": [250, 251], "last": [499], "pushed": [501],
           "every tile": list(range(5, 500, 32))}[where]
    for batch in (1, 160):  # a head spread over clusters, and one CTA per head
        q, k = with_low_scores(rng, heads, dim, tokens + pushes, low, depth)
        v = rng.standard_normal(k.shape).astype(np.float32)
        v[low, :, :64] *= np.float32(ratio)  # (the third group is an ordinary one)
        kv = QuantizedKvCache(ctx, batch, heads, dim, pushes, tokens, bits)
        rows = [dev(x.reshape(tokens + pushes, -1)) for x in (k, v)]
        for b in range(batch):
            kv.prefill(b, rows[0][:tokens], rows[1][:tokens])
        for i in range(tokens, tokens + pushes):
            kv.push(*(x[i:i + 1].repeat(batch, 1) for x in rows))
        out = host(kv.attention(dev(np.repeat(q.reshape(1, -1), batch, 0))))
        ctx.sync()
        check(kv, batch - 1, q, out[batch - 1], heads, dim, bits)
        assert np.array_equal(out, np.repeat(out[:1], batch, 0))
        kv.free()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("step", [1.5, -1.5, 1.0, -1.0, 0.07, -0.07])
def test_values_that_grow_and_shrink(ctx, bits, step):
    """Value sizes that rise or fall by a factor from token to token, far over the
    range of one fixed-point scale; some tokens' values are constant (no step)."""
    rng = np.random.default_rng(int(100 * abs(step)) + bits)
    heads, dim, tokens = 2, 64, 100 if abs(step) >= 1 else 1500
    size = np.exp2(np.clip(step * (np.arange(tokens) - tokens / 2), -80, 80))
    v = (rng.standard_normal((tokens, heads, dim)) * size[:, None, None]).astype(np.float32)
    v[::7, :, :32] = v[::7, :, :1]
    q = (0.3 * rng.standard_normal((1, heads, dim))).astype(np.float32)
    # the smaller a token's values, the larger its weight: all take part
    k = rng.standard_normal((tokens, heads, dim)).astype(np.float32)
    want = -np.log(size)[:, None] * np.sqrt(dim) / (q[0] * q[0]).sum(-1)
    k = (0.1 * k + want[:, :, None] * q).astype(np.float32)
    for batch in (1, 250):
        kv = QuantizedKvCache(ctx, batch, heads, dim, 1, tokens, bits)
        for b in range(batch):
            kv.prefill(b, dev(k.reshape(tokens, -1)), dev(v.reshape(tokens, -1)))
        out = host(kv.attention(dev(np.repeat(q.reshape(1, -1), batch, 0))))
        ctx.sync()
        check(kv, batch - 1, q[0], out[batch - 1], heads, dim, bits)
        kv.free()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("lengths,heads,dim", [((1517,), 10, 128), ((300, 40, 999), 3, 80), ((700,) * 64, 10, 64)])
def test_ordinary_draws_closely(ctx, bits, lengths, heads, dim):
    """Normal keys, values and queries: 1e-5 of sum p (s code + |m|).  A score is
    summed from minus the maximum in some 30 roundings of parts that stay below 8 in
    size (powers of two): as a walk, 3 sigma, 3 sqrt(30 / 3) 2^-25 8 = 2.3e-6; the
    weights' change and that of their sum make it 4.6e-6, exp, products and joins
    1e-6, the walk of the sums 3 sqrt(1517) 2^-24 of it at most: 7e-6."""
    rng = np.random.default_rng(sum(lengths) + dim + bits)
    kv, q, out = run_attention(ctx, rng, lengths, heads, dim, bits, 16, 3, 1.0, "normal")
    for b in (0, len(lengths) - 1):
        k, v = (host(t).reshape(-1, heads, dim) for t in kv.export(b))
        vm = held(v, bits)[2]
        scores = np.einsum("thd,hd->ht", k.astype(np.float64), q[b].reshape(heads, dim).astype(np.float64))
        p = np.exp((scores - scores.max(-1, keepdims=True)) / np.sqrt(dim))
        p /= p.sum(-1, keepdims=True)
        ref = np.einsum("ht,thd->hd", p, v.astype(np.float64))
        terms = np.einsum("ht,thd->hd", p, (v - vm) + np.abs(vm))
        off = np.abs(out[b].reshape(heads, dim) - ref)
        assert np.all(off <= 1e-5 * terms), np.max(off / terms)
    check_attention(kv, q, out, heads, dim, bits)
    kv.free()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("size", [30.0, 1e3, 1e5])
def test_outlying_channels_of_the_query(ctx, bits, size):
    """One channel of a query is far larger than the rest, and the keys are nearly
    (or exactly) zero there: scores within 2^-19 of sum |q| (|m| + R) / sqrt(dim),
    which moves the result by twice that of sum p (|m| + R) at most."""
    rng = np.random.default_rng(int(size) + bits)
    heads, dim, tokens = 4, 80, 700
    k, v = (rng.standard_normal((tokens, heads, dim)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((heads, dim)).astype(np.float32)
    q[:, 5], q[:, 70] = size, -size
    k = np.abs(k)
    k[:, :, 5] = 0.0
    k[:, :2, 70] *= np.float32(1 / size)
    kv = QuantizedKvCache(ctx, 1, heads, dim, 1, tokens, bits)
    kv.prefill(0, dev(k.reshape(tokens, -1)), dev(v.reshape(tokens, -1)))
    out = host(kv.attention(dev(q.reshape(1, -1)))).reshape(heads, dim)
    ctx.sync()
    (kh, ks, km), (vh, vs, vm) = held(k, bits), held(v, bits)
    levels = 2 ** bits - 1
    scores = np.einsum("thd,hd->ht", kh, q.astype(np.float64)) / np.sqrt(dim)
    off = 2.0 ** -19 * np.einsum("thd,hd->ht", np.abs(km) + levels * ks, np.abs(q)) / np.sqrt(dim)
    p = np.exp(scores - scores.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    ref = np.einsum("ht,thd->hd", p, vh)
    terms = np.einsum("ht,thd->hd", p, np.abs(vm) + levels * vs)
    move = np.expm1(2 * off.max(-1, keepdims=True)) + EPS * (100 + 3 * np.sqrt(tokens))
    assert np.all(np.abs(out - ref) <= move * terms), np.max(np.abs(out - ref) / (move * terms))
    kv.free()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("where", ["one", "first tiles", "last tiles", "all but one", "all but a pushed one"])
def test_scores_below_the_least_float(ctx, bits, where):
    """Scores of -inf weigh nothing, wherever they lie: as if their tokens were not there."""
    rng = np.random.default_rng(len(where) + bits)
    heads, dim, tokens, pushes = 3, 64, 400, 2
    low = np.zeros(tokens + pushes, bool)
    low[{"one": slice(7, 8), "first tiles": slice(0, 200), "last tiles": slice(100, tokens + pushes),
         "all but one": slice(0, tokens + pushes), "all but a pushed one": slice(0, tokens + pushes)}[where]] = True
    if where.startswith("all"):
        low[tokens + 1 if "pushed" in where else 333] = False
    big = np.float32(2.0 ** 30)
    q = np.full((heads, dim), big)
    k, v = (rng.standard_normal((tokens + pushes, heads, dim)).astype(np.float32) for _ in range(2))
    k /= 4 * big
    k[low, 1:] = -np.float32(2.0 ** 99)  # (the first head has no such score)
    rows = [x.reshape(tokens + pushes, -1) for x in (k, v)]
    for batch in (1, 260):  # a head spread over clusters, and one CTA per head
        kv = QuantizedKvCache(ctx, batch, heads, dim, pushes, tokens, bits)
        for b in range(batch):
            kv.prefill(b, dev(rows[0][:tokens]), dev(rows[1][:tokens]))
        for i in range(tokens, tokens + pushes):
            kv.push(*(dev(np.repeat(x[i:i + 1], batch, 0)) for x in rows))
        out = host(kv.attention(dev(np.repeat(q.reshape(1, -1), batch, 0)))).reshape(batch, heads, dim)
        ctx.sync()
        for h, there in ((0, np.ones_like(low)), (1, ~low), (2, ~low)):
            parts = ([t[:, None] for t in map(lambda t: t[there, h], held(x, bits))] for x in (k, v))
            ref, tol = reference(q[h:h + 1], *parts)
            assert np.all(np.abs(out[-1, h] - ref[0]) <= tol[0]), (h, np.max(np.abs(out[-1, h] - ref[0]) / tol[0]))
        kv.free()


@pytest.mark.parametrize("sign,where", [(1.0, "one"), (1.0, "first tiles"), (1.0, "last"), (1.0, "all"), (-1.0, "all")])
def test_scores_that_are_not_finite(ctx, sign, where):
    """One score of +inf, or nothing but -inf: NaN for that head alone, and Numerical."""
    rng = np.random.default_rng(len(where))
    heads, dim, tokens = 3, 64, 400
    low = {"one": slice(7, 8), "first tiles": slice(0, 70), "last": slice(399, 400), "all": slice(0, 400)}[where]
    q = np.full((1, heads * dim), np.float32(2.0 ** 30))
    k, v = (rng.standard_normal((tokens, heads, dim)).astype(np.float32) for _ in range(2))
    k *= np.float32(2.0 ** -32)
    k[low, 1] = np.float32(sign * 2.0 ** 99)
    for batch in (1, 260):
        kv = QuantizedKvCache(ctx, batch, heads, dim, 1, tokens, 4)
        for b in range(batch):
            kv.prefill(b, dev(k.reshape(tokens, -1)), dev(v.reshape(tokens, -1)))
        out = host(kv.attention(dev(np.repeat(q, batch, 0)))).reshape(batch, heads, dim)
        import uocr_q8
        with pytest.raises(uocr_q8.OcrError) as e:
            ctx.sync()
        assert e.value.kind == "Numerical"
        assert np.all(np.isnan(out[:, 1])) and np.all(np.isfinite(out[:, ::2]))
        kv.free()
