"""GPU tests of the KV cache held in 4 or 8 bits and of the attention over it,
against the definitions in 64 bits (numpy).

What a cache holds is compared exactly: codes are decided in 64 bits, and what
is read back is m + s * code rounded once.  Attention is FP32 with another
order of sums; its tolerance is derived in `attention_ref`.
"""
import numpy as np
import pytest

import oracle

pytestmark = pytest.mark.gpu


def QuantizedKvCache(*a):
    from uocr_q8.attention import QuantizedKvCache as Q
    return Q(*a)


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    return t.detach().cpu().numpy()


def raises(kind, call):
    import uocr_q8
    with pytest.raises(uocr_q8.OcrError) as e:
        call()
    assert e.value.kind == kind, e.value


# ---- the definition ---------------------------------------------------------------
def bf16_at_most(x):
    """Largest bf16 <= x (float32 values in, float64 out)."""
    u = np.float32(x).view(np.uint32)
    down = np.where(u >> 31, u + 0xFFFF, u) & np.uint32(0xFFFF0000)
    return down.astype(np.uint32).view(np.float32).astype(np.float64)


def bf16_at_least(t):
    """Smallest bf16 >= t (float64 values >= 0)."""
    f = t.astype(np.float32)
    f = np.where(f.astype(np.float64) < t, np.nextafter(f, np.float32(np.inf)), f).astype(np.float32)
    return ((f.view(np.uint32) + 0xFFFF) & np.uint32(0xFFFF0000)).astype(np.uint32).view(
        np.float32).astype(np.float64)


def held(x, bits):
    """(value in float64, step, least value per dim) of x [..., dim] float32."""
    levels = 2 ** bits - 1
    out, steps, least = (np.empty(x.shape, np.float64) for _ in range(3))
    for d in range(0, x.shape[-1], 32):
        g = x[..., d:d + 32]
        m = bf16_at_most(g.min(-1, keepdims=True))
        s = bf16_at_least((g.max(-1, keepdims=True).astype(np.float64) - m) / levels)
        with np.errstate(divide="ignore", invalid="ignore"):
            c = np.rint((g.astype(np.float64) - m) / s)
        c = np.clip(np.where(s > 0, c, 0), 0, levels)
        out[..., d:d + 32] = m + s * c
        steps[..., d:d + 32], least[..., d:d + 32] = s, m
    return out, steps, least


def attention_ref(q, k, v, heads):
    """softmax(q K^T / sqrt(d)) V in float64 of one query row over what a cache
    holds (k, v: `held`'s triples of [tokens, heads, dim]), and the tolerance.

    A score sums 2 dim terms of size |q| s code and |q| |m| (A in all), each
    sum rounded to 2^-24 of it: some 48 roundings in a row, whose errors add up
    like a walk, 3 sigma = 3 sqrt(48 / 3) = 12 steps of 2^-24 A.  A score that is
    off by e changes its weight by e and the sum of weights by at most as much:
    24 A.  exp's argument, score minus maximum (R), is rounded twice: 2 R; exp
    itself, the products and the joins: 16.  The weighted sum over T tokens walks
    as well: 3 sqrt(T).  All relative to sum p (s code + |m|)."""
    kv, ks, km = k
    vv, vs, vm = v
    tokens, _, dim = kv.shape
    q = q.reshape(heads, dim).astype(np.float64)
    scores = np.einsum("thd,hd->ht", kv, q) / np.sqrt(dim)
    p = np.exp(scores - scores.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    size = np.einsum("thd,hd->ht", (kv - km) + np.abs(km), np.abs(q)) / np.sqrt(dim)
    out = np.einsum("ht,thd->hd", p, vv)
    terms = np.einsum("ht,thd->hd", p, (vv - vm) + np.abs(vm))
    span = scores.max(-1) - scores.min(-1)
    tol = 2.0 ** -24 * (24 * size.max(-1) + 2 * span + 16 + 3 * np.sqrt(tokens))[:, None] * terms
    return out.reshape(-1), tol.reshape(-1)


def rows_of(rng, kind, tokens, heads, dim):
    x = rng.standard_normal((tokens, heads, dim))
    if kind == "offset":      # a group far from zero
        x = x * 0.01 + 100.0 * rng.standard_normal((tokens, heads, 1))
    elif kind == "constant":
        x = np.repeat(rng.standard_normal((tokens, heads, 1)), dim, -1)
    elif kind == "zero":
        x = x * 0.0
    elif kind == "tiny":      # steps below the smallest normal float
        x = x * 1e-39
    elif kind == "huge":
        x = x * 1e29
    elif kind == "mixed":     # channels of very different sizes
        x = x * np.exp(4 * rng.standard_normal((1, heads, dim)))
    elif kind == "borders":   # quotients on, and next to, the border between two codes
        x = rng.integers(0, 31, (tokens, heads, dim)) * 0.5
        x[..., 0], x[..., -1] = 0.0, 15.0
        x = np.where(rng.random(x.shape) < 0.5, x, np.nextafter(x.astype(np.float32), np.float32(1e9)))
    return x.astype(np.float32).reshape(tokens, heads * dim)


# ---- writing and reading back -------------------------------------------------------
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("tokens,heads,dim", [
    (1, 1, 1), (2, 3, 2), (5, 2, 31), (33, 1, 32), (31, 2, 33), (32, 3, 64), (100, 3, 80),
    (70, 2, 96), (40, 1, 127), (257, 10, 128), (33, 2, 129), (65, 1, 160), (34, 2, 200), (64, 2, 256)])
def test_prompt_reads_back(ctx, bits, tokens, heads, dim):
    rng = np.random.default_rng(tokens * 1000 + dim + bits)
    k, v = (rows_of(rng, "normal", tokens, heads, dim) for _ in range(2))
    kv = QuantizedKvCache(ctx, 1, heads, dim, 3, tokens, bits)
    kv.prefill(0, dev(k), dev(v))
    ko, vo = kv.read(0, 0, tokens)
    ctx.sync()
    for x, o in ((k, ko), (v, vo)):
        ref = held(x.reshape(tokens, heads, dim), bits)[0].reshape(tokens, -1)
        assert np.array_equal(host(o), ref.astype(np.float32))
    kv.free()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kind", ["offset", "constant", "zero", "tiny", "huge", "mixed", "borders"])
def test_values_read_back(ctx, bits, kind):
    rng = np.random.default_rng(len(kind) + bits)
    tokens, heads, dim = 150, 2, 112
    x = rows_of(rng, kind, tokens, heads, dim)
    kv = QuantizedKvCache(ctx, 1, heads, dim, 3, tokens, bits)
    kv.prefill(0, dev(x), dev(-x))
    for y, o in zip((x, -x), kv.read(0, 0, tokens)):
        ref, step, _ = (t.reshape(tokens, -1) for t in held(y.reshape(tokens, heads, dim), bits))
        assert np.array_equal(host(o), ref.astype(np.float32))
        # the code is the nearest: half a step, and the rounding of the value itself
        assert np.all(np.abs(host(o) - y.astype(np.float64))
                      <= step / 2 * (1 + 2.0 ** -40) + np.abs(ref) * 2.0 ** -24)
    ctx.sync()
    kv.free()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [33, 37, 65, 97])
def test_one_small_step_beside_others(ctx, bits, dim):
    """A group of few dims whose step is far below every other token's."""
    rng = np.random.default_rng(dim + bits)
    x = rng.standard_normal((64, 1, dim)).astype(np.float32)
    for t in range(64):
        if t % 4 == (t // 4) % 4:
            x[t, :, dim // 32 * 32:] = np.float32(2.0 ** -100) * (1 + np.arange(1, dim % 32 + 1) * np.float32(2.0 ** -10))
    rows = dev(x.reshape(64, -1))
    kv = QuantizedKvCache(ctx, 1, 1, dim, 1, 64, bits)
    kv.prefill(0, rows, rows)
    for got in kv.read(0, 0, 64):
        ctx.sync()
        assert np.array_equal(host(got), held(x, bits)[0].reshape(64, -1).astype(np.float32))
    kv.free()


def test_storage_bytes(ctx):
    """bits + 1 bits a dim at whole groups, in whole tiles of 32 tokens."""
    for bits in (4, 8):
        kv = QuantizedKvCache(ctx, 2, 10, 128, 128, 1920, bits)
        assert kv.storage_bytes() == 2 * 2 * 10 * 2048 * 128 * (bits + 1) // 8
        kv.free()


@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("heads,dim", [(2, 128), (3, 20), (2, 33)])
def test_rows_apart_and_unaligned(ctx, shift, heads, dim):
    """Slices of wider rows, starting at any float."""
    import torch
    rng = np.random.default_rng(dim + shift)
    tokens, width = 37, heads * dim
    wide = rng.standard_normal((tokens, 2 * width + 7)).astype(np.float32)
    t = dev(wide)
    k, v = t[:, shift:shift + width], t[:, width + shift + 1:2 * width + shift + 1]
    kv = QuantizedKvCache(ctx, 1, heads, dim, 3, tokens, 4)
    kv.prefill(0, k, v)
    out = torch.full((tokens * width * 2 + 8,), -7.0, device="cuda")
    ko = out[shift:shift + tokens * width].view(tokens, width)
    vo = out[tokens * width + shift + 1:2 * tokens * width + shift + 1].view(tokens, width)
    kv.read(0, 0, tokens, ko, vo)
    kv.push(k[:1], v[:1])
    kp, vp = kv.read(0, tokens, 1)
    ctx.sync()
    for x, o, p in ((k, ko, kp), (v, vo, vp)):
        ref = held(host(x).reshape(tokens, heads, dim), 4)[0].reshape(tokens, -1).astype(np.float32)
        assert np.array_equal(host(o), ref)
        assert np.array_equal(host(p), ref[:1])
    rest = np.ones(out.numel(), bool)
    rest[shift:shift + tokens * width] = rest[tokens * width + shift + 1:2 * tokens * width + shift + 1] = False
    assert np.all(host(out)[rest] == -7.0)
    kv.free()


@pytest.mark.parametrize("bits", [4, 8])
def test_ring_of_pushed_tokens(ctx, bits):
    """Slots and counters as LayerCache: prefix + generated % window."""
    rng = np.random.default_rng(bits)
    batch, heads, dim, window, lengths = 3, 2, 80, 5, (1, 30, 33)
    kv = QuantizedKvCache(ctx, batch, heads, dim, window, 40, bits)
    ref = []
    for b, n in enumerate(lengths):
        k, v = (rng.standard_normal((n, heads * dim)).astype(np.float32) for _ in range(2))
        kv.prefill(b, dev(k), dev(v))
        ref.append((list(k), list(v)))
    for step in range(13):
        k, v = (rng.standard_normal((batch, heads * dim)).astype(np.float32) for _ in range(2))
        kv.push(dev(k), dev(v))
        for b, n in enumerate(lengths):
            for rows, new in zip(ref[b], (k[b], v[b])):
                slot = n + step % window
                rows[slot:slot + 1] = [new]
    for b, n in enumerate(lengths):
        assert kv.state(b) == (n + window, n + 13)
        for rows, got in zip(ref[b], kv.export(b)):
            x = np.stack(rows)
            want = held(x.reshape(len(rows), heads, dim), bits)[0].reshape(len(rows), -1)
            assert np.array_equal(host(got), want.astype(np.float32))
        # a part of them
        part = host(kv.read(b, n - 1, 3)[1])
        assert np.array_equal(part, host(kv.export(b)[1])[n - 1:n + 2])
    kv.free()


@pytest.mark.parametrize("heads,dim", [(10, 128), (3, 20), (1, 2)])
def test_rope_push_equals_rope_then_push(ctx, heads, dim):
    from uocr_q8.attention import Rope
    rng = np.random.default_rng(dim)
    batch, width = 4, heads * dim
    rope = Rope(ctx, dim, 10000.0, 300)
    caches = [QuantizedKvCache(ctx, batch, heads, dim, 2, 40, 4) for _ in range(2)]
    for b in range(batch):
        k, v = (dev(rng.standard_normal((9 * b + 1, width)).astype(np.float32)) for _ in range(2))
        for c in caches:
            c.prefill(b, k, v)
    for step in range(3):
        qkv = rng.standard_normal((batch, 3 * width)).astype(np.float32)
        got = caches[0].rope_push_qkv(rope, dev(qkv))
        q, k, v = (dev(qkv[:, i * width:(i + 1) * width]) for i in range(3))
        caches[1].rope(rope, q, k)
        caches[1].push(k, v)
        ctx.sync()
        assert np.array_equal(host(got), host(q))
        for b in range(batch):
            assert np.array_equal(host(q)[b], oracle.rope(qkv[b, :width], dim, 9 * b + 1 + step))
            for x, y in zip(caches[0].export(b), caches[1].export(b)):
                assert np.array_equal(host(x), host(y))
    for c in caches:
        c.free()
    rope.free()


# ---- attention -----------------------------------------------------------------------
def run_attention(ctx, rng, lengths, heads, dim, bits, window, pushes, q_size=2.0, k_kind="mixed"):
    batch, width = len(lengths), heads * dim
    kv = QuantizedKvCache(ctx, batch, heads, dim, window, max(lengths), bits)
    size = np.exp(0.5 * rng.standard_normal(width)).astype(np.float32) if k_kind == "mixed" else 1.0
    for b, n in enumerate(lengths):
        kv.prefill(b, dev((rng.standard_normal((n, width)) * size).astype(np.float32)),
                   dev(rng.standard_normal((n, width)).astype(np.float32)))
    for _ in range(pushes):
        kv.push(dev((rng.standard_normal((batch, width)) * size).astype(np.float32)),
                dev(rng.standard_normal((batch, width)).astype(np.float32)))
    q = (q_size * rng.standard_normal((batch, width))).astype(np.float32)
    out = host(kv.attention(dev(q)))
    ctx.sync()
    return kv, q, out


def check_attention(kv, q, out, heads, dim, bits):
    for b in range(len(q)):
        # what the cache holds, quantised again, is what it holds: codes, step and
        # least value of the read rows give the terms of the tolerance
        k, v = (host(t).reshape(-1, heads, dim) for t in kv.export(b))
        parts = []
        for x in (k, v):
            _, s, m = held(x, bits)
            parts.append((x.astype(np.float64), s, m))
        ref, tol = attention_ref(q[b], *parts, heads)
        assert np.all(np.abs(out[b] - ref) <= tol), (b, np.max(np.abs(out[b] - ref) / tol))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("lengths,heads,dim,window,pushes", [
    ((1,), 1, 1, 1, 0),
    ((1,), 1, 32, 1, 0),
    ((1, 2, 3), 2, 64, 4, 0),
    ((31, 32, 33), 3, 128, 5, 1),
    ((7, 64, 65, 200), 3, 80, 5, 7),
    ((95, 1), 2, 96, 33, 40),
    ((129,), 5, 33, 3, 2),
    ((500, 10), 2, 127, 128, 3),
    ((300, 40), 1, 160, 16, 20),
    ((77, 260), 2, 192, 16, 1),
    ((65, 130), 2, 224, 8, 9),
    ((300, 3), 2, 256, 8, 9),
    ((1517,), 10, 128, 128, 130),
    (tuple(range(1, 65)), 4, 128, 8, 3),
])
def test_attention(ctx, bits, lengths, heads, dim, window, pushes):
    rng = np.random.default_rng(sum(lengths) + dim + bits)
    kv, q, out = run_attention(ctx, rng, lengths, heads, dim, bits, window, pushes)
    check_attention(kv, q, out, heads, dim, bits)
    kv.free()


@pytest.mark.parametrize("batch,tokens", [(1, 5000), (1, 32768), (3, 4001), (16, 700), (40, 300), (200, 64)])
def test_attention_sizes(ctx, batch, tokens):
    """Few and many sequences, short and long: every way the work is split."""
    rng = np.random.default_rng(batch + tokens)
    kv, q, out = run_attention(ctx, rng, (tokens,) * batch, 3, 128, 4, 16, 1)
    check_attention(kv, q, out, 3, 128, 4)
    kv.free()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("q_size", [0.0, 1e-20, 30.0])
def test_attention_flat_and_peaked(ctx, bits, q_size):
    """Uniform weights, and one token that takes nearly all of them."""
    rng = np.random.default_rng(int(q_size) + bits)
    kv, q, out = run_attention(ctx, rng, (700, 31), 2, 128, bits, 4, 2, q_size)
    check_attention(kv, q, out, 2, 128, bits)
    kv.free()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("size", [1e5, 1e7, 1e12, 1e29])
def test_attention_vast_scores(ctx, bits, size):
    """Scores of any size, negative ones alone among them: where the largest leads by
    more than a sum's rounding, its token takes all the weight.  (48 roundings of
    2^-24 of a score's terms at most: 2^-18 of them; the sum to L >= 1 and the two
    products of a value are three roundings, the weight's own 2^-30 and the least
    value's join three more: 2^-21 of s code + |m|.)"""
    rng = np.random.default_rng(int(np.log10(size)) + bits)
    heads, dim, tokens = 4, 96, 300
    kv = QuantizedKvCache(ctx, 1, heads, dim, 4, tokens, bits)
    k, v = (rng.standard_normal((tokens, heads, dim)).astype(np.float32) for _ in range(2))
    k *= np.float32(size)
    q = rng.standard_normal((heads, dim)).astype(np.float32)
    k[:, 2:] = np.abs(k[:, 2:])
    q[2:] = -np.abs(q[2:])
    kv.prefill(0, dev(k.reshape(tokens, -1)), dev(v.reshape(tokens, -1)))
    out = host(kv.attention(dev(q.reshape(1, -1)))).reshape(heads, dim)
    ctx.sync()
    (kh, ks, km), (vh, vs, vm) = held(k, bits), held(v, bits)
    scores = np.einsum("thd,hd->th", kh, q.astype(np.float64))
    terms = np.einsum("thd,hd->th", (kh - km) + np.abs(km), np.abs(q.astype(np.float64)))
    led = 0
    for h in range(heads):
        order = np.argsort(-scores[:, h])
        gap = (scores[order[0], h] - scores[order[1], h]) / np.sqrt(dim)
        if gap < 2.0 ** -17 * terms[:, h].max() / np.sqrt(dim) + 40:
            continue
        led += 1
        t = order[0]
        tol = 2.0 ** -21 * ((vh - vm) + np.abs(vm))[t, h] + tokens * np.exp(-40) * 8
        assert np.all(np.abs(out[h] - vh[t, h]) <= tol), (h, np.max(np.abs(out[h] - vh[t, h]) / tol))
    assert led >= 3
    kv.free()


@pytest.mark.parametrize("scale", [1e-25, 1e-12, 1e12])
def test_attention_value_sizes(ctx, scale):
    """Values of any size; keys of the inverse size of the queries."""
    rng = np.random.default_rng(3)
    heads, dim, tokens = 2, 64, 100
    kv = QuantizedKvCache(ctx, 1, heads, dim, 4, tokens, 4)
    k, v = (rng.standard_normal((tokens, heads * dim)) for _ in range(2))
    kv.prefill(0, dev((k / scale).astype(np.float32)), dev((v * scale).astype(np.float32)))
    q = (rng.standard_normal((1, heads * dim)) * scale).astype(np.float32)
    out = host(kv.attention(dev(q)))
    ctx.sync()
    check_attention(kv, q, out, heads, dim, 4)
    kv.free()


def test_attention_is_repeatable_and_leaves_the_cache(ctx):
    rng = np.random.default_rng(5)
    kv, q, out = run_attention(ctx, rng, (900, 33, 5), 4, 128, 4, 8, 3)
    before = [host(t) for t in kv.export(0)]
    for _ in range(5):
        assert np.array_equal(host(kv.attention(dev(q))), out)
    assert all(np.array_equal(x, host(y)) for x, y in zip(before, kv.export(0)))
    assert kv.state(0) == (903, 903)
    kv.free()


def test_reset_and_a_shorter_prompt(ctx):
    """Nothing of the tokens that were there before is left in the result."""
    rng = np.random.default_rng(6)
    heads, dim = 2, 128
    used = QuantizedKvCache(ctx, 1, heads, dim, 4, 400, 4)
    x = dev((1e3 * rng.standard_normal((400, heads * dim))).astype(np.float32))
    used.prefill(0, x, x)
    used.reset(0)
    raises("Shape", lambda: used.attention(x[:1]))
    fresh = QuantizedKvCache(ctx, 1, heads, dim, 4, 400, 4)
    k, v, q = (dev(rng.standard_normal((n, heads * dim)).astype(np.float32)) for n in (45, 45, 1))
    for c in (used, fresh):
        c.prefill(0, k, v)
        c.push(k[:1], v[:1])
    assert used.state(0) == (46, 46)
    assert np.array_equal(host(used.attention(q)), host(fresh.attention(q)))
    used.free()
    fresh.free()


def test_offsets_past_32_bits(ctx):
    """A cache of more than 2^33 bytes: the last sequence lies behind 2^32."""
    rng = np.random.default_rng(7)
    heads, dim, lengths = 4, 32, (5, 3, 70)
    kv = QuantizedKvCache(ctx, 3, heads, dim, 2, (1 << 24) - 2, 8)
    assert kv.storage_bytes() > 1 << 33
    rows = []
    for b, n in enumerate(lengths):
        k, v = (rng.standard_normal((n, heads * dim)).astype(np.float32) for _ in range(2))
        kv.prefill(b, dev(k), dev(v))
        rows.append((k, v))
    kv.push(dev(rows[2][0][:3]), dev(rows[2][1][:3]))
    q = rng.standard_normal((3, heads * dim)).astype(np.float32)
    out = host(kv.attention(dev(q)))
    for b, n in enumerate(lengths):
        got = kv.read(b, 0, n)
        for x, o in zip(rows[b], got):
            assert np.array_equal(host(o), held(x.reshape(n, heads, dim), 8)[0].reshape(n, -1).astype(np.float32))
    check_attention(kv, q, out, heads, dim, 8)
    kv.free()


# ---- what is refused, and what stays whole then -----------------------------------------
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 2.0 ** 100, -3e38])
def test_values_out_of_range(ctx, bad):
    rng = np.random.default_rng(8)
    heads, dim, n = 2, 128, 40
    k, v = (rng.standard_normal((n, heads * dim)).astype(np.float32) for _ in range(2))
    kv = QuantizedKvCache(ctx, 2, heads, dim, 3, n, 4)
    kv.prefill(0, dev(k), dev(v))
    ctx.sync()
    worse = v.copy()
    worse[33, 70] = bad  # token 33, head 0, group 2
    kv.prefill(1, dev(k), dev(worse))
    raises("Numerical", ctx.sync)
    ko, vo = (host(t) for t in kv.read(1, 0, n))
    ctx.sync()
    want = held(v.reshape(n, heads, dim), 4)[0].reshape(n, -1).astype(np.float32)
    lost = np.zeros_like(want, bool)
    lost[33, 64:96] = True
    assert np.all(np.isnan(vo[lost])) and np.array_equal(vo[~lost], want[~lost])
    assert np.all(np.isfinite(ko))
    # a value that is lost spoils its own dims; a key its whole head; no other sequence
    q = dev(rng.standard_normal((2, heads * dim)).astype(np.float32))
    out = host(kv.attention(q))
    ctx.sync()
    assert np.array_equal(np.isnan(out[1]), lost[33]) and np.all(np.isfinite(out[0]))
    worse = k[:2].copy()
    worse[1, 200] = bad
    kv.push(dev(worse), dev(v[:2]))
    raises("Numerical", ctx.sync)
    out = host(kv.attention(q))
    raises("Numerical", ctx.sync)
    assert np.all(np.isnan(out[1, 128:])) and np.all(np.isfinite(out[0]))
    assert np.array_equal(np.isnan(out[1, :128]), lost[33, :128])
    kv.free()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_queries_that_are_not_finite(ctx, bad):
    rng = np.random.default_rng(9)
    kv, q, out = run_attention(ctx, rng, (50, 20), 2, 64, 4, 4, 0)
    q[1, 100] = bad
    got = host(kv.attention(dev(q)))
    raises("Numerical", ctx.sync)
    assert np.array_equal(got[0], out[0]) and np.array_equal(got[1, :64], out[1, :64])
    assert np.all(np.isnan(got[1, 64:]))
    kv.free()


def test_order_of_calls(ctx):
    x = dev(np.ones((2, 64), np.float32))
    kv = QuantizedKvCache(ctx, 2, 2, 32, 3, 8, 4)
    raises("Shape", lambda: kv.push(x, x))
    raises("Shape", lambda: kv.attention(x))
    kv.prefill(0, x, x)
    raises("Shape", lambda: kv.push(x, x))
    raises("Shape", lambda: kv.prefill(0, x, x))
    raises("Resource", lambda: kv.prefill(1, *(dev(np.ones((9, 64), np.float32)),) * 2))
    kv.prefill(1, x, x)
    # slots that the window will hold, but that hold nothing yet
    out = [dev(np.full((3, 64), 5.0, np.float32)) for _ in range(2)]
    kv.read(1, 1, 3, *out)
    raises("Shape", ctx.sync)
    assert all(np.array_equal(host(o), np.repeat([[1.0], [5.0], [5.0]], 64, 1)) for o in out)
    raises("Shape", lambda: kv.read(1, 0, 6))
    assert [t.shape[0] for t in kv.read(1, 2, 0)] == [0, 0]
    kv.free()


def test_rows_of_another_shape_or_type(ctx):
    import torch
    kv = QuantizedKvCache(ctx, 2, 2, 32, 3, 8, 4)
    x = torch.ones((2, 64), device="cuda")
    kv.prefill(0, x, x)
    kv.prefill(1, x, x)
    for bad in (x.half(), x.cpu(), x[:1], x[:, :63], x.t(), torch.ones((64, 2), device="cuda").t()):
        raises("Shape", lambda: kv.push(bad, x))
        raises("Shape", lambda: kv.push(x, bad))
        raises("Shape", lambda: kv.attention(bad))
    wide = torch.ones((2, 80), device="cuda")
    raises("Shape", lambda: kv.attention(wide[:, :64]))
    kv.push(wide[:, :64], x)
    ctx.sync()
    kv.free()


def test_position_past_the_table(ctx):
    from uocr_q8.attention import Rope
    rope = Rope(ctx, 32, 10000.0, 4)
    kv = QuantizedKvCache(ctx, 1, 2, 32, 3, 8, 4)
    x = dev(np.ones((4, 64), np.float32))
    kv.prefill(0, x, x)
    kv.rope_push_qkv(rope, dev(np.ones((1, 192), np.float32)))
    raises("Resource", ctx.sync)
    kv.free()
    rope.free()


# ---- streams and graphs --------------------------------------------------------------
def test_captured_steps(ctx):
    """Push and attention in a graph, replayed past the ring's end, give what
    the same calls give one by one."""
    import torch
    rng = np.random.default_rng(10)
    heads, dim, batch, steps = 3, 128, 3, 9
    width = heads * dim
    caches = [QuantizedKvCache(ctx, batch, heads, dim, 4, 70, 4) for _ in range(2)]
    for b in range(batch):
        k, v = (dev(rng.standard_normal((20 * b + 30, width)).astype(np.float32)) for _ in range(2))
        for c in caches:
            c.prefill(b, k, v)
    rows = dev(rng.standard_normal((steps, 3, batch, width)).astype(np.float32))
    k, v, q = (torch.empty((batch, width), device="cuda") for _ in range(3))
    out = torch.empty_like(q)
    side, back = torch.cuda.Stream(), torch.cuda.current_stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    ctx.set_stream(side)
    try:
        with torch.cuda.graph(graph, stream=side):
            caches[0].push(k, v)
            caches[0].attention(q, out)
        for i in range(steps):
            for dst, src in zip((k, v, q), rows[i]):
                dst.copy_(src)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = host(out)
            ctx.set_stream(back)
            caches[1].push(rows[i, 0], rows[i, 1])
            want = host(caches[1].attention(rows[i, 2]))
            ctx.sync()
            assert np.array_equal(got, want), i
        assert caches[0].state(1) == caches[1].state(1) == (54, 59)
    finally:
        ctx.set_stream(back)
        del graph
    for c in caches:
        c.free()


def test_two_contexts_on_two_streams():
    """Two caches served at once on streams of their own."""
    import torch
    import uocr_q8
    rng = np.random.default_rng(11)
    heads, dim, batch = 2, 128, 2
    width = heads * dim
    made = []
    for _ in range(2):
        stream = torch.cuda.Stream()
        c = uocr_q8.GpuContext(0)
        c.set_stream(stream)
        kv = QuantizedKvCache(c, batch, heads, dim, 4, 3000, 4)
        rows = [dev(rng.standard_normal((3000, width)).astype(np.float32)) for _ in range(2)]
        q = dev(rng.standard_normal((batch, width)).astype(np.float32))
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        for b in range(batch):
            kv.prefill(b, rows[0], rows[1])
        kv.attention(q, out)
        c.sync()
        want = host(out)
        made.append((c, kv, rows, q, out, want))
    for _ in range(20):
        for c, kv, rows, q, out, want in made:
            kv.attention(q, out)
        for c, kv, rows, q, out, want in made:
            c.sync()
            assert np.array_equal(host(out), want)
            out.zero_()
        torch.cuda.synchronize()
    for c, kv, *_ in made:
        kv.free()
        c.close()


def test_first_calls_of_a_process_in_a_graph():
    """Nothing has to run before a capture but the calls that make the cache: the
    first push, attention and log probabilities of a process are captured."""
    import subprocess
    import sys
    from conftest import PKG
    code = f"""
import sys
sys.path.insert(0, {PKG!r})
import torch, uocr_q8
from uocr_q8.attention import QuantizedKvCache
from uocr_q8.decoder import token_logprobs_device
ctx = uocr_q8.GpuContext(0)
side = torch.cuda.Stream()
ctx.set_stream(side)
kv = QuantizedKvCache(ctx, 2, 2, 64, 4, 50, 4)
x = torch.randn(50, 128, device="cuda")
logits = torch.randn(150, 9000, device="cuda")
tokens = torch.arange(150, device="cuda")
out = torch.empty(2, 128, device="cuda")
torch.cuda.synchronize()
kv.prefill(0, x, x); kv.prefill(1, x, x)
ctx.sync()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    kv.push(x[:2], x[:2])
    kv.attention(x[:2], out)
    got = token_logprobs_device(ctx, logits, tokens, 3)
graph.replay()
torch.cuda.synchronize()
want = torch.log_softmax(logits, -1).gather(1, tokens[:, None])[:, 0]
assert (got.logprob - want).abs().max() < 1e-4
assert kv.state(1) == (51, 51) and torch.isfinite(out).all()
ctx.sync()
print("fine")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stdout + r.stderr


def test_in_place_and_out_of_order(ctx):
    """The result over its own queries; sequences filled in any order; one
    sequence emptied and filled again between steps of the others."""
    rng = np.random.default_rng(12)
    heads, dim = 2, 128
    width = heads * dim
    for tokens in (40, 9000):  # one CTA per head, and several clusters
        kv = QuantizedKvCache(ctx, 2, heads, dim, 4, tokens, 4)
        k, v = (dev(rng.standard_normal((tokens, width)).astype(np.float32)) for _ in range(2))
        kv.prefill(1, k, v)
        kv.prefill(0, k[:7], v[:7])
        kv.push(k[:2], v[:2])
        q = dev(rng.standard_normal((2, width)).astype(np.float32))
        want = host(kv.attention(q))
        assert kv.attention(q, q) is q
        assert np.array_equal(host(q), want)
        kv.reset(0)
        raises("Shape", lambda: kv.push(k[:2], v[:2]))
        kv.prefill(0, k[:33], v[:33])
        kv.push(k[:2], v[:2])
        assert kv.state(0) == (34, 34) and kv.state(1) == (tokens + 2, tokens + 2)
        q = rng.standard_normal((2, width)).astype(np.float32)
        out = host(kv.attention(dev(q)))
        ctx.sync()
        check_attention(kv, q, out, heads, dim, 4)
        kv.free()


@pytest.mark.parametrize("bits", [4, 8])
def test_many_heads(ctx, bits):
    """More (key or value) rows than a push has warps."""
    rng = np.random.default_rng(13)
    heads, dim, batch = 37, 48, 2
    kv, q, out = run_attention(ctx, rng, (70, 31), heads, dim, bits, 3, 5)
    check_attention(kv, q, out, heads, dim, bits)
    kv.free()
