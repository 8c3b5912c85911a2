"""Timed cases of the cache in 4 or 8 bits, of the attention over it and of the token log probabilities.

Each case is one pass of a user's program through one of them:

* ``write``: a prompt's keys and values are quantised into an empty cache and read back;
* ``decode``: one token per sequence is pushed into the cache, then every sequence's query attends to it;
* ``logprobs``: log probabilities of the given tokens, entropies and top alternatives of rows of logits.

``run`` computes them in plain torch operations, or with ``own`` set through the package's entry points.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 32          # dims that share a step and a least value
LIMIT = 64 * 2048 * 10 * 128  # cached elements (of keys) of the largest decode case


def _context():
    at = os.path.join(os.getcwd(), "unlimited-ocr-kernel_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import uocr_q8
    return uocr_q8.default_context(0)


def listed():
    return [
        # the first token of an empty prompt: what a write and a read cost at least
        {"name": "write 1 token, 4 bits", "kind": "write", "tokens": 1, "heads": 10, "dim": 128, "bits": 4},
        # the prompt of the fixed-work decoder benchmark
        {"name": "write 1517 tokens, 4 bits", "kind": "write", "tokens": 1517, "heads": 10, "dim": 128, "bits": 4},
        # a prompt that fills the maximum context
        {"name": "write 32768 tokens, 8 bits", "kind": "write", "tokens": 32768, "heads": 10, "dim": 128, "bits": 8},
        # a step of the fixed-work decoder benchmark: one sequence
        {"name": "decode 1 x 1517, 4 bits", "kind": "decode", "batch": 1, "tokens": 1517, "window": 128,
         "heads": 10, "dim": 128, "bits": 4, "ragged": False},
        # one sequence near the maximum context
        {"name": "decode 1 x 32640, 4 bits", "kind": "decode", "batch": 1, "tokens": 32640, "window": 128,
         "heads": 10, "dim": 128, "bits": 4, "ragged": False},
        # the batched decode step
        {"name": "decode 64 x 2048, 4 bits", "kind": "decode", "batch": 64, "tokens": 2048, "window": 128,
         "heads": 10, "dim": 128, "bits": 4, "ragged": False},
        {"name": "decode 64 x 2048, 8 bits", "kind": "decode", "batch": 64, "tokens": 2048, "window": 128,
         "heads": 10, "dim": 128, "bits": 8, "ragged": False},
        # sequences of different lengths, a head that is no multiple of 32, tiles that end early
        {"name": "decode 7 ragged, 3 x 80", "kind": "decode", "batch": 7, "tokens": 777, "window": 5,
         "heads": 3, "dim": 80, "bits": 4, "ragged": True},
        # one decoded token's alternatives
        {"name": "logprobs 1 row, top 20", "kind": "logprobs", "rows": 1, "vocab": 129280, "pad": 0, "top": 20,
         "grid": 0, "masked": 0.0},
        # a decode step of the whole batch
        {"name": "logprobs 64 rows, top 5", "kind": "logprobs", "rows": 64, "vocab": 129280, "pad": 0, "top": 5,
         "grid": 0, "masked": 0.0},
        # scoring every position of a prompt
        {"name": "logprobs 1517 rows, top 1", "kind": "logprobs", "rows": 1517, "vocab": 129280, "pad": 0, "top": 1,
         "grid": 0, "masked": 0.0},
        # odd vocabulary, rows apart from each other, ties among the logits, half of the tokens banned
        {"name": "logprobs 37 odd rows, top 32", "kind": "logprobs", "rows": 37, "vocab": 50021, "pad": 3, "top": 32,
         "grid": 64, "masked": 0.5},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["write", "decode", "decode", "logprobs"])
    if kind == "logprobs":
        vocab = _log_uniform(rng, 33, 200000)
        return {"kind": kind, "rows": _log_uniform(rng, 1, max(1, min(4096, 1517 * 129280 // vocab))), "vocab": vocab,
                "pad": rng.choice([0, 0, 1, 4, 7]), "top": rng.randint(0, 32), "grid": rng.choice([0, 0, 16, 256]),
                "masked": rng.choice([0.0, 0.0, 0.3, 0.9])}
    heads, dim, bits = rng.choice([1, 2, 3, 5, 8, 10, 10, 16]), rng.choice([16, 32, 64, 80, 96, 112, 128, 128, 160, 256]), rng.choice([4, 4, 8])
    if kind == "write":
        most = min(32768, 32768 * 1280 // (heads * dim))
        return {"kind": kind, "tokens": _log_uniform(rng, 1, most), "heads": heads, "dim": dim, "bits": bits}
    batch = _log_uniform(rng, 1, 64)
    most = min(32640, LIMIT // (batch * heads * dim))
    return {"kind": kind, "batch": batch, "tokens": _log_uniform(rng, 1, most), "window": rng.choice([1, 5, 33, 128]),
            "heads": heads, "dim": dim, "bits": bits, "ragged": rng.random() < 0.5}


def _lengths(case):
    """Prefix lengths of the sequences, the longest first."""
    n = case["batch"]
    return [max(1, case["tokens"] * (n - i) // n) if case["ragged"] else case["tokens"] for i in range(n)]


def work(case):
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (16 + 12 * case["top"]), "flops": 4 * n}
    groups = -(-case["dim"] // BLOCK)
    held = case["heads"] * (case["dim"] * case["bits"] / 8 + 4 * groups)  # bytes of one token's keys (or values)
    if case["kind"] == "write":  # rows read, codes written, codes read, rows written
        return {"bytes": case["tokens"] * 2 * (8 * case["heads"] * case["dim"] + 2 * held),
                "flops": 12 * case["tokens"] * case["heads"] * case["dim"]}
    present = sum(_lengths(case)) + case["batch"] * case["window"]
    row = 4 * case["heads"] * case["dim"]
    return {"bytes": present * 2 * held + case["batch"] * (4 * row + 2 * held),
            "flops": 4 * present * case["heads"] * case["dim"]}


# ---- the cache in its plain form: codes, steps and least values ------------------

def _to_bf16(x, up):
    """The nearest bf16 value at or above (or at or below) x, in 64 bits."""
    r = x.to(torch.float32).to(torch.bfloat16)
    inf = torch.full_like(r, math.inf if up else -math.inf)
    r = torch.where(r.double() < x if up else r.double() > x, torch.nextafter(r, inf), r)
    back = torch.nextafter(r, -inf)
    return torch.where(back.double() >= x if up else back.double() <= x, back, r).double()


def _quantize(x, bits):
    """Codes (0 .. 2^bits - 1), steps and least values of x [..., dim] in groups of 32 dims."""
    dim, top = x.shape[-1], 2 ** bits - 1
    fill = -dim % BLOCK
    x = x.double()
    lo = torch.nn.functional.pad(x, (0, fill), value=math.inf).unflatten(-1, (-1, BLOCK)).amin(-1)
    hi = torch.nn.functional.pad(x, (0, fill), value=-math.inf).unflatten(-1, (-1, BLOCK)).amax(-1)
    lo = _to_bf16(lo, False)
    step = _to_bf16((hi - lo) / top, True)
    wide_lo, wide = (v.repeat_interleave(BLOCK, -1)[..., :dim] for v in (lo, step))
    codes = torch.where(wide > 0, torch.round((x - wide_lo) / wide.clamp_min(1e-300)), 0.0).clamp(0, top)
    return codes.to(torch.uint8), step.to(torch.bfloat16), lo.to(torch.bfloat16)


def _values(codes, step, lo, dtype):
    dim = codes.shape[-1]
    step, lo = (v.to(dtype).repeat_interleave(BLOCK, -1)[..., :dim] for v in (step, lo))
    return codes.to(dtype) * step + lo


def _inputs(case, seed):
    """Keys, values (and for a decode step the new rows and the queries), on the GPU."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    width = case["heads"] * case["dim"]
    # keys have channels of their own size, as rotated keys do; values do not
    size = torch.exp(0.7 * torch.randn(width, generator=g, device="cuda"))
    rows = case["tokens"] if case["kind"] == "write" else sum(_lengths(case))
    got = {"k": torch.randn((rows, width), generator=g, device="cuda") * size,
           "v": torch.randn((rows, width), generator=g, device="cuda")}
    if case["kind"] == "decode":
        n = case["batch"]
        got["new_k"] = torch.randn((n, width), generator=g, device="cuda") * size
        got["new_v"] = torch.randn((n, width), generator=g, device="cuda")
        got["q"] = torch.randn((n, width), generator=g, device="cuda")
    return got


def _logits(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    rows, vocab = case["rows"], case["vocab"]
    x = 3.0 * torch.randn((rows, vocab + case["pad"]), generator=g, device="cuda")
    if case["grid"]:
        x = torch.round(x * case["grid"]) / case["grid"]
    if case["masked"]:
        ban = torch.rand(x.shape, generator=g, device="cuda") < case["masked"]
        ban[:, 0] = False  # something is left in every row
        x = x.masked_fill(ban, -math.inf)
    x = x[:, :vocab]
    return x, torch.randint(0, vocab, (rows,), generator=g, device="cuda")


def prepare(case, seed):
    if case["kind"] == "logprobs":
        logits, tokens = _logits(case, seed)
        return {"case": case, "logits": logits, "tokens": tokens}
    state = {"case": case, **_inputs(case, seed)}
    if case["kind"] == "write":
        if own:
            _context()
            from uocr_q8.attention import QuantizedKvCache
            state["cache"] = QuantizedKvCache(_context(), 1, case["heads"], case["dim"], 128, case["tokens"], case["bits"])
        return state
    # a decode step's cache: prompts of `lengths` tokens and a ring that already holds the row that every pass
    # pushes, so that a pass leaves the cache as it found it
    lengths, window = _lengths(case), case["window"]
    k, v = state.pop("k").split(lengths), state.pop("v").split(lengths)
    if own:
        ctx = _context()
        from uocr_q8.attention import QuantizedKvCache
        cache = QuantizedKvCache(ctx, case["batch"], case["heads"], case["dim"], window, case["tokens"], case["bits"])
        for b in range(case["batch"]):
            cache.prefill(b, k[b], v[b])
        for _ in range(window):
            cache.push(state["new_k"], state["new_v"])
        state["cache"] = cache
        return state
    shape = (case["batch"], case["tokens"] + window, case["heads"], case["dim"])
    groups = -(-case["dim"] // BLOCK)
    for name, rows, new in (("k", k, state["new_k"]), ("v", v, state["new_v"])):
        held = (torch.zeros(shape, dtype=torch.uint8, device="cuda"),
                *(torch.zeros((*shape[:3], groups), dtype=torch.bfloat16, device="cuda") for _ in range(2)))
        for b, n in enumerate(lengths):
            row = torch.cat([rows[b], new[b].expand(window, -1)]).view(-1, *shape[2:])
            for part, made in zip(held, _quantize(row, case["bits"])):
                part[b, : n + window] = made
        state["held_" + name] = held
    state["lengths"] = torch.tensor(lengths, device="cuda")
    state["pushed"] = torch.tensor(window, device="cuda")
    return state


# ---- one pass ------------------------------------------------------------------------

def _run_own(state):
    case = state["case"]
    if case["kind"] == "write":
        cache = state["cache"]
        cache.reset(0)
        cache.prefill(0, state["k"], state["v"])
        k, v = cache.read(0, 0, case["tokens"])
        return {"k": k, "v": v}
    if case["kind"] == "decode":
        state["cache"].push(state["new_k"], state["new_v"])
        return {"out": state["cache"].attention(state["q"])}
    from uocr_q8.decoder import token_logprobs_device
    got = token_logprobs_device(_context(), state["logits"], state["tokens"], case["top"])
    return {"logprob": got.logprob, "entropy": got.entropy, "top_ids": got.top_ids, "top_logprobs": got.top_logprobs}


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["kind"] == "logprobs":
        x = state["logits"]
        z = x - x.amax(-1, keepdim=True)
        e = z.exp()
        total = e.sum(-1, keepdim=True, dtype=torch.float64)  # sums over a whole vocabulary
        lse = total.log()
        entropy = lse[:, 0] - (e * z.clamp_min(-1000.0)).sum(-1, dtype=torch.float64) / total[:, 0]
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, : case["top"]]
        return {"logprob": (z.gather(-1, state["tokens"][:, None]) - lse)[:, 0].float(), "entropy": entropy.float(),
                "top_ids": order.contiguous(), "top_logprobs": (z.gather(-1, order) - lse).float()}
    shape = (-1, case["heads"], case["dim"])
    if case["kind"] == "write":
        k, v = (_values(*_quantize(state[n].view(shape), case["bits"]), torch.float32) for n in ("k", "v"))
        return {"k": k.flatten(1), "v": v.flatten(1)}
    lengths = state["lengths"]
    at = torch.arange(case["batch"], device="cuda")
    slot = lengths + state["pushed"] % case["window"]
    for held, new in ((state["held_k"], state["new_k"]), (state["held_v"], state["new_v"])):
        for part, made in zip(held, _quantize(new.view(shape), case["bits"])):
            part[at, slot] = made
    state["pushed"] += 1
    k, v = (_values(*state["held_" + n], torch.float32).transpose(1, 2) for n in ("k", "v"))
    q = state["q"].view(shape)
    scores = (k @ q[..., None])[..., 0] / math.sqrt(case["dim"])
    held = lengths + case["window"]
    scores = scores.masked_fill(torch.arange(scores.shape[-1], device="cuda") >= held[:, None, None], -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    return {"out": (p[:, :, None, :] @ v)[:, :, 0].flatten(1)}


# ---- the definitions in 64 bits -------------------------------------------------------

def _exact_held(x, bits):
    """The values that a cache of `bits` bits holds for rows x [rows, heads, dim], group by group."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for g in range(0, x.shape[-1], BLOCK):
        part = x[..., g : g + BLOCK].double()
        least, most = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        # bf16 values have 8 significant bits: multiples of 2^(e - 8) where frexp's exponent is e
        unit = torch.ldexp(torch.ones_like(least), torch.frexp(least).exponent - 8)
        least = torch.floor(least / unit) * unit
        step = (most - least) / (2 ** bits - 1)
        unit = torch.ldexp(torch.ones_like(step), torch.frexp(step).exponent - 8)
        step = torch.ceil(step / unit) * unit
        y = (part - least) / step
        code = torch.floor(y)
        rest = y - code
        code = code + ((rest > 0.5) | ((rest == 0.5) & (code % 2 == 1)))
        code = torch.where(step > 0, code, torch.zeros_like(code)).clamp(0, 2 ** bits - 1)
        out[..., g : g + BLOCK] = least + step * code
    return out


def exact(case, seed):
    if case["kind"] == "logprobs":
        logits, tokens = _logits(case, seed)
        k = case["top"]
        out = {"logprob": [], "entropy": [], "top_ids": None, "top_logprobs": []}
        for r in range(case["rows"]):
            x = logits[r].double()
            finite = x[x > -math.inf]
            lse = torch.logsumexp(finite, 0)
            out["logprob"].append(x[tokens[r]] - lse)
            p = torch.exp(finite - lse)
            out["entropy"].append((p * (lse - finite)).sum())
            out["top_logprobs"].append(torch.topk(x, k).values - lse)
        return {n: v if v is None else torch.stack(v) for n, v in out.items()}
    got = _inputs(case, seed)
    shape = (-1, case["heads"], case["dim"])
    if case["kind"] == "write":
        return {n: _exact_held(got[n].view(shape), case["bits"]).flatten(1) for n in ("k", "v")}
    out, first = [], 0
    for b, n in enumerate(_lengths(case)):
        k, v = (_exact_held(torch.cat([got[r][first : first + n].view(shape),
                                       got["new_" + r][b].view(shape).expand(case["window"], -1, -1)]), case["bits"])
                for r in ("k", "v"))
        first += n
        q = got["q"][b].view(shape[1:]).double()
        a = torch.softmax(torch.einsum("thd,hd->ht", k, q) / math.sqrt(case["dim"]), -1)
        out.append(torch.einsum("ht,thd->hd", a, v).flatten())
    return {"out": torch.stack(out)}
