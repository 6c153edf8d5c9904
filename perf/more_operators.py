"""Operators of one decode step of a served batch, as measurable cases.

Three operators, each with the inputs a serving program has in hand before the call:

* `prefix_attention` -- the new tokens of every sequence of a batch against a prefix that all sequences
  share, kept once, and each sequence's own cache.
* `quantized_rms_norm` -- the residual's addition, RMSNorm and an output in 8 bits with scales.
* `penalize_logits` -- repetition, presence and frequency penalties, biases, temperature and a grammar's
  bit mask on the logits of every sequence.

`run` is the plain form in elementary torch operations while `own` is false, the calls of
`neptune_opt_b200` while it is true.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EIGHT_BITS = {"e4m3": (torch.float8_e4m3fn, 448.0), "e5m2": (torch.float8_e5m2, 57344.0)}
SMALLEST_SCALE = 2.0 ** -126


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # One short conversation behind a short system prompt, on few heads: latency of the whole call.
        _attn("attn_one", "bfloat16", 1, 4, 1, 128, 200, 64, 1),
        # A batch of uneven conversations, a slot of it free, behind a system prompt.
        _attn("attn_chat", "bfloat16", 32, 32, 8, 128, 2048, 1024, 1, ragged=True),
        # Drafted tokens checked together: five new tokens a sequence, unshared heads, odd lengths.
        _attn("attn_draft", "float16", 16, 16, 16, 64, 4001, 777, 5, ragged=True),
        # A few questions about one very long document: the prefix's bytes count.
        _attn("attn_document", "bfloat16", 4, 32, 8, 128, 131072, 200, 1),
        # A large batch of short answers behind long instructions: products and bytes count.
        _attn("attn_wide", "bfloat16", 256, 32, 8, 128, 16384, 512, 1, ragged=True),
        # The rows of a small decode batch: latency.
        _norm("norm8_few", "bfloat16", 16, 2048, True, "e4m3", 0),
        # Odd width and row count in fp32, one scale a row.
        _norm("norm8_odd", "float32", 3003, 1001, True, "e4m3", 0),
        # The repository's RMSNorm shape (a prompt's tokens), one scale per 128 channels.
        _norm("norm8_batch", "bfloat16", 16384, 4096, True, "e4m3", 128),
        # A few sequences with all penalties, no mask: latency.
        _logits("logits_few", "float32", 8, 32000, 300, 0, False),
        # Odd vocabulary and row count in fp16, long histories, biases and a mask.
        _logits("logits_odd", "float16", 77, 50001, 2049, 100, True),
        # A large batch under a grammar, without a history.
        _logits("logits_grammar", "bfloat16", 512, 131072, 0, 0, True),
        # The repository's ultra-wide logits with everything at once.
        _logits("logits_wide", "bfloat16", 512, 262144, 4096, 32, True),
    ]


def _attn(name, dtype, batch, heads, kv_heads, dim, prefix, cache, new, ragged=False):
    return {"name": name, "op": "prefix_attention", "dtype": dtype, "batch": batch, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "prefix": prefix, "cache": cache, "new": new, "ragged": ragged}


def _norm(name, dtype, rows, width, residual, kind, group):
    return {"name": name, "op": "quantized_rms_norm", "dtype": dtype, "rows": rows, "width": width,
            "residual": residual, "kind": kind, "group": group}


def _logits(name, dtype, rows, vocab, history, biases, masked):
    return {"name": name, "op": "penalize_logits", "dtype": dtype, "rows": rows, "vocab": vocab,
            "history": history, "biases": biases, "masked": masked}


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["prefix_attention", "quantized_rms_norm", "penalize_logits"])
    if op == "prefix_attention":
        kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8, 16])
        dim, new = rng.choice([64, 128]), rng.choice([1, 1, 1, 2, 4, 7])
        prefix, cache = _log_int(rng, 1, 131072), max(new, _log_int(rng, 1, 8192))
        # No dearer than the largest listed ones: pairs of queries and keys, keys of the prefix and of all caches.
        pairs, keys = 256 * 32 * 16384 // (heads * new), 8 * 131072 * 128 // (kv_heads * dim)
        prefix = min(prefix, pairs, keys - cache)
        most = min(256, pairs // max(prefix, cache), (keys - prefix) // cache)
        case = _attn("", rng.choice(["bfloat16", "float16"]), _log_int(rng, 1, max(1, most)), heads, kv_heads, dim,
                     prefix, cache, new, rng.random() < 0.5)
    elif op == "quantized_rms_norm":
        group = rng.choice([0, 0, 32, 64, 128])
        width = _log_int(rng, 64, 16384)
        width = max(group, width // group * group) if group else width
        rows = _log_int(rng, 1, (16384 * 2048) // width)
        case = _norm("", rng.choice(list(DTYPES)), rows, width, rng.random() < 0.7, rng.choice(list(EIGHT_BITS)), group)
    else:
        vocab = _log_int(rng, 1000, 262144)
        rows = _log_int(rng, 1, min(1024, (256 * 262144) // vocab))
        case = _logits("", rng.choice(list(DTYPES)), rows, vocab, rng.choice([0, _log_int(rng, 1, 4096)]),
                       rng.choice([0, _log_int(rng, 1, 300)]), rng.random() < 0.6)
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(case):
    """Own tokens of each sequence, the new ones among them: full, none (a free slot), then a spread."""
    n, b = case["cache"], case["batch"]
    if not case["ragged"]:
        return [n] * b
    return [n if i == 0 else 0 if i == 1 else max(min(case["new"], n), int(n * ((0.618 * i) % 1.0))) for i in range(b)]


def prepare(case, seed):
    gen = _generator(seed)
    return {"prefix_attention": _prepare_attention, "quantized_rms_norm": _prepare_norm,
            "penalize_logits": _prepare_logits}[case["op"]](case, gen)


def _prepare_attention(case, gen):
    b, h, hk, d, dt = case["batch"], case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", dtype=dt, generator=gen)

    return {"case": case, "q": normal(b, h, case["new"], d), "pk": normal(hk, case["prefix"], d),
            "pv": normal(hk, case["prefix"], d), "k": normal(b, hk, case["cache"], d),
            "v": normal(b, hk, case["cache"], d), "scale": 1.0 / math.sqrt(d),
            "lens": torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None}


def _prepare_norm(case, gen):
    n, c, dt = case["rows"], case["width"], DTYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(*shape, device="cuda", dtype=dt, generator=gen) * std + mean

    # A residual stream with a few channels that stand far out of the others.
    residual = None
    if case["residual"]:
        residual = normal(n, c, std=2.0)
        residual[:, ::97] *= 8.0
    return {"case": case, "x": normal(n, c), "residual": residual, "weight": normal(c, mean=1.0, std=0.1), "eps": 1e-6}


def _prepare_logits(case, gen):
    n, v, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]

    def uniform(lo, hi):
        return torch.rand(n, device="cuda", generator=gen) * (hi - lo) + lo

    state = {"case": case, "logits": torch.randn(n, v, device="cuda", dtype=dt, generator=gen) * 3.0,
             "temperature": uniform(0.5, 1.5), "tokens": None, "token_lens": None, "prompt_lens": None,
             "repetition": None, "presence": None, "frequency": None, "bias_index": None, "bias_value": None,
             "allowed": None}
    if case["history"]:
        # Prompt and output tokens; some tokens come again and again.
        most = case["history"]
        state["tokens"] = (torch.rand(n, most, device="cuda", generator=gen) ** 4 * v).to(torch.int64).clamp(max=v - 1)
        lens = (uniform(0.3, 1.0) * most).to(torch.int32)
        lens[0] = most
        lens[n // 2] = 0
        state["token_lens"] = lens
        state["prompt_lens"] = (lens * uniform(0.0, 1.0)).to(torch.int32)
        state["repetition"], state["presence"], state["frequency"] = uniform(1.0, 1.3), uniform(0.0, 1.0), uniform(0.0, 0.5)
    if case["biases"]:
        # Distinct indices in every row: an arithmetic progression that does not wrap onto itself.
        m = min(case["biases"], v)
        first = torch.randint(0, v, (n, 1), device="cuda", generator=gen)
        stride = torch.randint(1, v // m + 1, (n, 1), device="cuda", generator=gen)
        state["bias_index"] = (first + stride * torch.arange(m, device="cuda")) % v
        state["bias_value"] = torch.randn(n, m, device="cuda", generator=gen) * 5.0
    if case["masked"]:
        # Words of 32 tokens: all allowed, about half, few, and (a grammar at a dead end) none.
        words = -(-v // 32)

        def bits():
            return torch.randint(-2 ** 31, 2 ** 31, (n, words), device="cuda", generator=gen, dtype=torch.int32)

        half = bits()
        few = half & bits() & bits() & bits()
        kind = torch.arange(n, device="cuda")[:, None] % 3
        allowed = torch.where(kind == 0, torch.full_like(half, -1), torch.where(kind == 1, half, few))
        allowed[n - 1] = 0
        state["allowed"] = allowed
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    return {"prefix_attention": _plain_attention, "quantized_rms_norm": _plain_norm,
            "penalize_logits": _plain_logits}[case["op"]](state, case)


def _run_own(state, case):
    import neptune_opt_b200 as NB

    if case["op"] == "prefix_attention":
        o, lse = NB.prefix_attention(state["q"], state["pk"], state["pv"], state["k"], state["v"], state["lens"],
                                     scale=state["scale"], return_lse=True)
        return {"o": o, "lse": lse}
    if case["op"] == "quantized_rms_norm":
        q, scale, y = NB.quantized_rms_norm(state["x"], state["weight"], state["residual"], group=case["group"] or None,
                                            dtype=EIGHT_BITS[case["kind"]][0], eps=state["eps"])
        return {"q": q, "scale": scale, "y": y}
    return NB.penalize_logits(state["logits"], state["tokens"], state["token_lens"], state["prompt_lens"],
                              repetition=state["repetition"], presence=state["presence"],
                              frequency=state["frequency"], bias_index=state["bias_index"],
                              bias_value=state["bias_value"], temperature=state["temperature"],
                              allowed=state["allowed"])


def _plain_attention(state, case):
    b, h, hk, d, t = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["new"]
    p, n, per = case["prefix"], case["cache"], h // hk
    q = state["q"].float().view(b, hk, per * t, d)
    # The prefix's scores for the queries of all sequences at once, [kv head, batch x head x token, prefix].
    rows = q.transpose(0, 1).reshape(hk, b * per * t, d)
    far = torch.matmul(rows, state["pk"].float().transpose(1, 2)) * state["scale"]
    near = torch.matmul(q, state["k"].float().transpose(2, 3)) * state["scale"]
    lens = state["lens"] if state["lens"] is not None else torch.full((b,), n, device="cuda", dtype=torch.int32)
    at = lens[:, None] - t + torch.arange(t, device="cuda")  # the queries' own positions
    seen = torch.arange(n, device="cuda") <= at[..., None]
    near = near.view(b, hk, per, t, n).masked_fill(~seen[:, None, None], -math.inf).view(b, hk, per * t, n)
    far = far.view(hk, b, per * t, p)
    top = torch.maximum(far.amax(-1).transpose(0, 1), near.amax(-1))
    far = torch.exp(far - top.transpose(0, 1)[..., None])
    near = torch.exp(near - top[..., None])
    total = far.sum(-1).transpose(0, 1) + near.sum(-1)
    o = torch.matmul(far.view(hk, b * per * t, p), state["pv"].float()).view(hk, b, per * t, d).transpose(0, 1)
    live = (torch.arange(n, device="cuda") < lens[:, None])[:, None, :, None]
    o = (o + torch.matmul(near, torch.where(live, state["v"].float(), 0.0))) / total[..., None]
    lse = top + torch.log(total)
    free = (at < 0)[:, None, None].expand(b, hk, per, t)
    o = o.view(b, hk, per, t, d).masked_fill(free[..., None], 0.0)
    lse = lse.view(b, hk, per, t).masked_fill(free, -math.inf)
    return {"o": o.reshape(b, h, t, d).to(state["q"].dtype), "lse": lse.reshape(b, h, t)}


def _plain_norm(state, case):
    kind, most = EIGHT_BITS[case["kind"]]
    rows, width = case["rows"], case["width"]
    y = state["x"].float()
    if state["residual"] is not None:
        y = y + state["residual"].float()
    h = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + state["eps"]) * state["weight"].float()
    h = h.view(rows, -1, case["group"] or width)
    scale = torch.clamp(h.abs().amax(-1, keepdim=True) / most, min=SMALLEST_SCALE)
    q = torch.clamp(h / scale, -most, most).view(rows, width).to(kind)
    return {"q": q, "scale": scale.squeeze(-1), "y": None if state["residual"] is None else y.to(state["x"].dtype)}


def _plain_logits(state, case):
    n, v = case["rows"], case["vocab"]
    x = state["logits"].float()
    if state["tokens"] is not None:
        place = torch.arange(case["history"], device="cuda")
        there = place < state["token_lens"][:, None]
        output = there & (place >= state["prompt_lens"][:, None])
        seen = torch.zeros(n, v, device="cuda", dtype=torch.int32).scatter_add_(1, state["tokens"], there.int())
        count = torch.zeros(n, v, device="cuda", dtype=torch.int32).scatter_add_(1, state["tokens"], output.int())
        rep = state["repetition"][:, None]
        x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
        x = x - state["frequency"][:, None] * count - state["presence"][:, None] * (count > 0)
    if state["bias_index"] is not None:
        x = x.scatter_add(1, state["bias_index"], state["bias_value"])
    x = x / state["temperature"][:, None]
    if state["allowed"] is not None:
        bit = torch.arange(32, device="cuda", dtype=torch.int32)
        ok = ((state["allowed"][..., None] >> bit) & 1).bool().view(n, -1)[:, :v]
        x = x.masked_fill(~ok, -math.inf)
    return x.to(state["logits"].dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "prefix_attention":
        b, h, hk, d, t = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["new"]
        lens = _lengths(case)
        live = sum(min(t, n) for n in lens)
        pairs = sum(max(0, n - t + i + 1) for n in lens for i in range(t))
        moved = 2 * hk * (case["prefix"] + sum(lens)) * d * size + 2 * b * h * t * d * size + b * h * t * 4 + b * 4
        return {"bytes": moved, "flops": 4 * d * h * (live * case["prefix"] + pairs)}
    if case["op"] == "quantized_rms_norm":
        n, c = case["rows"], case["width"]
        groups = c // case["group"] if case["group"] else 1
        return {"bytes": n * c * (size * (3 if case["residual"] else 1) + 1) + n * groups * 4 + c * size,
                "flops": 8 * n * c}
    n, v = case["rows"], case["vocab"]
    moved = 2 * n * v * size + n * case["history"] * 8 + n * case["biases"] * 12 + n * 24
    return {"bytes": moved + (n * -(-v // 32) * 4 if case["masked"] else 0), "flops": 5 * n * v}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"prefix_attention": _exact_attention, "quantized_rms_norm": _exact_norm,
            "penalize_logits": _exact_logits}[case["op"]](state, case)


def _exact_attention(state, case):
    """Sequence by sequence: the softmax over the prefix and the sequence's own tokens as one row of keys."""
    q, k, v, pk, pv = (state[n].double() for n in ("q", "k", "v", "pk", "pv"))
    b, h, t, d = q.shape
    per = h // case["kv_heads"]
    o = torch.zeros_like(q)
    lse = torch.full((b, h, t), -math.inf, device="cuda", dtype=torch.float64)
    for i, n in enumerate(_lengths(case)):
        for j in range(t):
            own_keys = n - t + j + 1
            if own_keys < 1:
                continue
            keys = torch.cat([pk, k[i, :, :own_keys]], 1)
            values = torch.cat([pv, v[i, :, :own_keys]], 1)
            s = torch.einsum("gpd,gkd->gpk", q[i, :, j].view(-1, per, d), keys) * state["scale"]
            lse[i, :, j] = torch.logsumexp(s, -1).flatten()
            o[i, :, j] = torch.softmax(s, -1).bmm(values).view(h, d)
    return {"o": o, "lse": lse}


def _exact_norm(state, case):
    """Through each row's root mean square; the quantised values are those of the 64-bit quotients."""
    kind, most = EIGHT_BITS[case["kind"]]
    y = state["x"].double() if state["residual"] is None else state["x"].double().add(state["residual"].double())
    rms = torch.sqrt(torch.einsum("nc,nc->n", y, y) / case["width"] + state["eps"])
    h = (state["weight"].double()[None] * y / rms[:, None]).unflatten(1, (-1, case["group"] or case["width"]))
    scale = (torch.linalg.vector_norm(h, math.inf, dim=-1) / most).clamp_min(SMALLEST_SCALE)
    q = (h / scale[..., None]).clamp(-most, most).flatten(1).to(kind).double()
    return {"q": q, "scale": scale, "y": None if state["residual"] is None else y}


def _exact_logits(state, case):
    """Token by token of each row: counts from sorted histories, one table of biases."""
    n, v = case["rows"], case["vocab"]
    x = state["logits"].double()
    if state["tokens"] is not None:
        for r in range(n):
            length, prompt = int(state["token_lens"][r]), int(state["prompt_lens"][r])
            seen = state["tokens"][r, :length].unique()
            rep = float(state["repetition"][r])
            picked = x[r, seen]
            x[r, seen] = torch.where(picked > 0, picked / rep, picked * rep)
            token, count = state["tokens"][r, prompt:length].unique(return_counts=True)
            x[r, token] -= float(state["frequency"][r]) * count.double() + float(state["presence"][r])
    if state["bias_index"] is not None:
        row = torch.arange(n, device="cuda")[:, None].expand_as(state["bias_index"])
        x.index_put_((row, state["bias_index"]), state["bias_value"].double(), accumulate=True)
    x /= state["temperature"].double()[:, None]
    if state["allowed"] is not None:
        for bit in range(32):
            shut = (state["allowed"].long() & (1 << bit)) == 0
            column = x[:, bit::32]
            column.masked_fill_(shut[:, :column.shape[1]], -math.inf)
    return x
