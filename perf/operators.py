"""Operators of one training step of a transformer block, as measurable cases.

Three operators, each with the inputs a training program has in hand before the call:

* `attention_backward` -- gradients of softmax(scale Q K^T [+ masks]) V from the saved output and
  log-sum-exp, the probabilities recomputed; shared key/value heads, causal mask, per-batch lengths.
* `gated_residual_norm` (forward and backward) -- RMSNorm after a block, its gate and residual
  scale, the residual sum and the RMSNorm before the next block in one pass.
* `distill_loss` (forward and backward) -- divergence of a student's full-vocabulary distribution
  from a teacher of which only the top logits were kept.

`run` is the plain form in elementary torch operations while `own` is false, the calls of
`neptune_opt_b200` while it is true.
"""
from __future__ import annotations

import math

import torch

own = False

HEAD_DIM = 128
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
CHUNK = 1 << 28  # elements of one temporary of the plain forms


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # One short prompt per head in an interactive fine-tuning step: latency of the whole call.
        _attn("attn_bwd_short", 2, 4, 4, 100, True),
        # A right-padded batch of uneven conversations (one of them empty), four query heads per
        # key/value head.
        _attn("attn_bwd_padded", 4, 16, 4, 1000, True, ragged=True),
        # One long document with grouped heads.
        _attn("attn_bwd_long", 1, 32, 8, 8192, True),
        # The repository's attention configuration, every key visible.
        _attn("attn_bwd_full", 8, 32, 32, 4096, False),
        # A handful of tokens: latency.
        _norm("norm_fwd_few", "forward", "bfloat16", 1, 16, 2048, "row", "none"),
        # The repository's RMSNorm shape as 8 sequences of 2048 tokens, one gate vector per sequence.
        _norm("norm_fwd_batch", "forward", "bfloat16", 8, 2048, 4096, "sequence", "tanh"),
        # Odd width and row count in fp32, one learnt gate vector (its gradient sums over all rows).
        _norm("norm_bwd_odd", "backward", "float32", 3, 1001, 1001, "channel", "none"),
        # Backward of the batch above.
        _norm("norm_bwd_batch", "backward", "bfloat16", 8, 2048, 4096, "sequence", "tanh"),
        # A few positions scored while drafting data: latency.
        _distill("distill_fwd_few", "forward", "float32", 8, 32000, 32, 1.0, False),
        # The repository's ultra-wide logits, teacher known with its own normaliser.
        _distill("distill_fwd_wide", "forward", "bfloat16", 512, 262144, 64, 2.0, True),
        # Odd vocabulary and row count in fp16.
        _distill("distill_bwd_odd", "backward", "float16", 1003, 50001, 20, 1.5, True),
        # The logits of one long-document step.
        _distill("distill_bwd_batch", "backward", "bfloat16", 4096, 131072, 64, 1.0, False),
    ]


def _attn(name, batch, heads, kv_heads, seq, causal, ragged=False):
    return {"name": name, "op": "attention_backward", "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "seq": seq, "causal": causal, "ragged": ragged}


def _norm(name, direction, dtype, batch, seq, width, gate, act):
    return {"name": name, "op": "gated_residual_norm", "direction": direction, "dtype": dtype, "batch": batch,
            "seq": seq, "width": width, "gate": gate, "act": act}


def _distill(name, direction, dtype, rows, vocab, top, temperature, normalised):
    return {"name": name, "op": "distill_loss", "direction": direction, "dtype": dtype, "rows": rows,
            "vocab": vocab, "top": top, "temperature": temperature, "normalised": normalised}


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attention_backward", "gated_residual_norm", "distill_loss"])
    if op == "attention_backward":
        seq = _log_int(rng, 1, 8192)
        kv_heads = rng.choice([1, 2, 3, 4, 8, 16, 32])
        heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 8) if g * kv_heads <= 32])
        most = max(1, min(8, (8 * 32 * 4096 * 4096) // (heads * seq * seq)))
        case = _attn("", rng.randint(1, most), heads, kv_heads, seq, rng.random() < 0.6, rng.random() < 0.4)
    elif op == "gated_residual_norm":
        width = _log_int(rng, 64, 8192)
        batch = rng.randint(1, 8)
        seq = _log_int(rng, 1, max(1, (16384 * 4096) // (width * batch)))
        case = _norm("", rng.choice(["forward", "backward"]), rng.choice(list(DTYPES)), batch, min(seq, 8192), width,
                     rng.choice(["none", "channel", "sequence", "row"]), rng.choice(["none", "tanh", "sigmoid"]))
    else:
        vocab = _log_int(rng, 1000, 262144)
        rows = _log_int(rng, 1, min(8192, (4096 * 131072) // (2 * vocab)))
        case = _distill("", rng.choice(["forward", "backward"]), rng.choice(list(DTYPES)), rows, vocab,
                        _log_int(rng, 1, 128), rng.choice([0.7, 1.0, 2.0, 4.0]), rng.random() < 0.5)
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(case):
    """Tokens of each batch element: full, empty, then a spread of shares of the padded length."""
    n, b = case["seq"], case["batch"]
    if not case["ragged"]:
        return [n] * b
    return [n if i == 0 else 0 if i == 1 else max(1, int(n * ((0.618 * i) % 1.0))) for i in range(b)]


def prepare(case, seed):
    if case["op"] == "attention_backward":
        return _prepare_attention(case, seed)
    if case["op"] == "gated_residual_norm":
        return _prepare_norm(case, seed)
    return _prepare_distill(case, seed)


def _prepare_attention(case, seed):
    gen = _generator(seed)
    b, h, hk, n, d = case["batch"], case["heads"], case["kv_heads"], case["seq"], HEAD_DIM

    def normal(heads):
        return torch.randn(b, heads, n, d, device="cuda", generator=gen).to(torch.bfloat16)

    q, k, v, grad = normal(h), normal(hk), normal(hk), normal(h)
    lens = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
    state = {"case": case, "q": q, "k": k, "v": v, "grad": grad, "lens": lens, "scale": 1.0 / math.sqrt(d)}
    # What the forward pass saved: its output and each row's log-sum-exp.
    out = torch.empty_like(q)
    lse = torch.empty(b, h, n, device="cuda")
    for i, j, group in _head_chunks(state):
        qc, kc, vc = q[i, group].float(), k[i, j].float(), v[i, j].float()
        s = torch.matmul(qc, kc.t()) * state["scale"]
        s = s.masked_fill(~_visible(state, i), -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
        total = p.sum(-1, keepdim=True)
        empty = total == 0
        out[i, group] = (torch.matmul(p, vc) / torch.where(empty, 1.0, total)).to(out.dtype)
        lse[i, group] = torch.where(empty, -math.inf, top + torch.log(total)).squeeze(-1)
    state.update(out=out, lse=lse)
    return state


def _head_chunks(state):
    """(batch, key/value head, query heads) pieces whose score matrices stay below CHUNK elements."""
    case = state["case"]
    per = case["heads"] // case["kv_heads"]
    step = max(1, min(per, CHUNK // max(1, case["seq"] ** 2)))
    for i in range(case["batch"]):
        for j in range(case["kv_heads"]):
            for g in range(0, per, step):
                yield i, j, slice(j * per + g, j * per + min(per, g + step))


def _visible(state, i):
    """[seq, seq] truth of which key each query of batch element i sees."""
    case = state["case"]
    pos = torch.arange(case["seq"], device="cuda")
    ok = torch.ones(case["seq"], case["seq"], dtype=torch.bool, device="cuda")
    if case["causal"]:
        ok = pos[None, :] <= pos[:, None]
    if state["lens"] is not None:
        ok = ok & (pos[None, :] < state["lens"][i]) & (pos[:, None] < state["lens"][i])
    return ok


def _prepare_norm(case, seed):
    gen = _generator(seed)
    b, n, c, dt = case["batch"], case["seq"], case["width"], DTYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * std + mean).to(dt)

    gate_shape = {"none": None, "channel": (c,), "sequence": (b, 1, c), "row": (b, n, c)}[case["gate"]]
    state = {"case": case, "x": normal(b, n, c), "residual": normal(b, n, c, std=2.0),
             "gate": None if gate_shape is None else normal(*gate_shape, mean=0.5, std=0.5),
             "post": normal(c, mean=1.0, std=0.1), "pre": normal(c, mean=1.0, std=0.1),
             "scale": 0.5, "eps": 1e-6}
    if case["direction"] == "backward":
        state["grad_res"], state["grad_norm"] = normal(b, n, c), normal(b, n, c)
        x = state["x"].float()
        r1 = torch.rsqrt((x * x).mean(-1) + state["eps"])
        y = state["residual"].float() + state["scale"] * _act(state) * x * r1[..., None] * state["post"].float()
        state["rstd"] = torch.stack([r1, torch.rsqrt((y * y).mean(-1) + state["eps"])], dim=-1)
    return state


def _act(state):
    if state["gate"] is None:
        return 1.0
    g = state["gate"].float()
    return {"none": lambda t: t, "tanh": torch.tanh, "sigmoid": torch.sigmoid}[state["case"]["act"]](g)


def _prepare_distill(case, seed):
    gen = _generator(seed)
    rows, vocab, top, dt = case["rows"], case["vocab"], min(case["top"], case["vocab"]), DTYPES[case["dtype"]]
    logits = torch.empty(rows, vocab, device="cuda", dtype=dt)
    step = max(1, CHUNK // vocab)
    for r in range(0, rows, step):
        logits[r:r + step] = torch.randn(min(step, rows - r), vocab, device="cuda", generator=gen) * 3.0
    # Distinct indices in every row: an arithmetic progression that does not wrap onto itself.
    first = torch.randint(0, vocab, (rows, 1), device="cuda", generator=gen)
    stride = torch.randint(1, vocab // top + 1, (rows, 1), device="cuda", generator=gen)
    index = (first + stride * torch.arange(top, device="cuda")) % vocab
    teacher = torch.randn(rows, top, device="cuda", generator=gen).mul_(2.0).add_(10.0)
    teacher = teacher.sort(-1, descending=True).values
    # The student is roughly right about the teacher's choices.
    noise = torch.randn(rows, top, device="cuda", generator=gen)
    logits.scatter_(1, index, (teacher + noise).to(dt))
    teacher = teacher.to(dt)
    # Rows with fewer kept logits, and prompt rows without any (index -1).
    kept = torch.randint(1, top + 1, (rows, 1), device="cuda", generator=gen)
    chance = torch.rand(rows, 1, device="cuda", generator=gen)
    kept = torch.where(chance < 0.1, 0, torch.where(chance < 0.3, kept, top))
    index = torch.where(torch.arange(top, device="cuda") < kept, index, -1)
    state = {"case": case, "logits": logits, "teacher": teacher, "index": index, "norm": None}
    if case["normalised"]:
        # Logits that were not kept add a share of the teacher's mass.
        scaled = teacher.float() / case["temperature"]
        state["norm"] = torch.logsumexp(scaled, -1) + 0.1 * torch.rand(rows, device="cuda", generator=gen)
    if case["direction"] == "backward":
        # The mean over rows; fp16 training scales its loss so that small gradients stay normal.
        weight = 65536.0 if case["dtype"] == "float16" else 1.0
        state["grad"] = torch.rand(rows, device="cuda", generator=gen) * (weight / rows)
        state["stats"] = _plain_distill_forward(state)[1]
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "attention_backward":
        return _plain_attention_backward(state)
    if case["op"] == "gated_residual_norm":
        return _plain_norm_forward(state) if case["direction"] == "forward" else _plain_norm_backward(state)
    return _plain_distill_forward(state) if case["direction"] == "forward" else _plain_distill_backward(state)


def _run_own(state, case):
    import neptune_opt_b200 as NB

    if case["op"] == "attention_backward":
        return NB.attention_backward(state["q"], state["k"], state["v"], state["out"], state["lse"], state["grad"],
                                     causal=case["causal"], scale=state["scale"], seq_lens=state["lens"])
    if case["op"] == "gated_residual_norm":
        kw = {"post_weight": state["post"], "pre_weight": state["pre"], "gate_act": case["act"],
              "residual_scale": state["scale"]}
        if case["direction"] == "forward":
            return NB.run_gated_residual_norm(state["x"], state["residual"], state["gate"], eps=state["eps"], **kw)
        return NB.gated_residual_norm_backward(state["grad_res"], state["grad_norm"], state["x"], state["residual"],
                                               state["gate"], state["rstd"], **kw)
    if case["direction"] == "forward":
        return NB.run_distill_loss(state["logits"], state["teacher"], state["index"],
                                   temperature=case["temperature"], teacher_lse=state["norm"])
    return NB.distill_loss_backward(state["grad"], state["logits"], state["teacher"], state["index"], state["stats"],
                                    temperature=case["temperature"])


def _plain_attention_backward(state):
    q, k, v = state["q"], state["k"], state["v"]
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    sums = None
    for i, j, group in _head_chunks(state):
        if group.start % (state["case"]["heads"] // state["case"]["kv_heads"]) == 0:
            sums = (torch.zeros(k.shape[2:], device="cuda"), torch.zeros(k.shape[2:], device="cuda"))
        qc, kc, vc = q[i, group].float(), k[i, j].float(), v[i, j].float()
        gc = state["grad"][i, group].float()
        seen = _visible(state, i)
        s = torch.matmul(qc, kc.t()) * state["scale"]
        p = torch.where(seen, torch.exp(s - state["lse"][i, group][..., None]), 0.0)
        delta = (gc * state["out"][i, group].float()).sum(-1, keepdim=True)
        ds = p * (torch.matmul(gc, vc.t()) - delta)
        dq[i, group] = (torch.matmul(ds, kc) * state["scale"]).to(dq.dtype)
        sums[0].add_(torch.matmul(ds.transpose(-1, -2), qc).sum(0))
        sums[1].add_(torch.matmul(p.transpose(-1, -2), gc).sum(0))
        dk[i, j] = (sums[0] * state["scale"]).to(dk.dtype)
        dv[i, j] = sums[1].to(dv.dtype)
    return dq, dk, dv


def _plain_norm_forward(state):
    x, dt = state["x"].float(), state["x"].dtype
    r1 = torch.rsqrt((x * x).mean(-1, keepdim=True) + state["eps"])
    y = state["residual"].float() + state["scale"] * _act(state) * (x * r1 * state["post"].float())
    r2 = torch.rsqrt((y * y).mean(-1, keepdim=True) + state["eps"])
    return y.to(dt), (y * r2 * state["pre"].float()).to(dt), torch.cat([r1, r2], dim=-1)


def _plain_norm_backward(state):
    x, dt, width = state["x"].float(), state["x"].dtype, state["case"]["width"]
    w1, w2 = state["post"].float(), state["pre"].float()
    r1, r2 = state["rstd"][..., :1], state["rstd"][..., 1:]
    a = _act(state)
    xhat = x * r1
    z = xhat * w1
    yhat = (state["residual"].float() + state["scale"] * a * z) * r2
    gh = state["grad_norm"].float()
    t = gh * w2
    dy = state["grad_res"].float() + r2 * (t - yhat * (t * yhat).mean(-1, keepdim=True))
    dpre = (gh * yhat).reshape(-1, width).sum(0)
    dz = state["scale"] * a * dy
    dpost = (dz * xhat).reshape(-1, width).sum(0)
    u = dz * w1
    dx = r1 * (u - xhat * (u * xhat).mean(-1, keepdim=True))
    dgate = None
    if state["gate"] is not None:
        slope = {"none": 1.0, "tanh": 1.0 - a * a, "sigmoid": a * (1.0 - a)}[state["case"]["act"]]
        dgate = state["scale"] * slope * z * dy
        if state["case"]["gate"] == "channel":
            dgate = dgate.reshape(-1, width).sum(0)
        elif state["case"]["gate"] == "sequence":
            dgate = dgate.sum(1, keepdim=True)
        dgate = dgate.to(dt)
    return dx.to(dt), dy.to(dt), dgate, dpost.to(dt), dpre.to(dt)


def _plain_distill_rows(state, rows):
    """Teacher probabilities of the kept logits (0 where there is none) and their normaliser."""
    valid = state["index"][rows] >= 0
    t = torch.where(valid, state["teacher"][rows].float() / state["case"]["temperature"], -math.inf)
    if state["norm"] is not None:
        norm = state["norm"][rows]
    else:
        top = t.amax(-1)
        top = torch.where(torch.isinf(top), 0.0, top)
        norm = top + torch.log(torch.exp(t - top[:, None]).sum(-1))
    p = torch.where(valid, torch.exp(t - norm[:, None]), 0.0)
    return valid, t, norm, p


def _row_chunks(state):
    rows, vocab = state["logits"].shape
    step = max(1, CHUNK // vocab)
    return [slice(r, min(rows, r + step)) for r in range(0, rows, step)]


def _plain_distill_forward(state):
    loss = torch.empty(state["logits"].shape[0], device="cuda")
    stats = torch.empty(state["logits"].shape[0], 3, device="cuda")
    for rows in _row_chunks(state):
        valid, t, norm, p = _plain_distill_rows(state, rows)
        x = state["logits"][rows].float() / state["case"]["temperature"]
        top = x.amax(-1, keepdim=True)
        lse = (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))).squeeze(-1)
        picked = torch.gather(x, 1, state["index"][rows].clamp(min=0))
        terms = p * ((t - norm[:, None]) - (picked - lse[:, None]))
        loss[rows] = torch.where(p > 0, terms, 0.0).sum(-1)
        stats[rows] = torch.stack([lse, norm, p.sum(-1)], dim=-1)
    return loss, stats


def _plain_distill_backward(state):
    out = torch.empty_like(state["logits"])
    for rows in _row_chunks(state):
        valid, t, _, _ = _plain_distill_rows(state, rows)
        lse, norm, mass = state["stats"][rows].unbind(-1)
        p = torch.where(valid, torch.exp(t - norm[:, None]), 0.0)
        x = state["logits"][rows].float() / state["case"]["temperature"]
        d = torch.exp(x - lse[:, None]) * mass[:, None]
        d.scatter_add_(1, state["index"][rows].clamp(min=0), -p)
        d *= (state["grad"][rows] / state["case"]["temperature"])[:, None]
        out[rows] = torch.where(valid.any(-1, keepdim=True), d, 0.0).to(out.dtype)
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "attention_backward":
        b, h, hk, n, d = case["batch"], case["heads"], case["kv_heads"], case["seq"], HEAD_DIM
        lens = _lengths(case)
        pairs = sum(t * (t + 1) // 2 if case["causal"] else t * t for t in lens)
        # q, o, dO and lse in, dQ out; k, v in, dK, dV out (gradients are written for every token).
        moved = sum(lens) * (3 * h * d * 2 + h * 4 + 2 * hk * d * 2) + b * n * (h + 2 * hk) * d * 2
        return {"bytes": moved, "flops": 10 * d * h * pairs}
    if case["op"] == "gated_residual_norm":
        b, n, c = case["batch"], case["seq"], case["width"]
        size = 4 if case["dtype"] == "float32" else 2
        rows, full = b * n, b * n * c * size
        gate = {"none": 0, "channel": c, "sequence": b * c, "row": rows * c}[case["gate"]] * size
        if case["direction"] == "forward":
            return {"bytes": 4 * full + gate + 2 * c * size + rows * 8, "flops": 10 * rows * c}
        return {"bytes": 6 * full + 2 * gate + 4 * c * size + rows * 8, "flops": 25 * rows * c}
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    size = 4 if case["dtype"] == "float32" else 2
    full, kept = rows * vocab * size, rows * top * (size + 8)
    if case["direction"] == "forward":
        return {"bytes": full + kept + rows * (16 + (4 if case["normalised"] else 0)), "flops": 4 * rows * vocab}
    return {"bytes": 2 * full + kept + rows * 16, "flops": 4 * rows * vocab}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attention_backward":
        return _exact_attention(state, case)
    if case["op"] == "gated_residual_norm":
        return _exact_norm(state, case)
    return _exact_distill(state, case)


def _exact_attention(state, case):
    """Per batch element and head over its own tokens only: the Jacobian of each softmax row,
    diag(p) - p p^T, in the saved output's terms."""
    q, k, v, g, o = (state[n].double() for n in ("q", "k", "v", "grad", "out"))
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    per = case["heads"] // case["kv_heads"]
    for i, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        hidden = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1) if case["causal"] else None
        for h in range(case["heads"]):
            j = h // per
            kk, vv, qq, gg = k[i, j, :n], v[i, j, :n], q[i, h, :n], g[i, h, :n]
            p = qq.mul(state["scale"]).mm(kk.T).sub_(state["lse"][i, h, :n, None].double()).exp_()
            if hidden is not None:
                p.masked_fill_(hidden, 0.0)
            dv[i, j, :n] += p.T.mm(gg)
            p.mul_(gg.mm(vv.T).sub_(torch.einsum("nd,nd->n", gg, o[i, h, :n])[:, None]))
            dq[i, h, :n] = p.mm(kk) * state["scale"]
            dk[i, j, :n] += p.T.mm(qq) * state["scale"]
    return dq, dk, dv


def _exact_norm(state, case):
    """Forward in 64 bits; backward by differentiating the same two normalisations row by row with
    the given reciprocal norms."""
    c = case["width"]
    wide = (case["batch"], case["seq"], c)
    x, r = state["x"].double(), state["residual"].double()
    w1, w2 = state["post"].double(), state["pre"].double()
    a, slope = torch.ones((), dtype=torch.float64, device="cuda"), None
    if state["gate"] is not None:
        a = state["gate"].double()
        if case["act"] == "tanh":
            a = 1.0 - 2.0 / (torch.exp(2.0 * a) + 1.0)
            slope = 1.0 - a ** 2
        elif case["act"] == "sigmoid":
            a = 1.0 / (1.0 + torch.exp(-a))
            slope = a - a ** 2
        else:
            slope = torch.ones_like(a)
    if case["direction"] == "forward":
        n1 = 1.0 / torch.sqrt(x.pow(2).sum(-1) / c + state["eps"])
        y = r + state["scale"] * (a * w1 * x) * n1[..., None]
        n2 = 1.0 / torch.sqrt(y.pow(2).sum(-1) / c + state["eps"])
        return y, y * n2[..., None] * w2, torch.stack([n1, n2], -1)
    n1, n2 = (t[..., None] for t in state["rstd"].double().unbind(-1))
    y = r + state["scale"] * (a * w1 * x) * n1
    gh = state["grad_norm"].double()
    dy = state["grad_res"].double() + gh * w2 * n2 - y * n2 ** 3 * ((gh * w2 * y).sum(-1, keepdim=True) / c)
    dpre = torch.einsum("bsc,bsc,bs->c", gh, y, n2[..., 0])
    da = state["scale"] * n1 * x * dy * w1
    dpost = torch.einsum("bsc,bsc,bs->c", a.expand(wide) * x, dy, n1[..., 0]) * state["scale"]
    u = state["scale"] * a * w1 * dy
    dx = u * n1 - x * n1 ** 3 * ((u * x).sum(-1, keepdim=True) / c)
    dgate = None
    if state["gate"] is not None:
        dgate = da * slope
        if case["gate"] == "channel":
            dgate = dgate.flatten(0, 1).sum(0)
        elif case["gate"] == "sequence":
            dgate = dgate.sum(1, keepdim=True)
    return dx, dy, dgate, dpost, dpre


def _exact_distill(state, case):
    rows, vocab = state["logits"].shape
    inv = 1.0 / case["temperature"]
    valid = state["index"] >= 0
    t = (state["teacher"].double() * inv).masked_fill(~valid, -math.inf)
    if case["direction"] == "forward":
        norm = torch.logsumexp(t, -1) if state["norm"] is None else state["norm"].double()
        lse = torch.empty(rows, dtype=torch.float64, device="cuda")
        picked = torch.empty_like(t)
        for r in range(rows):
            row = state["logits"][r].double() * inv
            lse[r] = torch.logsumexp(row, 0)
            picked[r] = row[state["index"][r].clamp(min=0)]
        logp = (t - norm[:, None]).masked_fill(~valid, -math.inf)
        p = logp.exp()
        gap = (logp - picked + lse[:, None]).masked_fill(~valid, 0.0)
        return (p * gap).sum(-1), torch.stack([lse, norm, p.sum(-1)], -1)
    lse, norm, mass = state["stats"].double().unbind(-1)
    p = (t - norm[:, None]).exp().masked_fill(~valid, 0.0)
    weight = state["grad"].double() * inv
    out = torch.empty(rows, vocab, dtype=torch.float64, device="cuda")
    for r in range(rows):
        out[r] = (state["logits"][r].double() * inv - lse[r]).exp_() * (mass[r] * weight[r])
    keep = valid.nonzero()
    out.index_put_((keep[:, 0], state["index"][valid]), -(p * weight[:, None])[valid], accumulate=True)
    return out
