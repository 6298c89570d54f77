"""Cases for the operators of the catalogue head: the softmax cross entropy over a whole item table with its gradients, table rows
held in 8 bits, and scores as 8-bit integer products.

`own` chooses between the plain form (elementary torch operations in 32 bits) and the framework's entry points.

Ranges: 1 .. 8,192 rows per call (one user .. a large training batch), 1,000 .. 1,000,000 items, widths 16 .. 128 (50 and 100 are the
presets' widths, 128 the large tables'), float32 / float16 / bfloat16; scores also with products up to 4,096 deep.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PIECE = 1 << 29          # logits of one piece of a plain form, in elements


def listed():
    return [
        # one user's next item over a CiteULike-sized catalogue: an online update, bound by latency
        dict(name="xent-1x17000-f32", op="xent", n=1, c=17000, d=100, dtype="f32", reduction="mean", bias=False, weight=False, ragged=False),
        # a training step at the 'best' preset's width and batch
        dict(name="xent-512x17000-f32", op="xent", n=512, c=17000, d=100, dtype="f32", reduction="mean", bias=False, weight=False, ragged=False),
        # the default preset's width; odd sizes, item bias with items left out, row weights, padding rows in the batch
        dict(name="xent-509x16981-d50-f32", op="xent", n=509, c=16981, d=50, dtype="f32", reduction="none", bias=True, weight=True, ragged=True),
        # a large batch against bfloat16 copies of the tables
        dict(name="xent-8192x16980-bf16", op="xent", n=8192, c=16980, d=100, dtype="bf16", reduction="mean", bias=False, weight=False, ragged=False),
        # float16 tables, a popularity correction as item bias, a ragged last batch
        dict(name="xent-1000x50021-f16", op="xent", n=1000, c=50021, d=96, dtype="f16", reduction="sum", bias=True, weight=False, ragged=True),
        # the million-item table in full precision
        dict(name="xent-4096x1000000-f32", op="xent", n=4096, c=1000000, d=128, dtype="f32", reduction="mean", bias=False, weight=False, ragged=False),
        # a batch of user rows to 8 bits and back
        dict(name="rows-512x50-bf16", op="rows", n=512, k=50, dtype="bf16"),
        # the million-item table to 8 bits and back
        dict(name="rows-1000000x128-f32", op="rows", n=1000000, k=128, dtype="f32"),
        # one user served from a CiteULike-sized table in 8 bits
        dict(name="scores-1x17000-f32", op="scores", m=1, c=17000, k=100, dtype="f32", out="f32", bias=False),
        # one user served from the million-item table
        dict(name="scores-1x1000000-bf16", op="scores", m=1, c=1000000, k=128, dtype="bf16", out="f32", bias=True),
        # all users against all candidates, as an evaluation pass scores them
        dict(name="scores-16000x16980-f32", op="scores", m=16000, c=16980, k=100, dtype="f32", out="f32", bias=True),
        # deep products (wide concatenated rows), 16-bit scores out
        dict(name="scores-2000x16384-k4096-bf16", op="scores", m=2000, c=16384, k=4096, dtype="bf16", out="bf16", bias=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["xent", "xent", "rows", "scores"])
    if op == "xent":
        n = _log(rng, 1, 8192)
        c = _log(rng, 1000, min(1000000, 4096 * 1000000 // n))
        return dict(op=op, n=n, c=c, d=_log(rng, 16, 128), dtype=rng.choice(["f32", "f32", "f16", "bf16"]),
                    reduction=rng.choice(["mean", "sum", "none"]), bias=rng.random() < 0.5, weight=rng.random() < 0.3,
                    ragged=rng.random() < 0.3)
    if op == "rows":
        k = _log(rng, 16, 4096)
        return dict(op=op, n=_log(rng, 1, min(1000000, 128000000 // k)), k=k, dtype=rng.choice(["f32", "f16", "bf16"]))
    k = _log(rng, 16, 4096)
    m = _log(rng, 1, 16000)
    c = _log(rng, 1000, max(1001, min(1000000, 16000 * 16980 // m, 2000 * 16384 * 4096 // (m * k), 512000000 // k)))
    return dict(op=op, m=m, c=c, k=k, dtype=rng.choice(["f32", "f16", "bf16"]), out=rng.choice(["f32", "f32", "f16", "bf16"]),
                bias=rng.random() < 0.5)


def _xent_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, c, d, dt = case["n"], case["c"], case["d"], DTYPES[case["dtype"]]
    table = torch.randn(c, d, generator=g, device="cuda") / math.sqrt(d)
    # popular items more often, as in a link list; a row leans towards its item, from not at all to confidently
    target = (c * torch.rand(n, generator=g, device="cuda") ** 3).long().clamp_(max=c - 1)
    lean = 2 * torch.rand(n, 1, generator=g, device="cuda")
    rows = lean * table[target] + 0.5 * torch.randn(n, d, generator=g, device="cuda") / math.sqrt(d)
    bias = weight = None
    if case["bias"]:
        bias = 0.5 * torch.randn(c, generator=g, device="cuda")
        out = torch.rand(c, generator=g, device="cuda") < 0.01      # items that are not on offer
        out[target] = False
        bias[out] = -math.inf
    if case["weight"]:
        weight = 0.5 + torch.rand(n, generator=g, device="cuda")
    if case["ragged"]:
        pad = torch.rand(n, generator=g, device="cuda") < 0.1
        pad[0] = False
        target = torch.where(pad, -1, target)
    return dict(rows=rows.to(dt), table=table.to(dt), target=target.int(), bias=bias, weight=weight)


def _float_rows(n, k, dt, g):
    # row magnitudes spread as those of embedding rows that were trained for different lengths of time
    x = torch.randn(n, k, generator=g, device="cuda")
    x *= 0.05 + torch.rand(n, 1, generator=g, device="cuda")
    return x.to(dt)


def prepare(case, seed):
    if case["op"] == "xent":
        return dict(case=case, **_xent_inputs(case, seed))
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "rows":
        return dict(case=case, x=_float_rows(case["n"], case["k"], dt, g))
    x = _float_rows(case["m"], case["k"], dt, g)
    table = _float_rows(case["c"], case["k"], torch.float32, g)
    bias = 0.5 * torch.randn(case["c"], generator=g, device="cuda") if case["bias"] else None
    state = dict(case=case, x=x, bias=bias)
    if own:      # the table is laid out once and served from many times
        from nncf_amd import catalogue
        state["table"] = catalogue.quantize_rows(table)
    else:
        state["table"] = _plain_quantize(table)
    return state


def run(state):
    case = state["case"]
    if case["op"] == "xent":
        if own:
            from nncf_amd import catalogue
            r = catalogue.softmax_xent(state["rows"], state["table"], state["target"], bias=state["bias"], weight=state["weight"],
                                       scale=10.0, reduction=case["reduction"])
            return dict(loss=r.loss, lse=r.lse, d_rows=r.d_rows, d_table=r.d_table, d_bias=r.d_bias)
        return _plain_xent(state, 10.0, case["reduction"])
    if case["op"] == "rows":
        if own:
            from nncf_amd import catalogue
            r = catalogue.quantize_rows(state["x"])
            return dict(values=r.dequantize(), scale=r.scale)
        q, scale = _plain_quantize(state["x"])
        return dict(values=q.float() * scale[:, None], scale=scale)
    out = DTYPES[case["out"]]
    if own:
        from nncf_amd import catalogue
        return catalogue.int8_scores(state["x"], state["table"], col_bias=state["bias"], dtype=out)
    return _plain_scores(state["x"], *state["table"], state["bias"], out)


# ---- plain forms ---------------------------------------------------------------------------------------------------------------


def _plain_xent(state, scale, reduction):
    rows, table, target = state["rows"].float(), state["table"].float(), state["target"].long()
    n, c = rows.shape[0], table.shape[0]
    valid = target >= 0
    left_out = torch.isinf(state["bias"]) if state["bias"] is not None else None
    if left_out is not None:
        table = torch.where(left_out[:, None], torch.zeros_like(table), table)
    g = valid.float()
    if state["weight"] is not None:
        g = g * state["weight"]
    share = g / valid.sum().clamp(min=1) if reduction == "mean" else g
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    d_rows, d_table = torch.empty_like(rows), torch.zeros_like(table)
    d_bias = torch.zeros(c, device="cuda") if state["bias"] is not None else None
    step = max(1, PIECE // c)
    for i in range(0, n, step):
        u, v, t = rows[i:i + step], valid[i:i + step], target[i:i + step].clamp(min=0)[:, None]
        z = (u @ table.t()) * scale
        if state["bias"] is not None:
            z = z + state["bias"]
        # the target's part is kept apart: p_t - 1 = -(sum of the others), which 1 - p_t would lose for a confident row
        z_t = z.gather(1, t)
        z.scatter_(1, t, torch.full_like(z_t, -math.inf))
        top = z.max(1, keepdim=True).values
        p = (z - top).exp()
        others = p.sum(1, keepdim=True)
        apart = top + others.log() - z_t                       # log of (the others' sum / the target's)
        each = apart.clamp(min=0) + torch.log1p((-apart.abs()).exp())
        loss[i:i + step] = g[i:i + step] * each[:, 0]
        lse[i:i + step] = torch.where(v, (z_t + each)[:, 0], 0.0)
        miss = 1 / (1 + (-apart).exp())                        # 1 - p_t
        p *= miss / others
        p.scatter_(1, t, -miss)
        p *= share[i:i + step, None]
        mean = torch.zeros(u.shape, dtype=torch.float64, device="cuda")      # a sum over up to a million items
        for j in range(0, c, 32768):
            mean += p[:, j:j + 32768] @ table[j:j + 32768]
        d_rows[i:i + step] = mean * scale
        d_table += (p.t() @ u) * scale
        if d_bias is not None:
            d_bias += p.sum(0)
    if reduction != "none":
        loss = loss.sum()
        if reduction == "mean":
            loss = loss / valid.sum().clamp(min=1)
    return dict(loss=loss, lse=lse, d_rows=d_rows.to(state["rows"].dtype), d_table=d_table.to(state["table"].dtype), d_bias=d_bias)


def _plain_quantize(x):
    x = x.float()
    top = x.abs().amax(1)
    full = torch.full_like(top, 127.0)      # a tensor: divisions by and of Python numbers are not rounded as divisions
    inverse = torch.where(top > 0, full / top, torch.zeros_like(top))
    return torch.round(x * inverse[:, None]).to(torch.int8), top / full


def _plain_scores(x, q_table, s_table, bias, dtype):
    q, s = _plain_quantize(x)
    m, k = q.shape
    total = None
    for j in range(0, k, 1024):      # sums of 1,024 products of two 8-bit values are whole numbers below 2^24
        part = q[:, j:j + 1024].float() @ q_table[:, j:j + 1024].float().t()
        total = part if total is None else total.double() + part
    out = total.float() * s[:, None] * s_table
    if bias is not None:
        out = out + bias
    return out.to(dtype)


def work(case):
    if case["op"] == "xent":
        n, c, d, e = case["n"], case["c"], case["d"], 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * (n + c) * d * e + n * (4 + 4 + 4) + (8 * c if case["bias"] else 0), "flops": 6.0 * n * c * d}
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rows":     # x in, 8 bits out and in again, 32 bits out; a scale per row each time
        n, k = case["n"], case["k"]
        return {"bytes": n * k * (e + 1 + 1 + 4) + 8 * n, "flops": 4.0 * n * k}
    m, c, k = case["m"], case["c"], case["k"]
    o = 4 if case["out"] == "f32" else 2
    return {"bytes": m * k * e + c * k + 4 * c + m * c * o + (4 * c if case["bias"] else 0), "flops": 2.0 * m * c * k}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------


def _exact_xent(case, seed):
    """Piece by piece of the catalogue: a first pass for the normaliser, a second for the gradients."""
    s = _xent_inputs(case, seed)
    u, v, t = s["rows"].double(), s["table"].double(), s["target"].long()
    n, c = case["n"], case["c"]
    keep = t >= 0
    beta = s["bias"].double() if s["bias"] is not None else torch.zeros(c, dtype=torch.float64, device="cuda")
    w = s["weight"].double() if s["weight"] is not None else torch.ones(n, dtype=torch.float64, device="cuda")
    w = torch.where(keep, w, 0.0)
    count = max(1, int(keep.sum()))
    step = max(1, (PIECE // 4) // n)
    pieces = [(j, min(c, j + step)) for j in range(0, c, step)]
    logit = lambda a, b: torch.addmm(beta[a:b][None, :], u, v[a:b].t(), alpha=10.0)      # noqa: E731
    norm = torch.full((n,), -math.inf, dtype=torch.float64, device="cuda")
    for a, b in pieces:
        norm = torch.logaddexp(norm, torch.logsumexp(logit(a, b), 1))
    at = t.clamp(min=0)
    each = w * (norm - 10.0 * (u * v[at]).sum(1) - beta[at])
    g = w / count if case["reduction"] == "mean" else w
    du, dv, db = torch.zeros_like(u), torch.empty_like(v), torch.empty(c, dtype=torch.float64, device="cuda")
    for a, b in pieces:
        coef = torch.exp(logit(a, b) - norm[:, None])
        inside = (at >= a) & (at < b)
        coef[inside.nonzero()[:, 0], at[inside] - a] -= 1.0
        coef *= g[:, None]
        du += 10.0 * (coef @ v[a:b])
        dv[a:b] = 10.0 * (coef.t() @ u)
        db[a:b] = coef.sum(0)
    loss = each if case["reduction"] == "none" else each.sum() / (count if case["reduction"] == "mean" else 1)
    return dict(loss=loss, lse=torch.where(keep, norm, 0.0), d_rows=du, d_table=dv, d_bias=db if s["bias"] is not None else None)


def _exact_codes(x):
    """The 8-bit codes, whose definition rounds to 32 bits twice, and the scales."""
    x = x.double()
    top = torch.linalg.vector_norm(x, ord=math.inf, dim=1)
    inverse = (127.0 / top).float().double()
    codes = (x * inverse[:, None]).float().double().round()
    return codes, top / 127.0


def exact(case, seed):
    if case["op"] == "xent":
        return _exact_xent(case, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "rows":
        codes, scale = _exact_codes(_float_rows(case["n"], case["k"], dt, g))
        return dict(values=codes * scale[:, None], scale=scale)
    x = _float_rows(case["m"], case["k"], dt, g)
    table = _float_rows(case["c"], case["k"], torch.float32, g)
    bias = 0.5 * torch.randn(case["c"], generator=g, device="cuda") if case["bias"] else None
    (a, sa), (b, sb) = _exact_codes(x), _exact_codes(table)
    out = torch.empty(case["m"], case["c"], dtype=torch.float64, device="cuda")
    for j in range(0, case["c"], 65536):
        out[:, j:j + 65536] = ((a * sa[:, None]) @ (b[j:j + 65536] * sb[j:j + 65536, None]).t())
    return out if bias is None else out + bias.double()
