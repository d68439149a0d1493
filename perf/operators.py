"""The operators over rows of logits, as cases to measure: the k best logits of every row
(device.top_k), distillation from a teacher's stored best logits, forward and backward
(device.distill_loss, device.distill_grad), and sampling (device.sample).

run() computes a case in its plain form (elementary torch operations), or with `own` by the
library's calls.  exact() restates the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one sequence asks for its eight best continuations: latency is what counts
        dict(name="top_k one row", op="top_k", rows=1, vocab=32000, dtype="bf16", k=8, temperature=1.0, pad=0),
        # a teacher's answer for one batch of 4096 tokens, to be stored
        dict(name="top_k teacher batch", op="top_k", rows=4096, vocab=32000, dtype="bf16", k=64, temperature=2.0, pad=0),
        # fp32 logits of a large vocabulary, many kept
        dict(name="top_k wide f32", op="top_k", rows=1024, vocab=131072, dtype="f32", k=256, temperature=1.0, pad=0),
        # odd row length behind a padded row stride: no row but the first starts on a vector
        dict(name="top_k odd f16", op="top_k", rows=777, vocab=50001, dtype="f16", k=33, temperature=1.0, pad=6),
        # a few tokens: the smallest training call
        dict(name="distill few tokens", op="distill", rows=16, vocab=32000, dtype="f32", k=16, temperature=1.0,
             pad=0, calls=1, mass=False),
        # one micro-batch of a training step, loss and gradient in one call
        dict(name="distill step", op="distill", rows=4096, vocab=32000, dtype="bf16", k=64, temperature=2.0,
             pad=0, calls=1, mass=False),
        # forward call, then the backward call with the incoming gradient of every row; the
        # teacher's probabilities keep the mass they have over the whole vocabulary
        dict(name="distill two calls f32", op="distill", rows=1000, vocab=50001, dtype="f32", k=33, temperature=1.0,
             pad=7, calls=2, mass=True),
        # large vocabulary, long batch
        dict(name="distill large", op="distill", rows=4096, vocab=131072, dtype="bf16", k=64, temperature=1.0,
             pad=0, calls=1, mass=True),
        # one request being decoded
        dict(name="sample one row", op="sample", rows=1, vocab=131072, dtype="bf16", kind="top_k+top_p", masked=False, pad=0),
        # a serving batch, every request with settings of its own
        dict(name="sample batch mixed", op="sample", rows=256, vocab=131072, dtype="bf16", kind="mixed", masked=False, pad=0),
        # temperature alone, the vocabulary restricted by a grammar
        dict(name="sample masked f32", op="sample", rows=64, vocab=50001, dtype="f32", kind="temperature", masked=True, pad=3),
        # many sequences at once (several samples per prompt), nucleus only
        dict(name="sample nucleus f16", op="sample", rows=1024, vocab=131072, dtype="f16", kind="top_p", masked=False, pad=0),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["top_k", "distill", "sample"])
    vocab = spread(1000, 131072) | rng.choice([0, 1])
    rows = spread(1, min(4096, (1 << 27) // vocab))
    case = dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["f16", "bf16", "f32"]),
                pad=rng.choice([0, 0, 1, 8, 61]))
    if op == "top_k":
        case.update(k=spread(1, 256), temperature=rng.choice([1.0, 1.0, 0.5, 2.0]))
    elif op == "distill":
        case.update(k=spread(1, 256), temperature=rng.choice([1.0, 2.0, 4.0]), calls=rng.choice([1, 2]),
                    mass=rng.choice([False, True]))
    else:
        case.update(kind=rng.choice(["top_k+top_p", "mixed", "temperature", "top_p", "min_p", "top_k"]),
                    masked=rng.choice([False, True]))
    return case


# ---- inputs -------------------------------------------------------------------------------------


def _rows(case, gen):
    """[rows, vocab] of a bulk of unlikely tokens, as a view of rows `pad` elements longer."""
    full = torch.empty(case["rows"], case["vocab"] + case["pad"], dtype=DTYPES[case["dtype"]], device="cuda")
    step = max(1, (1 << 28) // full.shape[1])
    for at in range(0, case["rows"], step):
        part = full[at:at + step]
        part.copy_(1.5 * torch.randn(part.shape, device="cuda", generator=gen))
    return full[:, :case["vocab"]]


def _places(case, n, gen):
    """n different tokens for every row, in no order."""
    r, v = case["rows"], case["vocab"]
    first = torch.randint(0, v, (r, 1), device="cuda", generator=gen)
    step = torch.randint(1, max(2, v // n), (r, 1), device="cuda", generator=gen)
    return (first + step * torch.arange(n, device="cuda")) % v


def _likely(case, n, gen, low, high):
    """Logits of n likely tokens a row: they fall off as a power of the rank, from a height between
    `low` and `high` that says how sure the model is at this position."""
    top = low + (high - low) * torch.rand(case["rows"], 1, device="cuda", generator=gen)
    rank = torch.arange(1, n + 1, device="cuda", dtype=torch.float32)
    return top - 1.2 * rank.log() + 0.5 * torch.randn(case["rows"], n, device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r, v = case["rows"], case["vocab"]
    s = dict(case=case, x=_rows(case, gen))
    if case["op"] == "distill":
        k = case["k"]
        idx = _places(case, k, gen)
        t = _likely(case, k, gen, 8.0, 16.0)
        s["x"].scatter_(1, idx, (t + torch.randn(r, k, device="cuda", generator=gen)).to(s["x"].dtype))
        t, order = t.sort(dim=1, descending=True)
        idx = idx.gather(1, order)
        # every eighth row has a shorter list, every thirtieth position is padding without a teacher
        row = torch.arange(r, device="cuda")[:, None]
        used = torch.where(row % 30 == 29, 0, torch.where(row % 8 == 7, (k + 1) // 2, k))
        idx = torch.where(torch.arange(k, device="cuda") < used, idx, -1)
        s["t"] = t.to(s["x"].dtype)
        s["idx"] = idx.to(torch.int32).contiguous()
        # the teacher's own normaliser: its list holds 0.95 of the mass
        s["teacher_lse"] = ((s["t"].float() / case["temperature"]).logsumexp(1) - math.log(0.95)) if case["mass"] else None
        s["scale"] = case["temperature"] ** 2 / r
        s["row_grad"] = 0.5 + torch.rand(r, device="cuda", generator=gen) if case["calls"] == 2 else None
        s["loss"] = torch.empty(r, device="cuda")
        s["stats"] = torch.empty(r, 2, device="cuda")
        s["grad"] = torch.empty(r, v, dtype=s["x"].dtype, device="cuda")
        return s
    n = min(100, v // 2)
    s["x"].scatter_(1, _places(case, n, gen), _likely(case, n, gen, 12.5, 20.0).to(s["x"].dtype))
    if case["op"] == "top_k":
        s["values"] = torch.empty(r, case["k"], dtype=s["x"].dtype, device="cuda")
        s["indices"] = torch.empty(r, case["k"], dtype=torch.int32, device="cuda")
        s["lse"] = torch.empty(r, device="cuda")
        return s
    row, kind = torch.arange(r, device="cuda"), case["kind"]
    mode = {"mixed": row % 5, "top_k+top_p": row * 0 + 1, "top_p": row * 0 + 2, "min_p": row * 0 + 3,
            "temperature": row * 0 + 4, "top_k": row * 0 + 5}[kind]
    # mode 0 is greedy, 4 is temperature alone
    warm = 0.6 + 0.8 * torch.rand(r, device="cuda", generator=gen)
    s["temperature"] = torch.where(mode == 0, torch.zeros_like(warm), warm)
    s["top_k"] = torch.where((mode == 1) | (mode == 5), 20 + row % 60, 0).to(torch.int32)
    s["top_p"] = torch.where((mode == 1) | (mode == 2), 0.8 + 0.15 * torch.rand(r, device="cuda", generator=gen),
                             torch.ones_like(warm))
    s["min_p"] = torch.where(mode == 3, 0.02 + 0.1 * torch.rand(r, device="cuda", generator=gen), torch.zeros_like(warm))
    s["u"] = torch.rand(r, device="cuda", generator=gen)
    s["allowed"] = None
    if case["masked"]:  # about half of the vocabulary, one bit a token, 32 to a word
        words = (v + 31) // 32
        s["allowed"] = torch.randint(-2**31, 2**31, (r, words), device="cuda", generator=gen).to(torch.int32)
    s["token"] = torch.empty(r, dtype=torch.int32, device="cuda")
    s["logprob"] = torch.empty(r, device="cuda")
    return s


# ---- one pass -----------------------------------------------------------------------------------


def _top_k(s):
    x = s["x"].float()
    values, order = x.sort(dim=1, descending=True, stable=True)
    k = s["case"]["k"]
    y = x / s["case"]["temperature"]
    m = y.amax(1, keepdim=True)
    lse = (y - m).exp().sum(1).log() + m[:, 0]
    return {"values": values[:, :k].to(s["x"].dtype), "indices": order[:, :k].to(torch.int32), "lse": lse}


def _distill(s):
    inv_t = 1.0 / s["case"]["temperature"]
    used = s["idx"] >= 0
    idx = torch.where(used, s["idx"], 0).long()
    t = torch.where(used, s["t"].float() * inv_t, -math.inf)
    norm = s["teacher_lse"]
    if norm is None:
        m = torch.where(used.any(1), t.amax(1), 0.0)
        norm = (t - m[:, None]).exp().sum(1).log() + m
    log_p = torch.where(used, t - norm[:, None], 0.0)
    p = torch.where(used, log_p.exp(), 0.0)
    z = s["x"].float()
    m = z.amax(1, keepdim=True)
    e = ((z - m) * inv_t).exp()
    total = e.sum(1, keepdim=True)
    log_q = (z.gather(1, idx) - m) * inv_t - total.log()
    loss = s["scale"] * torch.where(used, p * (log_p - log_q), 0.0).sum(1)
    c = torch.full_like(loss, s["scale"] * inv_t) if s["row_grad"] is None else s["row_grad"] * (s["scale"] * inv_t)
    grad = e * (c[:, None] * p.sum(1, keepdim=True) / total)
    grad.scatter_add_(1, idx, -c[:, None] * p)
    return {"loss": loss, "grad": grad.to(s["x"].dtype)}


def _sample(s):
    x = s["x"].double()
    v = x.shape[1]
    ok = x > -math.inf
    if s["allowed"] is not None:
        token = torch.arange(v, device=x.device)
        ok = ok & ((s["allowed"][:, token // 32] >> (token % 32)) & 1).bool()
    greedy = s["temperature"] <= 0
    temperature = torch.where(greedy, 1.0, s["temperature"].double())
    keep_k = torch.where(greedy, 1, torch.where(s["top_k"] > 0, s["top_k"], v))
    y, order = torch.where(ok, x / temperature[:, None], -math.inf).sort(dim=1, descending=True, stable=True)
    top = torch.where(y[:, :1] > -math.inf, y[:, :1], 0.0)
    w = (y - top).exp()
    w = torch.where(torch.arange(v, device=x.device) < keep_k[:, None], w, 0.0)
    before = w.cumsum(1) - w
    w = torch.where(before < s["top_p"].double()[:, None] * w.sum(1, keepdim=True), w, 0.0)
    w = torch.where(w >= s["min_p"].double()[:, None], w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)  # back into the order of the vocabulary
    c = w.cumsum(1)
    total = c[:, -1:]
    token = (c <= s["u"].double()[:, None] * total).sum(1)
    last = (w > 0).long().cumsum(1).argmax(1)  # the last token that is kept
    token = torch.minimum(token, last)
    logprob = (w.gather(1, token[:, None]) / total).log()[:, 0]
    some = total[:, 0] > 0
    return {"token": torch.where(some, token, -1).to(torch.int32),
            "logprob": torch.where(some, logprob, -math.inf).float()}


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"top_k": _top_k, "distill": _distill, "sample": _sample}[case["op"]](s)
    from raft_amd import device
    if case["op"] == "top_k":
        device.top_k(s["x"], s["values"], s["indices"], s["lse"], temperature=case["temperature"])
        return {"values": s["values"], "indices": s["indices"], "lse": s["lse"]}
    if case["op"] == "distill":
        how = dict(temperature=case["temperature"], scale=s["scale"], teacher_lse=s["teacher_lse"])
        if case["calls"] == 1:
            device.distill_loss(s["x"], s["t"], s["idx"], s["loss"], grad=s["grad"], **how)
        else:
            device.distill_loss(s["x"], s["t"], s["idx"], s["loss"], s["stats"], **how)
            device.distill_grad(s["x"], s["t"], s["idx"], s["stats"], s["grad"], row_grad=s["row_grad"], **how)
        return {"loss": s["loss"], "grad": s["grad"]}
    device.sample(s["x"], s["u"], s["token"], s["logprob"], temperature=s["temperature"], top_k=s["top_k"],
                  top_p=s["top_p"], min_p=s["min_p"], allowed=s["allowed"])
    return {"token": s["token"], "logprob": s["logprob"]}


def work(case):
    n = case["rows"] * case["vocab"]
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "top_k":  # a comparison and the sum of exponentials
        return {"bytes": n * es + case["rows"] * (case["k"] * (es + 4) + 4), "flops": 4 * n}
    if case["op"] == "distill":  # read once, written once; the sum of exponentials and the scaled exponential
        return {"bytes": 2 * n * es + case["rows"] * (case["k"] * (es + 4) + 4), "flops": 8 * n}
    return {"bytes": n * es + (n // 8 if case["masked"] else 0) + case["rows"] * 28, "flops": 6 * n}


# ---- the definitions in 64 bits -------------------------------------------------------------------


def _chunks(state):
    rows, vocab = state["x"].shape
    step = max(1, (1 << 25) // vocab)
    for at in range(0, rows, step):
        yield slice(at, min(rows, at + step))


def _log_sum_exp(y):
    m = y.max(dim=1).values
    m = torch.where(m > -math.inf, m, 0.0)
    return m + torch.log(torch.exp(y - m[:, None]).sum(1))


def exact(case, seed):
    s = prepare(case, seed)
    found = []
    if case["op"] == "top_k":
        for at in _chunks(s):
            x = s["x"][at].double()
            found.append((x.topk(case["k"], dim=1).values, _log_sum_exp(x / case["temperature"])))
        return {"values": torch.cat([f[0] for f in found]), "indices": None, "lse": torch.cat([f[1] for f in found])}
    if case["op"] == "distill":
        grad = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda")
        for at in _chunks(s):
            y = s["x"][at].double() / case["temperature"]
            log_q = y - _log_sum_exp(y)[:, None]
            valid = s["idx"][at] >= 0
            rows, cols = valid.nonzero(as_tuple=True)
            entry = s["idx"][at][rows, cols].long()
            t = s["t"][at].double() / case["temperature"]
            if case["mass"]:
                norm = s["teacher_lse"][at].double()
            else:
                norm = _log_sum_exp(t.masked_fill(~valid, -math.inf))
            log_p = (t - norm[:, None])[rows, cols]
            p = log_p.exp()
            loss = torch.zeros(valid.shape[0], dtype=torch.float64, device="cuda")
            loss.index_add_(0, rows, p * (log_p - log_q[rows, entry]))
            mass = torch.zeros_like(loss).index_add_(0, rows, p)
            d = mass[:, None] * log_q.exp()
            d.index_put_((rows, entry), -p, accumulate=True)
            up = 1.0 if s["row_grad"] is None else s["row_grad"][at].double()[:, None]
            grad[at] = d * (up * s["scale"] / case["temperature"])
            found.append(loss * s["scale"])
        return {"loss": torch.cat(found), "grad": grad}
    for at in _chunks(s):
        found.append(_exact_logprob(s, at))
    return {"token": None, "logprob": torch.cat(found)}


def _exact_logprob(s, at):
    """log of the chosen token's share, by way of probabilities in rank order."""
    x = s["x"][at].double()
    rows, v = x.shape
    x = x.masked_fill(x.isnan(), -math.inf)
    if s["allowed"] is not None:
        bit = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
        word = s["allowed"][at].long() & 0xFFFFFFFF
        x = x.masked_fill(((word[:, :, None] & bit) == 0).reshape(rows, -1)[:, :v], -math.inf)
    t = s["temperature"][at].double()[:, None]
    value, token = x.sort(dim=1, descending=True, stable=True)
    best = torch.where(value[:, :1] > -math.inf, value[:, :1], 0.0)
    p = torch.exp((value - best) / torch.where(t > 0, t, 1.0))
    p = p / p.sum(1, keepdim=True)
    rank = torch.arange(v, device="cuda").expand(rows, v)
    limit = s["top_k"][at].long()[:, None]
    limit = torch.where(t > 0, torch.where(limit > 0, limit, v), 1)
    p = p.masked_fill(rank >= limit, 0.0)
    p = p / p.sum(1, keepdim=True)
    ahead = torch.cat([torch.zeros(rows, 1, dtype=p.dtype, device="cuda"), p.cumsum(1)[:, :-1]], 1)
    drop = (ahead >= s["top_p"][at].double()[:, None]) | (p < s["min_p"][at].double()[:, None] * p[:, :1])
    p = p.masked_fill(drop, 0.0)
    p = p / p.sum(1, keepdim=True)
    token, order = token.sort(dim=1)
    p = p.gather(1, order)
    reach = p.cumsum(1)
    # the cumulative probability passes u first at the chosen token
    place = torch.searchsorted(reach, s["u"][at].double()[:, None], right=True).clamp(max=v - 1)
    return p.gather(1, place)[:, 0].log()
