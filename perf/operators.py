"""What the operators between tokens and rows are measured on.

Three groups, which share the vocabulary as their axis:
  embedding_lookup / embedding_grad             token numbers -> scaled rows, and the table's gradient
  distill_loss / distill_grad / .._loss_and_grad   loss against a teacher's top logits, and its gradient
  sample                                        one token a row from temperature, top-k, top-p and min-p, and its log probability

`run` computes them in elementary torch operations, or (own = True) through
moderngpu_amd's calls.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # One decode step of a small batch: the latency of one launch counts.
        dict(name="lookup_decode", op="lookup", tokens=16, vocab=32768, dim=4096, dtype="bf16", scale=1.0),
        # A prompt or a training batch of a wide model with scaled embeddings.
        dict(name="lookup_prompt", op="lookup", tokens=16384, vocab=131072, dim=4096, dtype="bf16", scale=64.0),
        # Sizes that nothing divides, 32-bit rows.
        dict(name="lookup_odd", op="lookup", tokens=4099, vocab=50021, dim=1023, dtype="f32", scale=0.5),
        # The gradient of a training batch, as a whole table.
        dict(name="grad_batch", op="grad", tokens=16384, vocab=65536, dim=2048, dtype="bf16", out="bf16", scale=1.0),
        # Two micro-batches into one 32-bit gradient: the first writes it, the second adds.
        dict(name="grad_two_steps", op="grad_steps", tokens=16384, vocab=32768, dim=4096, dtype="bf16", out="f32", scale=64.0),
        # A short odd batch in 32 bits.
        dict(name="grad_odd", op="grad", tokens=1537, vocab=10007, dim=515, dtype="f32", out="f32", scale=2.0),
        # A training step's rows, 64 teacher logits each, prompt rows masked.
        dict(name="distill_batch", op="distill_step", rows=4096, vocab=32768, top=64, dtype="bf16", tau=2.0, masked=0.2),
        # A wide vocabulary: a row is longer than what one thread group keeps in shared memory.
        dict(name="distill_wide", op="distill_step", rows=2048, vocab=131072, top=128, dtype="bf16", tau=1.0, masked=0.0),
        # Loss first, gradient later from what the loss kept: rows that start at odd addresses.
        dict(name="distill_odd", op="distill_pair", rows=333, vocab=50021, top=17, dtype="f32", tau=1.5, masked=0.1),
        # One answer being written: a single row.
        dict(name="sample_one", op="sample", rows=1, vocab=131072, dtype="bf16", mode="all"),
        # A full serving batch without top-k: every logit's probability counts.
        dict(name="sample_batch", op="sample", rows=256, vocab=131072, dtype="bf16", mode="top_p"),
        # Requests with settings of their own, 32-bit logits, odd row length.
        dict(name="sample_odd", op="sample", rows=33, vocab=50021, dtype="f32", mode="mixed"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high, step):
    n = _log_int(rng, low, high)
    return max(low, n // step * step) if rng.random() < 0.5 else n


def _draw(rng):
    op = rng.choice(["lookup", "grad", "grad_steps", "distill_step", "distill_pair", "sample"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op in ("lookup", "grad", "grad_steps"):
        c = dict(op=op, tokens=_size(rng, 1, 16384, 64), vocab=_size(rng, 1000, 131072, 64),
                 dim=_size(rng, 64, 8192, 64), dtype=dtype, scale=rng.choice([1.0, 0.25, 45.25]))
        if op != "lookup":
            c["out"] = rng.choice([dtype, "f32"])
        return c
    if op == "sample":
        return dict(op=op, rows=_size(rng, 1, 256, 8), vocab=_size(rng, 1000, 131072, 64), dtype=dtype,
                    mode=rng.choice(["all", "top_k", "top_p", "min_p", "mixed", "free"]))
    return dict(op=op, rows=_size(rng, 1, 4096, 64), vocab=_size(rng, 1000, 131072, 64), top=_size(rng, 1, 256, 8),
                dtype=dtype, tau=rng.choice([1.0, 2.0, 0.7]), masked=rng.choice([0.0, 0.1, 0.5]))


def draw(rng):
    while True:
        c = _draw(rng)
        if work(c)["bytes"] <= 1.05e9:
            return c


# ---- inputs ----------------------------------------------------------------

def _token_weights(vocab):
    """Frequencies of tokens in text: rank r about 1 / (r + 2.7)."""
    w = 1.0 / (np.arange(vocab, dtype=np.float64) + 2.7)
    return w / w.sum()


def _tokens(case, gen, dev):
    cdf = torch.from_numpy(np.cumsum(_token_weights(case["vocab"]))).to(dev)
    u = torch.rand(case["tokens"], generator=gen, device=dev, dtype=torch.float64)
    rank = torch.searchsorted(cdf, u).clamp_(max=case["vocab"] - 1)
    places = torch.randperm(case["vocab"], generator=gen, device=dev)     # frequent tokens lie anywhere
    return places[rank].to(torch.int32)


def _places(rows, count, vocab, gen, dev):
    """`count` distinct columns a row, in no order."""
    width = vocab // count
    at = torch.arange(count, device=dev) * width + torch.randint(0, width, (rows, count), generator=gen, device=dev)
    return at.gather(1, torch.rand((rows, count), generator=gen, device=dev).argsort(1))


def _normal(shape, gen, dev, dtype, std=1.0):
    return torch.empty(shape, device=dev, dtype=dtype).normal_(0.0, std, generator=gen)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    op, dtype = case["op"], TYPES[case["dtype"]]
    s = {"op": op}
    if op == "lookup":
        s["table"] = _normal((case["vocab"], case["dim"]), gen, dev, dtype, 0.02)
        s["ids"] = _tokens(case, gen, dev)
        s["scale"] = case["scale"]
    elif op in ("grad", "grad_steps"):
        steps = 2 if op == "grad_steps" else 1
        s["grads"] = [_normal((case["tokens"], case["dim"]), gen, dev, dtype, 0.1) for _ in range(steps)]
        s["ids"] = [_tokens(case, gen, dev) for _ in range(steps)]
        s["scale"], s["vocab"], s["out_type"] = case["scale"], case["vocab"], TYPES[case["out"]]
        # the parameter's gradient buffer, which a training program holds on to
        s["out"] = torch.zeros((case["vocab"], case["dim"]), device=dev, dtype=TYPES[case["out"]])
    elif op in ("distill_step", "distill_pair"):
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        logits = _normal((rows, vocab), gen, dev, dtype, 2.0)
        ids = _places(rows, top, vocab, gen, dev)
        teacher = _normal((rows, top), gen, dev, torch.float32, 2.0).sort(dim=1, descending=True).values
        # a student that has learnt something: the teacher's tokens stand out
        logits.scatter_(1, ids, (teacher + 5.0 + _normal((rows, top), gen, dev, torch.float32)).to(dtype))
        # some rows have fewer teacher tokens than there is room for
        kept = torch.randint(max(1, top // 2), top + 1, (rows, 1), generator=gen, device=dev)
        ids = torch.where(torch.arange(top, device=dev)[None] < kept, ids, torch.full_like(ids, -1))
        weights = torch.rand(rows, generator=gen, device=dev) + 0.5
        off = torch.randperm(rows, generator=gen, device=dev)[:int(case["masked"] * rows)]
        weights[off] = 0.0
        weights *= (4096.0 if case["dtype"] == "f16" else 1.0) / rows       # a mean over rows; 16-bit floats train with a loss scale
        s.update(logits=logits, ids=ids.to(torch.int32), teacher=teacher, weights=weights, tau=case["tau"],
                 incoming=torch.rand(rows, generator=gen, device=dev) + 0.5)
    elif op == "sample":
        rows, vocab, mode = case["rows"], case["vocab"], case["mode"]
        logits = _normal((rows, vocab), gen, dev, dtype, 2.0)
        peaks = _places(rows, 48, vocab, gen, dev)
        logits.scatter_(1, peaks, _normal((rows, 48), gen, dev, torch.float32, 2.5).add_(8.0).to(dtype))
        banned = torch.randint(0, vocab, (rows, 16), generator=gen, device=dev)      # tokens that a grammar rules out
        logits.scatter_(1, banned, -math.inf)
        pick = torch.randint(0, 4, (rows,), generator=gen, device=dev)
        full = lambda v, t: torch.full((rows,), v, dtype=t, device=dev)  # noqa: E731
        temperature, top_k, top_p, min_p = full(0.8, torch.float32), full(0, torch.int32), full(1.0, torch.float32), full(0.0, torch.float32)
        if mode == "mixed":
            temperature = torch.tensor([0.0, 0.6, 1.0, 1.3], device=dev)[pick]
            pick = torch.randint(0, 4, (rows,), generator=gen, device=dev)
            top_k = torch.tensor([0, 1, 40, 1000], device=dev, dtype=torch.int32)[pick]
            pick = torch.randint(0, 4, (rows,), generator=gen, device=dev)
            top_p = torch.tensor([1.0, 0.5, 0.9, 0.99], device=dev)[pick]
            min_p = torch.tensor([0.0, 0.05, 0.0, 0.001], device=dev)[pick]
        if mode in ("all", "top_k"):
            top_k = full(50, torch.int32)
        if mode in ("all", "top_p"):
            top_p = full(0.95, torch.float32)
        if mode in ("all", "min_p"):
            min_p = full(0.02, torch.float32)
        s.update(logits=logits, uniform=torch.rand(rows, generator=gen, device=dev), temperature=temperature,
                 top_k=top_k, top_p=top_p, min_p=min_p)
    return s


# ---- one pass ---------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state["op"]](state)


def _run_own(s):
    import moderngpu_amd as m
    op = s["op"]
    if op == "lookup":
        return m.embedding_lookup(s["table"], s["ids"], scale=s["scale"])
    if op in ("grad", "grad_steps"):
        out = m.embedding_grad(s["grads"][0], s["ids"][0], scale=s["scale"], out=s["out"])
        if op == "grad_steps":
            m.embedding_grad(s["grads"][1], s["ids"][1], scale=s["scale"], out=out, accumulate=True)
        return out
    if op == "distill_step":
        loss, grad = m.distill_loss_and_grad(s["logits"], s["ids"], s["teacher"], temperature=s["tau"], weights=s["weights"])
        return {"loss": loss, "grad": grad}
    if op == "distill_pair":
        loss, lse = m.distill_loss(s["logits"], s["ids"], s["teacher"], temperature=s["tau"], weights=s["weights"])
        grad = m.distill_grad(s["logits"], lse, s["ids"], s["teacher"], s["weights"] * s["incoming"], temperature=s["tau"])
        return {"loss": loss, "grad": grad}
    token, logprob = m.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return {"token": token, "logprob": logprob}


def _plain_lookup(s):
    table = s["table"]
    return (table[s["ids"].long()].float() * s["scale"]).to(table.dtype)


def _plain_sum(grad, ids, scale, vocab):
    total = torch.zeros((vocab, grad.shape[1]), dtype=torch.float32, device=grad.device)
    return total.index_add_(0, ids.long(), grad.float()).mul_(scale)


def _plain_grad(s):
    return _plain_sum(s["grads"][0], s["ids"][0], s["scale"], s["vocab"]).to(s["out_type"])


def _plain_grad_steps(s):
    first = _plain_grad(s)
    second = _plain_sum(s["grads"][1], s["ids"][1], s["scale"], s["vocab"])
    return (first.float() + second).to(s["out_type"])


def _plain_distill(s, coefficients):
    tau, w = s["tau"], s["weights"]
    z = s["logits"].float() / tau
    vocab = z.shape[1]
    ids = s["ids"].long()
    valid = (ids >= 0) & (ids < vocab)
    at = ids.clamp(0, vocab - 1)
    a = torch.where(valid, s["teacher"].float() / tau, torch.full_like(s["teacher"], -math.inf))
    a = a - a.amax(1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(a)
    total = p.sum(1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    top = z.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    log_p = torch.log(torch.where(p > 0, p, torch.ones_like(p)))
    term = torch.where(p > 0, p * (log_p - (z.gather(1, at) - lse)), torch.zeros_like(p))
    loss = torch.where(w != 0, w * tau * tau * term.sum(1), torch.zeros_like(w))
    q = torch.exp(z - lse) * (total > 0)
    diff = q.scatter_add_(1, at, -p)
    c = coefficients[:, None]
    grad = torch.where(c != 0, c * tau * diff, torch.zeros_like(diff))
    return {"loss": loss, "grad": grad.to(s["logits"].dtype)}


def _plain_sample(s):
    # 64 bits: a sum next to a border decides which token is drawn.
    z = s["logits"].double()
    z = torch.where(torch.isnan(z), torch.full_like(z, -math.inf), z).clamp_(max=torch.finfo(torch.float32).max)
    rows, vocab = z.shape
    order_z, order = torch.sort(z, dim=1, descending=True, stable=True)
    temperature = s["temperature"].double()[:, None]
    greedy = ~(temperature > 0)
    scaled = (order_z - order_z[:, :1]) / torch.where(greedy, torch.ones_like(temperature), temperature)
    mass = torch.exp(torch.where(torch.isneginf(order_z), order_z, scaled))
    rank = torch.arange(vocab, device=z.device)[None]
    k = s["top_k"].long()[:, None]
    k = torch.where((k <= 0) | greedy, torch.where(greedy, torch.ones_like(k), torch.full_like(k, vocab)), k)
    mass = mass * (rank < k)
    before = torch.cumsum(mass, 1) - mass
    top_p = s["top_p"].double()[:, None]
    keep = (before < top_p * mass.sum(1, keepdim=True)) | (top_p >= 1) | (rank == 0)
    keep &= (mass >= s["min_p"].double()[:, None]) | (rank == 0)
    kept = torch.zeros_like(mass).scatter_(1, order, mass * keep)       # back in the order of the tokens
    sums = torch.cumsum(kept, 1)
    last = torch.where(kept > 0, rank, torch.full_like(rank, -1)).amax(1)
    token = (sums <= s["uniform"].double()[:, None] * sums[:, -1:]).sum(1)
    token = torch.minimum(token, last)[:, None]
    share = kept.gather(1, token) / sums[:, -1:]
    return {"token": token[:, 0].to(torch.int32), "logprob": torch.log(share[:, 0]).float()}


_PLAIN = {"lookup": _plain_lookup, "grad": _plain_grad, "grad_steps": _plain_grad_steps,
          "distill_step": lambda s: _plain_distill(s, s["weights"]),
          "distill_pair": lambda s: _plain_distill(s, s["weights"] * s["incoming"]), "sample": _plain_sample}


# ---- what a pass cannot do without ------------------------------------------

def _distinct(case):
    """Expected number of distinct tokens of a batch."""
    return float(-np.expm1(case["tokens"] * np.log1p(-_token_weights(case["vocab"]))).sum())


def work(case):
    op, e = case["op"], SIZE[case["dtype"]]
    if op == "lookup":
        t, d = case["tokens"], case["dim"]
        return {"bytes": 4 * t + _distinct(case) * d * e + t * d * e, "flops": t * d}
    if op in ("grad", "grad_steps"):
        t, d, o = case["tokens"], case["dim"], SIZE[case["out"]]
        whole = 4 * t + t * d * e + case["vocab"] * d * o
        if op == "grad":
            return {"bytes": whole, "flops": 2 * t * d}
        return {"bytes": whole + 4 * t + t * d * e + 2 * _distinct(case) * d * o, "flops": 4 * t * d}
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * e + 28 * case["rows"], "flops": 4 * n}
    # Rows of weight zero are not read; their gradient is written all the same.
    live = case["rows"] - int(case["masked"] * case["rows"])
    reads = 2 if op == "distill_pair" else 1
    n, k = live * case["vocab"], live * case["top"]
    return {"bytes": reads * (n * e + 8 * k) + case["rows"] * (case["vocab"] * e + 12), "flops": 8 * n + 12 * k}


# ---- the definitions in 64 bits -----------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "lookup":
        return torch.index_select(s["table"], 0, s["ids"]).double().mul_(s["scale"])
    if op in ("grad", "grad_steps"):
        total = None
        for grad, ids in zip(s["grads"], s["ids"]):
            step = _exact_sum(grad, ids, s["vocab"]) * s["scale"]
            total = step if total is None else total + step
        return total
    if op == "sample":
        names = ("logits", "uniform", "temperature", "top_k", "top_p", "min_p")
        h = {n: (s[n].float() if s[n].dtype.is_floating_point else s[n]).cpu().numpy() for n in names}
        drawn = [_exact_token(*(h[n][r] for n in names)) for r in range(case["rows"])]
        return {"token": torch.tensor([t for t, _ in drawn], dtype=torch.int32), "logprob": torch.tensor([p for _, p in drawn], dtype=torch.float64)}
    c = s["weights"] * s["incoming"] if op == "distill_pair" else s["weights"]
    parts = [_exact_distill(s, c, r, min(r + 256, case["rows"])) for r in range(0, case["rows"], 256)]
    return {"loss": torch.cat([p[0] for p in parts]), "grad": torch.cat([p[1] for p in parts])}


def _exact_sum(grad, ids, vocab):
    """Differences of running sums over the tokens in sorted order."""
    ids, order = torch.sort(ids.long(), stable=True)
    tokens = torch.arange(vocab, device=ids.device)
    begin, end = torch.searchsorted(ids, tokens), torch.searchsorted(ids, tokens, right=True)
    out = torch.empty((vocab, grad.shape[1]), dtype=torch.float64, device=grad.device)
    for c in range(0, grad.shape[1], 512):
        sums = torch.nn.functional.pad(grad[:, c:c + 512].double()[order].cumsum(0), (0, 0, 1, 0))
        out[:, c:c + 512] = sums[end] - sums[begin]
    return out


def _exact_distill(s, coefficients, r0, r1):
    tau, vocab = s["tau"], s["logits"].shape[1]
    log_q = torch.log_softmax(s["logits"][r0:r1].double() / tau, dim=1)
    ids, w, c = s["ids"][r0:r1].long(), s["weights"][r0:r1].double(), coefficients[r0:r1].double()
    ok = (ids >= 0) & (ids < vocab)
    log_p = torch.log_softmax(s["teacher"][r0:r1].double().masked_fill(~ok, -1e300) / tau, dim=1)
    p = log_p.exp() * ok
    target = torch.zeros_like(log_q).index_put_(
        (torch.arange(r1 - r0, device=ids.device)[:, None].expand_as(ids)[ok], ids[ok]), p[ok], accumulate=True)
    cross = (p * (log_p - log_q.gather(1, ids.masked_fill(~ok, 0))).masked_fill(~ok, 0.0)).sum(1)
    return w * tau ** 2 * cross, (c * tau)[:, None] * (log_q.exp() - target)


def _exact_token(z, u, temperature, top_k, top_p, min_p):
    z = z.astype(np.float64)
    if not temperature > 0:
        return int(np.argmax(z)), 0.0
    p = np.exp((z - z.max()) / np.float64(temperature))
    order = np.argsort(-z, kind="stable")
    if 0 < top_k < z.size:
        order = order[:top_k]
    in_front = np.concatenate([[0.0], np.cumsum(p[order])])
    if top_p < 1:
        order = order[:max(1, int(np.searchsorted(in_front[:-1], np.float64(top_p) * in_front[-1], side="left")))]
    order = np.sort(order[(p[order] >= np.float64(min_p)) | (order == order[0])])
    sums = np.cumsum(p[order])
    at = int(np.searchsorted(sums, np.float64(u) * sums[-1], side="right"))
    token = int(order[min(at, order.size - 1)])
    return token, float((z[token] - z.max()) / np.float64(temperature) - np.log(sums[-1]))
