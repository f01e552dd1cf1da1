"""What is measured of the operators on row tables and score rows (vectordb_amd.ops), with their plain forms.

A table is a matrix of rows (a vocabulary's embeddings, or the vectors of a collection); a score row holds one value
for every row of a table (the logits of one position or query).  Five directions of four operators:

  lookup        rows of a table by number, scaled
  lookup_grad   the gradient of that table: the rows of an upstream gradient summed by row number
  distill       divergence of a score row from a teacher's top scores, as a top-k search returns them
  distill_grad  its gradient
  distill_step  both in one call, where the weight of every score row is known beforehand
  sample        one row number drawn from each score row: temperature, top-k, top-p, min-p, row filter

`own` False computes them from elementary torch operations, True through vectordb_amd.ops.
"""

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # the vectors behind one answer of ten rows, out of a small collection: latency
        {"name": "lookup, one answer", "op": "lookup", "n": 10, "dim": 128, "rows": 10_000, "dtype": "f32", "out": "f32", "scale": 1.0},
        # the input rows of a long training batch, scaled by sqrt(dim)
        {"name": "lookup, training batch", "op": "lookup", "n": 131_072, "dim": 2048, "rows": 131_072, "dtype": "bf16", "out": "bf16",
         "scale": 45.25},
        # ten answers for each of 1024 queries: a gradient for 10240 of 100k rows
        {"name": "lookup_grad, answers of a batch", "op": "lookup_grad", "n": 10_240, "dim": 384, "rows": 100_000, "dtype": "f32", "out": "f32",
         "scale": 1.0},
        # a training batch whose row numbers are distributed as words are: a few rows take most of the sum
        {"name": "lookup_grad, training batch", "op": "lookup_grad", "n": 131_072, "dim": 2048, "rows": 131_072, "dtype": "bf16", "out": "f32",
         "scale": 45.25},
        # 100 queries against a collection of 10k rows, the teacher's ten best of each
        {"name": "distill, small collection", "op": "distill", "n": 100, "vocab": 10_000, "k": 10, "dtype": "f32", "temperature": 1.0, "whole": False},
        # a training batch over a large vocabulary
        {"name": "distill, training batch", "op": "distill", "n": 4096, "vocab": 131_072, "k": 64, "dtype": "bf16", "temperature": 2.0, "whole": False},
        # the gradients of the same two kinds of work; a vocabulary of odd size
        {"name": "distill_grad, small collection", "op": "distill_grad", "n": 100, "vocab": 10_000, "k": 10, "dtype": "f32", "temperature": 1.0,
         "whole": False},
        {"name": "distill_grad, odd vocabulary", "op": "distill_grad", "n": 2048, "vocab": 50_021, "k": 32, "dtype": "f16", "temperature": 1.0,
         "whole": True},
        # loss and gradient of a training step in one call
        {"name": "distill_step, few rows", "op": "distill_step", "n": 16, "vocab": 32_768, "k": 16, "dtype": "f32", "temperature": 1.0, "whole": False},
        {"name": "distill_step, training batch", "op": "distill_step", "n": 4096, "vocab": 32_768, "k": 64, "dtype": "bf16", "temperature": 1.0,
         "whole": True},
        # the next token of one request: latency
        {"name": "sample, one request", "op": "sample", "n": 1, "vocab": 32_768, "dtype": "f32", "filters": "mixed", "masked": False},
        # the next tokens of a full serving batch, every request with settings of its own
        {"name": "sample, serving batch", "op": "sample", "n": 256, "vocab": 131_072, "dtype": "bf16", "filters": "mixed", "masked": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "distill", "distill_grad", "distill_step", "sample"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op in ("lookup", "lookup_grad"):
        dim = _log(rng, 16, 2048)
        rows = min(_log(rng, 1000, 1_000_000), 131_072 * 2048 // dim)
        out = rng.choice([dtype, "f32"])
        return {"op": op, "n": _log(rng, 1, 131_072), "dim": dim, "rows": rows, "dtype": dtype, "out": out, "scale": rng.choice([1.0, 0.125, 22.6])}
    vocab = _log(rng, 1000, 200_000)
    if op == "sample":
        return {"op": op, "n": min(_log(rng, 1, 1024), 256 * 131_072 // vocab), "vocab": vocab, "dtype": dtype,
                "filters": rng.choice(["none", "top_k", "top_p", "min_p", "mixed"]), "masked": rng.random() < 0.3}
    most = {"distill": 4096 * 65_536, "distill_grad": 4096 * 16_384, "distill_step": 4096 * 16_384}[op]
    return {"op": op, "n": min(_log(rng, 1, 8192), most // vocab), "vocab": vocab, "k": _log(rng, 1, 256), "dtype": dtype,
            "temperature": rng.choice([0.7, 1.0, 2.0]), "whole": rng.random() < 0.4}


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1_000_003 * (seed + 1))
    op, n, t = case["op"], case["n"], TYPES[case["dtype"]]

    def uniform(*shape):
        return torch.rand(shape, device="cuda", generator=g)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, device="cuda", generator=g, dtype=dtype)

    s = dict(case)
    if op in ("lookup", "lookup_grad"):
        # row numbers by rank, P(rank) ~ 1 / rank, the ranks spread over the table; one in 64 is the -1 of a slot that a
        # search could not fill
        rank = (case["rows"] ** uniform(n).double() - 1).long().clamp_(0, case["rows"] - 1)
        at = torch.randperm(case["rows"], device="cuda", generator=g)[rank]
        s["at"] = torch.where(uniform(n) < 1 / 64, torch.full_like(at, -1), at)
        if op == "lookup":
            s["table"] = normal(case["rows"], case["dim"], dtype=t)
        else:
            s["grad"] = normal(n, case["dim"], dtype=t)
        return s
    v = case["vocab"]
    z = normal(n, v, dtype=t).mul_(2.5)
    if op == "sample":
        # a row as a language model leaves it: a broad bulk and a few scores that stand out
        z.scatter_(1, torch.randint(0, v, (n, 16), device="cuda", generator=g), (4.0 + 10.0 * uniform(n, 16)).to(t))

        def choose(*values):
            return torch.tensor(values, device="cuda")[torch.randint(0, len(values), (n,), device="cuda", generator=g)]

        f = case["filters"]
        mixed = f == "mixed"
        s.update(logits=z, uniforms=uniform(n), temperature=(choose(0.0, 0.6, 0.8, 1.0, 1.0, 1.3) if mixed else 0.5 + uniform(n)).float(),
                 top_k=choose(0, 1, 20, 50, 50, 400).int() if mixed else choose(1, 10, 50, 100, 1000).int() if f == "top_k" else None,
                 top_p=choose(1.0, 0.95, 0.9, 0.5).float() if mixed else choose(0.99, 0.95, 0.9, 0.8, 0.5).float() if f == "top_p" else None,
                 min_p=choose(0.0, 0.0, 0.05).float() if mixed else choose(0.01, 0.05, 0.1, 0.2).float() if f == "min_p" else None,
                 words=None)
        if case["masked"]:
            # a filter of its own for each request, seven rows in eight pass
            a, b, c = (torch.randint(-2 ** 31, 2 ** 31, (n, (v + 31) // 32), device="cuda", generator=g).int() for _ in range(3))
            s["words"] = a | b | c
        return s
    k = min(case["k"], v)
    # the teacher's best rows, scores falling; one list in four is shorter than k, one in 32 is empty (padding)
    first = torch.randint(0, v, (n, 1), device="cuda", generator=g)
    step = torch.randint(1, max(v // k, 1) + 1, (n, 1), device="cuda", generator=g)
    slot = torch.arange(k, device="cuda")
    at = (first + slot * step) % v
    filled = torch.where(uniform(n, 1) < 0.25, (uniform(n, 1) * (k + 1)).long(), k)
    filled = torch.where(uniform(n, 1) < 1 / 32, 0, filled)
    tl = 12.0 - (0.2 * uniform(n, k)).cumsum(1)
    # where the teacher scores high, the student leans that way
    z.scatter_add_(1, at, (0.5 * tl).to(t))
    s.update(logits=z, teacher=torch.where(slot < filled, tl, -math.inf), at=torch.where(slot < filled, at, -1),
             teacher_lse=(tl.amax(1) / case["temperature"] + math.log(k) + 0.5 * uniform(n)) if case["whole"] else None)
    if op != "distill":
        # the mean over the rows, one row in 16 left out; half-precision gradients are trained with a loss scale
        s["weight"] = torch.where(uniform(n) < 1 / 16, 0.0, 0.5 + uniform(n)) * ((4096.0 if case["dtype"] == "f16" else 1.0) / n)
    if op == "distill_grad":
        # what the forward pass left: the largest score of each row and the logarithm of the sum behind it
        zf = z.float()
        top = zf.amax(1)
        s["stats"] = torch.stack([top, ((zf - top[:, None]) / case["temperature"]).exp().sum(1).log()], 1)
    return s


# ---------------------------------------------------------------- plain forms
def _lookup(s):
    known = (s["at"] >= 0) & (s["at"] < s["rows"])
    x = s["table"][torch.where(known, s["at"], 0)].float() * s["scale"]
    return torch.where(known[:, None], x, 0.0).to(TYPES[s["out"]])


def _lookup_grad(s):
    known = (s["at"] >= 0) & (s["at"] < s["rows"])
    x = torch.where(known[:, None], s["grad"].float(), 0.0)
    total = torch.zeros((s["rows"], s["dim"]), device=x.device).index_add_(0, torch.where(known, s["at"], 0), x)
    return (total * s["scale"]).to(TYPES[s["out"]])


def _teacher(s):
    """Probabilities of the teacher's slots and their logarithms: over the filled slots, or over its whole vocabulary."""
    tau, v = s["temperature"], s["logits"].shape[1]
    filled = (s["at"] >= 0) & (s["at"] < v) & (s["teacher"] > -math.inf)
    t = torch.where(filled, s["teacher"] / tau, -math.inf)
    if s["teacher_lse"] is not None:
        logp = t - s["teacher_lse"][:, None]
    else:
        top = t.amax(1, keepdim=True)
        top = torch.where(top > -math.inf, top, 0.0)
        logp = t - top - torch.exp(t - top).sum(1, keepdim=True).clamp_min(1e-30).log()
    return torch.where(filled, torch.exp(logp), 0.0), logp, torch.where(filled, s["at"], 0)


def _stats(s):
    z = s["logits"].float()
    top = z.amax(1)
    return torch.stack([top, torch.exp((z - top[:, None]) / s["temperature"]).sum(1).log()], 1)


def _distill(s, stats):
    tau = s["temperature"]
    p, logp, at = _teacher(s)
    logq = (s["logits"].gather(1, at).float() - stats[:, :1]) / tau - stats[:, 1:]
    return tau * tau * torch.where(p > 0, p * (logp - logq), 0.0).sum(1)


def _distill_grad(s, stats):
    tau = s["temperature"]
    p, _, at = _teacher(s)
    q = torch.exp((s["logits"].float() - stats[:, :1]) / tau - stats[:, 1:])
    w = (s["weight"] * tau)[:, None]
    grad = (w * (q * p.sum(1, keepdim=True))).scatter_add_(1, at, -w * p)
    return torch.where(w != 0, grad, 0.0).to(s["logits"].dtype)


def _sample(s):
    """In 64 bits: a draw next to a border belongs to the row that the exact sums say."""
    x = s["logits"].double()
    n, v = x.shape
    x = torch.where(torch.isnan(x), -math.inf, x)
    if s["words"] is not None:
        number = torch.arange(v, device=x.device)
        x = torch.where((s["words"][:, number // 32] >> (number % 32)) & 1 == 1, x, -math.inf)
    ranked, order = torch.sort(x, dim=1, descending=True, stable=True)
    best, rank = ranked[:, :1], torch.arange(v, device=x.device)
    tau = s["temperature"].double()[:, None]
    w = torch.where(ranked == best, 1.0, torch.exp((ranked - best) / tau))
    # a weight below 2^-40 of the largest counts as nothing
    w = torch.where((ranked > -math.inf) & (w >= 2.0 ** -40), w, 0.0)
    most = torch.full_like(best, v) if s["top_k"] is None else torch.where(s["top_k"] > 0, s["top_k"], v)[:, None]
    w = torch.where(rank < torch.where(tau > 0, most, 1), w, 0.0)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        before = w.cumsum(1) - w
        w = torch.where((before < p * w.sum(1, keepdim=True)) | (p >= 1) | (rank == 0), w, 0.0)
    if s["min_p"] is not None:
        w = torch.where(w >= s["min_p"].double()[:, None].clamp_max(1.0), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    running = w.cumsum(1)
    total = running[:, -1:]
    drawn = (running <= s["uniforms"].double()[:, None] * total).sum(1, keepdim=True).clamp_max(v - 1)
    some = best > -math.inf
    logp = torch.where(some, torch.log(w.gather(1, drawn) / total), -math.inf)
    return torch.where(some, drawn, -1)[:, 0], logp[:, 0].float()


def run(s):
    op = s["op"]
    if own:
        from vectordb_amd import ops
        if op == "lookup":
            return ops.lookup(s["table"], s["at"], scale=s["scale"], dtype=TYPES[s["out"]])
        if op == "lookup_grad":
            return ops.lookup_grad(s["grad"], s["at"], s["rows"], scale=s["scale"], dtype=TYPES[s["out"]])
        if op == "sample":
            return ops.sample(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                              mask_words=s["words"])
        settings = {"temperature": s["temperature"], "teacher_lse": s["teacher_lse"]}
        if op == "distill":
            return ops.distill(s["logits"], s["teacher"], s["at"], **settings)
        if op == "distill_grad":
            return ops.distill_grad(s["logits"], s["teacher"], s["at"], s["stats"], s["weight"], **settings)
        return ops.distill_step(s["logits"], s["teacher"], s["at"], s["weight"], **settings)
    if op == "lookup":
        return _lookup(s)
    if op == "lookup_grad":
        return _lookup_grad(s)
    if op == "sample":
        return _sample(s)
    if op == "distill":
        stats = _stats(s)
        return _distill(s, stats), stats
    if op == "distill_grad":
        return _distill_grad(s, s["stats"])
    stats = _stats(s)
    return _distill(s, stats), _distill_grad(s, stats)


def work(case):
    n, b = case["n"], BYTES[case["dtype"]]
    if case["op"] in ("lookup", "lookup_grad"):
        dim, o = case["dim"], BYTES[case["out"]]
        if case["op"] == "lookup":
            return {"bytes": n * 8 + min(n, case["rows"]) * dim * b + n * dim * o, "flops": n * dim}
        return {"bytes": n * 8 + n * dim * b + case["rows"] * dim * o, "flops": n * dim}
    v = case["vocab"]
    if case["op"] == "sample":
        return {"bytes": n * v * b + (n * ((v + 31) // 32) * 4 if case["masked"] else 0) + n * 32, "flops": 4 * n * v}
    lists = n * min(case["k"], v) * 12 + n * 16
    if case["op"] == "distill":
        return {"bytes": n * v * b + lists, "flops": 4 * n * v}
    return {"bytes": 2 * n * v * b + lists, "flops": (4 if case["op"] == "distill_grad" else 8) * n * v}


# ---------------------------------------------------------------- the definitions, in 64 bits
def _exact_sample(s):
    """One row after the other: sort, cut, add up, look where the uniform number falls."""
    z = s["logits"].double().cpu().numpy()
    n, v = z.shape
    got, logs = np.full(n, -1, np.int64), np.full(n, -np.inf)
    take = {k: None if s[k] is None else s[k].cpu().numpy() for k in ("top_k", "top_p", "min_p", "words", "temperature", "uniforms")}
    for i in range(n):
        usable = np.isfinite(z[i])
        if take["words"] is not None:
            usable &= np.unpackbits(take["words"][i].view(np.uint8), bitorder="little")[:v].astype(bool)
        place = np.flatnonzero(usable)
        if len(place) == 0:
            continue
        place = place[np.argsort(-z[i, place], kind="stable")]
        tau = float(take["temperature"][i])
        limit = 1 if tau <= 0 else int(take["top_k"][i]) if take["top_k"] is not None and take["top_k"][i] > 0 else v
        place = place[:limit]
        weight = np.exp((z[i, place] - z[i, place[0]]) / (tau if tau > 0 else 1.0))
        weight[weight < 2.0 ** -40] = 0.0
        count = len(place)
        if take["top_p"] is not None and take["top_p"][i] < 1:
            reach = np.concatenate([[0.0], np.cumsum(weight)])
            count = max(1, int(np.searchsorted(reach[:-1], float(take["top_p"][i]) * reach[-1], side="left")))
        if take["min_p"] is not None:
            count = min(count, int((weight >= min(float(take["min_p"][i]), 1.0)).sum()))
        by_number = np.argsort(place[:count], kind="stable")
        place, weight = place[by_number], weight[by_number]
        reach = np.cumsum(weight)
        j = min(int(np.searchsorted(reach, float(take["uniforms"][i]) * reach[-1], side="right")), count - 1)
        got[i], logs[i] = place[j], math.log(weight[j] / reach[-1])
    return torch.from_numpy(got), torch.from_numpy(logs)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "sample":
        return _exact_sample(s)
    if op == "lookup":
        x = torch.cat([s["table"], torch.zeros_like(s["table"][:1])])[s["at"]].double()       # -1 is the row of zeros behind the table
        return x * case["scale"]
    if op == "lookup_grad":
        total = torch.zeros((case["rows"] + 1, case["dim"]), device="cuda", dtype=torch.float64)
        total.index_put_((s["at"] % (case["rows"] + 1),), s["grad"].double() * case["scale"], accumulate=True)
        return total[:-1]
    tau, rows, v = case["temperature"], case["n"], case["vocab"]
    logq = torch.log_softmax(s["logits"].double() / tau, 1)
    t = s["teacher"].double() / tau
    empty = (s["at"] < 0).all(1)
    norm = s["teacher_lse"].double() if case["whole"] else torch.logsumexp(t, 1)
    p = torch.exp(t - torch.where(empty, 0.0, norm)[:, None])                                 # an unfilled slot: exp(-inf) = 0
    at = s["at"] % v
    gap = torch.where(p > 0, p.clamp_min(1e-300).log() - logq.gather(1, at), 0.0)
    loss = tau ** 2 * (p * gap).sum(1)
    if op == "distill":
        top = s["logits"].double().amax(1)
        return loss, torch.stack([top, torch.logsumexp(s["logits"].double() / tau, 1) - top / tau], 1)
    target = torch.zeros((rows, v), device="cuda", dtype=torch.float64).scatter_add_(1, at, p)
    grad = (logq.exp_().mul_(p.sum(1, keepdim=True)).sub_(target)).mul_((tau * s["weight"].double())[:, None])
    return grad if op == "distill_grad" else (loss, grad)
