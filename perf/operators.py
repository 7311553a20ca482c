"""What the token-model operators are timed on: layer norm, embedding lookup and sampling, each in the calls that a program makes.

A case names a kind of call and its sizes.  With `own`, `run` calls the framework's entry points; without it, it computes the same
outputs from elementary torch operations in 32 bits (64 where a value lies next to a border), rounded once at the end.

Kinds
  norm_fwd   layer norm of each row: y = (x - mean) * rstd * gamma + beta, with the rows' mean and rstd where they are kept
  norm_bwd   its backward pass: the gradients of x, gamma and beta
  embed_fwd  rows of a table by token: out[t] = scale * table[ids[t]]; an id outside the table is padding and gives a row of zeros
  embed_bwd  the table's gradient: grad[v] = scale * sum of dout[t] over the tokens of v, written whole or added to what is there
  sample     one token per row of logits: temperature, top-k, top-p and min-p, drawn with a given number from [0, 1)
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # generating one token: one row through a norm, nothing kept for a backward pass
        {"name": "norm_fwd_token", "kind": "norm_fwd", "dtype": "bf16", "rows": 1, "cols": 4096, "keep": False},
        # the activations of the benchmark's batch in training, f32
        {"name": "norm_fwd_train", "kind": "norm_fwd", "dtype": "f32", "rows": 16384, "cols": 4096, "keep": True},
        # a small model's training batch: a few microseconds of work
        {"name": "norm_bwd_small", "kind": "norm_bwd", "dtype": "f32", "rows": 384, "cols": 256},
        # rows that start at any element, rows and columns multiples of nothing
        {"name": "norm_bwd_ragged", "kind": "norm_bwd", "dtype": "f16", "rows": 4099, "cols": 1001},
        # a large model's training batch in 16-bit storage
        {"name": "norm_bwd_train", "kind": "norm_bwd", "dtype": "bf16", "rows": 16384, "cols": 4096},
        # the tokens of a small serving batch
        {"name": "embed_fwd_serve", "kind": "embed_fwd", "dtype": "bf16", "tokens": 64, "vocab": 32000, "dim": 4096, "pad": 0.0},
        # a training batch of short rows of odd length, some of it padding
        {"name": "embed_fwd_ragged", "kind": "embed_fwd", "dtype": "f32", "tokens": 30011, "vocab": 50021, "dim": 777, "pad": 0.1},
        # the gradient of a training batch added to the table's gradient, which the update has left at zero
        {"name": "embed_bwd_add", "kind": "embed_bwd", "dtype": "f32", "tokens": 8192, "vocab": 32000, "dim": 1024, "pad": 0.05, "add": True},
        # the largest: a long batch, the gradient written whole
        {"name": "embed_bwd_train", "kind": "embed_bwd", "dtype": "bf16", "tokens": 32768, "vocab": 32000, "dim": 4096, "pad": 0.0, "add": False},
        # one request's next token, with every filter
        {"name": "sample_token", "kind": "sample", "dtype": "f32", "rows": 1, "cols": 32000, "filters": "all"},
        # a serving batch over a large vocabulary of odd size, requests with filters of their own
        {"name": "sample_serve", "kind": "sample", "dtype": "bf16", "rows": 256, "cols": 128003, "filters": "mixed"},
        # many continuations drawn at a temperature alone
        {"name": "sample_plain", "kind": "sample", "dtype": "f32", "rows": 512, "cols": 32000, "filters": "none"},
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]: any whole number, or a multiple of 8 or 64."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    g = rng.choice((1, 8, 64))
    return max(lo, min(hi, (v + g - 1) // g * g if v >= g else v))


def draw(rng):
    kind = rng.choice(("norm_fwd", "norm_bwd", "embed_fwd", "embed_bwd", "sample"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    if kind in ("norm_fwd", "norm_bwd"):
        cols = _size(rng, 16, 16384)
        rows = min(_size(rng, 1, 32768), 60_000_000 // cols)
        case = {"kind": kind, "dtype": dtype, "rows": rows, "cols": cols}
        return {**case, "keep": rng.random() < 0.5} if kind == "norm_fwd" else case
    if kind in ("embed_fwd", "embed_bwd"):
        dim = _size(rng, 16, 8192)
        case = {"kind": kind, "dtype": dtype, "tokens": min(_size(rng, 1, 65536), 60_000_000 // dim),
                "vocab": min(_size(rng, 100, 200_000), 60_000_000 // dim), "dim": dim, "pad": rng.choice((0.0, 0.1, 0.3))}
        return {**case, "add": rng.random() < 0.5} if kind == "embed_bwd" else case
    cols = _size(rng, 50, 150_000)
    return {"kind": kind, "dtype": dtype, "rows": min(_size(rng, 1, 512), 30_000_000 // cols), "cols": cols,
            "filters": rng.choice(("none", "all", "mixed"))}


# ---- inputs ----
def _inputs(case, seed):
    """The input tensors of a case, a function of the seed alone."""
    gen, kind = torch.Generator(device="cuda").manual_seed(1_000_003 * int(seed) + 29), case["kind"]
    dt = DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")   # noqa: E731
    uniform = lambda *shape: torch.rand(shape, generator=gen, device="cuda")   # noqa: E731
    if kind in ("norm_fwd", "norm_bwd"):
        rows, cols = case["rows"], case["cols"]
        # a residual stream: rows of different sizes, off zero
        x = (normal(rows, cols) * (0.5 + 2.0 * uniform(rows, 1)) + normal(rows, 1)).to(dt)
        t = {"x": x, "gamma": (1.0 + 0.1 * normal(cols)).to(dt), "beta": (0.1 * normal(cols)).to(dt)}
        if kind == "norm_bwd":
            t["dy"] = normal(rows, cols).to(dt)
            v, m = torch.var_mean(x.float(), 1, correction=0)
            t["mean"], t["rstd"] = m, torch.rsqrt(v + _EPS)
        return t
    if kind in ("embed_fwd", "embed_bwd"):
        n, vocab, dim = case["tokens"], case["vocab"], case["dim"]
        # words fall off with their rank; the padding of a batch stands at the end of it
        ids = torch.exp(uniform(n).double() * math.log(vocab)).floor().long() - 1
        ids = ids.clamp_(0, vocab - 1).int()
        ids[n - int(n * case["pad"]):] = -1
        if kind == "embed_fwd":
            return {"ids": ids, "table": normal(vocab, dim).to(dt)}
        return {"ids": ids, "dout": normal(n, dim).to(dt)}
    rows, cols = case["rows"], case["cols"]
    logits = normal(rows, cols) * 2.5
    logits.masked_fill_(uniform(rows, cols) < 0.1, -math.inf)          # tokens that the request forbids
    t = {"logits": logits.to(dt), "u": uniform(rows)}
    if case["filters"] == "none":
        return {**t, "temperature": 0.7 + 0.6 * uniform(rows)}
    t["temperature"] = 0.6 + 0.6 * uniform(rows)
    t["top_k"] = (10 + 90 * uniform(rows)).int()
    t["top_p"] = 0.7 + 0.29 * uniform(rows)
    t["min_p"] = 0.1 * uniform(rows)
    if case["filters"] == "mixed":                                     # each request sets some of them, some none, some ask for the largest
        t["temperature"][uniform(rows) < 0.1] = 0.0
        t["top_k"][uniform(rows) < 0.5] = 0
        t["top_p"][uniform(rows) < 0.5] = 1.0
        t["min_p"][uniform(rows) < 0.5] = 0.0
    return t


_EPS, _SCALE = 1e-5, 1.5


def prepare(case, seed):
    t, kind = _inputs(case, seed), case["kind"]
    new = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="cuda")   # noqa: E731
    if kind == "norm_fwd":
        out = {"y": torch.empty_like(t["x"])}
        if case["keep"]:
            out.update(mean=new(case["rows"]), rstd=new(case["rows"]))
    elif kind == "norm_bwd":
        out = {"dx": torch.empty_like(t["x"]), "dgamma": torch.empty_like(t["gamma"]), "dbeta": torch.empty_like(t["beta"])}
    elif kind == "embed_fwd":
        out = {"out": new(case["tokens"], case["dim"], dtype=t["table"].dtype)}
    elif kind == "embed_bwd":
        out = {"grad": torch.zeros((case["vocab"], case["dim"]), dtype=t["dout"].dtype, device="cuda")}
    else:
        out = {"token": new(case["rows"], dtype=torch.int32), "prob": new(case["rows"])}
    torch.cuda.synchronize()
    return {"case": case, "in": t, "out": out, "at": {k: v.data_ptr() for k, v in {**t, **out}.items()}}


_context = None


def _ctx():
    """One context per process, as a program has."""
    global _context
    if _context is None:
        from ferrograd_b200 import GpuContext
        _context = GpuContext(0)
    return _context


def run(state):
    case, o = state["case"], state["out"]
    if not own:
        with torch.no_grad():
            o.update(_plain(case, state["in"], o))
        return o
    c, p, kind = _ctx(), state["at"], case["kind"]
    if kind == "norm_fwd":
        c.layernorm_fwd(p["x"], p["gamma"], p["beta"], p["y"], case["rows"], case["cols"], eps=_EPS, mean=p.get("mean"), rstd=p.get("rstd"),
                        dtype=case["dtype"])
    elif kind == "norm_bwd":
        c.layernorm_bwd(p["x"], p["dy"], p["gamma"], p["mean"], p["rstd"], case["rows"], case["cols"], dx=p["dx"], dgamma=p["dgamma"],
                        dbeta=p["dbeta"], dtype=case["dtype"])
    elif kind == "embed_fwd":
        c.embedding_fwd(p["table"], p["ids"], p["out"], case["tokens"], case["vocab"], case["dim"], scale=_SCALE, dtype=case["dtype"])
    elif kind == "embed_bwd":
        c.embedding_bwd(p["ids"], p["dout"], p["grad"], case["tokens"], case["vocab"], case["dim"], scale=_SCALE, accumulate=case["add"],
                        dtype=case["dtype"])
    else:
        c.sample(p["logits"], p["u"], p["token"], case["rows"], case["cols"], temperature=p["temperature"], top_k=p.get("top_k"),
                 top_p=p.get("top_p"), min_p=p.get("min_p"), prob=p["prob"], dtype=case["dtype"])
    return o


# ---- the plain form ----
def _plain(case, t, o):
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    if kind == "norm_fwd":
        x = t["x"].float()
        mean = x.mean(1, keepdim=True)
        d = x - mean
        rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + _EPS)
        y = (d * rstd * t["gamma"].float() + t["beta"].float()).to(dt)
        return {"y": y, "mean": mean[:, 0], "rstd": rstd[:, 0]} if case["keep"] else {"y": y}
    if kind == "norm_bwd":
        dy, rstd = t["dy"].float(), t["rstd"][:, None]
        xhat = (t["x"].float() - t["mean"][:, None]) * rstd
        g = dy * t["gamma"].float()
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        return {"dx": dx.to(dt), "dgamma": (dy * xhat).sum(0).to(dt), "dbeta": dy.sum(0).to(dt)}
    if kind in ("embed_fwd", "embed_bwd"):
        ids = t["ids"].long()
        inside = (ids >= 0) & (ids < case["vocab"])
        at = torch.where(inside, ids, 0)
        if kind == "embed_fwd":
            return {"out": torch.where(inside[:, None], t["table"][at].float() * _SCALE, 0.0).to(dt)}
        rows = torch.where(inside[:, None], t["dout"].float() * _SCALE, 0.0)
        grad = torch.zeros((case["vocab"], case["dim"]), device="cuda").index_add_(0, at, rows)
        if case["add"]:
            return {"grad": o["grad"].copy_(o["grad"].float() + grad)}
        return {"grad": grad.to(dt)}
    x = t["logits"].double()
    rows, cols = x.shape
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    rank = torch.arange(cols, device="cuda")
    temperature = t["temperature"].double()[:, None]
    w = torch.exp((x - x[:, :1]) / torch.where(temperature > 0, temperature, 1.0))
    keep = torch.where(temperature > 0, True, rank == 0)
    if case["filters"] != "none":
        k = t["top_k"].long()[:, None]
        keep = keep & ((k == 0) | (rank < k))
        kept = w * keep
        before = kept.cumsum(1) - kept
        p = t["top_p"].double()[:, None]
        keep = keep & ((p >= 1) | (before < p * kept.sum(1, keepdim=True)))
        keep = keep & (w >= t["min_p"].double()[:, None])
    kept = torch.zeros_like(x).scatter_(1, order, w * keep)
    cdf = kept.cumsum(1)
    token = (cdf <= t["u"].double()[:, None] * cdf[:, -1:]).sum(1, keepdim=True).clamp_(max=cols - 1)
    return {"token": token[:, 0].int(), "prob": (kept.gather(1, token) / cdf[:, -1:])[:, 0].float()}


# ---- what a call cannot do without ----
def _inside(case):
    return case["tokens"] - int(case["tokens"] * case["pad"])


def _used(case):
    """Rows of the table that the tokens name, on average: the rank r (from 1) is drawn with log(1 + 1/r) / log(vocab)."""
    r = np.arange(1, case["vocab"] + 1, dtype=np.float64)
    return float(-np.expm1(_inside(case) * np.log1p(-np.minimum(np.log1p(1.0 / r) / math.log(case["vocab"]), 1 - 1e-12))).sum())


def work(case):
    """Bytes: every input read once, every output written once (of a table, the rows that are used).  flops: the arithmetic of the
    formulas, an exponential as one."""
    kind, size = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind in ("norm_fwd", "norm_bwd"):
        n, rows, cols = case["rows"] * case["cols"], case["rows"], case["cols"]
        if kind == "norm_fwd":
            return {"bytes": size * (2 * n + 2 * cols) + (8 * rows if case["keep"] else 0), "flops": 8 * n}
        return {"bytes": size * (3 * n + 3 * cols) + 8 * rows, "flops": 14 * n}
    if kind == "embed_fwd":
        return {"bytes": 4 * case["tokens"] + size * case["dim"] * (_used(case) + case["tokens"]), "flops": case["tokens"] * case["dim"]}
    if kind == "embed_bwd":
        table = 2 * _used(case) if case["add"] else case["vocab"]
        return {"bytes": 4 * case["tokens"] + size * case["dim"] * (_inside(case) + table), "flops": 2 * _inside(case) * case["dim"]}
    n = case["rows"] * case["cols"]
    return {"bytes": size * n + 16 * case["rows"], "flops": 4 * n}


# ---- the same outputs in 64 bits ----
def exact(case, seed):
    kind, t = case["kind"], _inputs(case, seed)
    d = {k: v.double() for k, v in t.items() if v.is_floating_point()}
    if kind == "norm_fwd":
        var, mean = torch.var_mean(d["x"], 1, correction=0)
        rstd = (var + _EPS) ** -0.5
        y = torch.addcmul(d["beta"], (d["x"] - mean[:, None]) * rstd[:, None], d["gamma"])
        return {"y": y, "mean": mean, "rstd": rstd} if case["keep"] else {"y": y}
    if kind == "norm_bwd":
        # dL/dx of y = h(x) gamma through the projection that a normalised row is: (I - 1 1'/n - h h'/n) rstd
        h = (d["x"] - d["mean"][:, None]) * d["rstd"][:, None]
        g, n = d["dy"] * d["gamma"], case["cols"]
        dx = g - torch.einsum("rc->r", g)[:, None] / n - h * (torch.einsum("rc,rc->r", g, h) / n)[:, None]
        return {"dx": dx * d["rstd"][:, None], "dgamma": torch.einsum("rc,rc->c", d["dy"], h), "dbeta": torch.einsum("rc->c", d["dy"])}
    if kind == "embed_fwd":
        table = torch.cat([d["table"], torch.zeros((1, case["dim"]), dtype=torch.float64, device="cuda")])
        return {"out": _SCALE * torch.nn.functional.embedding(t["ids"].long() % (case["vocab"] + 1), table)}
    if kind == "embed_bwd":
        ids, order = torch.sort(t["ids"].long() % (case["vocab"] + 1))
        rows, count = torch.unique_consecutive(ids, return_counts=True)
        sums = torch.segment_reduce(d["dout"][order], "sum", lengths=count, axis=0)
        grad = torch.zeros((case["vocab"] + 1, case["dim"]), dtype=torch.float64, device="cuda")
        grad[rows] = _SCALE * sums
        return {"grad": grad[:-1]}
    rows, cols = case["rows"], case["cols"]
    host = {k: v.cpu().numpy() for k, v in {**d, "top_k": t.get("top_k", d["u"])}.items()}
    token, prob = np.zeros(rows, np.int32), np.zeros(rows)
    for r in range(rows):
        x = host["logits"][r]
        temperature = host["temperature"][r]
        if temperature <= 0:
            token[r], prob[r] = int(np.argmax(x)), 1.0
            continue
        allowed = np.flatnonzero(np.isfinite(x))
        w = np.exp((x[allowed] - x.max()) / temperature)
        if case["filters"] != "none":
            # the most likely first, of equal ones the first; a weight below min_p of the largest is out in any case
            down = np.argsort(-x[allowed], kind="stable")
            k = int(host["top_k"][r])
            down = down[:k] if k else down
            mass, p = np.cumsum(w[down]), host["top_p"][r]
            down = down[:1 + int(np.searchsorted(mass, p * mass[-1], side="left"))] if p < 1 else down
            chosen = np.sort(down[w[down] >= host["min_p"][r]])
            allowed, w = allowed[chosen], w[chosen]
        mass = np.cumsum(w)
        i = min(int(np.searchsorted(mass, host["u"][r] * mass[-1], side="right")), len(w) - 1)
        token[r], prob[r] = allowed[i], w[i] / mass[-1]
    return {"token": torch.from_numpy(token), "prob": torch.from_numpy(prob)}
