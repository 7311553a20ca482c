"""What the operators of a decoder block and of its policy loss are timed on: attention, root-mean-square norm and log probabilities.

A case names a kind of call and its sizes.  With `own`, `run` calls the framework's entry points; without it, it computes the same
outputs from elementary torch operations in 32 bits, rounded once at the end.

Kinds
  attend        softmax(scale * q k') v per head over packed sequences, query heads in groups that share a head of k and v; causal: the last
                query of a sequence sees all of its keys, the one before all but the last, and so on.  lse: log of each row's sum, kept for training
  attend_bwd    its backward pass: the gradients of q, k and v
  rms           h = x + residual, y = h * rstd * gamma with rstd = 1 / sqrt(mean(h * h) + eps)
  rms8          the same with y in e4m3 and a scale per group of columns (group 0: the row): largest |y| / 448
  rms_bwd       its backward pass: the gradients of h (which is that of x and of the residual) and of gamma
  logprobs      log softmax(scale * logits) at the row's target, the entropy of the row and its `top` largest with their log probabilities
  logprobs_bwd  the gradient of the logits, of given gradients of log probability and entropy
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-5


def listed():
    return [
        # one request's next token, over what it has so far
        {"name": "attend_token", "kind": "attend", "dtype": "bf16", "seqs": 1, "queries": 1, "keys": 1000, "heads": 16, "kv_heads": 4, "dim": 64,
         "causal": True, "keep": False},
        # the next token of every request of a serving batch, over caches of different lengths
        {"name": "attend_serve", "kind": "attend", "dtype": "bf16", "seqs": 64, "queries": 64, "keys": 250007, "heads": 32, "kv_heads": 8, "dim": 128,
         "causal": True, "keep": False},
        # prompts of different lengths packed into one batch, narrow heads
        {"name": "attend_prompts", "kind": "attend", "dtype": "f16", "seqs": 13, "queries": 11003, "keys": 11003, "heads": 16, "kv_heads": 4, "dim": 64,
         "causal": True, "keep": False},
        # one long document in training
        {"name": "attend_long", "kind": "attend", "dtype": "bf16", "seqs": 1, "queries": 16384, "keys": 16384, "heads": 16, "kv_heads": 2, "dim": 128,
         "causal": True, "keep": True},
        # a small model's training batch, f32
        {"name": "attend_bwd_small", "kind": "attend_bwd", "dtype": "f32", "seqs": 3, "queries": 501, "keys": 501, "heads": 6, "kv_heads": 6, "dim": 48,
         "causal": True},
        # a training batch of packed documents
        {"name": "attend_bwd_train", "kind": "attend_bwd", "dtype": "bf16", "seqs": 5, "queries": 16384, "keys": 16384, "heads": 32, "kv_heads": 8,
         "dim": 128, "causal": True},
        # a serving batch's rows before an 8-bit product
        {"name": "rms8_serve", "kind": "rms8", "dtype": "bf16", "rows": 256, "cols": 8192, "group": 128},
        # the activations of the benchmark's batch in training, f32 and with the residual's addition
        {"name": "rms_train", "kind": "rms", "dtype": "f32", "rows": 16384, "cols": 4096, "keep": True},
        # a large model's training batch in 16-bit storage
        {"name": "rms_bwd_train", "kind": "rms_bwd", "dtype": "bf16", "rows": 16384, "cols": 4096},
        # a serving batch's logits with the alternatives that a request asks for, vocabulary of odd size
        {"name": "logprobs_serve", "kind": "logprobs", "dtype": "bf16", "rows": 64, "cols": 128003, "top": 20, "entropy": False},
        # a policy's loss over a training batch, and its gradient
        {"name": "logprobs_train", "kind": "logprobs", "dtype": "f32", "rows": 8192, "cols": 32000, "top": 0, "entropy": True},
        {"name": "logprobs_bwd_train", "kind": "logprobs_bwd", "dtype": "bf16", "rows": 8192, "cols": 32000, "entropy": True},
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]: any whole number, or a multiple of 8 or 64."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    g = rng.choice((1, 8, 64))
    return max(lo, min(hi, (v + g - 1) // g * g if v >= g else v))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend_bwd", "rms", "rms8", "rms_bwd", "logprobs", "logprobs_bwd"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    if kind in ("attend", "attend_bwd"):
        kv = rng.choice((1, 2, 4, 8))
        case = {"kind": kind, "dtype": dtype, "heads": kv * rng.choice((1, 2, 4, 8)), "kv_heads": kv,
                "dim": rng.choice((32, 40, 64, 64, 80, 96, 128, 128)), "causal": rng.random() < 0.75}
        if kind == "attend" and rng.random() < 0.5:      # serving: one to a few queries per sequence
            seqs = _size(rng, 1, 128)
            case.update(seqs=seqs, queries=seqs * rng.choice((1, 1, 1, 2, 5)), keys=seqs * _size(rng, 1, min(16384, 200_000 // seqs)), keep=False)
            return case
        tokens = _size(rng, 16, 12000)
        seqs = min(_size(rng, 1, 24), tokens)
        # what the largest listed case computes, and what its matrices of weights take, are not exceeded (f32 runs outside of the tensor cores)
        most = 4e8 if dtype == "f32" else 1.5e9
        while seqs * case["heads"] * max(_lengths(tokens, seqs)) ** 2 > most:
            tokens = max(seqs, tokens * 3 // 4)
        case.update(seqs=seqs, queries=tokens, keys=tokens)
        return {**case, "keep": rng.random() < 0.5} if kind == "attend" else case
    if kind in ("rms", "rms8", "rms_bwd"):
        cols = _size(rng, 16, 16384)
        case = {"kind": kind, "dtype": dtype, "rows": min(_size(rng, 1, 32768), 60_000_000 // cols), "cols": cols}
        return {**case, "keep": rng.random() < 0.5} if kind == "rms" else {**case, "group": rng.choice((0, 128))} if kind == "rms8" else case
    cols = _size(rng, 50, 150_000)
    case = {"kind": kind, "dtype": dtype, "rows": min(_size(rng, 1, 8192), 100_000_000 // cols), "cols": cols, "entropy": rng.random() < 0.5}
    return {**case, "top": rng.choice((0, 1, 5, 20))} if kind == "logprobs" else case


# ---- sizes of sequences ----
def _lengths(total, n):
    """n lengths with this sum, up to five times apart."""
    w = [0.25 + 0.618034 * (i + 1) % 1.0 for i in range(n)]
    lengths = [max(1, int(total * x / sum(w))) for x in w]
    lengths[lengths.index(max(lengths))] += total - sum(lengths)
    return lengths


def _own_tokens(case):
    """Whether the keys are those of the queries' own tokens (training, prompts), and not a cache."""
    return case["queries"] == case["keys"]


def _pairs(case):
    """(query, key) pairs that the mask leaves, of one head."""
    n, total = case["seqs"], 0
    ks = _lengths(case["keys"], n)
    qs = ks if _own_tokens(case) else [case["queries"] // n] * n
    for q, k in zip(qs, ks):
        seen = min(q, k)      # queries that see a key at all
        total += seen * k - seen * (seen - 1) // 2 if case["causal"] else q * k
    return total


# ---- inputs ----
def _inputs(case, seed):
    """The input tensors of a case, a function of the seed alone."""
    gen, kind = torch.Generator(device="cuda").manual_seed(1_000_003 * int(seed) + 31), case["kind"]
    dt = DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda")   # noqa: E731
    uniform = lambda *shape: torch.rand(shape, generator=gen, device="cuda")   # noqa: E731
    if kind in ("attend", "attend_bwd"):
        n, heads, kv, dim = case["seqs"], case["heads"], case["kv_heads"], case["dim"]
        order = torch.randperm(n, generator=gen, device="cuda")
        lengths = torch.tensor(_lengths(case["keys"], n), device="cuda")[order]
        starts = lambda x: torch.nn.functional.pad(x.cumsum(0), (1, 0)).int()   # noqa: E731
        t = {"k_starts": starts(lengths)}
        if _own_tokens(case):      # one product makes q, k and v, a row of them per token
            t["qkv"] = normal(case["queries"], (heads + 2 * kv) * dim).to(dt)
            t["q_starts"] = t["k_starts"]
        else:                      # a cache has room for more: each sequence's keys stand in a slot
            slot = int(lengths.max()) + 5
            t["k_starts"] = (torch.arange(n + 1, device="cuda") * slot).int()
            t["k_lengths"] = lengths.int()
            t["q"] = normal(case["queries"], heads * dim).to(dt)
            t["k"], t["v"] = normal(n * slot, kv * dim).to(dt), normal(n * slot, kv * dim).to(dt)
            t["q_starts"] = starts(torch.full((n,), case["queries"] // n, device="cuda"))
        if kind == "attend_bwd":
            t["dout"] = normal(case["queries"], heads * dim).to(dt)
            with torch.no_grad():
                f = _attend(case, t)
            t["out"], t["lse"] = f["out"], f["lse"]
        return t
    rows, cols = case["rows"], case["cols"]
    if kind in ("rms", "rms8", "rms_bwd"):
        # a residual stream: rows of different sizes, a few columns much larger than the others
        x = normal(rows, cols) * (0.5 + 2.0 * uniform(rows, 1)) * torch.where(uniform(cols) < 0.01, 8.0, 1.0)
        t = {"gamma": (1.0 + 0.1 * normal(cols)).to(dt), "x": x.to(dt)}
        if kind == "rms_bwd":
            h = t["x"].float()
            t.update(dy=normal(rows, cols).to(dt), dsum=normal(rows, cols).to(dt), rstd=torch.rsqrt((h * h).mean(1) + _EPS))
        else:
            t["residual"] = normal(rows, cols).to(dt)
        return t
    logits = (normal(rows, cols) * 2.5).to(dt)
    t = {"logits": logits, "targets": (uniform(rows) * cols).int().clamp_(max=cols - 1)}
    t["targets"][uniform(rows) < 0.05] = -1      # padding
    if kind == "logprobs_bwd":
        f = _logprobs(case, t)
        t.update(lse=f["lse"], entropy=f["entropy"], dlogprob=normal(rows) / rows, dentropy=0.01 * normal(rows) / rows)
    return t


_SCALE = 1.25      # of logits: 1 / temperature


def prepare(case, seed):
    t, kind = _inputs(case, seed), case["kind"]
    new = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="cuda")   # noqa: E731
    if kind == "attend":
        out = {"out": new(case["queries"], case["heads"] * case["dim"], dtype=DTYPES[case["dtype"]])}
        if case["keep"]:
            out["lse"] = new(case["heads"], case["queries"])
    elif kind == "attend_bwd":
        out = {"dqkv": torch.empty_like(t["qkv"])}
    elif kind == "rms":
        out = {"y": torch.empty_like(t["x"]), "sum": torch.empty_like(t["x"])}
        if case["keep"]:
            out["rstd"] = new(case["rows"])
    elif kind == "rms8":
        out = {"y": new(case["rows"], case["cols"], dtype=torch.float8_e4m3fn), "sum": torch.empty_like(t["x"]),
               "scale": new(case["rows"], _groups(case))}
    elif kind == "rms_bwd":
        out = {"dx": torch.empty_like(t["x"]), "dgamma": torch.empty_like(t["gamma"])}
    elif kind == "logprobs":
        out = {"logprob": new(case["rows"])}
        if case["entropy"]:
            out.update(entropy=new(case["rows"]), lse=new(case["rows"]))
        if case["top"]:
            out.update(top_ids=new(case["rows"], case["top"], dtype=torch.int32), top_logprobs=new(case["rows"], case["top"]))
    else:
        out = {"dlogits": torch.empty_like(t["logits"])}
    torch.cuda.synchronize()
    return {"case": case, "in": t, "out": out, "at": {k: v.data_ptr() for k, v in {**t, **out}.items()}}


def _groups(case):
    return -(-case["cols"] // case["group"]) if case["group"] else 1


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
            f = _plain(case, state["in"])
            return {k: f[k] for k in o}
    c, p, kind, dtype = _ctx(), state["at"], case["kind"], case["dtype"]
    if kind in ("attend", "attend_bwd"):
        heads, kv, dim, size = case["heads"], case["kv_heads"], case["dim"], 4 if dtype == "f32" else 2
        sizes = (case["seqs"], case["queries"], state["in"]["k"].shape[0] if "k" in p else case["keys"], heads, kv, dim)
        if "qkv" in p:
            q, row = p["qkv"], (heads + 2 * kv) * dim
            k, v = q + heads * dim * size, q + (heads + kv) * dim * size
        else:
            q, k, v, row = p["q"], p["k"], p["v"], 0
        lay = dict(q_stride=row, k_stride=row, v_stride=row, k_lengths=p.get("k_lengths"), causal=case["causal"], dtype=dtype)
        if kind == "attend":
            c.attention_fwd(q, k, v, p["out"], p["q_starts"], p["k_starts"], *sizes, lse=p.get("lse"), **lay)
        else:
            dq = p["dqkv"]
            c.attention_bwd(q, k, v, p["out"], p["lse"], p["dout"], p["q_starts"], p["k_starts"], *sizes, dq=dq, dk=dq + heads * dim * size,
                            dv=dq + (heads + kv) * dim * size, **lay)
    elif kind == "rms":
        c.rmsnorm_fwd(p["x"], p["gamma"], p["y"], case["rows"], case["cols"], eps=_EPS, residual=p["residual"], sum=p["sum"], rstd=p.get("rstd"),
                      dtype=dtype)
    elif kind == "rms8":
        c.rmsnorm_fwd_e4m3(p["x"], p["gamma"], p["y"], p["scale"], case["rows"], case["cols"], group=case["group"], eps=_EPS,
                           residual=p["residual"], sum=p["sum"], dtype=dtype)
    elif kind == "rms_bwd":
        c.rmsnorm_bwd(p["x"], p["dy"], p["gamma"], p["rstd"], case["rows"], case["cols"], dx=p["dx"], dgamma=p["dgamma"], dsum=p["dsum"], dtype=dtype)
    elif kind == "logprobs":
        c.logprobs_fwd(p["logits"], p["targets"], p["logprob"], case["rows"], case["cols"], scale=_SCALE, entropy=p.get("entropy"), lse=p.get("lse"),
                       top=case["top"], top_ids=p.get("top_ids"), top_logprobs=p.get("top_logprobs"), dtype=dtype)
    else:
        c.logprobs_bwd(p["logits"], p["targets"], p["lse"], case["rows"], case["cols"], p["dlogits"], scale=_SCALE, dlogprob=p["dlogprob"],
                       entropy=p["entropy"] if case["entropy"] else None, dentropy=p["dentropy"] if case["entropy"] else None, dtype=dtype)
    return o


# ---- the plain form ----
def _plain(case, t):
    kind = case["kind"]
    if kind == "attend":
        return _attend(case, t)
    if kind == "attend_bwd":
        return _attend_bwd(case, t)
    if kind in ("rms", "rms8"):
        return _rms(case, t)
    if kind == "rms_bwd":
        h, rstd, dy = t["x"].float(), t["rstd"][:, None], t["dy"].float()
        n = h * rstd
        g = dy * t["gamma"].float()
        dx = t["dsum"].float() + rstd * (g - n * (g * n).mean(1, keepdim=True))
        return {"dx": dx.to(t["x"].dtype), "dgamma": (dy * n).sum(0).to(t["gamma"].dtype)}
    if kind == "logprobs":
        return _logprobs(case, t)
    p = torch.exp(t["logits"].float() * _SCALE - t["lse"][:, None])
    there = t["targets"] >= 0
    g = p * -t["dlogprob"][:, None]
    g.scatter_add_(1, t["targets"].long().clamp_(min=0)[:, None], t["dlogprob"][:, None])
    if case["entropy"]:
        logp = t["logits"].float() * _SCALE - t["lse"][:, None]
        g = g - t["dentropy"][:, None] * p * (logp + t["entropy"][:, None])
    return {"dlogits": torch.where(there[:, None], _SCALE * g, 0.0).to(t["logits"].dtype)}


def _qkv(case, t):
    """q [tokens, heads, dim], k and v [tokens, kv_heads, dim]."""
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    q, k, v = t["qkv"].split((h * d, kv * d, kv * d), 1) if "qkv" in t else (t["q"], t["k"], t["v"])
    return q.reshape(-1, h, d), k.reshape(-1, kv, d), v.reshape(-1, kv, d)


def _slots(case, t):
    """Where the tokens of each sequence stand, filled up to the longest: indices [seqs, longest], whether there is one, of queries and of keys;
    and the pairs that the mask leaves [seqs, longest, longest]."""
    n = case["seqs"]
    ks = _lengths(case["keys"], n)
    most_q, most_k = max(ks) if _own_tokens(case) else case["queries"] // n, max(ks)
    q0, k0 = t["q_starts"].long(), t["k_starts"].long()
    q_len, k_len = q0[1:] - q0[:-1], t["k_lengths"].long() if "k_lengths" in t else k0[1:] - k0[:-1]
    i, j = torch.arange(most_q, device="cuda"), torch.arange(most_k, device="cuda")
    q_in, k_in = i < q_len[:, None], j < k_len[:, None]
    pairs = q_in[:, :, None] & k_in[:, None, :]
    if case["causal"]:
        pairs = pairs & (j[None, None, :] - (k_len - q_len)[:, None, None] <= i[None, :, None])
    return torch.where(q_in, q0[:-1, None] + i, 0), q_in, torch.where(k_in, k0[:-1, None] + j, 0), k_in, pairs


def _grouped(case, x):
    """[seqs, longest, heads, dim] as [seqs, kv_heads, group * longest, dim]: the queries that share a head of keys."""
    b, n, h, d = x.shape
    return x.reshape(b, n, case["kv_heads"], -1, d).permute(0, 2, 3, 1, 4).reshape(b, case["kv_heads"], -1, d)


def _apart(case, x, n):
    """The way back, of rows [seqs, kv_heads, group * n, ...] to [seqs, n, heads, ...]."""
    b = x.shape[0]
    x = x.reshape(b, case["kv_heads"], -1, n, *x.shape[3:])
    return x.permute(0, 3, 1, 2, *range(4, x.dim())).reshape(b, n, case["heads"], *x.shape[4:])


def _scores(case, t):
    """scale * q k' where the mask allows it, -inf elsewhere: [seqs, kv_heads, group * longest, longest]; and what it was made of."""
    q, k, v = _qkv(case, t)
    q_at, q_in, k_at, k_in, pairs = _slots(case, t)
    q = _grouped(case, q[q_at].float())
    k = k[k_at].float().transpose(1, 2)
    v = torch.where(k_in[:, :, None, None], v[k_at].float(), 0.0).transpose(1, 2)
    s = q @ k.transpose(2, 3)
    s.mul_(case["dim"] ** -0.5)
    b, kv, rows, m = s.shape
    s.view(b, kv, -1, q_at.shape[1], m).masked_fill_(~pairs[:, None, None], -math.inf)
    return s, q, k, v, q_at, q_in, k_at, k_in


def _attend(case, t):
    s, _, _, v, q_at, q_in, _, _ = _scores(case, t)
    top = s.amax(-1, keepdim=True)
    top.masked_fill_(top == -math.inf, 0.0)      # a row without a key
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    lse = top + torch.log(total)
    n, dt = q_at.shape[1], DTYPES[case["dtype"]]
    out, lse = _apart(case, out, n)[q_in], _apart(case, lse, n)[q_in]
    return {"out": out.reshape(case["queries"], -1).to(dt), "lse": lse[:, :, 0].t().contiguous()}


def _attend_bwd(case, t):
    s, q, k, v, q_at, q_in, k_at, k_in = _scores(case, t)
    scale, n, dt = case["dim"] ** -0.5, q_at.shape[1], DTYPES[case["dtype"]]
    heads = lambda x: x.reshape(x.shape[0], case["heads"], -1)   # noqa: E731
    there = q_in[:, :, None, None]
    lse = _grouped(case, torch.where(there, heads(t["lse"].t())[q_at], 0.0))
    p = s.sub_(torch.where(lse > -math.inf, lse, 0.0)).exp_()
    dout = torch.where(there, heads(t["dout"]).float()[q_at], 0.0)
    delta = _grouped(case, (dout * heads(t["out"]).float()[q_at]).sum(-1, keepdim=True))
    dout = _grouped(case, dout)
    dv = p.transpose(2, 3) @ dout
    ds = (dout @ v.transpose(2, 3)).sub_(delta).mul_(p).mul_(scale)
    dq = _apart(case, ds @ k, n)[q_in].reshape(case["queries"], -1)
    dk = (ds.transpose(2, 3) @ q).transpose(1, 2)[k_in].reshape(case["keys"], -1)
    dv = dv.transpose(1, 2)[k_in].reshape(case["keys"], -1)
    return {"dqkv": torch.cat([dq, dk, dv], 1).to(dt)}


def _rms(case, t):
    dt = t["x"].dtype
    total = (t["x"].float() + t["residual"].float()).to(dt)
    h = total.float()
    rstd = torch.rsqrt((h * h).mean(1, keepdim=True) + _EPS)
    y = h * rstd * t["gamma"].float()
    if case["kind"] == "rms":
        return {"y": y.to(dt), "sum": total, "rstd": rstd[:, 0]}
    rows, cols = y.shape
    group = case["group"] or cols
    wide = torch.nn.functional.pad(y, (0, _groups(case) * group - cols)).reshape(rows, -1, group)
    scale = wide.abs().amax(2, keepdim=True) / 448.0
    q = wide / torch.where(scale > 0, scale, 1.0)
    return {"y": q.reshape(rows, -1)[:, :cols].contiguous().to(torch.float8_e4m3fn), "sum": total, "scale": scale[:, :, 0]}


def _logprobs(case, t):
    x = t["logits"].float() * _SCALE
    target = t["targets"].long()[:, None]
    there = target[:, 0] >= 0
    top = x.amax(1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    logprob = d.gather(1, target.clamp(min=0)) - torch.log(total)
    entropy = torch.log(total) - (e * d).sum(1, keepdim=True) / total
    f = {"logprob": torch.where(there, logprob[:, 0], 0.0), "lse": torch.where(there, lse[:, 0], 0.0), "entropy": torch.where(there, entropy[:, 0], 0.0)}
    n = case.get("top", 0)
    if n:
        best, ids = torch.sort(t["logits"], dim=1, descending=True, stable=True)      # the logits themselves: of equal ones the lowest index first
        f["top_ids"] = torch.where(there[:, None], ids[:, :n], -1).int()
        f["top_logprobs"] = torch.where(there[:, None], best[:, :n].float() * _SCALE - lse, -math.inf)
    return f


# ---- what a call cannot do without ----
def work(case):
    """Bytes: every input read once, every output written once.  flops: the arithmetic of the formulas, an exponential as one; of attention, the pairs
    that the mask leaves."""
    kind, size = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind in ("attend", "attend_bwd"):
        d, h, pairs = case["dim"], case["heads"], _pairs(case)
        q, kv = case["queries"] * h * d * size, 2 * case["keys"] * case["kv_heads"] * d * size
        if kind == "attend":
            return {"bytes": 2 * q + kv + (4 * h * case["queries"] if case["keep"] else 0), "flops": h * pairs * (4 * d + 4)}
        return {"bytes": 4 * q + 2 * kv + 4 * h * case["queries"], "flops": h * pairs * (10 * d + 6)}
    n, rows, cols = case["rows"] * case["cols"], case["rows"], case["cols"]
    if kind == "rms":
        return {"bytes": size * (4 * n + cols) + (4 * rows if case["keep"] else 0), "flops": 5 * n}
    if kind == "rms8":
        return {"bytes": size * (3 * n + cols) + n + 4 * rows * _groups(case), "flops": 7 * n}
    if kind == "rms_bwd":
        return {"bytes": size * (4 * n + 2 * cols) + 4 * rows, "flops": 11 * n}
    if kind == "logprobs":
        return {"bytes": size * n + 4 * rows * (2 + (2 if case["entropy"] else 0) + 2 * case["top"]), "flops": n * (6 if case["entropy"] else 4)}
    return {"bytes": 2 * size * n + 20 * rows, "flops": n * (9 if case["entropy"] else 5)}


# ---- the same outputs in 64 bits ----
def exact(case, seed):
    kind, t = case["kind"], _inputs(case, seed)
    d = {k: v.double() for k, v in t.items() if v.is_floating_point()}
    if kind in ("attend", "attend_bwd"):
        return _exact_attention(case, t, d)
    if kind in ("rms", "rms8"):
        total = (d["x"] + d["residual"]).to(t["x"].dtype).double()      # what the norm is taken of
        rms = torch.sqrt(total.pow(2).mean(1) + _EPS)
        y = torch.einsum("rc,c,r->rc", total, d["gamma"], 1.0 / rms)
        if kind == "rms":
            o = {"y": y, "sum": d["x"] + d["residual"], "rstd": 1.0 / rms}
            return o if case["keep"] else {k: o[k] for k in ("y", "sum")}
        group = case["group"] or case["cols"]
        scale = torch.stack([c.abs().max(1).values for c in y.split(group, 1)], 1) / 448.0
        return {"y": y / torch.repeat_interleave(scale, group, 1)[:, :case["cols"]].clamp(min=1e-300), "sum": d["x"] + d["residual"], "scale": scale}
    if kind == "rms_bwd":
        # dL/dh of y = n(h) gamma through the projection that a normalised row is: (I - n n'/cols) rstd
        n = d["x"] * d["rstd"][:, None]
        g = d["dy"] * d["gamma"]
        along = torch.einsum("rc,rc->r", g, n) / case["cols"]
        return {"dx": torch.addcmul(d["dsum"], g - along[:, None] * n, d["rstd"][:, None]), "dgamma": torch.einsum("rc,rc->c", d["dy"], n)}
    there = t["targets"] >= 0
    at = torch.where(there, t["targets"], 0).long()
    if kind == "logprobs":
        logp = torch.log_softmax(d["logits"] * _SCALE, 1)
        o = {"logprob": torch.where(there, logp[torch.arange(case["rows"], device="cuda"), at], 0.0)}
        if case["entropy"]:
            o.update(entropy=torch.where(there, -(logp.exp() * logp).sum(1), 0.0), lse=torch.where(there, torch.logsumexp(d["logits"] * _SCALE, 1), 0.0))
        if case["top"]:
            order = torch.argsort(-d["logits"], dim=1, stable=True)[:, :case["top"]]
            o.update(top_ids=torch.where(there[:, None], order, -1).int(), top_logprobs=torch.where(there[:, None], logp.gather(1, order), -math.inf))
        return o
    x = d["logits"].requires_grad_()
    logp = torch.log_softmax(x * _SCALE, 1)
    loss = (logp[torch.arange(case["rows"], device="cuda"), at] * d["dlogprob"])[there].sum()
    if case["entropy"]:
        loss = loss - ((logp.exp() * logp).sum(1) * d["dentropy"])[there].sum()
    return {"dlogits": torch.autograd.grad(loss, x)[0]}


def _exact_attention(case, t, d):
    """Sequence by sequence and head by head, the gradients by differentiation."""
    bwd = case["kind"] == "attend_bwd"
    if _pairs(case) * case["heads"] * case["dim"] > 4e12:
        return None
    q, k, v = (x.contiguous() for x in _qkv(case, d))
    group = case["heads"] // case["kv_heads"]
    out, lse = torch.zeros_like(q), torch.full((case["heads"], case["queries"]), -math.inf, dtype=torch.float64, device="cuda")
    grads = tuple(torch.zeros_like(x) for x in (q, k, v))
    q0, k0 = t["q_starts"].tolist(), t["k_starts"].tolist()
    for b in range(case["seqs"]):
        nk = int(t["k_lengths"][b]) if "k_lengths" in t else k0[b + 1] - k0[b]
        i, j = slice(q0[b], q0[b + 1]), slice(k0[b], k0[b] + nk)
        nq = q0[b + 1] - q0[b]
        first = max(0, nq - nk) if case["causal"] else (0 if nk else nq)      # rows before it see nothing
        mask = torch.ones((nq, nk), dtype=torch.bool, device="cuda").tril(nk - nq)[first:] if case["causal"] else None
        for h in range(case["heads"]):
            rows = [x.detach().requires_grad_(bwd) for x in (q[i, h][first:], k[j, h // group], v[j, h // group])]
            s = rows[0] @ rows[1].T * case["dim"] ** -0.5
            s = s if mask is None else s.masked_fill(~mask, -math.inf)
            o = torch.softmax(s, 1) @ rows[2]
            if bwd:
                g = torch.autograd.grad(o, rows, d["dout"].view_as(q)[i, h][first:])
                grads[0][i, h][first:] = g[0]
                grads[1][j, h // group] += g[1]
                grads[2][j, h // group] += g[2]
            else:
                out[i, h][first:] = o
                lse[h, i][first:] = torch.logsumexp(s, 1)
    if bwd:
        return {"dqkv": torch.cat([g.reshape(g.shape[0], -1) for g in grads], 1)}
    out = out.reshape(case["queries"], -1)
    return {"out": out, "lse": lse} if case["keep"] else {"out": out}
