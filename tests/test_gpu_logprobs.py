"""Log probabilities, entropies and largest entries of rows of logits against the formulas in 64 bits.

Bounds, with U = 2^-24, h the half step of the storage type, z = scale * x, m the largest z, d = z - m and n = cols / 32 + 64 (the longest
chain of additions in a row's sum):
  weight   relative e_w = U (2 |z| + 2 |m| + 3 |d|) + 2^-21
  lse      sum of p e_w, n U, 4 U (|lse| + |m|)
  logprob  that of lse - m, and U (2 |z_t| + 2 |m| + 2 |logprob|)
  entropy  that of log l, sum p e_w |d| and sum p e_w times sum p |d|, 2 n U sum p |d|, U (2 |z| + 2 |m|) p, 4 U
  dlogits  p with e_w + U (2 |z| + 3 |lse|); U (2 |z| + 3 |lse| + 3 |H|) for log p + H; 8 U of each term; h of the result
"""
import numpy as np
import pytest

from token_ops import check, empty, HALF_ULP, Placed, rounded, TINY, U

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]
PAD = 0xffffffff
NO_TOKEN = 0xffffffff


@pytest.fixture()
def ctx():
    from ferrograd_b200 import GpuContext
    c = GpuContext(0)
    yield c
    assert c.device_status() == 0
    c.destroy()


def rng(*key):
    return np.random.Generator(np.random.Philox(key))


def case(seed, rows, cols, dtype, spread=2.5, forbidden=0.1):
    r = rng(seed, rows, cols)
    x = r.standard_normal((rows, cols)) * spread
    x[r.random((rows, cols)) < forbidden] = -np.inf
    t = r.integers(0, cols, rows).astype(np.uint32)
    t[r.random(rows) < 0.1] = PAD
    return rounded(x, dtype), t


def forward64(x, t, scale):
    scale = float(np.float32(scale))
    z = x.astype(np.float64) * scale
    cols = x.shape[1]
    m = z.max(1, keepdims=True)
    there = np.isfinite(m)
    m0 = np.where(there, m, 0.0)
    d = np.where(np.isfinite(z), z - m0, 0.0)
    w = np.where(np.isfinite(z), np.exp(d), 0.0)
    l = w.sum(1, keepdims=True)
    l0 = np.where(there, l, 1.0)
    p = w / l0
    zf = np.where(np.isfinite(z), z, 0.0)
    e_w = U * (2 * np.abs(zf) + 2 * np.abs(m0) + 3 * np.abs(d)) + 2.0 ** -21
    n = cols / 32 + 64
    lse = np.where(there, m0 + np.log(l0), -np.inf)[:, 0]
    e_log = (p * e_w).sum(1) + n * U + 4 * U * np.abs(np.log(l0[:, 0]))
    e_lse = e_log + 4 * U * np.where(there, np.abs(np.where(there, lse[:, None], 0.0)) + np.abs(m0), 0.0)[:, 0]
    at = np.where(t < cols, t, 0).astype(int)
    zt = z[np.arange(len(t)), at]
    with np.errstate(invalid="ignore"):
        logp = np.where(there[:, 0], zt - np.where(there[:, 0], lse, 0.0), -np.inf)
    f = lambda a: np.where(np.isfinite(a), np.abs(a), 0.0)   # noqa: E731
    e_logp = e_log + U * (2 * f(zt) + 2 * np.abs(m0[:, 0]) + 2 * f(logp))
    pd = (p * np.abs(d)).sum(1)
    ent = np.where(there[:, 0], np.log(l0[:, 0]) + pd, 0.0)
    e_ent = e_log + (p * e_w * np.abs(d)).sum(1) + (p * e_w).sum(1) * pd + 2 * n * U * pd + (p * U * (2 * np.abs(zf) + 2 * np.abs(m0))).sum(1) + 4 * U * (1 + ent)
    return {"lse": lse, "logprob": logp, "entropy": ent}, {"lse": e_lse, "logprob": e_logp, "entropy": e_ent}, p, z


def same(got, want, bound, what):
    inf = np.isneginf(want)
    assert np.array_equal(np.isneginf(got), inf), what
    if (~inf).any():
        check(got[~inf], want[~inf], bound[~inf], what)


def top64(x, top):
    order = np.argsort(-x.astype(np.float64), axis=1, kind="stable")[:, :top]
    return np.where(np.isneginf(np.take_along_axis(x, order, 1)), NO_TOKEN, order).astype(np.uint32)


def run(ctx, x, t, dtype, scale=1.0, top=0, shift=0, entropy=True):
    rows, cols = x.shape
    o = {n: empty(ctx, (rows,)) for n in ("logprob", "lse")}
    if entropy:
        o["entropy"] = empty(ctx, (rows,))
    ids, lps = (empty(ctx, (rows, top), "u32"), empty(ctx, (rows, top))) if top else (None, None)
    ctx.logprobs_fwd(Placed(ctx, x, dtype, shift), Placed(ctx, t, "u32"), o["logprob"], rows, cols, scale=scale, entropy=o.get("entropy"), lse=o["lse"], top=top,
                     top_ids=ids, top_logprobs=lps, dtype=dtype)
    got = {n: v.get() for n, v in o.items()}
    return (got, ids.get(), lps.get()) if top else (got, None, None)


def check_forward(x, t, scale, top, got, ids, lps):
    cols = x.shape[1]
    want, bound, _, z = forward64(x, t, scale)
    live = t < cols
    for n, v in got.items():
        assert (v[~live] == 0).all(), n
        same(v[live], want[n][live], bound[n][live], n)
    if top:
        assert (ids[~live] == NO_TOKEN).all() and np.isneginf(lps[~live]).all()
        assert np.array_equal(ids[live], top64(x, top)[live])
        for i in range(top):
            w, b, _, _ = forward64(x, np.where(ids[:, i] == NO_TOKEN, 0, ids[:, i]), scale)
            some = live & (ids[:, i] != NO_TOKEN)
            same(lps[some, i], w["logprob"][some], b["logprob"][some], f"top {i}")
            assert np.isneginf(lps[live & ~some, i]).all()


SIZES = [(1, 1), (3, 2), (1, 50), (40, 333), (7, 1000), (64, 4096), (2, 32000), (300, 777), (5, 50257), (1, 128003), (3, 200000), (600, 129), (160, 32000)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top", [0, 1, 20])
def test_forward(ctx, rows, cols, dtype, top):
    top = min(top, cols)
    x, t = case(1, rows, cols, dtype)
    for shift in (0, 1):
        check_forward(x, t, 1.25, top, *run(ctx, x, t, dtype, 1.25, top, shift))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top", [2, 31, 32, 33, 64])
def test_many_alternatives(ctx, dtype, top):
    x, t = case(2, 9, 3001, dtype)
    check_forward(x, t, 1.0, top, *run(ctx, x, t, dtype, 1.0, top, entropy=False))


@pytest.mark.parametrize("dtype", TYPES)
def test_ties(ctx, dtype):
    # few values, so the order is that of the indices; zeros of both signs are equal; rising and falling rows
    r = rng(3)
    x = np.stack([r.integers(-2, 3, 5000), np.zeros(5000), np.where(r.random(5000) < 0.5, 0.0, -0.0), np.arange(5000) // 64, -(np.arange(5000) // 64), np.full(5000, -7.0)])
    x = rounded(x, dtype)
    t = np.arange(6, dtype=np.uint32)
    check_forward(x, t, 1.0, 64, *run(ctx, x, t, dtype, 1.0, 64))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_with_little(ctx, dtype):
    # nothing, one entry, fewer than asked for, one that has all of the weight, entries of the lowest number
    x = np.full((6, 700), -np.inf, np.float32)
    x[1, 699] = 3.0
    x[2, 5:9] = 1.0
    x[3] = -50.0
    x[3, 300] = 60.0
    x[4] = rounded(np.float32(-60000.0 if dtype == "f16" else -3.3e38), dtype)
    x[4, 10:20] = 0.5
    x[5] = rounded(np.float32(-60000.0 if dtype == "f16" else -3.3e38), dtype)
    x = rounded(x, dtype)
    t = np.array([3, 699, 4, 300, 11, 0], np.uint32)
    check_forward(x, t, 1.0, 20, *run(ctx, x, t, dtype, 1.0, 20))


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_and_infinity(ctx, dtype):
    x, t = case(4, 5, 900, dtype, forbidden=0.0)
    t[:] = [1, 2, 3, 4, 5]
    clean = x.copy()
    x[1, 400] = np.nan
    x[2, 500] = np.inf
    x[4] = -np.inf
    x[4, 600] = np.nan
    got, ids, lps = run(ctx, x, t, dtype, 1.0, 5)
    for n, v in got.items():
        assert np.isnan(v[1]) and np.isnan(v[4]) and (np.isnan(v[2]) or (n == "lse" and np.isposinf(v[2]))), n
    assert 400 not in ids[1] and ids[2, 0] == 500 and np.isnan(lps[1]).all()
    rest = [0, 3]
    check_forward(clean[rest], t[rest], 1.0, 5, {n: v[rest] for n, v in got.items()}, ids[rest], lps[rest])


@pytest.mark.parametrize("dtype", TYPES)
def test_some_outputs(ctx, dtype):
    x, t = case(5, 30, 1003, dtype)
    want, bound, _, _ = forward64(x, t, 0.7)
    d, dt = Placed(ctx, x, dtype), Placed(ctx, t, "u32")
    live = t < 1003
    for n in ("logprob", "entropy", "lse"):
        o = empty(ctx, (30,))
        ctx.logprobs_fwd(d, dt, o if n == "logprob" else None, 30, 1003, scale=0.7, dtype=dtype, **({n: o} if n != "logprob" else {}))
        same(o.get()[live], want[n][live], bound[n][live], n)
    o, e, ids, lps = empty(ctx, (30,)), empty(ctx, (30,)), empty(ctx, (30, 3), "u32"), empty(ctx, (30, 3))
    ctx.logprobs_fwd(d, None, None, 30, 1003, scale=0.7, entropy=e, top=3, top_ids=ids, top_logprobs=lps, dtype=dtype)      # no targets: no padding
    same(e.get(), want["entropy"], bound["entropy"], "entropy")
    assert np.array_equal(ids.get(), top64(x, 3))


def backward64(x, t, scale, lse, ent, gl, ge):
    want, _, _, z = forward64(x, t, scale)
    rows, cols = x.shape
    scale = float(np.float32(scale))
    lse, ent = lse.astype(np.float64)[:, None], ent.astype(np.float64)[:, None]
    gl, ge = (np.zeros((rows, 1)) if g is None else g.astype(np.float64)[:, None] for g in (gl, ge))
    ok = np.isfinite(lse)
    zf = np.where(np.isfinite(z), z, 0.0)
    logp = np.where(np.isfinite(z) & ok, zf - np.where(ok, lse, 0.0), -1e4)
    p = np.exp(logp)
    one = np.arange(cols)[None] == t[:, None]
    live = ok & (t[:, None] < cols)
    g = np.where(live, scale * (gl * (one - p) - ge * p * (logp + ent)), 0.0)
    e_z = U * (3 * np.abs(zf) + 4 * np.abs(np.where(ok, lse, 0.0)))
    e = scale * (p * (np.abs(gl) + np.abs(ge * (logp + ent))) * (e_z + 2.0 ** -20) + p * np.abs(ge) * (e_z + 4 * U * (np.abs(ent) + np.abs(logp))) + 8 * U * np.abs(gl) * one)
    return g, e + 8 * U * np.abs(g) + 2.0 ** -126 * scale * (np.abs(gl) + 100 * np.abs(ge))


@pytest.mark.parametrize("rows,cols", SIZES + [(1000, 1024)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_backward(ctx, rows, cols, dtype, shift):
    x, t = case(6, rows, cols, dtype)
    r = rng(7, rows, cols)
    gl, ge = r.standard_normal(rows).astype(np.float32), r.standard_normal(rows).astype(np.float32)
    f = forward64(x, t, 1.25)[0]
    lse, ent = f["lse"].astype(np.float32), f["entropy"].astype(np.float32)
    dev = {n: Placed(ctx, v) for n, v in (("lse", lse), ("ent", ent), ("gl", gl), ("ge", ge))}
    d, dt = Placed(ctx, x, dtype, shift), Placed(ctx, t, "u32")
    for with_l, with_e in ((True, True), (True, False), (False, True)):
        g = empty(ctx, (rows, cols), dtype, shift)
        ctx.logprobs_bwd(d, dt, dev["lse"], rows, cols, g, scale=1.25, dlogprob=dev["gl"] if with_l else None, entropy=dev["ent"] if with_e else None,
                         dentropy=dev["ge"] if with_e else None, dtype=dtype)
        want, bound = backward64(x, t, 1.25, lse, ent, gl if with_l else None, ge if with_e else None)
        check(g.get(), want, bound + HALF_ULP[dtype] * np.abs(want) + TINY[dtype], "dlogits")
    ctx.logprobs_bwd(d, dt, dev["lse"], rows, cols, d, scale=1.25, dlogprob=dev["gl"], dtype=dtype)      # in place
    want, bound = backward64(x, t, 1.25, lse, ent, gl, None)
    check(d.get(), want, bound + HALF_ULP[dtype] * np.abs(want) + TINY[dtype], "dlogits")


def test_differences(ctx):
    x, t = case(8, 20, 300, "f32", forbidden=0.0)
    r = rng(9)
    gl, ge = r.standard_normal(20).astype(np.float32), r.standard_normal(20).astype(np.float32)
    got, _, _ = run(ctx, x, t, "f32", 0.8)
    g = empty(ctx, x.shape)
    ctx.logprobs_bwd(Placed(ctx, x), Placed(ctx, t, "u32"), Placed(ctx, got["lse"]), 20, 300, g, scale=0.8, dlogprob=Placed(ctx, gl), entropy=Placed(ctx, got["entropy"]),
                     dentropy=Placed(ctx, ge))
    step = r.standard_normal(x.shape)
    live = t < 300

    def loss(x):
        f = forward64(x, t, 0.8)[0]
        return (f["logprob"] * gl + f["entropy"] * ge)[live].sum()

    slope = (loss(x + 1e-6 * step) - loss(x - 1e-6 * step)) / 2e-6
    assert abs((g.get() * step).sum() - slope) <= 2e-5 * (np.abs(g.get()) * np.abs(step)).sum()


@pytest.mark.parametrize("dtype", TYPES)
def test_same_bits_and_recorded(ctx, dtype):
    rows, cols, top = 33, 40001, 10
    x, t = case(10, rows, cols, dtype)
    d, dt = Placed(ctx, x, dtype), Placed(ctx, t, "u32")
    r = rng(11)
    gl, ge = Placed(ctx, r.standard_normal(rows)), Placed(ctx, r.standard_normal(rows))
    outputs = lambda: [empty(ctx, (rows,)) for _ in range(3)] + [empty(ctx, (rows, top), "u32"), empty(ctx, (rows, top)), empty(ctx, (rows, cols), dtype)]   # noqa: E731

    def step(o):
        ctx.logprobs_fwd(d, dt, o[0], rows, cols, entropy=o[1], lse=o[2], top=top, top_ids=o[3], top_logprobs=o[4], dtype=dtype)
        ctx.logprobs_bwd(d, dt, o[2], rows, cols, o[5], dlogprob=gl, entropy=o[1], dentropy=ge, dtype=dtype)

    a, b = outputs(), outputs()
    step(a)
    ctx.plan_begin()
    step(b)
    plan = ctx.plan_end()
    for _ in range(3):
        step(a)
        plan.launch()
    ctx.sync()
    for p, q in zip(a, b):
        assert np.array_equal(p.bits(), q.bits())
    plan.destroy()


def test_refusals(ctx):
    from ferrograd_b200.backend import FgError
    x, g = Placed(ctx, np.zeros((4, 80))), Placed(ctx, np.zeros((4, 80)))
    t, v, w, u = Placed(ctx, np.zeros(4), "u32"), Placed(ctx, np.zeros(4)), Placed(ctx, np.zeros(4)), Placed(ctx, np.zeros(4))
    ids, lps = Placed(ctx, np.zeros((4, 80)), "u32"), Placed(ctx, np.zeros((4, 80)))
    f = lambda x=x, t=t, logprob=v, rows=4, cols=80, **k: ctx.logprobs_fwd(x, t, logprob, rows, cols, **k)   # noqa: E731
    b = lambda x=x, t=t, lse=v, cols=80, g=g, **k: ctx.logprobs_bwd(x, t, lse, 4, cols, g, **k)   # noqa: E731
    f(entropy=w, lse=u, top=5, top_ids=ids, top_logprobs=lps)
    b(dlogprob=w)
    f(rows=0)
    bad = [lambda: f(x=None), lambda: f(t=None), lambda: f(cols=0), lambda: f(rows=1 << 31, cols=1 << 31), lambda: f(scale=0.0), lambda: f(scale=-1.0), lambda: f(scale=float("nan")),
           lambda: f(scale=float("inf")), lambda: f(logprob=None), lambda: f(top=65, top_ids=ids, top_logprobs=lps), lambda: f(cols=4, top=5, top_ids=ids, top_logprobs=lps),
           lambda: f(top=5, top_ids=ids), lambda: f(top=5, top_logprobs=lps), lambda: f(logprob=x), lambda: f(logprob=t), lambda: f(entropy=v), lambda: f(lse=v.ptr + 4),
           lambda: f(top=5, top_ids=ids, top_logprobs=ids), lambda: f(x=x.ptr + 2), lambda: f(logprob=v.ptr + 1),
           lambda: b(x=None, dlogprob=w), lambda: b(lse=None, dlogprob=w), lambda: b(g=None, dlogprob=w), lambda: b(), lambda: b(t=None, dlogprob=w), lambda: b(dentropy=w),
           lambda: b(cols=0, dlogprob=w), lambda: b(dlogprob=w, scale=0.0), lambda: b(g=x.ptr + 4, dlogprob=w), lambda: b(g=v, dlogprob=w), lambda: b(g=w, dlogprob=w),
           lambda: b(g=t, dlogprob=w)]
    for i, call in enumerate(bad):
        with pytest.raises(FgError) as err:
            call()
        assert err.value.kind == "FG_ERR_INVALID_ARGUMENT", i
    assert ctx.device_status() == 0
