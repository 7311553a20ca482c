"""Sampling against the definition in 64 bits: tokens have to be equal.  A token of the definition could only differ where u times the total lies
within 1e-11 of a border between two tokens (the weights' rounding), which is no chance to speak of for the rows here; the share of a token
is off by half a step of f32."""
import numpy as np
import pytest

from token_ops import Placed, empty, rounded

pytestmark = pytest.mark.gpu
TYPES = ("f32", "f16", "bf16")
NONE = 0xffffffff


@pytest.fixture(scope="module")
def ctx():
    from ferrograd_b200 import GpuContext
    c = GpuContext(0)
    yield c
    assert c.device_status() == 0
    c.destroy()


def definition(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, share) of one row."""
    x = x.astype(np.float64)
    allowed = np.flatnonzero(x > -np.inf)          # neither -inf nor NaN
    if not allowed.size:
        return NONE, 0.0
    x = x[allowed]
    m = x.max()
    if not temperature > 0:
        return allowed[np.argmax(x)], 1.0
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        w = np.where(x == m, 1.0, np.exp((x - m) / np.float64(temperature)) if m < np.inf else 0.0)
    down = np.argsort(-x, kind="stable")
    if 0 < top_k < down.size:
        down = down[:top_k]
    if top_p < 1:
        mass = np.cumsum(w[down])
        down = down[:1 + np.searchsorted(mass, max(top_p, 0.0) * mass[-1], side="left")]
    if min_p > 0:
        down = down[w[down] >= min(np.float64(min_p), 1.0)]
    kept = np.sort(down)
    mass = np.cumsum(w[kept])
    u = np.float64(min(u, np.float32(0.99999994))) if u > 0 else 0.0
    i = np.searchsorted(mass, u * mass[-1], side="right")
    return allowed[kept[i]], w[kept[i]] / mass[-1]


def run(ctx, x, u, dtype="f32", shift=0, **params):
    rows, cols = x.shape
    args = {k: Placed(ctx, v, "u32" if k == "top_k" else "f32", shift) for k, v in params.items() if v is not None}
    token, prob = empty(ctx, (rows,), "u32", shift), empty(ctx, (rows,), "f32", shift)
    ctx.sample(Placed(ctx, x, dtype, shift), Placed(ctx, u, "f32", shift), token, rows, cols, prob=prob, dtype=dtype, **args)
    got, share = token.get(), prob.get()
    for r in range(rows):
        want = definition(x[r], np.float32(u[r]), **{k: v[r] for k, v in params.items() if v is not None})
        assert got[r] == want[0], f"row {r}: token {got[r]} for {want[0]}, u {u[r]}, " + ", ".join(f"{k} {v[r]}" for k, v in params.items() if v is not None)
        assert abs(share[r] - want[1]) <= 2.0 ** -24 * 1.01 * want[1] + 2.0 ** -149, f"row {r}: share {share[r]} for {want[1]}"
    again, _ = empty(ctx, (rows,), "u32"), None
    ctx.sample(Placed(ctx, x, dtype, shift), Placed(ctx, u, "f32", shift), again, rows, cols, dtype=dtype, **args)
    assert np.array_equal(again.get(), got)
    return got


FILTERS = {"none": (), "temperature": ("temperature",), "top_k": ("top_k",), "top_p": ("top_p",), "min_p": ("min_p",), "k_and_p": ("top_k", "top_p"),
           "p_and_min": ("temperature", "top_p", "min_p"), "all": ("temperature", "top_k", "top_p", "min_p")}


def params_of(names, rows, cols, r):
    every = {"temperature": (0.3 + 1.5 * r.random(rows)).astype(np.float32), "top_k": r.integers(0, max(2, min(cols + 2, 120)), rows).astype(np.uint32),
             "top_p": r.random(rows).astype(np.float32) * np.float32(1.05), "min_p": (r.random(rows) ** 3).astype(np.float32)}
    return {k: every[k] for k in names}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(3, 1), (5, 2), (7, 31), (40, 100), (300, 1000), (9, 1024), (6, 8193), (4, 32000), (3, 50257), (200, 5001), (2, 131072), (1, 300001)])
@pytest.mark.parametrize("filters", sorted(FILTERS))
@pytest.mark.parametrize("spread,shift", [(2.5, 0), (0.05, 1), (40.0, 0)])
def test_random_rows(ctx, dtype, rows, cols, filters, spread, shift):
    r = np.random.Generator(np.random.Philox(rows * 7 + cols))
    x = r.standard_normal((rows, cols)) * spread
    x[r.random((rows, cols)) < 0.1] = -np.inf
    run(ctx, rounded(x, dtype), r.random(rows).astype(np.float32), dtype, shift, **params_of(FILTERS[filters], rows, cols, r))


@pytest.mark.parametrize("cols", [1, 3, 40, 1000, 4099, 40000, 200000])
def test_equal_logits(ctx, cols):
    # every weight is one: sums are whole, borders are hit exactly, and the first of the equal ones are kept
    u = np.array([0.0, 0.5, 0.25, 0.999, 0.99999994, 2.0 ** -30, 0.75, 0.125], np.float32)
    n = len(u)
    x = np.full((n, cols), 1.5, np.float32)
    run(ctx, x, u)
    run(ctx, x, u, top_k=np.array([1, 2, 3, 0, cols, cols + 5, max(1, cols // 2), 0xffffffff], np.uint32))
    p = np.array([0.0, 0.5, 0.25, 1.0, 0.75, 2.0, -1.0, 0.125], np.float32)
    run(ctx, x, u, top_p=p)
    run(ctx, x, u, top_p=p, top_k=np.full(n, max(1, cols // 3), np.uint32))
    run(ctx, x, u, min_p=np.array([0, 1, 2, 0.5, -1, 1, 1, 0], np.float32))
    # two values, the larger one rare
    x[:, ::3] = 2.5
    run(ctx, x, u, top_k=np.array([1, 2, 3, 0, cols, cols // 3 + 1, max(1, cols // 2), cols // 3 + 2], np.uint32), top_p=p)
    # few values, as 16-bit logits have
    r = np.random.Generator(np.random.Philox(cols))
    x = r.integers(-4, 5, (n, cols)).astype(np.float32)
    x[x == 0] *= -1.0          # -0 is 0
    for dtype in TYPES:
        run(ctx, x, u, dtype, top_k=r.integers(0, cols + 1, n).astype(np.uint32), top_p=r.random(n).astype(np.float32))
        run(ctx, x, u, dtype, top_p=r.random(n).astype(np.float32))


@pytest.mark.parametrize("cols", [5, 100, 2000, 33000])
def test_values_out_of_the_ordinary(ctx, cols):
    r = np.random.Generator(np.random.Philox(cols))
    x = r.standard_normal((16, cols)).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2] = -np.inf
    x[2, cols // 2] = -3.0                       # one allowed
    x[3, 1] = np.inf
    x[4, [1, cols - 1]] = np.inf                 # two that are infinite
    x[5, ::2] = np.nan
    x[6] = -3.4e38                               # the lowest number is a number
    x[7, :] = np.where(np.arange(cols) % 2, -3.4028235e38, -np.inf)
    x[8, 0], x[8, 1] = 3.4e38, -3.4e38
    x[9] = 0.0
    x[9, ::2] = -0.0
    x[10] = 1e-45
    x[11, :3] = 30000.0
    u = r.random(16).astype(np.float32)
    none = dict()
    for params in (none, dict(top_k=np.full(16, 2, np.uint32)), dict(top_p=np.full(16, 0.6, np.float32)), dict(min_p=np.full(16, 0.3, np.float32)),
                   dict(temperature=np.zeros(16, np.float32)), dict(temperature=np.full(16, np.inf, np.float32)), dict(temperature=np.full(16, 1e-40, np.float32)),
                   dict(temperature=np.full(16, 3e38, np.float32), top_k=np.full(16, 3, np.uint32)), dict(temperature=np.full(16, 0.7, np.float32),
                   top_k=np.full(16, 3, np.uint32), top_p=np.full(16, 0.5, np.float32), min_p=np.full(16, 0.01, np.float32))):
        run(ctx, x, u, **params)
    # parameters out of their ranges
    y = np.repeat(x[12:13], 16, 0)
    odd = np.array([np.nan, -1, 0, 5, np.inf, -np.inf, 1e-30, 0.5] * 2, np.float32)
    run(ctx, y, u, temperature=odd)
    run(ctx, y, u, top_p=odd)
    run(ctx, y, u, min_p=odd)
    run(ctx, y, odd)


def test_border_of_top_k_among_equals(ctx):
    # the k-th largest value occurs on both sides of the cut: the first ones are kept, wherever they lie
    for cols in (50, 3000, 70000):
        x = np.zeros((64, cols), np.float32)
        r = np.random.Generator(np.random.Philox(cols))
        for i in range(64):
            x[i, r.permutation(cols)[:10]] = 3.0
            x[i, r.permutation(cols)[:15]] = 2.0
        run(ctx, x, r.random(64).astype(np.float32), top_k=r.integers(5, 30, 64).astype(np.uint32), min_p=np.full(64, 0.2, np.float32))


@pytest.mark.parametrize("dtype,rows,cols", [("f32", 2, 500_001), ("f16", 2, 1_000_003), ("bf16", 1, 2_097_152)])
def test_rows_that_no_cluster_holds(ctx, dtype, rows, cols):
    r = np.random.Generator(np.random.Philox(cols))
    x = r.standard_normal((rows, cols)) * 3
    x[r.random((rows, cols)) < 0.2] = -np.inf
    x, u = rounded(x, dtype), r.random(rows).astype(np.float32)
    for names in ((), ("top_k",), ("top_p",), ("top_k", "top_p", "min_p"), ("temperature", "min_p")):
        run(ctx, x, u, dtype, 1, **params_of(names, rows, cols, r))


@pytest.mark.parametrize("cols,k", [(5000, 2500), (20000, 300), (20000, 3000), (50000, 49_999), (130000, 1500), (130000, 20_000)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_wide_filters(ctx, cols, k, dtype):
    # more candidates than a list has room for, and nuclei of most of a row
    r = np.random.Generator(np.random.Philox(cols + k))
    x, u = rounded(r.standard_normal((4, cols)) * 2, dtype), r.random(4).astype(np.float32)
    x[2] *= np.float32(0.0625)          # nearly flat
    x[3] = np.sort(x[3])                # all that counts is in the last CTA
    run(ctx, x, u, dtype, top_k=np.full(4, k, np.uint32))
    run(ctx, x, u, dtype, top_k=np.full(4, k, np.uint32), top_p=np.full(4, 0.97, np.float32))
    for p in (0.05, 0.5, 0.95, 0.999, 0.9999999):
        run(ctx, x, u, dtype, top_p=np.full(4, p, np.float32), min_p=np.array([0, 0.01, 0, 0.1], np.float32))


def test_draws_follow_the_weights(ctx):
    # 4096 draws from one row: each count within five deviations of its share
    cols, rows = 50, 4096
    r = np.random.Generator(np.random.Philox(2))
    x = np.repeat(r.standard_normal((1, cols)).astype(np.float32), rows, 0)
    got = run(ctx, x, ((np.arange(rows) + 0.5) / rows).astype(np.float32))
    w = np.exp(x[0].astype(np.float64))
    # evenly spaced numbers: a token's count is its share to within one
    assert np.abs(np.bincount(got, minlength=cols) - rows * w / w.sum()).max() <= 1.01
    assert np.all(np.diff(got.astype(np.int64)) >= 0)


@pytest.mark.parametrize("rows,cols", [(1, 32000), (70, 3000), (20, 150000)])
def test_captured(ctx, rows, cols):
    r = np.random.Generator(np.random.Philox(rows))
    x = Placed(ctx, np.zeros((rows, cols)))
    p = {k: Placed(ctx, np.zeros(rows), "u32" if k == "top_k" else "f32") for k in ("u", "temperature", "top_k", "top_p", "min_p")}
    token, prob = empty(ctx, (rows,), "u32"), empty(ctx, (rows,))
    args = (x, p["u"], token, rows, cols, p["temperature"], p["top_k"], p["top_p"], p["min_p"], prob)
    ctx.sample(*args)
    ctx.plan_begin()
    ctx.sample(*args)
    plan = ctx.plan_end()
    for k in range(4):
        values = (3 * r.standard_normal((rows, cols))).astype(np.float32)
        given = params_of(FILTERS["all"], rows, cols, r) | {"u": r.random(rows).astype(np.float32)}
        if k == 2:
            given["temperature"][:] = 0
        if k == 3:
            given["top_p"][:], given["top_k"][:], given["min_p"][:] = 1, 0, 0
        ctx.upload(x.t.data, values)
        for name, v in given.items():
            ctx.upload(p[name].t.data, v)
        plan.launch()
        u = given.pop("u")
        want = [definition(values[i], u[i], **{n: v[i] for n, v in given.items()}) for i in range(rows)]
        assert np.array_equal(token.get(), np.array([w[0] for w in want], np.uint32))
    plan.destroy()


def test_empty_and_refusals(ctx):
    from ferrograd_b200 import FgError
    t = ctx.new_tensor((256,))
    p = t.ptr
    ctx.sample(p, p, p, 0, 4)

    def refuse(**kw):
        a = dict(logits=p, u=p + 512, token=p + 600, rows=2, cols=4) | kw
        with pytest.raises(FgError) as e:
            ctx.sample(**a)
        assert e.value.kind == "FG_ERR_INVALID_ARGUMENT"

    for kw in (dict(logits=None), dict(u=None), dict(token=None), dict(cols=0), dict(cols=2097153), dict(logits=p + 2), dict(u=p + 514), dict(token=p + 602),
               dict(temperature=p + 1), dict(top_k=p + 2), dict(top_p=p + 3), dict(min_p=p + 6), dict(prob=p + 6)):
        refuse(**kw)
    assert ctx.lib.fg_sample(ctx.handle, 3, 1, 4, p, p, None, None, None, None, p, None) == 1


def test_outputs_that_overlap_are_refused(ctx):
    from ferrograd_b200 import FgError
    p = ctx.new_tensor((64,)).ptr      # 2 x 4 logits: 32 bytes; the others 8 bytes each
    given = dict(logits=p, u=p + 32, token=p + 128, rows=2, cols=4, temperature=p + 40, top_k=p + 48, top_p=p + 56, min_p=p + 64, prob=p + 136)
    for at in (0, 28, 32, 36, 44, 52, 60, 68):
        for out in ("token", "prob"):
            with pytest.raises(FgError) as e:
                ctx.sample(**(given | {out: p + at}))
            assert e.value.kind == "FG_ERR_INVALID_ARGUMENT"
    for kw in (dict(prob=p + 128), dict(prob=p + 132), dict(token=p + 140)):
        with pytest.raises(FgError):
            ctx.sample(**(given | kw))
    ctx.sample(**given)


@pytest.mark.parametrize("dtype,cols", [("f32", 360_001), ("bf16", 730_001), ("f16", 730_008)])
@pytest.mark.parametrize("spread", [0.0, 0.02, 1.0, 3.0])
def test_wide_nuclei_of_the_longest_rows_held(ctx, dtype, cols, spread):
    # the largest sums that a CTA adds up in parts: 46000 and 92000 weights of up to one, and lists that no CTA has room for
    r = np.random.Generator(np.random.Philox(cols + int(100 * spread)))
    x = rounded(r.standard_normal((3, cols)) * spread, dtype)
    x[1, r.random(cols) < 0.5] = -np.inf
    u = r.random(3).astype(np.float32)
    for p in (0.3, 0.9, 0.9999, 0.99999):
        run(ctx, x, u, dtype, top_p=np.full(3, p, np.float32), min_p=np.array([0, 0, 0.05], np.float32))
    run(ctx, x, u, dtype, top_p=np.full(3, 0.9, np.float32), top_k=np.array([cols // 2, cols // 3, 5000], np.uint32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(64, 1), (64, 50), (64, 3000), (24, 40000), (2, 750_001)])
def test_min_p_of_one_keeps_the_largest(ctx, dtype, rows, cols):
    # at any temperature, with every other filter: the largest logit, and those equal to it, are all that is left
    r = np.random.Generator(np.random.Philox(rows + cols))
    x = rounded(r.standard_normal((rows, cols)) * 3 + 4 * r.standard_normal((rows, 1)), dtype)
    x[::5, cols // 2] = x[::5].max(1)
    u = r.random(rows).astype(np.float32)
    given = {"temperature": (0.3 + 1.2 * r.random(rows)).astype(np.float32), "min_p": r.choice([1.0, 2.0, 0.99999994, np.inf], rows).astype(np.float32)}
    k, p = r.integers(1, 60, rows).astype(np.uint32), r.random(rows).astype(np.float32)
    for more in ({}, {"top_k": k}, {"top_p": p}, {"top_k": k, "top_p": p}):
        got = run(ctx, x, u, dtype, **given, **more)
        assert (x[np.arange(rows), got] == x.max(1)).all()


@pytest.mark.parametrize("dtype,cols,spread,temperature", [("bf16", 700_001, 0.02, 1.0), ("f32", 1_048_576, 0.02, 1.0), ("f16", 1_048_576, 0.1, 1.0), ("bf16", 1_500_000, 0.02, 1.0),
                                                           ("f32", 2_097_152, 0.0, 1.0), ("bf16", 2_097_152, 0.02, 0.7), ("f32", 600_001, 1.0, 30.0)])
def test_nuclei_of_the_longest_flat_rows(ctx, dtype, cols, spread, temperature):
    # more columns near one weight than 32 bits count in parts of 2^-13
    r = np.random.Generator(np.random.Philox(cols))
    x = rounded(r.standard_normal((4, cols)) * spread, dtype)
    x[3, r.permutation(cols)[:cols // 3]] = -1e9 if dtype != "f16" else -6e4          # masks that are numbers
    u, t = r.random(4).astype(np.float32), np.full(4, temperature, np.float32)
    run(ctx, x, u, dtype, temperature=t, top_p=np.array([0.1, 0.3, 0.6, 0.6], np.float32))
    run(ctx, x, u, dtype, temperature=t, top_p=np.array([0.9, 0.5, 0.99, 0.3], np.float32), min_p=np.array([0, 0, 0.5, 1], np.float32))


def test_long_and_short_rows_at_once():
    # two host threads, a context each: neither's shared memory is limited by the other's call
    import threading

    from ferrograd_b200 import GpuContext
    sizes, calls, failed = (300_001, 40_000), 1500, []
    contexts = [GpuContext(0) for _ in sizes]
    r = np.random.Generator(np.random.Philox(8))
    x = [r.standard_normal((1, cols)).astype(np.float32) for cols in sizes]
    u = np.array([0.37], np.float32)
    given = [(Placed(c, a), Placed(c, u), empty(c, (1,), "u32")) for c, a in zip(contexts, x)]

    def work(c, logits, u, token, cols):
        try:
            for _ in range(calls):
                c._check(c.lib.fg_sample(c.handle, 0, 1, cols, logits.ptr, u.ptr, None, None, None, None, token.ptr, None))
        except Exception as e:   # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(c, *g, cols)) for c, g, cols in zip(contexts, given, sizes)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for c, (_, _, token), a in zip(contexts, given, x):
        assert token.get()[0] == definition(a[0], u[0])[0]
        assert c.device_status() == 0
        c.destroy()


def test_long_and_short_rows_in_one_plan(ctx):
    r = np.random.Generator(np.random.Philox(9))
    x = [r.standard_normal((2, cols)).astype(np.float32) for cols in (300_001, 40_000, 100)]
    u = r.random(2).astype(np.float32)
    given = [(Placed(ctx, a), Placed(ctx, u), empty(ctx, (2,), "u32")) for a in x]
    ctx.plan_begin()
    for (logits, ud, token), a in zip(given, x):
        ctx.sample(logits, ud, token, *a.shape)
    plan = ctx.plan_end()
    ctx.sample(*given[1], *x[1].shape)
    plan.launch()
    for (_, _, token), a in zip(given, x):
        assert np.array_equal(token.get(), [definition(a[i], u[i])[0] for i in range(2)])
    plan.destroy()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [40, 2500, 17074, 46571, 300_000])
def test_equal_logits_far_from_zero(ctx, dtype, cols):
    # equal weights that are not quite 2^42, and whose sums 53 bits do not hold: borders at u and top_p times the total are hit exactly all the same
    r = np.random.Generator(np.random.Philox(cols))
    n = 24 if cols < 100_000 else 6
    x = np.repeat(rounded(r.choice([-1.0, 1.0], (n, 1)) * (300 + 3000 * r.random((n, 1))), dtype), cols, 1)
    given = {"temperature": (0.05 + r.random(n)).astype(np.float32)}
    u = r.choice(np.array([0.5, 0.25, 0.75, 0.125, 0.99999994, 2.0 ** -30], np.float32), n)
    p = r.choice(np.array([0.5, 0.25, 0.75, 0.375], np.float32), n)
    run(ctx, x, u, dtype, **given)
    run(ctx, x, u, dtype, **given, top_p=p)
    run(ctx, x, u, dtype, **given, top_p=p, min_p=np.full(n, 1, np.float32), top_k=np.full(n, max(1, cols // 2), np.uint32))
