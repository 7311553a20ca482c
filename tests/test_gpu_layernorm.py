"""Layer norm, forward and backward, against 64-bit formulas: the three storage types, rows that start at any element, one row to many,
one column to rows that no block holds.

Bounds.  A thread adds at most cols / 32 values in a chain (a warp per row is the fewest threads) and 32 more join them: a sum of n terms
is off by (cols / 32 + 32) u of the sum of their sizes, u = 2^-24.  Along a column no chain is longer than rows / 16 + 64.  Every further
operation adds u, the result half a step of its type."""
import numpy as np
import pytest

from token_ops import HALF_ULP, TINY, U, Placed, check, empty, rounded

pytestmark = pytest.mark.gpu
TYPES = ("f32", "f16", "bf16")


@pytest.fixture(scope="module")
def ctx():
    from ferrograd_b200 import GpuContext
    c = GpuContext(0)
    yield c
    assert c.device_status() == 0
    c.destroy()


def make(rows, cols, dtype, offset=1.0):
    r = np.random.Generator(np.random.Philox(rows * 100003 + cols))
    x = r.standard_normal((rows, cols)) * (0.5 + 2 * r.random((rows, 1))) + offset * r.standard_normal((rows, 1))
    return [rounded(a, dtype) for a in (x, r.standard_normal((rows, cols)), 1 + 0.2 * r.standard_normal(cols), 0.3 * r.standard_normal(cols))]


def forward64(x, eps):
    x = x.astype(np.float64)
    mean = x.mean(1, keepdims=True)
    d = x - mean
    mean, d = mean + d.mean(1, keepdims=True), d - d.mean(1, keepdims=True)
    return mean[:, 0], 1 / np.sqrt((d * d).mean(1) + float(np.float32(eps)))


def check_forward(got_y, got_mean, got_rstd, x, gamma, beta, eps, dtype, what=""):
    mean, rstd = forward64(x, eps)
    h = (x - mean[:, None]) * rstd[:, None]
    y = h * gamma.astype(np.float64) + beta
    n = x.shape[1]
    chain = (n / 32 + 48) * U
    if got_mean is not None:
        d = np.abs(x - mean[:, None]).mean(1)
        check(got_mean, mean, 2 * U * np.abs(mean) + chain * d, what + "mean")
        check(got_rstd, rstd, chain * rstd, what + "rstd")
    check(got_y, y, (1 + 4 * U) * (chain * (np.abs(h) + 1) * np.abs(gamma) + 2 * U * np.abs(y)) + HALF_ULP[dtype] * np.abs(y) * 1.001 + TINY[dtype], what + "y")


SHAPES = [(1, 1), (3, 2), (5, 7), (1, 33), (37, 100), (9, 256), (33, 257), (16, 768), (7, 1001), (300, 1024), (5, 2047), (20, 4096), (3, 4100),
          (2, 8192), (3, 8200), (2, 16384), (2, 20001), (1, 32768), (2, 33000), (1, 70001), (700, 65)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_forward_and_backward(ctx, dtype, rows, cols, shift):
    x, dy, gamma, beta = make(rows, cols, dtype)
    put = lambda a, s=shift: Placed(ctx, a, dtype, s)   # noqa: E731
    xd, dyd, gd, bd = put(x), put(dy), put(gamma, 2 * shift), put(beta, shift)
    y, mean, rstd = empty(ctx, x.shape, dtype, shift), empty(ctx, (rows,), "f32", shift), empty(ctx, (rows,))
    eps = 1e-5
    ctx.layernorm_fwd(xd, gd, bd, y, rows, cols, eps=eps, mean=mean, rstd=rstd, dtype=dtype)
    check_forward(y.get(), mean.get(), rstd.get(), x, gamma, beta, eps, dtype)
    run_backward(ctx, dtype, x, dy, gamma, mean.get(), rstd.get(), xd, dyd, gd, mean, rstd, shift)


def backward64(x, dy, gamma, mean, rstd):
    m, s = mean.astype(np.float64)[:, None], rstd.astype(np.float64)[:, None]
    h, g = (x - m) * s, dy.astype(np.float64) * gamma
    dx = s * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True))
    return dx, (dy * h).sum(0), dy.astype(np.float64).sum(0), h, g, s


def bounds(x, dy, gamma, mean, rstd, dtype):
    rows, cols = x.shape
    dx, dgamma, dbeta, h, g, s = backward64(x, dy, gamma, mean, rstd)
    chain, column = (cols / 32 + 48) * U, (rows / 16 + 80) * U
    half = HALF_ULP[dtype] * 1.001
    return (chain * s * (np.abs(g) + np.abs(g).mean(1, keepdims=True) + np.abs(h) * np.abs(g * h).mean(1, keepdims=True)) + half * np.abs(dx) + TINY[dtype],
            column * np.abs(dy * h).sum(0) + half * np.abs(dgamma) + TINY[dtype], column * np.abs(dy).sum(0) + half * np.abs(dbeta) + TINY[dtype])


def run_backward(ctx, dtype, x, dy, gamma, mean, rstd, xd, dyd, gd, meand, rstdd, shift, **kw):
    rows, cols = x.shape
    want, bound = backward64(x, dy, gamma, mean, rstd)[:3], bounds(x, dy, gamma, mean, rstd, dtype)
    outs = [empty(ctx, x.shape, dtype, shift), empty(ctx, (cols,), dtype, shift), empty(ctx, (cols,), dtype, 0)]
    ctx.layernorm_bwd(xd, dyd, gd, meand, rstdd, rows, cols, dx=outs[0], dgamma=outs[1], dbeta=outs[2], dtype=dtype)
    for o, w, b, name in zip(outs, want, bound, ("dx", "dgamma", "dbeta")):
        check(o.get(), w, b, name)
    return outs


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,shift", [(40, 64, 0), (40, 63, 1), (70, 1024, 0), (3, 9000, 0), (5, 40001, 0), (700, 320, 0)])
def test_parts_of_the_backward_pass(ctx, dtype, rows, cols, shift):
    # each output alone, accumulated, in place; no gamma
    x, dy, gamma, beta = make(rows, cols, dtype)
    mean, rstd = (v.astype(np.float32) for v in forward64(x, 1e-5))
    xd, dyd, gd, md, rd = Placed(ctx, x, dtype, shift), Placed(ctx, dy, dtype, shift), Placed(ctx, gamma, dtype, shift), Placed(ctx, mean), Placed(ctx, rstd)
    want, bound = backward64(x, dy, gamma, mean, rstd)[:3], bounds(x, dy, gamma, mean, rstd, dtype)
    names, shapes = ("dx", "dgamma", "dbeta"), (x.shape, (cols,), (cols,))
    for i, name in enumerate(names):
        o = empty(ctx, shapes[i], dtype, shift)
        ctx.layernorm_bwd(xd, dyd, gd, md, rd, rows, cols, dtype=dtype, **{name: o})
        check(o.get(), want[i], bound[i], name + " alone")
    base = [rounded(np.full(s, 0.75), dtype) for s in shapes]
    for adx, apar in ((1, 0), (0, 1), (1, 1)):
        outs = [Placed(ctx, b, dtype, shift) for b in base]
        ctx.layernorm_bwd(xd, dyd, gd, md, rd, rows, cols, dx=outs[0], dgamma=outs[1], dbeta=outs[2], accumulate_dx=adx, accumulate_params=apar, dtype=dtype)
        for o, w, b, add, name in zip(outs, want, bound, (adx, apar, apar), names):
            check(o.get(), w + 0.75 * add, b + 2 * HALF_ULP[dtype] * (0.75 + np.abs(w)) * add, f"{name} accumulated {adx} {apar}")
    for over in ("x", "dy"):
        a, b = Placed(ctx, x, dtype, shift), Placed(ctx, dy, dtype, shift)
        dg = empty(ctx, (cols,), dtype)
        ctx.layernorm_bwd(a, b, gd, md, rd, rows, cols, dx=a if over == "x" else b, dgamma=dg, dtype=dtype)
        check((a if over == "x" else b).get(), want[0], bound[0], "dx in place of " + over)
        check(dg.get(), want[1], bound[1], "dgamma beside dx in place of " + over)
    ones = np.ones(cols, np.float32)
    o = empty(ctx, x.shape, dtype, shift)
    ctx.layernorm_bwd(xd, dyd, None, md, rd, rows, cols, dx=o, dtype=dtype)
    check(o.get(), backward64(x, dy, ones, mean, rstd)[0], bounds(x, dy, ones, mean, rstd, dtype)[0], "dx without gamma")
    for g, b in ((None, None), (gamma, None), (None, beta)):
        y = empty(ctx, x.shape, dtype, shift)
        ctx.layernorm_fwd(xd, gd if g is not None else None, Placed(ctx, beta, dtype, shift) if b is not None else None, y, rows, cols, dtype=dtype)
        check_forward(y.get(), None, None, x, ones if g is None else g, 0 * ones if b is None else b, 1e-5, dtype)
    y = Placed(ctx, x, dtype, shift)
    ctx.layernorm_fwd(y, gd, None, y, rows, cols, dtype=dtype)
    check_forward(y.get(), None, None, x, gamma, 0 * ones, 1e-5, dtype, "in place: ")


def test_many_rows(ctx):
    # more rows than blocks, an odd number: every row, and sums over all of them
    for dtype, rows, cols in (("bf16", 5003, 512), ("f32", 20011, 40), ("f16", 1031, 3000), ("f32", 1500, 1001), ("f32", 70001, 3)):
        x, dy, gamma, beta = make(rows, cols, dtype)
        xd, dyd, gd, bd = (Placed(ctx, a, dtype) for a in (x, dy, gamma, beta))
        y, mean, rstd = empty(ctx, x.shape, dtype), empty(ctx, (rows,)), empty(ctx, (rows,))
        ctx.layernorm_fwd(xd, gd, bd, y, rows, cols, mean=mean, rstd=rstd, dtype=dtype)
        check_forward(y.get(), mean.get(), rstd.get(), x, gamma, beta, 1e-5, dtype)
        outs = run_backward(ctx, dtype, x, dy, gamma, mean.get(), rstd.get(), xd, dyd, gd, mean, rstd, 0)
        again = [empty(ctx, o.shape, dtype) for o in outs]
        ctx.layernorm_bwd(xd, dyd, gd, mean, rstd, rows, cols, dx=again[0], dgamma=again[1], dbeta=again[2], dtype=dtype)
        for o, b in zip(outs, again):
            assert np.array_equal(o.bits(), b.bits()), "the same call gives the same bits"


@pytest.mark.parametrize("cols", [8, 100, 4096, 10000, 40000])
def test_rows_far_from_zero(ctx, cols):
    # a mean 1e4 times the deviation: what rounding leaves of the mean is put right
    x, _, gamma, beta = make(6, cols, "f32", offset=0.0)
    x = (x + 10000).astype(np.float32)
    y, mean, rstd = empty(ctx, x.shape), empty(ctx, (6,)), empty(ctx, (6,))
    ctx.layernorm_fwd(Placed(ctx, x), Placed(ctx, gamma), Placed(ctx, beta), y, 6, cols, mean=mean, rstd=rstd)
    check_forward(y.get(), mean.get(), rstd.get(), x, gamma, beta, 1e-5, "f32")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [5, 128, 1000, 6000, 50000])
def test_values_out_of_the_ordinary(ctx, dtype, cols):
    # a constant row has no deviation: y = beta, with 1 / sqrt(eps); infinities and NaN stay in their row
    x, dy, gamma, beta = make(5, cols, dtype)
    x[0], x[2, cols // 2], x[3, 0] = 3.0, np.inf, np.nan
    y, mean, rstd = empty(ctx, x.shape, dtype), empty(ctx, (5,)), empty(ctx, (5,))
    args = Placed(ctx, x, dtype), Placed(ctx, gamma, dtype), Placed(ctx, beta, dtype)
    ctx.layernorm_fwd(*args, y, 5, cols, mean=mean, rstd=rstd, dtype=dtype)
    g = y.get()
    assert np.array_equal(g[0], beta) and mean.get()[0] == 3.0
    check(rstd.get()[:1], [1 / np.sqrt(np.float64(np.float32(1e-5)))], 4 * U * 320, "rstd of a constant row")
    assert np.isnan(g[2]).all() and np.isnan(g[3]).all()
    ok = [1, 4]
    check_forward(g[ok], mean.get()[ok], rstd.get()[ok], x[ok], gamma, beta, 1e-5, dtype)
    dx = empty(ctx, x.shape, dtype)
    ctx.layernorm_bwd(args[0], Placed(ctx, dy, dtype), args[1], mean, rstd, 5, cols, dx=dx, dtype=dtype)
    want, bound = backward64(x[ok], dy[ok], gamma, mean.get()[ok], rstd.get()[ok])[0], bounds(x[ok], dy[ok], gamma, mean.get()[ok], rstd.get()[ok], dtype)[0]
    assert np.isnan(dx.get()[3]).all()
    check(dx.get()[ok], want, bound, "dx beside rows that are not numbers")


def test_gradient_against_differences(ctx):
    # L = sum(w * y) at x + t e and x - t e, the forward pass alone
    rows, cols, t = 3, 40, 2.0 ** -6
    x, w, gamma, beta = make(rows, cols, "f32")

    def loss(x, gamma, beta):
        y = empty(ctx, x.shape)
        ctx.layernorm_fwd(Placed(ctx, x), Placed(ctx, gamma), Placed(ctx, beta), y, rows, cols)
        return (y.get().astype(np.float64) * w).sum()

    y, mean, rstd = empty(ctx, x.shape), empty(ctx, (rows,)), empty(ctx, (rows,))
    ctx.layernorm_fwd(Placed(ctx, x), Placed(ctx, gamma), Placed(ctx, beta), y, rows, cols, mean=mean, rstd=rstd)
    dx, dg, db = empty(ctx, x.shape), empty(ctx, (cols,)), empty(ctx, (cols,))
    ctx.layernorm_bwd(Placed(ctx, x), Placed(ctx, w), Placed(ctx, gamma), mean, rstd, rows, cols, dx=dx, dgamma=dg, dbeta=db)
    for i, (a, g) in enumerate(((x, dx), (gamma, dg), (beta, db))):
        for at in range(0, a.size, 17):
            args = [x.copy(), gamma.copy(), beta.copy()]
            args[i].ravel()[at] += t
            up = loss(*args)
            args[i].ravel()[at] -= 2 * t
            # f32 results: 120 of them off by 2^-23 at most, over 2 t = 2^-5; the third derivative times t^2 / 6
            assert abs((up - loss(*args)) / (2 * t) - g.get().ravel()[at]) < 120 * 2.0 ** -21 * 2.0 ** 5 + 20 * t * t


def test_empty_and_captured(ctx):
    rows, cols = 600, 640
    x, dy, gamma, beta = make(rows, cols, "f32")
    xd, dyd, gd, bd = (Placed(ctx, a) for a in (x, dy, gamma, beta))
    y, mean, rstd = empty(ctx, x.shape), empty(ctx, (rows,)), empty(ctx, (rows,))
    dg, db = empty(ctx, (cols,)), Placed(ctx, np.ones(cols))
    ctx.layernorm_fwd(xd, gd, bd, y, 0, cols)
    ctx.layernorm_bwd(xd, dyd, gd, mean, rstd, 0, cols, dgamma=dg)
    ctx.layernorm_bwd(xd, dyd, gd, mean, rstd, 0, cols, dbeta=db, accumulate_params=True)
    assert np.isnan(y.get()).all() and (dg.get() == 0).all() and (db.get() == 1).all()
    dx = empty(ctx, x.shape)
    ctx.layernorm_bwd(xd, dyd, gd, mean, rstd, rows, cols, dx=dx, dgamma=dg, dbeta=db)      # the arena is there before the recording
    ctx.plan_begin()
    ctx.layernorm_fwd(xd, gd, bd, y, rows, cols, mean=mean, rstd=rstd)
    ctx.layernorm_bwd(xd, dyd, gd, mean, rstd, rows, cols, dx=dx, dgamma=dg, dbeta=db)
    plan = ctx.plan_end()
    for k in range(3):
        ctx.upload(xd.t.data, np.concatenate([(x + k).ravel().view(np.uint32), np.full(37, xd.fill, np.uint32)]))
        plan.launch()
        check_forward(y.get(), mean.get(), rstd.get(), x + np.float32(k), gamma, beta, 1e-5, "f32")
        want, bound = backward64(x + np.float32(k), dy, gamma, mean.get(), rstd.get())[:3], bounds(x + np.float32(k), dy, gamma, mean.get(), rstd.get(), "f32")
        for o, w, b, name in zip((dx, dg, db), want, bound, ("dx", "dgamma", "dbeta")):
            check(o.get(), w, b, f"replay {k}: {name}")
    plan.destroy()


def test_refusals(ctx):
    from ferrograd_b200 import FgError
    t = ctx.new_tensor((64,))
    p = t.ptr

    def refuse(f):
        with pytest.raises(FgError) as e:
            f()
        assert e.value.kind == "FG_ERR_INVALID_ARGUMENT"

    for kw in (dict(x=None), dict(y=None), dict(cols=0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(x=p + 2), dict(y=p + 1),
               dict(mean=p + 2), dict(rows=1 << 31, cols=1 << 31), dict(y=p + 4), dict(gamma=p + 1), dict(gamma=p + 140), dict(beta=p + 120)):
        a = dict(x=p, gamma=None, beta=None, y=p + 128, rows=2, cols=4, eps=1e-5, mean=None) | kw
        refuse(lambda: ctx.layernorm_fwd(**a))
    for kw in (dict(x=None), dict(dy=None), dict(mean=None), dict(rstd=None), dict(cols=0), dict(dx=p + 4), dict(dx=p, accumulate_dx=True), dict(dx=p + 36),
               dict(dgamma=p + 1), dict(rows=1 << 31, cols=1 << 31), dict(dx=None), dict(dgamma=p + 8), dict(dbeta=p + 40), dict(dgamma=p + 156), dict(gamma=p + 132),
               dict(dgamma=p + 192, dbeta=p + 204), dict(gamma=p + 192, dgamma=p + 192)):
        a = dict(x=p, dy=p + 32, gamma=None, mean=p + 64, rstd=p + 80, rows=2, cols=4, dx=p + 128) | kw
        refuse(lambda: ctx.layernorm_bwd(**a))
    with pytest.raises(KeyError):
        ctx.layernorm_fwd(p, None, None, p, 1, 4, dtype="f64")
    assert ctx.lib.fg_layernorm_fwd(ctx.handle, 3, 1, 4, p, None, None, 1e-5, p, None, None) == 1
    assert ctx.lib.fg_layernorm_bwd(ctx.handle, -1, 1, 4, p, p, None, p, p, p, None, None, 0, 0) == 1


def test_statistics_that_overlap_are_refused(ctx):
    from ferrograd_b200 import FgError
    p = ctx.new_tensor((64,)).ptr      # x: 32 bytes at 0, y or dx at 128, lines of 16 bytes
    forward = dict(x=p, gamma=p + 64, beta=p + 80, y=p + 128, rows=2, cols=4, mean=p + 192, rstd=p + 200)
    for kw in (dict(mean=p + 28), dict(mean=p + 124), dict(rstd=p + 156), dict(mean=p + 76), dict(rstd=p + 92), dict(rstd=p + 196), dict(mean=p + 200)):
        with pytest.raises(FgError) as e:
            ctx.layernorm_fwd(**(forward | kw))
        assert e.value.kind == "FG_ERR_INVALID_ARGUMENT"
    ctx.layernorm_fwd(**forward)
    backward = dict(x=p, dy=p + 32, gamma=None, mean=p + 192, rstd=p + 200, rows=2, cols=4, dx=p + 128, dgamma=p + 160, dbeta=p + 176)
    for kw in (dict(mean=p + 156), dict(rstd=p + 124), dict(mean=p + 172), dict(rstd=p + 188)):
        with pytest.raises(FgError) as e:
            ctx.layernorm_bwd(**(backward | kw))
        assert e.value.kind == "FG_ERR_INVALID_ARGUMENT"
    ctx.layernorm_bwd(**backward)


# Rows whose starts lie at 8, 4, 2 places of a 16-byte word, more of them than are worked on at a time, and a word or an element over a border.
RAGGED = [("f16", 6001, 129), ("bf16", 5003, 257), ("f16", 2501, 1001), ("bf16", 3001, 1002), ("f16", 3000, 1004), ("bf16", 1203, 4097), ("f16", 700, 8191),
          ("f32", 5003, 257), ("f32", 2600, 777), ("f32", 1300, 1002), ("f32", 701, 4099), ("bf16", 4001, 5), ("f32", 3001, 1), ("bf16", 650, 9001),
          ("f32", 310, 12001), ("f16", 310, 16001), ("f32", 300, 8194)]


@pytest.mark.parametrize("dtype,rows,cols", RAGGED)
def test_many_ragged_rows(ctx, dtype, rows, cols):
    x, dy, gamma, beta = make(rows, cols, dtype)
    xd, dyd, gd, bd = Placed(ctx, x, dtype), Placed(ctx, dy, dtype), Placed(ctx, gamma, dtype, 1), Placed(ctx, beta, dtype, 3)
    y, mean, rstd = empty(ctx, x.shape, dtype), empty(ctx, (rows,)), empty(ctx, (rows,))
    ctx.layernorm_fwd(xd, gd, bd, y, rows, cols, mean=mean, rstd=rstd, dtype=dtype)
    check_forward(y.get(), mean.get(), rstd.get(), x, gamma, beta, 1e-5, dtype)
    outs = run_backward(ctx, dtype, x, dy, gamma, mean.get(), rstd.get(), xd, dyd, gd, mean, rstd, 0)
    # in place: words at the ends of rows are read for one row while another's elements are written
    over = Placed(ctx, x, dtype)
    ctx.layernorm_fwd(over, gd, bd, over, rows, cols, dtype=dtype)
    assert np.array_equal(over.bits(), y.bits())
    for place in range(2):
        a = [Placed(ctx, x, dtype), Placed(ctx, dy, dtype)]
        dg, db = empty(ctx, (cols,), dtype), empty(ctx, (cols,), dtype, 1)
        ctx.layernorm_bwd(*a, gd, mean, rstd, rows, cols, dx=a[place], dgamma=dg, dbeta=db, dtype=dtype)
        for got, want in zip((a[place], dg, db), outs):
            assert np.array_equal(got.bits(), want.bits())
    # dx alone, and added to
    base = rounded(np.full(x.shape, 0.75), dtype)
    alone, added = empty(ctx, x.shape, dtype), Placed(ctx, base, dtype)
    ctx.layernorm_bwd(xd, dyd, gd, mean, rstd, rows, cols, dx=alone, dtype=dtype)
    ctx.layernorm_bwd(xd, dyd, gd, mean, rstd, rows, cols, dx=added, accumulate_dx=True, dtype=dtype)
    want, bound = backward64(x, dy, gamma, mean.get(), rstd.get())[0], bounds(x, dy, gamma, mean.get(), rstd.get(), dtype)[0]
    check(alone.get(), want, bound, "dx alone")
    check(added.get(), want + 0.75, bound + 2 * HALF_ULP[dtype] * (0.75 + np.abs(want)), "dx added")


@pytest.mark.parametrize("dtype,rows,cols", [("f16", 2500, 1001), ("bf16", 3001, 257), ("f32", 1300, 777), ("bf16", 640, 4097), ("f32", 900, 3), ("f16", 40, 9)])
def test_ragged_rows_beside_values_out_of_the_ordinary(ctx, dtype, rows, cols):
    # every third row is inf or NaN: the others come out as if it were not
    x, dy, gamma, beta = make(rows, cols, dtype)
    gd, bd = Placed(ctx, gamma, dtype), Placed(ctx, beta, dtype)

    def run(x, dy):
        xd, dyd = Placed(ctx, x, dtype), Placed(ctx, dy, dtype)
        y, dx, mean, rstd = empty(ctx, x.shape, dtype), empty(ctx, x.shape, dtype), empty(ctx, (rows,)), empty(ctx, (rows,))
        ctx.layernorm_fwd(xd, gd, bd, y, rows, cols, mean=mean, rstd=rstd, dtype=dtype)
        ctx.layernorm_bwd(xd, dyd, gd, mean, rstd, rows, cols, dx=dx, dtype=dtype)
        return [t.bits().copy() for t in (y, dx, mean, rstd)]

    plain = run(x, dy)
    bad, bad_dy = x.copy(), dy.copy()
    bad[0::3], bad_dy[0::3] = np.where(np.arange(len(bad[0::3]))[:, None] % 2, np.inf, np.nan), np.nan
    for a, b in zip(plain, run(bad, bad_dy)):
        assert np.array_equal(a[1::3], b[1::3]) and np.array_equal(a[2::3], b[2::3])


def test_gradients_of_the_most_columns():
    # one row of 2^32 - 1 columns: the grids over its columns are no 32-bit sums
    from ferrograd_b200 import GpuContext
    ctx, cols = GpuContext(0), (1 << 32) - 1
    x, dgamma = (ctx.new_tensor((cols,), np.uint16) for _ in range(2))
    r, at = np.random.Generator(np.random.Philox(6)), (0, cols // 3, cols - 300)
    parts = [r.integers(-8, 9, 300).astype(np.float16) for _ in at]
    got = np.empty(300, np.float16)
    ctx.memset_zero(x, 2 * cols)
    for i, part in zip(at, parts):
        ctx.upload(x.data, part, dst_off=2 * i)
        ctx.upload(dgamma.data, np.full(300, np.nan, np.float16), dst_off=2 * i)
    ctx.layernorm_bwd(x, x, None, Placed(ctx, [0.5]), Placed(ctx, [2.0]), 1, cols, dgamma=dgamma, dtype="f16")
    for i, part in zip(at, parts):
        ctx.download(dgamma.data, got, src_off=2 * i)
        assert np.array_equal(got, part * (part - np.float16(0.5)) * 2)          # whole numbers: exact
    assert ctx.device_status() == 0
    for t in (x, dgamma):
        t.data.free()
    ctx.destroy()


def test_a_refused_workspace_leaves_the_next_call_alone():
    from ferrograd_b200 import FgError, GpuContext
    ctx = GpuContext(0)
    x, y = Placed(ctx, [[1.0, 3.0]]), empty(ctx, (1, 2))
    for refused in (lambda: ctx.alloc(1 << 46), lambda: ctx.reserve_workspace(1 << 46)):          # 64 TB
        with pytest.raises(FgError) as e:
            refused()
        assert e.value.kind == "FG_ERR_OUT_OF_MEMORY"
        ctx.layernorm_fwd(x, None, None, y, 1, 2, eps=0.0)
        assert np.array_equal(y.get(), [[-1.0, 1.0]])
    ctx.destroy()
