"""Root-mean-square norm against the formulas in 64 bits.

Bounds, with U = 2^-24, h the half step of the storage type and d = cols / 32 + 32 (the longest chain of additions in a row's sum: a warp
at least shares it):
  sum    x + residual in f32, rounded: equal
  rstd   (d / 2 + 4) U
  y      (d / 2 + 8) U |y| + h |y|
  e4m3   scale (d / 2 + 8) U; a value 2^-4 of it, or half of the smallest step 2^-9, and the error of y / scale
  dx     rstd (8 U |g| + |n| (d + 8) U mean |g n|) + 2 U |dx|, and h |dx|
  dgamma (rows + 8) U sum |dy n|, and h
"""
import numpy as np
import pytest

from token_ops import check, empty, HALF_ULP, Placed, rounded, TINY, U

pytestmark = pytest.mark.gpu
EPS = 1e-5
TYPES = ["f32", "f16", "bf16"]


@pytest.fixture()
def ctx():
    from ferrograd_b200 import GpuContext
    c = GpuContext(0)
    yield c
    assert c.device_status() == 0
    c.destroy()


def rng(*key):
    return np.random.Generator(np.random.Philox(key))


def chain(cols):
    return cols / 32 + 32


def matrix(r, rows, cols, dtype, size=1.0):
    return rounded(size * r.standard_normal((rows, cols)) * (0.5 + r.random((rows, 1))), dtype)


def forward64(h, gamma):
    h = h.astype(np.float64)
    rstd = 1 / np.sqrt((h * h).mean(1) + EPS)
    return h * rstd[:, None] * (1.0 if gamma is None else gamma.astype(np.float64)), rstd


def total(x, residual, dtype):
    return x if residual is None else rounded(x.astype(np.float32) + residual.astype(np.float32), dtype)


ROWS = [(1, 4096), (3, 1), (2, 7), (5, 33), (300, 256), (64, 1001), (700, 777), (17, 8192), (9, 8200), (4, 20000), (2, 70001), (1500, 96), (33, 5001), (600, 2048)]


@pytest.mark.parametrize("rows,cols", ROWS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_forward(ctx, rows, cols, dtype, shift):
    r = rng(rows, cols)
    x, res = matrix(r, rows, cols, dtype), matrix(r, rows, cols, dtype)
    gamma = rounded(1 + 0.1 * r.standard_normal(cols), dtype)
    dx, dres, dg = Placed(ctx, x, dtype, shift), Placed(ctx, res, dtype, shift), Placed(ctx, gamma, dtype, 0 if shift else 0)
    for with_res, with_gamma in ((True, True), (False, True), (True, False)):
        y, s, rstd = empty(ctx, (rows, cols), dtype, shift), empty(ctx, (rows, cols), dtype, shift), empty(ctx, (rows,))
        ctx.rmsnorm_fwd(dx, dg if with_gamma else None, y, rows, cols, eps=EPS, residual=dres if with_res else None, sum=s if with_res else None, rstd=rstd, dtype=dtype)
        h = total(x, res if with_res else None, dtype)
        if with_res:
            assert np.array_equal(s.get(), h)
        want, want_rstd = forward64(h, gamma if with_gamma else None)
        check(rstd.get(), want_rstd, (chain(cols) / 2 + 4) * U * want_rstd, "rstd")
        check(y.get(), want, ((chain(cols) / 2 + 8) * U + HALF_ULP[dtype]) * np.abs(want) + TINY[dtype], "y")
    y = empty(ctx, (rows, cols), dtype, shift)      # without what may be left out
    ctx.rmsnorm_fwd(dx, dg, y, rows, cols, eps=EPS, residual=dres, dtype=dtype)
    want, _ = forward64(total(x, res, dtype), gamma)
    check(y.get(), want, ((chain(cols) / 2 + 8) * U + HALF_ULP[dtype]) * np.abs(want) + TINY[dtype], "y")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(40, 512), (7, 1001), (3, 30000)])
def test_in_place(ctx, dtype, rows, cols):
    r = rng(rows, cols, 1)
    x, res = matrix(r, rows, cols, dtype), matrix(r, rows, cols, dtype)
    gamma = rounded(1 + 0.1 * r.standard_normal(cols), dtype)
    g = Placed(ctx, gamma, dtype)
    h = total(x, res, dtype)
    want, _ = forward64(h, gamma)
    bound = ((chain(cols) / 2 + 8) * U + HALF_ULP[dtype]) * np.abs(want) + TINY[dtype]
    a, b = Placed(ctx, x, dtype), Placed(ctx, res, dtype)
    ctx.rmsnorm_fwd(a, g, a, rows, cols, eps=EPS, residual=b, sum=b, dtype=dtype)      # y in x, the sum in the residual
    assert np.array_equal(b.get(), h)
    check(a.get(), want, bound, "y")
    a, b = Placed(ctx, x, dtype), Placed(ctx, res, dtype)
    ctx.rmsnorm_fwd(a, g, b, rows, cols, eps=EPS, residual=b, sum=a, dtype=dtype)      # the other way round
    assert np.array_equal(a.get(), h)
    check(b.get(), want, bound, "y")


def e4m3_values():
    v = np.zeros(256)
    for b in range(256):
        s, e, m = b >> 7, b >> 3 & 15, b & 7
        v[b] = np.nan if e == 15 and m == 7 else (-1) ** s * (m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return v


class Bytes:
    """A byte tensor on the device with a pattern before and behind it."""

    def __init__(self, ctx, n, shift):
        self.ctx, self.n, self.shift = ctx, n, shift
        self.t = ctx.new_tensor((shift + n + 37,), np.uint8)
        ctx.upload(self.t.data, np.full(shift + n + 37, 0xa5, np.uint8))
        self.ptr = self.t.ptr + shift

    def get(self):
        b = self.ctx.to_numpy(self.t)
        assert (b[:self.shift] == 0xa5).all() and (b[self.shift + self.n:] == 0xa5).all(), "written outside the tensor"
        return b[self.shift:self.shift + self.n]


@pytest.mark.parametrize("rows,cols", [(1, 4096), (3, 1), (2, 31), (300, 256), (64, 1001), (33, 777), (17, 8192), (5, 16384), (4, 20000), (300, 4096), (70, 129), (2, 70001)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [0, 32, 64, 128, 256])
def test_e4m3(ctx, rows, cols, dtype, group):
    r = rng(rows, cols, 2, group)
    x, res = matrix(r, rows, cols, dtype), matrix(r, rows, cols, dtype)
    if rows > 2:
        x[1] = res[1] = 0.0                     # a row of zeros
        x[2, :cols // 2] = res[2, :cols // 2] = 0.0
    gamma = rounded(1 + 0.1 * r.standard_normal(cols), dtype)
    groups = -(-cols // group) if group else 1
    for shift in (0, 1):
        a, b, g = Placed(ctx, x, dtype, shift), Placed(ctx, res, dtype, shift), Placed(ctx, gamma, dtype, shift)
        q, scale, s, rstd = Bytes(ctx, rows * cols, shift), empty(ctx, (rows, groups)), empty(ctx, (rows, cols), dtype, shift), empty(ctx, (rows,))
        ctx.rmsnorm_fwd_e4m3(a, g, q, scale, rows, cols, group=group, eps=EPS, residual=b, sum=s, rstd=rstd, dtype=dtype)
        h = total(x, res, dtype)
        assert np.array_equal(s.get(), h)
        want, want_rstd = forward64(h, gamma)
        check(rstd.get(), want_rstd, (chain(cols) / 2 + 4) * U * want_rstd, "rstd")
        each = group or cols
        wide = np.zeros((rows, groups * each))
        wide[:, :cols] = want
        most = np.abs(wide.reshape(rows, groups, each)).max(2)
        check(scale.get(), most / 448, (chain(cols) / 2 + 8) * U * most / 448 + 2.0 ** -149, "scale")
        got = e4m3_values()[q.get()].reshape(rows, cols)
        by = np.repeat(most / 448, each, 1)[:, :cols]
        ref = np.where(by > 0, want / np.where(by > 0, by, 1.0), 0.0)
        check(got, ref, (2.0 ** -4 + (chain(cols) + 16) * U) * np.abs(ref) + 2.0 ** -10, "y")
    q2, scale2 = Bytes(ctx, rows * cols, 0), empty(ctx, (rows, groups))      # no residual, no gamma
    ctx.rmsnorm_fwd_e4m3(a, None, q2, scale2, rows, cols, group=group, eps=EPS, dtype=dtype)
    want, _ = forward64(x, None)
    wide[:, :cols] = want
    most = np.abs(wide.reshape(rows, groups, each)).max(2)
    check(scale2.get(), most / 448, (chain(cols) / 2 + 8) * U * most / 448 + 2.0 ** -149, "scale")


@pytest.mark.parametrize("dtype", TYPES)
def test_e4m3_extremes(ctx, dtype):
    # the largest of a group is 448 exactly, and numbers far below it become zero; tiny rows keep their values
    cols = 64
    x = np.zeros((3, cols), np.float32)
    x[0, :4] = 1.0, -1.0, 2.0 ** -10, 2.0 ** -20
    x[1, :2] = rounded([1e-30 if dtype != "f16" else 1e-7, 0.0], dtype)
    x[2] = 1.0
    a, q, scale = Placed(ctx, x, dtype), Bytes(ctx, 3 * cols, 0), empty(ctx, (3, 1))
    ctx.rmsnorm_fwd_e4m3(a, None, q, scale, 3, cols, eps=EPS, dtype=dtype)
    v = e4m3_values()[q.get()].reshape(3, cols)
    assert v[0, 0] == 448 and v[0, 1] == -448 and v[0, 2] == 0.4375 and v[0, 3] == 0
    assert v[1, 0] == 448 and (v[1, 1:] == 0).all() and (v[2] == 448).all()


def backward64(x, dy, gamma, rstd, dsum):
    x, dy, rstd = x.astype(np.float64), dy.astype(np.float64), rstd.astype(np.float64)[:, None]
    cols = x.shape[1]
    n = x * rstd
    g = dy * (1.0 if gamma is None else gamma.astype(np.float64))
    m = (g * n).mean(1, keepdims=True)
    dx = rstd * (g - n * m) + (0.0 if dsum is None else dsum.astype(np.float64))
    e = rstd * (8 * U * np.abs(g) + np.abs(n) * (chain(cols) + 8) * U * np.abs(g * n).mean(1, keepdims=True)) + 4 * U * np.abs(dx)
    return dx, e, (dy * n).sum(0), np.abs(dy * n).sum(0)


@pytest.mark.parametrize("rows,cols", ROWS + [(4099, 64), (2000, 1024), (1, 16384), (900, 12288), (513, 9999)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_backward(ctx, rows, cols, dtype, shift):
    r = rng(rows, cols, 3)
    x, dy, dsum = (matrix(r, rows, cols, dtype) for _ in range(3))
    gamma = rounded(1 + 0.1 * r.standard_normal(cols), dtype)
    rstd = forward64(x, None)[1].astype(np.float32)
    dev = [Placed(ctx, t, dtype, shift) for t in (x, dy, dsum, gamma)]
    drstd = Placed(ctx, rstd)
    half, tiny = HALF_ULP[dtype], TINY[dtype]
    for with_sum, with_gamma, params, add in ((True, True, True, False), (False, True, True, True), (True, False, False, False), (False, True, None, False)):
        start = rounded(r.standard_normal(cols), dtype)
        dx = empty(ctx, (rows, cols), dtype, shift) if params is not None else None
        dg = Placed(ctx, start, dtype, shift) if add else empty(ctx, (cols,), dtype, shift) if params is not False else None
        ctx.rmsnorm_bwd(dev[0], dev[1], dev[3] if with_gamma else None, drstd, rows, cols, dx=dx, dgamma=dg, dsum=dev[2] if with_sum else None,
                        accumulate_params=add, dtype=dtype)
        want, bound, want_g, size_g = backward64(x, dy, gamma if with_gamma else None, rstd, dsum if with_sum else None)
        if dx is not None:
            check(dx.get(), want, bound + half * np.abs(want) + tiny, "dx")
        if dg is not None:
            ref = want_g + (start if add else 0.0)
            check(dg.get(), ref, (rows + 8) * U * size_g + (half + 4 * U) * np.abs(ref) + tiny, "dgamma")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(200, 512), (33, 1001), (40, 20000)])
def test_backward_in_place(ctx, dtype, rows, cols):
    r = rng(rows, cols, 4)
    x, dy, dsum = (matrix(r, rows, cols, dtype) for _ in range(3))
    gamma = rounded(1 + 0.1 * r.standard_normal(cols), dtype)
    rstd = forward64(x, None)[1].astype(np.float32)
    want, bound, want_g, size_g = backward64(x, dy, gamma, rstd, dsum)
    for which in range(3):
        dev = [Placed(ctx, t, dtype) for t in (x, dy, dsum)]
        dg = empty(ctx, (cols,), dtype)
        ctx.rmsnorm_bwd(dev[0], dev[1], Placed(ctx, gamma, dtype), Placed(ctx, rstd), rows, cols, dx=dev[which], dgamma=dg, dsum=dev[2], dtype=dtype)
        check(dev[which].get(), want, bound + HALF_ULP[dtype] * np.abs(want) + TINY[dtype], "dx")
        check(dg.get(), want_g, (rows + 8) * U * size_g + (HALF_ULP[dtype] + 4 * U) * np.abs(want_g) + TINY[dtype], "dgamma")


def test_differences(ctx):
    # the gradient along a direction against the difference of the loss in 64 bits, through the sum
    rows, cols = 12, 300
    r = rng(5)
    x, dy, dsum = (matrix(r, rows, cols, "f32") for _ in range(3))
    gamma = rounded(1 + 0.1 * r.standard_normal(cols), "f32")
    loss = lambda h, g: (forward64(h, g)[0] * dy).sum() + (h * dsum).sum()   # noqa: E731
    dx, dg = empty(ctx, (rows, cols)), empty(ctx, (cols,))
    rstd = forward64(x, None)[1].astype(np.float32)
    ctx.rmsnorm_bwd(Placed(ctx, x), Placed(ctx, dy), Placed(ctx, gamma), Placed(ctx, rstd), rows, cols, dx=dx, dgamma=dg, dsum=Placed(ctx, dsum))
    for name, got, at in (("x", dx.get(), x), ("gamma", dg.get(), gamma)):
        step = r.standard_normal(at.shape)
        moved = [(x + s * step, gamma) if name == "x" else (x, gamma + s * step) for s in (1e-6, -1e-6)]
        slope = (loss(*moved[0]) - loss(*moved[1])) / 2e-6
        assert abs((got * step).sum() - slope) <= 2e-5 * (np.abs(got) * np.abs(step)).sum(), name


@pytest.mark.parametrize("dtype", TYPES)
def test_zeros_and_nan(ctx, dtype):
    cols = 500
    x = np.zeros((4, cols), np.float32)
    x[1] = 1.0
    x[2, 17] = np.nan
    x[3] = 2.0
    y, rstd = empty(ctx, (4, cols), dtype), empty(ctx, (4,))
    ctx.rmsnorm_fwd(Placed(ctx, x, dtype), None, y, 4, cols, eps=EPS, rstd=rstd, dtype=dtype)
    got = y.get()
    assert (got[0] == 0).all() and np.isnan(got[2]).all() and np.isnan(rstd.get()[2])
    check(got[[1, 3]], forward64(x[[1, 3]], None)[0], 2 * HALF_ULP[dtype], "y")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(2000, 1024), (100, 999)])
def test_same_bits_and_recorded(ctx, dtype, rows, cols):
    r = rng(rows, cols, 6)
    x, dy, dsum = (Placed(ctx, matrix(r, rows, cols, dtype), dtype) for _ in range(3))
    gamma = Placed(ctx, rounded(1 + 0.1 * r.standard_normal(cols), dtype), dtype)

    def outputs():
        return [empty(ctx, (rows, cols), dtype) for _ in range(3)] + [empty(ctx, (cols,), dtype), empty(ctx, (rows,)), Bytes(ctx, rows * cols, 0), empty(ctx, (rows, 1))]

    def step(o):
        ctx.rmsnorm_fwd(x, gamma, o[0], rows, cols, residual=dy, sum=o[1], rstd=o[4], dtype=dtype)
        ctx.rmsnorm_bwd(o[1], dy, gamma, o[4], rows, cols, dx=o[2], dgamma=o[3], dsum=dsum, dtype=dtype)
        ctx.rmsnorm_fwd_e4m3(x, gamma, o[5], o[6], rows, cols, residual=dy, dtype=dtype)

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
        assert np.array_equal(p.get() if isinstance(p, Bytes) else p.bits(), q.get() if isinstance(q, Bytes) else q.bits())
    plan.destroy()


def test_no_rows(ctx):
    g = Placed(ctx, np.ones(8))
    x = Placed(ctx, np.ones((1, 8)))
    ctx.rmsnorm_fwd(x, g, x, 0, 8)
    d = empty(ctx, (8,))
    ctx.rmsnorm_bwd(x, x, g, g, 0, 8, dgamma=d)
    assert (d.get() == 0).all()
    a = Placed(ctx, np.ones(8))
    ctx.rmsnorm_bwd(x, x, g, g, 0, 8, dgamma=a, accumulate_params=True)
    assert (a.get() == 1).all() and (x.get() == 1).all()


def test_refusals(ctx):
    from ferrograd_b200.backend import FgError
    rows, cols = 4, 64
    x, res, y, s, dy = (Placed(ctx, np.ones((rows, cols))) for _ in range(5))
    g, rstd, scale, dg = Placed(ctx, np.ones(cols)), Placed(ctx, np.ones(rows)), Placed(ctx, np.ones((rows, 2))), Placed(ctx, np.ones(cols))
    q = Bytes(ctx, rows * cols, 0)
    f = lambda x=x, g=g, y=y, rows=rows, cols=cols, **k: ctx.rmsnorm_fwd(x, g, y, rows, cols, **k)   # noqa: E731
    e = lambda y=q, scale=scale, group=32, **k: ctx.rmsnorm_fwd_e4m3(x, g, y, scale, rows, cols, group=group, **k)   # noqa: E731
    b = lambda x=x, dy=dy, g=g, rstd=rstd, cols=cols, dx=y, dgamma=dg, **k: ctx.rmsnorm_bwd(x, dy, g, rstd, rows, cols, dx=dx, dgamma=dgamma, **k)   # noqa: E731
    f(residual=res, sum=s, rstd=rstd)
    e()
    b()
    bad = [lambda: f(x=None), lambda: f(y=None), lambda: f(cols=0), lambda: f(eps=-1.0), lambda: f(eps=0.0), lambda: f(eps=1e-40), lambda: f(eps=float("nan")), lambda: f(eps=float("inf")),
           lambda: f(rows=1 << 20, cols=1 << 20), lambda: f(sum=s), lambda: f(y=x.ptr + 4), lambda: f(residual=res, y=res.ptr + 8), lambda: f(residual=res, sum=y),
           lambda: f(y=g), lambda: f(rstd=x), lambda: f(rstd=y.ptr), lambda: f(x=x.ptr + 2),
           lambda: e(group=48), lambda: e(group=1), lambda: e(group=512), lambda: e(scale=None), lambda: e(y=None), lambda: e(y=x), lambda: e(scale=x), lambda: e(scale=q),
           lambda: e(scale=scale.ptr + 2), lambda: e(rstd=scale),
           lambda: b(x=None), lambda: b(dy=None), lambda: b(rstd=None), lambda: b(cols=0), lambda: b(dx=None, dgamma=None), lambda: b(dx=x.ptr + 4), lambda: b(dsum=s, dx=s.ptr + 4),
           lambda: b(dgamma=g), lambda: b(dgamma=x), lambda: b(dgamma=y), lambda: b(dx=g), lambda: b(dx=rstd), lambda: b(dgamma=rstd)]
    for i, call in enumerate(bad):
        with pytest.raises(FgError) as err:
            call()
        assert err.value.kind == "FG_ERR_INVALID_ARGUMENT", i
    assert ctx.device_status() == 0
