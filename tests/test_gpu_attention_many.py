"""Attention outside of the tensor cores' 16-bit path where there are rows enough for its large tiles: f32, head sizes that the tensor cores do not take as they lie,
tensors off 16-byte boundaries, heads of more than 128 columns.  Formulas and bounds are those of the other sizes."""
import numpy as np
import pytest

from test_gpu_attention import Case, check_backward, check_forward, compare, OnDevice, SELF
from token_ops import bits, Placed, rounded

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ctx():
    from ferrograd_b200 import GpuContext
    c = GpuContext(0)
    yield c
    assert c.device_status() == 0
    c.destroy()


# 16 heads over 4: more than two tiles of 64 rows for each of 148 SMs.
LENGTHS = {"own tokens": SELF(611, 1, 700, 0, 93), "others": [(400, 900), (611, 130), (0, 70), (300, 40), (101, 102)]}


@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,dim,shift", [("f32", 64, 0), ("f32", 40, 1), ("f32", 100, 0), ("f32", 128, 0), ("f32", 192, 0), ("f32", 256, 0),
                                             ("bf16", 36, 0), ("f16", 100, 0), ("bf16", 128, 1), ("f16", 64, 1), ("bf16", 256, 0)])
def test_many_rows(ctx, dtype, dim, shift, causal, lengths):
    d = OnDevice(ctx, Case(50, dtype, dim, 16, 4, LENGTHS[lengths], causal, gap=(3, 5), tail=(2, 9)), shift=shift)
    d.forward()
    check_forward(d)
    check_backward(ctx, d)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv", [(16, 16), (48, 1), (15, 5)])
def test_heads(ctx, dim, heads, kv):
    # columns of one tensor, heads of all groupings
    d = OnDevice(ctx, Case(51, "f32", dim, heads, kv, SELF(700, 29, 600)), fused=True, pad=5)
    d.forward()
    check_forward(d)
    check_backward(ctx, d)


@pytest.mark.parametrize("dim", [64, 128])
def test_same_bits_and_recorded(ctx, dim):
    c = Case(52, "f32", dim, 16, 4, SELF(611, 700))
    a, b = OnDevice(ctx, c), OnDevice(ctx, c)
    out, lse, _, _ = c.forward()
    t = Placed(ctx, rounded(out, "f32")), Placed(ctx, lse.astype(np.float32)), Placed(ctx, c.dout)

    def both(d):
        d.forward()
        d.backward(*t)

    both(a)
    ctx.plan_begin()
    both(b)
    plan = ctx.plan_end()
    for _ in range(2):
        both(a)
        plan.launch()
    ctx.sync()
    assert (a.out.bits() == b.out.bits()).all() and (a.lse.bits() == b.lse.bits()).all()
    for x, y in zip(a.g, b.g):
        assert (x.bits() == y.bits()).all()
    plan.destroy()


def test_large_scores(ctx):
    # scores of hundreds that rise along a row: what was summed so far is multiplied down again and again
    for dim in (64, 128):
        c = Case(53, "f32", dim, 16, 4, SELF(1300), scale=1.0, size=3.0)
        c.k *= np.linspace(0.2, 2.0, 1300)[:, None, None]
        c.k = rounded(c.k, "f32")
        d = OnDevice(ctx, c)
        d.forward()
        check_forward(d)
        check_backward(ctx, d)


@pytest.mark.parametrize("dtype,dim,heads,kv", [("bf16", 128, 4, 1), ("f16", 64, 4, 2), ("f32", 64, 4, 2), ("f32", 128, 16, 4)])
@pytest.mark.parametrize("first,then,slot", [([(300, 300), (40, 40), (900, 900)], [(0, 0), (1210, 1210), (30, 30)], None), ([(1, 700), (1, 3), (1, 0)], [(1, 2), (1, 0), (1, 5000)], 5000),
                                             ([(2, 30), (1, 900), (0, 7)], [(0, 0), (3, 1200), (0, 1200)], 1200)], ids=["prompts", "tokens", "moved"])
def test_recorded_with_new_lengths(ctx, dtype, dim, heads, kv, first, then, slot):
    # starts and lengths are read when the kernels run: a plan of one batch, played for another
    a, b = (Case(54, dtype, dim, heads, kv, lens, slot=slot) for lens in (first, then))
    d = OnDevice(ctx, a)

    def both():
        d.forward()
        d.backward(*t)

    def given(c):
        out, lse, _, _ = c.forward()
        return Placed(ctx, rounded(out, dtype), dtype), Placed(ctx, lse.astype(np.float32)), Placed(ctx, c.dout, dtype)

    t, u = given(a), given(b)
    both()
    ctx.sync()
    ctx.plan_begin()
    both()
    plan = ctx.plan_end()
    plan.launch()
    check_forward(d)
    for x, y in zip(t, u):
        ctx.upload(x.t.data, ctx.to_numpy(y.t))
    ctx.upload(d.q_starts.t.data, ctx.to_numpy(Placed(ctx, np.asarray(b.q_starts), "u32").t))
    ctx.upload(d.k_starts.t.data, ctx.to_numpy(Placed(ctx, np.asarray(b.k_starts), "u32").t))
    if slot:
        ctx.upload(d.k_lengths.t.data, ctx.to_numpy(Placed(ctx, np.asarray(b.k_lengths), "u32").t))
    for x in (d.out, d.lse, *d.g):      # NaN where the new batch has nothing
        ctx.upload(x.t.data, cleared(x, ctx))
    d.c = b
    plan.launch()
    ctx.sync()
    check_forward(d)
    want, bound = b.backward(rounded(b.forward()[0], dtype), b.forward()[1].astype(np.float32))
    rows = b.rows
    for n, got in d.gradients().items():
        compare(got, want[n], bound[n], rows[0] if n == "dq" else rows[1], n)
    plan.destroy()


def cleared(x, ctx):
    whole = ctx.to_numpy(x.t).copy()
    whole[x.shift:x.shift + x.n] = bits(np.full(x.n, np.nan), x.dtype)
    return whole
