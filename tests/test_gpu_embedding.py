"""Embedding lookup and the gradient of its table, against 64-bit sums: the three storage types, tables and outputs that start at any element,
one token to many, tokens that all differ, that are all one, and padding.

Bounds: a product is off by half a step of its type; a row's sum of k terms by k u of the sum of their sizes (u = 2^-24) whatever the order,
its scaling and the addition to what was there by u each."""
import numpy as np
import pytest

from token_ops import HALF_ULP, TINY, U, Placed, check, empty, rounded

pytestmark = pytest.mark.gpu
TYPES = ("f32", "f16", "bf16")
PAD = 0xffffffff


@pytest.fixture(scope="module")
def ctx():
    from ferrograd_b200 import GpuContext
    c = GpuContext(0)
    yield c
    assert c.device_status() == 0
    c.destroy()


def tokens_of(kind, n, vocab, r):
    if kind == "one":
        return np.full(n, vocab - 1, np.uint32)
    if kind == "all":
        return (r.permutation(max(n, vocab))[:n] % vocab).astype(np.uint32)
    ids = np.minimum(np.exp(r.random(n) * np.log(vocab + 1)) - 1, vocab - 1).astype(np.uint32)
    if kind == "padded":
        ids[r.random(n) < 0.3] = PAD
        ids[r.random(n) < 0.1] = vocab          # just outside
    if kind == "padding":
        ids[:] = PAD
    return ids


SHAPES = [(1, 1, 1), (1, 10, 4096), (5, 3, 7), (33, 100, 64), (64, 1000, 777), (100, 50, 8), (257, 31, 1000), (1000, 5000, 129), (1025, 300, 256),
          (2500, 40, 520), (4097, 70000, 16), (20000, 1000, 24), (7, 2, 20001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,dim", SHAPES)
@pytest.mark.parametrize("kind,shift", [("words", 0), ("words", 1), ("padded", 0), ("padded", 3), ("one", 0), ("all", 0), ("padding", 0)])
def test_lookup_and_gradient(ctx, dtype, n, vocab, dim, kind, shift):
    r = np.random.Generator(np.random.Philox(n + vocab + dim))
    ids = tokens_of(kind, n, vocab, r)
    inside = ids < vocab
    scale = float(np.float32(1.7))
    idd = Placed(ctx, ids, "u32", shift)
    if vocab * dim <= 3_000_000:
        table = rounded(r.standard_normal((vocab, dim)), dtype)
        out = empty(ctx, (n, dim), dtype, shift)
        ctx.embedding_fwd(Placed(ctx, table, dtype, 2 * shift), idd, out, n, vocab, dim, scale=scale, dtype=dtype)
        want = np.where(inside[:, None], scale * table[np.where(inside, ids, 0)].astype(np.float64), 0.0)
        got = out.get()
        check(got, want, HALF_ULP[dtype] * 1.001 * np.abs(want) + TINY[dtype] * (want != 0), "lookup")
        assert not got[~inside].any()
    dout = rounded(r.standard_normal((n, dim)), dtype)
    doutd = Placed(ctx, dout, dtype, shift)
    base = rounded(r.standard_normal((vocab, dim)), dtype)
    sums, sizes, count = np.zeros((vocab, dim)), np.zeros((vocab, dim)), np.bincount(ids[inside], minlength=vocab)[:, None]
    np.add.at(sums, ids[inside], dout[inside].astype(np.float64))
    np.add.at(sizes, ids[inside], np.abs(dout[inside]).astype(np.float64))
    for add in (False, True):
        grad = Placed(ctx, base, dtype, 2 * shift) if add else empty(ctx, (vocab, dim), dtype, 2 * shift)
        ctx.embedding_bwd(idd, doutd, grad, n, vocab, dim, scale=scale, accumulate=add, dtype=dtype)
        want = scale * sums + (base if add else 0.0)
        bound = (count + 2) * U * scale * sizes + U * np.abs(want) + HALF_ULP[dtype] * 1.001 * np.abs(want) + TINY[dtype]
        got = grad.get()
        check(got, want, bound, f"gradient, accumulate {add}")
        idle = count[:, 0] == 0
        assert np.array_equal(got[idle], base[idle] if add else np.zeros_like(base[idle]))
        if not add:
            again = empty(ctx, (vocab, dim), dtype, 2 * shift)
            ctx.embedding_bwd(idd, doutd, again, n, vocab, dim, scale=scale, dtype=dtype)
            assert np.array_equal(grad.bits(), again.bits()), "the same call gives the same bits"


@pytest.mark.parametrize("n,vocab,kind", [(70000, 200000, "words"), (70001, 9, "words"), (300000, 1 << 24, "all"), (300001, 4, "one"), (150000, 65537, "padded")])
def test_long_batches(ctx, n, vocab, kind):
    # whole numbers: every order of a sum gives the same, so the table is compared exactly
    r = np.random.Generator(np.random.Philox(n))
    ids, dim = tokens_of(kind, n, vocab, r), 4
    dout = r.integers(-8, 9, (n, dim)).astype(np.float32)
    grad = empty(ctx, (vocab, dim))
    ctx.embedding_bwd(Placed(ctx, ids, "u32"), Placed(ctx, dout), grad, n, vocab, dim)
    inside = ids < vocab
    want = np.stack([np.bincount(ids[inside], weights=dout[inside, c], minlength=vocab) for c in range(dim)], 1)
    assert np.array_equal(grad.get(), want.astype(np.float32))


@pytest.mark.parametrize("dtype,vocab,dim,shift", [("f32", 20011, 777, 1), ("f16", 30000, 1024, 0), ("bf16", 700, 40001, 3)])
@pytest.mark.parametrize("kind", ["words", "padded", "one"])
def test_large_tables(ctx, dtype, vocab, dim, shift, kind):
    # tables whose rows are cleared in both launches; sums of whole numbers, rounded once
    r = np.random.Generator(np.random.Philox(vocab))
    n = 1500
    ids, dout = tokens_of(kind, n, vocab, r), r.integers(-2, 3, (n, dim)).astype(np.float32)
    if kind == "words":
        ids[:700] = r.permutation(vocab)[:700]
    dout[200:] *= kind != "one"
    grad = empty(ctx, (vocab, dim), dtype, shift)
    ctx.embedding_bwd(Placed(ctx, ids, "u32"), Placed(ctx, dout, dtype, shift), grad, n, vocab, dim, dtype=dtype)
    inside = ids < vocab
    want = np.zeros((vocab, dim), np.float32)
    np.add.at(want, ids[inside], dout[inside])
    assert np.array_equal(grad.get(), rounded(want, dtype))


def test_values_out_of_the_ordinary(ctx):
    # an infinity or NaN in a padded place is not read; in a used one it stays in its row and column
    ids = np.array([2, PAD, 0, 2], np.uint32)
    dout = np.ones((4, 16), np.float32)
    dout[1], dout[3, 5] = np.nan, np.inf
    grad = empty(ctx, (4, 16))
    ctx.embedding_bwd(Placed(ctx, ids, "u32"), Placed(ctx, dout), grad, 4, 4, 16)
    want = np.array([[1.0], [0.0], [2.0], [0.0]]) * np.ones((4, 16))
    want[2, 5] = np.inf
    assert np.array_equal(grad.get(), want.astype(np.float32))
    table = np.ones((4, 16), np.float32)
    table[2, 3], table[3] = np.nan, np.inf
    out = empty(ctx, (4, 16))
    ctx.embedding_fwd(Placed(ctx, table), Placed(ctx, ids, "u32"), out, 4, 4, 16, scale=0.5)
    got = out.get()
    assert np.isnan(got[[0, 3], 3]).all() and np.isnan(got).sum() == 2 and not got[1].any() and (got[2] == 0.5).all()


def test_far_offsets(ctx):
    # rows of a table beyond 2^32 bytes, and 2^31 elements
    vocab, dim = 300_000, 8192
    rows = np.array([0, 1, 262_143, 262_144, 299_999, PAD, 299_999], np.uint32)
    table = ctx.new_tensor((vocab * dim // 2,), np.float32)          # bf16 elements in pairs
    r = np.random.Generator(np.random.Philox(5))
    from ferrograd_b200.backend import to_bf16_bits, from_bf16_bits
    values = to_bf16_bits(r.standard_normal((len(rows), dim)).astype(np.float32)).reshape(len(rows), dim)
    values[6] = values[4]
    for i, v in enumerate(rows):
        if v != PAD:
            ctx.upload(table.data, values[i], dst_off=int(v) * dim * 2)
    ids, out = Placed(ctx, rows, "u32"), empty(ctx, (len(rows), dim), "bf16")
    ctx.embedding_fwd(table, ids, out, len(rows), vocab, dim, dtype="bf16")
    want = values.copy()
    want[5] = 0
    assert np.array_equal(out.bits(), want)
    ctx.memset_zero(table, vocab * dim * 2)
    ctx.embedding_bwd(ids, out, table, len(rows), vocab, dim, accumulate=True, dtype="bf16")
    got = np.empty(dim, np.uint16)
    for i in (0, 1, 2, 3, 4):
        ctx.download(table.data, got, src_off=int(rows[i]) * dim * 2)
        assert np.array_equal(from_bf16_bits(got), from_bf16_bits(values[i]) * (2 if i == 4 else 1))
    table.data.free()


@pytest.mark.parametrize("n,vocab,dim", [(40, 100, 64), (3000, 500, 100), (40000, 3000, 8)])
def test_captured(ctx, n, vocab, dim):
    r = np.random.Generator(np.random.Philox(n))
    all_ids = [tokens_of(k, n, vocab, r) for k in ("words", "one", "padded", "padding")]
    dout = r.integers(-8, 9, (n, dim)).astype(np.float32)
    idd, doutd, grad, out = Placed(ctx, all_ids[0], "u32"), Placed(ctx, dout), empty(ctx, (vocab, dim)), empty(ctx, (n, dim))
    ctx.embedding_bwd(idd, doutd, grad, n, vocab, dim)          # the arena is there before the recording
    ctx.plan_begin()
    ctx.embedding_bwd(idd, doutd, grad, n, vocab, dim)
    ctx.embedding_fwd(grad, idd, out, n, vocab, dim)
    plan = ctx.plan_end()
    for ids in all_ids:
        ctx.upload(idd.t.data, ids)
        plan.launch()
        want, inside = np.zeros((vocab, dim), np.float32), ids < vocab
        np.add.at(want, ids[inside], dout[inside])
        assert np.array_equal(grad.get(), want)
        assert np.array_equal(out.get(), np.where(inside[:, None], want[np.where(inside, ids, 0)], 0))
    plan.destroy()


def test_empty_and_refusals(ctx):
    from ferrograd_b200 import FgError
    t, g = ctx.new_tensor((256,)), Placed(ctx, np.ones((4, 4)))
    p = t.ptr
    ctx.embedding_fwd(p, p, p + 512, 0, 4, 4)
    ctx.embedding_bwd(p, p, g, 0, 4, 4, accumulate=True)
    assert (g.get() == 1).all()
    ctx.embedding_bwd(p, p, g, 0, 4, 4)
    assert (g.get() == 0).all()

    def refuse(f):
        with pytest.raises(FgError) as e:
            f()
        assert e.value.kind == "FG_ERR_INVALID_ARGUMENT"

    for kw in (dict(table=None), dict(ids=None), dict(out=None), dict(vocab=0), dict(dim=0), dict(table=p + 2), dict(ids=p + 514), dict(out=p + 257),
               dict(out=p + 16), dict(vocab=1 << 31, dim=1 << 31), dict(ids=p + 260)):
        a = dict(table=p, ids=p + 512, out=p + 256, tokens=2, vocab=4, dim=4) | kw
        refuse(lambda: ctx.embedding_fwd(**a))
    for kw in (dict(dout=None), dict(ids=None), dict(dtable=None), dict(vocab=0), dict(dim=0), dict(dtable=p + 2), dict(ids=p + 514), dict(dout=p + 257),
               dict(dtable=p + 272), dict(vocab=1 << 31, dim=1 << 31), dict(ids=p + 60), dict(tokens=1 << 31)):
        a = dict(ids=p + 512, dout=p + 256, dtable=p, tokens=2, vocab=4, dim=4) | kw
        refuse(lambda: ctx.embedding_bwd(**a))
    assert ctx.lib.fg_embedding_fwd(ctx.handle, 3, 1, 4, 4, p, p + 64, 1.0, p + 256) == 1
    assert ctx.lib.fg_embedding_bwd(ctx.handle, -1, 1, 4, 4, p, p + 64, 1.0, p + 256, 0) == 1


def test_rows_of_the_most_columns():
    # one row of 2^32 - 1 columns: the number of its tiles is no 32-bit sum
    from ferrograd_b200 import GpuContext
    from ferrograd_b200.backend import to_bf16_bits
    ctx, dim = GpuContext(0), (1 << 32) - 1
    source, grad = (ctx.new_tensor((dim,), np.uint16) for _ in range(2))
    r, at = np.random.Generator(np.random.Philox(4)), (0, dim // 3, dim - 300)
    parts = [to_bf16_bits(r.integers(1, 9, 300).astype(np.float32)) for _ in at]
    ids, got = Placed(ctx, [0], "u32"), np.empty(300, np.uint16)

    def expect(times):
        for i, part in zip(at, parts):
            ctx.download(grad.data, got, src_off=2 * i)
            assert np.array_equal(got, to_bf16_bits(times * (part.astype(np.uint32) << 16).view(np.float32)))

    ctx.memset_zero(source, 2 * dim)
    for i, part in zip(at, parts):
        ctx.upload(source.data, part, dst_off=2 * i)
        ctx.upload(grad.data, np.full(300, 0x7fc0, np.uint16), dst_off=2 * i)          # NaN
    ctx.embedding_fwd(source, ids, grad, 1, 1, dim, scale=2.0, dtype="bf16")
    expect(2)
    ctx.embedding_bwd(ids, source, grad, 1, 1, dim, dtype="bf16")
    expect(1)
    ctx.embedding_bwd(ids, source, grad, 1, 1, dim, accumulate=True, dtype="bf16")
    expect(2)
    assert ctx.device_status() == 0
    for t in (source, grad):
        t.data.free()
    ctx.destroy()
