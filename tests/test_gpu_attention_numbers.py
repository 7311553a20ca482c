"""Attention with numbers that are none, infinities and the largest ones inside of a sequence: what the formulas make of them has to come out.

A NaN or an infinity in v, and backward in any tensor, may reach the rows of its own sequence that do not see it; so each test names what must not be a number,
and what must be one: the other sequence.  Both signs of the NaN whose bits are all set are tried beside the usual one: the first is what arithmetic on the
device makes."""
import numpy as np
import pytest

from test_gpu_attention import Case, check_forward, compare, OnDevice, SELF
from token_ops import bits, Placed, rounded

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ctx():
    from ferrograd_b200 import GpuContext
    c = GpuContext(0)
    yield c
    assert c.device_status() == 0
    c.destroy()


# Few tiles of rows and many: the kernels of 64 columns and fewer, of up to 128 and of more; 16-bit heads that the tensor cores do not take as they lie, and some that they do.
FEW, MANY = (SELF(70, 90), 4, 2), (SELF(600, 640), 16, 4)
FORMS = [(size, dtype, dim) for size in ("few", "many") for dtype, dim in (("f32", 64), ("f32", 100), ("f32", 128), ("f32", 200), ("bf16", 36), ("f16", 100))]
FORMS += [("few", "bf16", 64), ("few", "f16", 128)]
NAN = {"f32": (0x7fffffff, 0xffffffff, 0x7fc00000, 0x7f800001), "bf16": (0x7fff, 0xffff, 0x7fc0), "f16": (0x7fff, 0xffff, 0x7e00)}


def case(size, dtype, dim, causal=True):
    lens, heads, kv = FEW if size == "few" else MANY
    return Case(40, dtype, dim, heads, kv, lens, causal)


class WithBits(Placed):
    """A tensor with one element of given bits."""

    def __init__(self, ctx, a, dtype, at, word):
        super().__init__(ctx, a, dtype)
        b = bits(a, dtype).copy().reshape(np.shape(a))
        b[at] = word
        whole = self.ctx.to_numpy(self.t).copy()
        whole[:self.n] = b.ravel()
        ctx.upload(self.t.data, whole)


def place(c, which, i=None, j=None, h=1, col=3):
    """Where the element of a tensor goes: query i or key j of the first sequence, query head h or its head of k and v."""
    w = h * c.kv // c.heads
    return {"q": (i, h, col), "dout": (i, h, col), "out": (i, h, col), "k": (j, w, col), "v": (j, w, col), "lse": (h, i)}[which]


@pytest.mark.parametrize("size,dtype,dim", FORMS)
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_forward(ctx, size, dtype, dim, which):
    c = case(size, dtype, dim)
    d = OnDevice(ctx, c)
    d.forward()
    ctx.sync()
    clean = d.out.get()
    nq = c.seqs[0][1]
    i, j, h, col = 2 * nq // 3, nq // 4, 1, 3
    group = c.heads // c.kv
    heads = range(h // group * group, h // group * group + group)
    for word in NAN[dtype]:
        t = WithBits(ctx, getattr(c, which), dtype, place(c, which, i, j, h, col), word)
        d.__dict__.update({which: t.ptr, "out": Placed(ctx, np.zeros(c.q.shape), dtype), "lse": Placed(ctx, np.zeros((c.heads, c.n)))})
        d.forward()
        out, lse = d.out.get(), d.lse.get()
        if which == "q":
            assert np.isnan(out[i, h]).all() and np.isnan(lse[h, i]), hex(word)
        else:
            for g in heads:
                seen = out[j:nq, g] if which == "k" else out[j:nq, g, col]
                assert np.isnan(seen).all(), (hex(word), g)
                assert np.isnan(lse[g, j:nq]).all() if which == "k" else np.isfinite(lse[g, :nq]).all()
            if which == "k":      # not seen by the rows before
                assert np.array_equal(out[:j, h], clean[:j, h])
        assert np.array_equal(out[nq:], clean[nq:]) and np.isfinite(lse[:, nq:]).all()
        others = [g for g in range(c.heads) if g not in heads]
        assert np.array_equal(out[:, others], clean[:, others])


@pytest.mark.parametrize("size,dtype,dim", FORMS)
@pytest.mark.parametrize("which", ["q", "k", "v", "dout", "out", "lse"])
def test_backward(ctx, size, dtype, dim, which):
    c = case(size, dtype, dim)
    d = OnDevice(ctx, c)
    out, lse, _, _ = c.forward()
    host = {"q": c.q, "k": c.k, "v": c.v, "dout": c.dout, "out": rounded(out, dtype), "lse": lse.astype(np.float32)}
    t = {n: Placed(ctx, host[n], "f32" if n == "lse" else dtype) for n in ("out", "lse", "dout")}
    d.backward(t["out"], t["lse"], t["dout"])
    clean = d.gradients()
    nq = c.seqs[0][1]
    i, j, h, col = 2 * nq // 3, nq // 4, 1, 3
    w, group = h * c.kv // c.heads, c.heads // c.kv
    for word in NAN["f32" if which == "lse" else dtype]:
        x = WithBits(ctx, host[which], "f32" if which == "lse" else dtype, place(c, which, i, j, h, col), word)
        more = dict(t)
        if which in t:
            more[which] = x
        else:
            setattr(d, which, x.ptr)
        d.backward(more["out"], more["lse"], more["dout"])
        g = d.gradients()
        what = (which, hex(word))
        if which in ("k", "v"):
            for head in range(w * group, (w + 1) * group):
                assert np.isnan(g["dq"][j:nq, head]).all(), what
            assert np.isnan(g["dk"][j, w]).all(), what
            assert np.isnan(g["dv"][j, w]).all() or which == "v", what
        else:
            assert np.isnan(g["dq"][i, h]).all(), what
            assert np.isnan(g["dk"][:i + 1, w]).all(), what
            if which in ("q", "lse"):
                assert np.isnan(g["dv"][:i + 1, w]).all(), what
            elif which == "dout":
                assert np.isnan(g["dv"][:i + 1, w, col]).all(), what
        for n in g:
            assert np.isfinite(g[n][nq:]).all(), (what, n)
            others = [k for k in range(g[n].shape[1]) if (k // group if n == "dq" else k) != w]
            if dtype != "f16":
                assert np.array_equal(g[n][:, others], clean[n][:, others]), (what, n)
            assert np.isfinite(g[n][:, others]).all(), (what, n)


@pytest.mark.parametrize("size,dtype,dim", FORMS)
@pytest.mark.parametrize("sign", [1, -1])
def test_infinite_value(ctx, size, dtype, dim, sign):
    # v of infinity: the rows that see it have it, in its column
    c = case(size, dtype, dim)
    nq = c.seqs[0][1]
    j, w, col = nq // 4, 0, 5
    c.v[j, w, col] = sign * np.inf
    d = OnDevice(ctx, c)
    d.forward()
    out = d.out.get()
    for h in range(c.heads // c.kv):
        assert (out[j:nq, h, col] == sign * np.inf).all()
        assert np.isfinite(np.delete(out[:, h], col, 1)).all()
    assert np.isfinite(out[nq:]).all()


@pytest.mark.parametrize("size,dim", [(s, d) for s in ("few", "many") for d in (64, 128)])
def test_infinite_gradient(ctx, size, dim):
    # dout of infinity: dv of the keys that are seen has it, in its column; dp and delta are infinities, whose difference is one or no number, by the signs of v and out
    c = case(size, "f32", dim)
    out, lse, _, _ = c.forward()
    nq = c.seqs[0][1]
    i, h, col = 2 * nq // 3, 1, 5
    c.dout[i, h, col] = np.inf
    d = OnDevice(ctx, c)
    d.backward(Placed(ctx, rounded(out, "f32")), Placed(ctx, lse.astype(np.float32)), Placed(ctx, c.dout))
    g = d.gradients()
    assert (g["dv"][:i + 1, 0, col] == np.inf).all()
    sign = np.sign(c.v[:i + 1, 0, col])
    ds = np.where(sign == np.sign(out[i, h, col]), np.nan, sign * np.inf)
    assert np.isnan(ds).any() and np.isnan(g["dq"][i, h]).all()
    assert np.array_equal(g["dk"][:i + 1, 0], ds[:, None] * c.q[i, h], equal_nan=True)
    for n in g:
        assert np.isfinite(g[n][nq:]).all() and np.isfinite(np.delete(g[n], h if n == "dq" else 0, 1)).all()


@pytest.mark.parametrize("size,dim", [(s, d) for s in ("few", "many") for d in (64, 128, 200)])
@pytest.mark.parametrize("largest", [0x7f7fffff, 0x7f7ff000, 0x7f7fefff, 0xff7fffff])
def test_largest_numbers(ctx, size, dim, largest):
    # f32's largest numbers where the sums stay below them: a value with the weights of its rows, a query whose column of k is zero
    x = np.uint32(largest).view(np.float32)
    c = case(size, "f32", dim)
    nq = c.seqs[0][1]
    c.v[nq // 4, 0, 5] = x
    d = OnDevice(ctx, c)
    d.forward()
    check_forward(d)
    c = case(size, "f32", dim)
    c.k[:, 0, 3] = 0.0
    c.q[2 * nq // 3, 1, 3] = x
    c.dout = rounded(0.01 * c.dout, "f32")
    out, lse, _, _ = c.forward()
    out, lse = rounded(out, "f32"), lse.astype(np.float32)
    d = OnDevice(ctx, c)
    d.backward(Placed(ctx, out), Placed(ctx, lse), Placed(ctx, c.dout))
    want, bound = c.backward(out, lse)
    rows = c.rows
    far = (np.abs(want["dk"]) + bound["dk"]).max()
    assert far < 3.4e38, "the formula's own gradient is beyond the largest number"
    for n, got in d.gradients().items():
        compare(got, want[n], bound[n], rows[0] if n == "dq" else rows[1], n)


@pytest.mark.parametrize("size", ["few", "many"])
@pytest.mark.parametrize("dim", [32, 128])
def test_infinite_scores(ctx, size, dim):
    # a key whose score is -inf has no weight, whichever kernel multiplies; a row with no other is empty
    c = case(size, "f32", dim)
    c.q[:, :, 0] = np.abs(c.q[:, :, 0]) + 1
    c.k[:5, :, 0] = -np.inf
    d = OnDevice(ctx, c)
    d.forward()
    got, lse = d.out.get(), d.lse.get()
    assert (got[:5] == 0).all() and np.isneginf(lse[:, :5]).all()
    rest = case(size, "f32", dim)
    rest.q = c.q
    (q0, nq, k0, nk), other = rest.seqs
    rest.seqs = [(5, nq - 5, 5, nk - 5), other]
    out, _, bound, _ = rest.forward()
    assert (np.abs(got[5:] - out[5:]) <= bound[5:]).all()


CACHES = [("f32", 64, 4, 2), ("f32", 200, 2, 1), ("bf16", 128, 8, 2), ("f16", 64, 4, 4), ("f16", 128, 20, 1), ("bf16", 64, 40, 1), ("bf16", 36, 4, 2)]


@pytest.mark.parametrize("dtype,dim,heads,kv", CACHES)
@pytest.mark.parametrize("lens", [[(1, 1), (1, 1), (1, 1)], [(1, 40), (1, 100), (1, 30)], [(1, 30), (1, 5000), (1, 4000)], [(2, 70), (3, 9000)]],
                         ids=["one key", "one share", "shares", "more tokens"])
def test_generated_tokens(ctx, dtype, dim, heads, kv, lens):
    # a query that is no number, and a key: the rows that see it are none, and their lse is none; the others are what they are without it
    c = Case(41, dtype, dim, heads, kv, lens)
    d = OnDevice(ctx, c)
    d.forward()
    check_forward(d)
    out, lse, e_out, e_lse = c.forward()
    q0, nq, k0, nk = c.seqs[1]
    h, group = heads // 2, heads // kv
    w = h // group
    for word in NAN[dtype]:
        for which, at in (("q", (q0 + nq - 1, h, 3)), ("k", (k0 + nk // 2, w, 3)), ("k", (k0 + nk - 1, w, 3))):
            x = WithBits(ctx, getattr(c, which), dtype, at, word)
            e = OnDevice(ctx, c)
            setattr(e, which, x.ptr)
            e.forward()
            got, got_lse = e.out.get(), e.lse.get()
            bad = np.zeros((c.n, heads), bool)
            if which == "q":
                bad[q0 + nq - 1, h] = True
            else:
                first = at[0] - k0 - (nk - nq)          # the first query that sees the key
                bad[q0 + max(first, 0):q0 + nq, w * group:(w + 1) * group] = True
            assert np.isnan(got[bad]).all() and np.isnan(got_lse.T[bad]).all(), (which, hex(word))
            assert (np.abs(got[~bad] - out[~bad]) <= e_out[~bad]).all() and (np.abs(got_lse.T[~bad] - lse.T[~bad]) <= e_lse.T[~bad]).all(), (which, hex(word))


@pytest.mark.parametrize("dtype,dim,heads,kv", CACHES)
def test_generated_tokens_infinite_scores(ctx, dtype, dim, heads, kv):
    # all scores of a row -inf: zeros and -inf, in one share and in several; a score of +inf has no weights
    for n in (1, 50, 5000):
        c = Case(42, dtype, dim, heads, kv, [(1, n), (1, n)])
        c.q[:, :, 0] = np.abs(c.q[:, :, 0]) + 1
        c.k[n:, :, 0] = -np.inf
        d = OnDevice(ctx, c)
        d.forward()
        out, lse = d.out.get(), d.lse.get()
        assert (out[1] == 0).all() and np.isneginf(lse[:, 1]).all() and np.isfinite(out[0]).all() and np.isfinite(lse[:, 0]).all()
        c.k[n:, :, 0] = np.inf
        d = OnDevice(ctx, c)
        d.forward()
        out, lse = d.out.get(), d.lse.get()
        assert np.isnan(out[1]).all() and np.isnan(lse[:, 1]).all() and np.isfinite(out[0]).all() and np.isfinite(lse[:, 0]).all()


# f16 gradients of the scores are multiplied in f16, by a power of two that brings them into its range.
def one_head(c, b, w):
    """Sequence b's heads that share head w of k and v, as a case by itself."""
    q0, nq, k0, nk = c.seqs[b]
    group = c.heads // c.kv
    x = Case(0, c.dtype, c.dim, group, 1, [(nq, nk)], c.causal, scale=c.scale)
    i, j, h = slice(q0, q0 + nq), slice(k0, k0 + nk), slice(w * group, (w + 1) * group)
    x.q, x.dout, x.k, x.v = c.q[i, h], c.dout[i, h], c.k[j, w:w + 1], c.v[j, w:w + 1]
    return x, i, j, h


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens", [SELF(300, 200), [(300, 300), (500, 70), (40, 200)]], ids=["few", "more"])
@pytest.mark.parametrize("infinite", [False, True])
def test_factors_of_sequences_and_heads(ctx, dim, lens, infinite):
    # dout up to 4 * 10^5 times as large in one sequence, or head of k and v, as in another: each is as exact as it is alone; an infinity, too, is its own sequence's and head's
    c = Case(43, "f16", dim, 4, 2, lens)
    for b, (q0, nq, _, _) in enumerate(c.seqs):
        for w in range(2):
            c.dout[q0:q0 + nq, 2 * w:2 * w + 2] *= (8000.0, 0.02)[(b + w) % 2]
    c.dout = rounded(c.dout, "f16")
    out, lse, _, _ = c.forward()
    out, lse = rounded(out, "f16"), lse.astype(np.float32)
    dout = c.dout.copy()
    if infinite:
        dout[17, 1, 3] = np.inf
    d = OnDevice(ctx, c)
    d.backward(Placed(ctx, out, "f16"), Placed(ctx, lse), Placed(ctx, dout, "f16"))
    got = d.gradients()
    for b in range(len(lens)):
        for w in range(2):
            if infinite and b == w == 0:
                continue
            x, i, j, h = one_head(c, b, w)
            want, bound = x.backward(out[i, h], lse[h, i])
            for n, mine in (("dq", got["dq"][i, h]), ("dk", got["dk"][j, w:w + 1]), ("dv", got["dv"][j, w:w + 1])):
                assert np.abs(want[n]).max() < 6e4
                compare(mine, want[n], bound[n], np.ones(len(mine), bool), f"{n} of {b}, {w}")
