"""Attention over packed sequences against the formulas in 64 bits.

Bounds, with U = 2^-24 (a sum of n f32 terms is off by at most n U of the sum of their sizes) and h the half step of the storage type.  An f32 product
on the tensor cores is three of numbers of 11 bits: x = hi + lo + r with |r| <= 2^-22 |x|, and lo lo, at most 2^-22 |x y|, is left out, so it is off by
3 * 2^-22 |x y| = 12 U |x y|; their sums, three instructions for 8 terms that each cut less than 2 U of the sum, stay within U a term.
  score      e_s = (dim + 20) U scale (|q|.|k|): its products and sum, the factor, the difference from the row's largest, lse
  weight     relative e_p = e_s + 2^-20 + 4 U |lse| (the exponential, the sums that normalise it), and h where the weights are rounded to 16 bits;
             f16 weights below 2^-14 of the largest are off by 2^-25 of it; weights below 2^-126 are zero
  out        sum of p e_p (|v| + |out|), (n + 20) U sum of p |v|, and h |out|
  ds         p (e_p |dp - delta| + (dim + 16) U (|dout|.|v| + |dout|.|out|)), and h |ds| rounded to 16 bits (f16: and 2^-24 of what the largest dout
             and v can give, the operands being scaled by a power of two with that)
  gradients  the sums of these with |k|, |q| and |dout|, (n + 20) U of the sums of sizes, and h of the result
"""
import numpy as np
import pytest

from token_ops import empty, HALF_ULP, Placed, rounded, TINY, U

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ctx():
    from ferrograd_b200 import GpuContext
    c = GpuContext(0)
    yield c
    assert c.device_status() == 0
    c.destroy()


def rng(*key):
    return np.random.Generator(np.random.Philox(key))


class Case:
    """Tensors on the host, and where the sequences lie in them: (first query, queries, first key, keys)."""

    def __init__(self, seed, dtype, dim, heads, kv, lens, causal=True, slot=None, gap=(0, 0), tail=(0, 0), scale=None, size=1.0):
        r = rng(seed, dim, heads, kv, len(lens))
        self.dtype, self.dim, self.heads, self.kv, self.causal = dtype, dim, heads, kv, causal
        self.scale = np.float32(dim ** -0.5 if scale is None else scale)
        q_lens, k_lens = [a for a, _ in lens], [b for _, b in lens]
        self.q_starts = np.cumsum([gap[0]] + q_lens)
        self.k_lengths = None
        if slot is None:
            self.k_starts = np.cumsum([gap[1]] + k_lens)
        else:
            self.k_starts = gap[1] + np.arange(len(lens) + 1) * slot
            self.k_lengths = np.array(k_lens)
        self.n = int(self.q_starts[-1]) + tail[0]
        self.m = int(self.k_starts[-1]) + tail[1]
        self.seqs = [(int(self.q_starts[b]), q_lens[b], int(self.k_starts[b]), k_lens[b]) for b in range(len(lens))]
        make = lambda *s: rounded(size * r.standard_normal(s), dtype)   # noqa: E731
        self.q, self.dout = make(self.n, heads, dim), make(self.n, heads, dim)
        self.k, self.v = make(self.m, kv, dim), make(self.m, kv, dim)

    @property
    def rows(self):
        """Which queries and which keys belong to a sequence."""
        a, b = np.zeros(self.n, bool), np.zeros(self.m, bool)
        for q0, nq, k0, nk in self.seqs:
            a[q0:q0 + nq] = True
            b[k0:k0 + nk] = True
        return a, b

    def tensor_cores(self):
        return self.dtype != "f32" and self.dim % 8 == 0 and self.dim <= 128

    def weights(self, b, h):
        """p, lse and the bound of p's relative error, of one sequence and head."""
        q0, nq, k0, nk = self.seqs[b]
        q, k = self.q[q0:q0 + nq, h].astype(np.float64), self.k[k0:k0 + nk, h * self.kv // self.heads].astype(np.float64)
        s = float(self.scale) * (q @ k.T)
        seen = np.ones((nq, nk), bool)
        if self.causal:
            seen = np.arange(nk)[None] <= np.arange(nq)[:, None] + nk - nq
        s = np.where(seen, s, -np.inf)
        top = s.max(1, initial=-np.inf)
        e = np.exp(s - np.where(np.isfinite(top), top, 0.0)[:, None])
        total = e.sum(1)
        with np.errstate(divide="ignore"):
            lse = np.where(total > 0, top + np.log(total), -np.inf)
        p = e / np.where(total > 0, total, 1.0)[:, None]
        e_s = (self.dim + 20) * U * abs(float(self.scale)) * (np.abs(q) @ np.abs(k).T)
        return p, lse, e_s + 2.0 ** -20 + 4 * U * np.where(np.isfinite(lse), np.abs(lse), 0.0)[:, None]

    def forward(self, few=False):
        """out, lse and the bounds of their errors."""
        half = HALF_ULP[self.dtype]
        tc = self.tensor_cores()
        out, lse = np.zeros((self.n, self.heads, self.dim)), np.full((self.heads, self.n), -np.inf)
        e_out, e_lse = np.zeros_like(out), np.zeros_like(lse)
        for b, (q0, nq, k0, nk) in enumerate(self.seqs):
            for h in range(self.heads):
                v = self.v[k0:k0 + nk, h * self.kv // self.heads].astype(np.float64)
                p, lse[h, q0:q0 + nq], e_p = self.weights(b, h)
                o = p @ v
                out[q0:q0 + nq, h] = o
                e = p * (e_p + (half if tc else 0.0)) + 2.0 ** -126 * (p > 0)
                if tc and self.dtype == "f16":
                    e = e + p.max(1, initial=0.0)[:, None] * 2.0 ** -24 * (p > 0)
                e_out[q0:q0 + nq, h] = e @ np.abs(v) + np.abs(o) * e.sum(1)[:, None] + (nk + 20) * U * (p @ np.abs(v)) + half * np.abs(o) + TINY[self.dtype]
                e_lse[h, q0:q0 + nq] = (p * e_p).sum(1) + (nk + 8) * U + 4 * U * np.where(np.isfinite(lse[h, q0:q0 + nq]), np.abs(lse[h, q0:q0 + nq]), 0.0)
        return out, lse, e_out, e_lse

    def backward(self, out, lse):
        """dq, dk, dv of these (rounded) out and lse, and the bounds of their errors."""
        half = HALF_ULP[self.dtype]
        tc, sc = self.tensor_cores(), abs(float(self.scale))
        g = {"dq": np.zeros(self.q.shape), "dk": np.zeros(self.k.shape), "dv": np.zeros(self.v.shape)}
        e = {n: np.zeros_like(x) for n, x in g.items()}
        a, c = self.rows
        most = 2.0 ** -24 * 8 * self.dim * float(np.abs(self.dout[a]).max(initial=0.0)) * float(np.abs(self.v[c]).max(initial=0.0)) * 2.0 ** -13
        for b, (q0, nq, k0, nk) in enumerate(self.seqs):
            i, j = slice(q0, q0 + nq), slice(k0, k0 + nk)
            for h in range(self.heads):
                w = h * self.kv // self.heads
                q, k, v, do, o = (x.astype(np.float64) for x in (self.q[i, h], self.k[j, w], self.v[j, w], self.dout[i, h], out[i, h]))
                p, true_lse, e_p = self.weights(b, h)
                given = lse[h, i].astype(np.float64)
                ok = np.isfinite(true_lse)
                p = p * np.exp(np.where(ok, true_lse - np.where(ok, given, 0.0), 0.0))[:, None]
                dp, delta = do @ v.T, (do * o).sum(1)[:, None]
                ds = p * (dp - delta)
                e_ds = p * (e_p * np.abs(dp - delta) + (self.dim + 16) * U * (np.abs(do) @ np.abs(v).T + (np.abs(do) * np.abs(o)).sum(1)[:, None]))
                e_ds = e_ds + 2.0 ** -126 * np.abs(dp - delta) * (p > 0)
                e_pp = p * e_p + 2.0 ** -126 * (p > 0)
                if tc:
                    e_ds = e_ds + half * np.abs(ds) + (most * (p > 0) if self.dtype == "f16" else 0.0)
                    e_pp = e_pp + half * p + (2.0 ** -24 * (p > 0) if self.dtype == "f16" else 0.0)
                g["dq"][i, h] += float(self.scale) * ds @ k
                g["dk"][j, w] += float(self.scale) * ds.T @ q
                g["dv"][j, w] += p.T @ do
                e["dq"][i, h] += sc * (e_ds @ np.abs(k) + (nk + 20) * U * np.abs(ds) @ np.abs(k))
                e["dk"][j, w] += sc * (e_ds.T @ np.abs(q) + (nq * self.heads + 20) * U * np.abs(ds).T @ np.abs(q))
                e["dv"][j, w] += e_pp.T @ np.abs(do) + (nq * self.heads + 20) * U * p.T @ np.abs(do)
        for n in g:
            e[n] += half * np.abs(g[n]) + TINY[self.dtype]
        return g, e


class OnDevice:
    """The case's tensors on the device: dense, or q, k and v as columns of one tensor (fused: queries and keys are the same tokens)."""

    def __init__(self, ctx, c, fused=False, shift=0, pad=0):
        self.ctx, self.c, self.fused = ctx, c, fused
        size = 4 if c.dtype == "f32" else 2
        ql, kl = c.heads * c.dim, c.kv * c.dim
        u32 = lambda a: Placed(ctx, np.asarray(a, np.uint32), "u32")   # noqa: E731
        self.q_starts, self.k_starts = u32(c.q_starts), u32(c.k_starts)
        self.k_lengths = None if c.k_lengths is None else u32(c.k_lengths)
        self.pad = pad
        if fused:
            row = ql + 2 * kl + pad
            whole = np.full((c.n, row), np.nan, np.float32)
            whole[:, :ql + 2 * kl] = np.concatenate([x.reshape(c.n, -1) for x in (c.q, c.k, c.v)], 1)
            self.qkv = Placed(ctx, whole, c.dtype, shift)
            self.grad = empty(ctx, (c.n, row), c.dtype, shift)
            place = lambda t: (t.ptr, t.ptr + ql * size, t.ptr + (ql + kl) * size)   # noqa: E731
            self.q, self.k, self.v = place(self.qkv)
            self.dq, self.dk, self.dv = place(self.grad)
            self.strides = dict(q_stride=row, k_stride=row, v_stride=row)
        else:
            lay = lambda x: Placed(ctx, np.concatenate([x.reshape(len(x), x.shape[1] * c.dim), np.full((len(x), pad), np.nan, np.float32)], 1), c.dtype, shift)   # noqa: E731
            self.t = [lay(x) for x in (c.q, c.k, c.v)]
            self.q, self.k, self.v = (x.ptr for x in self.t)
            self.g = [empty(ctx, (len(x), x.shape[1] * c.dim + pad), c.dtype, shift) for x in (c.q, c.k, c.v)]
            self.dq, self.dk, self.dv = (x.ptr for x in self.g)
            self.strides = dict(q_stride=ql + pad, k_stride=kl + pad, v_stride=kl + pad) if pad else {}
        self.out, self.lse = empty(ctx, (c.n, c.heads, c.dim), c.dtype, shift), empty(ctx, (c.heads, c.n))
        self.sizes = (len(c.seqs), c.n, c.m, c.heads, c.kv, c.dim)
        self.more = dict(scale=float(c.scale), causal=c.causal, k_lengths=self.k_lengths, dtype=c.dtype, **self.strides)

    def forward(self, lse=True):
        self.ctx.attention_fwd(self.q, self.k, self.v, self.out, self.q_starts, self.k_starts, *self.sizes, lse=self.lse if lse else None, **self.more)

    def backward(self, out, lse, dout, parts=("dq", "dk", "dv")):
        self.ctx.attention_bwd(self.q, self.k, self.v, out, lse, dout, self.q_starts, self.k_starts, *self.sizes,
                               **{n: getattr(self, n) for n in parts}, **self.more)

    def gradients(self):
        c = self.c
        if self.fused:
            ql, kl = c.heads * c.dim, c.kv * c.dim
            g = self.grad.get()
            assert self.pad == 0 or np.isnan(g[:, ql + 2 * kl:]).all(), "written between rows"
            parts = (g[:, :ql], g[:, ql:ql + kl], g[:, ql + kl:ql + 2 * kl])
        else:
            parts = [x.get() for x in self.g]
            for x in parts:
                assert self.pad == 0 or np.isnan(x[:, x.shape[1] - self.pad:]).all(), "written between rows"
            parts = [x[:, :x.shape[1] - self.pad] for x in parts]
        return {n: x.reshape(s.shape) for n, x, s in zip(("dq", "dk", "dv"), parts, (c.q, c.k, c.v))}


def compare(got, want, bound, rows, what):
    """Inside the sequences within the bound; outside of them as it was (NaN)."""
    assert np.isnan(got[~rows]).all(), f"{what}: written outside the sequences"
    got, want, bound = got[rows].astype(np.float64), want[rows], bound[rows]
    assert np.isfinite(got).all(), f"{what}: not finite"
    over = np.abs(got - want) - bound
    if over.size:
        i = np.unravel_index(np.argmax(over), over.shape)
        assert over[i] <= 0, f"{what}: {got[i]} for {want[i]} at {i}, off by {abs(got[i] - want[i]):.3g} of {bound[i]:.3g}"


def check_forward(d):
    c = d.c
    out, lse, e_out, e_lse = c.forward()
    rows = c.rows[0]
    compare(d.out.get(), out, e_out, rows, "out")
    got = d.lse.get()
    assert np.isnan(got[:, ~rows]).all()
    empty_rows = np.isneginf(lse) & rows[None]
    assert np.isneginf(got[empty_rows]).all(), "lse of a row that sees nothing"
    there = ~empty_rows & rows[None]
    assert (np.abs(got[there] - lse[there]) <= e_lse[there]).all(), "lse"


def check_backward(ctx, d, **how):
    c = d.c
    out, lse, _, _ = c.forward()
    out, lse = rounded(out, c.dtype), lse.astype(np.float32)
    t = Placed(ctx, out, c.dtype), Placed(ctx, lse), Placed(ctx, c.dout, c.dtype)
    d.backward(*t, **how)
    want, bound = c.backward(out, lse)
    rows = c.rows
    for n, got in d.gradients().items():
        if n in how.get("parts", want):
            compare(got, want[n], bound[n], rows[0] if n == "dq" else rows[1], n)
        else:
            assert np.isnan(got).all(), n


SELF = lambda *n: [(x, x) for x in n]   # noqa: E731
LENGTHS = {
    "one": SELF(1), "short": SELF(7, 1, 0, 30), "tile": SELF(128), "over": SELF(129, 64, 65), "long": SELF(700), "ragged": SELF(300, 5, 0, 128, 211),
    "chunk": [(40, 333), (129, 130), (3, 500)], "fewer keys": [(60, 20), (5, 0), (200, 131)], "many": SELF(*range(1, 40)),
}


@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("dtype,dim,heads,kv", [("f32", 64, 2, 2), ("bf16", 128, 4, 1), ("f16", 64, 4, 2), ("bf16", 40, 3, 1), ("f32", 33, 2, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(ctx, lengths, dtype, dim, heads, kv, causal):
    d = OnDevice(ctx, Case(1, dtype, dim, heads, kv, LENGTHS[lengths], causal))
    d.forward()
    check_forward(d)
    check_backward(ctx, d)


@pytest.mark.parametrize("dim", [1, 8, 16, 24, 32, 48, 63, 72, 80, 96, 100, 104, 112, 120, 128, 136, 192, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_dims(ctx, dim, dtype):
    d = OnDevice(ctx, Case(2, dtype, dim, 2, 1, SELF(150, 33)))
    d.forward()
    check_forward(d)
    check_backward(ctx, d)


@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 8), (8, 1), (15, 3), (7, 1), (64, 2), (130, 1), (128, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_heads(ctx, heads, kv, dtype):
    d = OnDevice(ctx, Case(3, dtype, 64, heads, kv, SELF(70, 140)))
    d.forward()
    check_forward(d)
    check_backward(ctx, d)


@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("bf16", 128), ("f16", 80), ("f16", 64)])
@pytest.mark.parametrize("shift,pad", [(0, 0), (0, 8), (0, 24), (8, 0), (1, 0), (0, 3)])
def test_layouts(ctx, dtype, dim, shift, pad):
    # one tensor of q, k and v, rows apart, tensors off 16-byte boundaries
    for fused in (True, False):
        d = OnDevice(ctx, Case(4, dtype, dim, 4, 2, SELF(100, 31, 140)), fused, shift, pad)
        d.forward()
        check_forward(d)
        check_backward(ctx, d)


@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("bf16", 128), ("f16", 64)])
def test_outside_of_sequences(ctx, dtype, dim):
    # rows before the first sequence and behind the last, slots that are not full: NaN there reaches nothing, and nothing is written there
    c = Case(5, dtype, dim, 4, 2, [(20, 20), (150, 170), (0, 9), (33, 140)], slot=200, gap=(3, 5), tail=(9, 50))
    a, b = c.rows
    c.q[~a] = c.dout[~a] = np.nan
    c.k[~b] = c.v[~b] = np.nan
    d = OnDevice(ctx, c)
    d.forward()
    check_forward(d)
    clean = OnDevice(ctx, c)
    check_backward(ctx, clean)


TOKENS = [("bf16", 128, 32, 8), ("bf16", 64, 8, 8), ("f16", 128, 8, 1), ("f16", 64, 6, 2), ("f32", 64, 4, 2), ("f32", 128, 8, 1), ("bf16", 80, 16, 1), ("bf16", 36, 4, 2),
          ("f16", 256, 4, 2), ("bf16", 96, 24, 1)]


@pytest.mark.parametrize("dtype,dim,heads,kv", TOKENS)
@pytest.mark.parametrize("queries", [1, 2, 5])
def test_single_tokens(ctx, dtype, dim, heads, kv, queries):
    # a cache with slots, NaN behind what is used
    lens = [(queries, n) for n in (1, 700, 64, 65, 3, 2500, 128, 0, 1023)]
    for causal in (True, False):
        c = Case(6, dtype, dim, heads, kv, lens, causal, slot=2600)
        b = c.rows[1]
        c.k[~b] = c.v[~b] = np.nan
        d = OnDevice(ctx, c)
        d.forward()
        check_forward(d)
        d.forward(lse=False)


@pytest.mark.parametrize("dtype,dim,heads,kv", TOKENS[:6])
def test_one_long_sequence(ctx, dtype, dim, heads, kv):
    # one query over many keys: as many shares as there are, some of them behind the end
    for keys, slot in ((30000, None), (1, 20000), (12345, 40000)):
        c = Case(7, dtype, dim, heads, kv, [(1, keys)], slot=slot)
        d = OnDevice(ctx, c)
        d.forward()
        check_forward(d)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_one_sequence_much_longer(ctx, dtype):
    # few queries on average, but one sequence has many, and one has most of the keys
    c = Case(8, dtype, 64, 2, 1, [(1, 40)] * 60 + [(70, 3000)] + [(1, 9)] * 5)
    d = OnDevice(ctx, c)
    d.forward()
    check_forward(d)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_large_scores(ctx, dtype):
    # scores of hundreds: the largest rises again and again along a row, most weights are zero
    c = Case(9, dtype, 64, 2, 2, SELF(400), scale=1.0, size=3.0)
    c.k *= np.linspace(0.2, 2.0, 400)[:, None, None]
    c.k = rounded(c.k, dtype)
    d = OnDevice(ctx, c)
    d.forward()
    check_forward(d)
    check_backward(ctx, d)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scales(ctx, scale, dtype):
    d = OnDevice(ctx, Case(10, dtype, 64, 2, 1, SELF(200), scale=scale))
    d.forward()
    check_forward(d)
    check_backward(ctx, d)


@pytest.mark.parametrize("dtype,dim", [("f32", 32), ("f32", 160), ("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_few_keys_many_rows(ctx, dtype, dim, causal):
    # a head of keys for many heads of queries: the rows of a tile of keys go in shares, some of them empty
    for lens in (SELF(700), [(500, 70), (300, 200), (0, 9), (40, 40)]):
        check_backward(ctx, OnDevice(ctx, Case(23, dtype, dim, 16, 1, lens, causal)))


def test_small_gradients_f16(ctx):
    # dout of 1e-4: the gradients of the scores are far below the smallest normal number of f16
    c = Case(11, "f16", 64, 2, 1, SELF(300))
    c.dout = rounded(c.dout * 1e-4, "f16")
    d = OnDevice(ctx, c)
    check_backward(ctx, d)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_parts_of_the_gradient(ctx, dtype):
    for parts in (("dq",), ("dk", "dv")):
        check_backward(ctx, OnDevice(ctx, Case(12, dtype, 64, 4, 2, SELF(140, 9))), parts=parts)


@pytest.mark.parametrize("dtype,dim", [("f32", 32), ("bf16", 64), ("f16", 128)])
def test_infinite_scores(ctx, dtype, dim):
    # a key whose score is -inf has no weight, a row with no other is empty
    c = Case(13, dtype, dim, 1, 1, SELF(140))
    c.q[:, :, 0] = np.abs(c.q[:, :, 0]) + 1
    c.k[:5, :, 0] = -np.inf
    d = OnDevice(ctx, c)
    d.forward()
    got, lse = d.out.get(), d.lse.get()
    assert (got[:5] == 0).all() and np.isneginf(lse[:, :5]).all()
    rest = Case(13, dtype, dim, 1, 1, SELF(140))
    rest.q = c.q
    rest.seqs = [(5, 135, 5, 135)]
    out, _, bound, _ = rest.forward()
    assert (np.abs(got[5:] - out[5:]) <= bound[5:]).all()


@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("bf16", 128), ("f16", 64)])
def test_neighbours_stay_apart(ctx, dtype, dim):
    # NaN and infinities of one sequence reach no other
    c = Case(14, dtype, dim, 2, 1, SELF(100, 60, 90))
    bad = slice(100, 160)
    for x in (c.q, c.k, c.v, c.dout):
        x[bad] = np.nan
        x[bad, :, ::2] = np.inf
    d = OnDevice(ctx, c)
    d.forward()
    clean = Case(14, dtype, dim, 2, 1, SELF(100, 60, 90))
    clean.seqs = [s for s in clean.seqs if s[0] != 100]
    rows = clean.rows[0]
    out, lse, e_out, _ = clean.forward()
    got = d.out.get()
    assert (np.abs(got[rows] - out[rows]) <= e_out[rows]).all()
    out, lse = rounded(out, dtype), lse.astype(np.float32)
    d.backward(Placed(ctx, out, dtype), Placed(ctx, lse), Placed(ctx, c.dout, dtype))
    want, bound = clean.backward(out, lse)
    for n, got in d.gradients().items():
        assert (np.abs(got[rows] - want[n][rows]) <= bound[n][rows]).all(), n


@pytest.mark.parametrize("dtype,dim", [("f32", 32), ("bf16", 64), ("f16", 128)])
def test_differences(ctx, dtype, dim):
    # the gradient along a direction against the difference of the forward pass in 64 bits
    c = Case(15, dtype, dim, 4, 2, SELF(50, 90))
    r = rng(15)
    out, lse, _, _ = c.forward()
    out, lse = rounded(out, dtype), lse.astype(np.float32)
    d = OnDevice(ctx, c)
    d.backward(Placed(ctx, out, dtype), Placed(ctx, lse), Placed(ctx, c.dout, dtype))
    got = d.gradients()
    want, bound = c.backward(out, lse)
    for name, attr in (("dq", "q"), ("dk", "k"), ("dv", "v")):
        x = getattr(c, attr).astype(np.float64)
        step = r.standard_normal(x.shape)
        loss = []
        for sign in (1, -1):
            setattr(c, attr, x + sign * 1e-5 * step)
            loss.append((c.forward()[0] * c.dout).sum())
        setattr(c, attr, x.astype(np.float32))
        slope = (loss[0] - loss[1]) / 2e-5
        # out was rounded on the way to delta: that moves ds by p times what the rounding moves delta
        moved = HALF_ULP[dtype] * (np.abs(c.dout) * np.abs(out)).sum() * float(c.scale) * 8
        far = (np.abs(bound[name]) * np.abs(step)).sum() + (0.0 if name == "dv" else moved) + 1e-5 * abs(slope) + 1e-4
        assert abs((got[name] * step).sum() - slope) <= far, name


@pytest.mark.parametrize("dtype,dim,heads,kv,lens", [("bf16", 128, 4, 1, SELF(300, 140)), ("f32", 64, 2, 2, SELF(300)), ("bf16", 64, 8, 2, [(1, 900), (1, 5000)])])
def test_same_bits_again_and_recorded(ctx, dtype, dim, heads, kv, lens):
    c = Case(16, dtype, dim, heads, kv, lens)
    a, b = OnDevice(ctx, c), OnDevice(ctx, c)
    out, lse, _, _ = c.forward()
    t = Placed(ctx, rounded(out, dtype), dtype), Placed(ctx, lse.astype(np.float32)), Placed(ctx, c.dout, dtype)

    def both(d):
        d.forward()
        d.backward(*t)

    both(a)
    ctx.sync()
    ctx.plan_begin()
    both(b)
    plan = ctx.plan_end()
    for _ in range(3):
        both(a)
        plan.launch()
    assert (a.out.bits() == b.out.bits()).all() and (a.lse.bits() == b.lse.bits()).all()
    for x, y in zip(a.g, b.g):
        assert (x.bits() == y.bits()).all()
    plan.destroy()
    check_forward(b)


def test_two_contexts_at_once():
    from ferrograd_b200 import GpuContext
    work = []
    for seed, lens in ((17, SELF(900, 300)), (18, [(1, 3000)] * 7)):
        ctx = GpuContext(0)
        work.append((ctx, OnDevice(ctx, Case(seed, "bf16", 128, 8, 2, lens))))
    for _ in range(5):
        for _, d in work:
            d.forward()
    for ctx, d in work:
        check_forward(d)
        assert ctx.device_status() == 0
        ctx.destroy()


def test_starts_that_do_not_fit(ctx):
    # starts beyond the tensors are held to their sizes, starts that decrease give empty sequences
    c = Case(19, "bf16", 64, 2, 1, SELF(100, 60))
    d = OnDevice(ctx, c)
    for starts in ([0, 100, 500], [0, 100, 0xffffffff]):
        d.q_starts = d.k_starts = Placed(ctx, np.array(starts, np.uint32), "u32")
        d.forward()
        check_forward(d)
    d.out = empty(ctx, (c.n, c.heads, c.dim), c.dtype)
    for starts in ([160, 100, 60], [0xffffffff, 0xfffffff0, 5], [0xffffffff] * 3):
        d.q_starts = d.k_starts = Placed(ctx, np.array(starts, np.uint32), "u32")
        d.forward()
        d.backward(Placed(ctx, np.zeros((c.n, c.heads, c.dim)), c.dtype), Placed(ctx, np.zeros((c.heads, c.n))), Placed(ctx, c.dout, c.dtype))
    ctx.sync()
    assert np.isnan(d.out.get()).all()


def test_many_sequences(ctx):
    lens = SELF(*rng(20).integers(0, 4, 3000).tolist())
    c = Case(20, "bf16", 32, 1, 1, lens)
    d = OnDevice(ctx, c)
    d.forward()
    check_forward(d)
    check_backward(ctx, d)


def test_nothing_to_do(ctx):
    c = Case(21, "f32", 16, 1, 1, SELF(4))
    d = OnDevice(ctx, c)
    before = d.out.bits().copy()
    sizes = list(d.sizes)
    sizes[0] = 0
    ctx.attention_fwd(d.q, d.k, d.v, d.out, d.q_starts, d.k_starts, *sizes, dtype="f32")
    ctx.attention_fwd(None, None, None, None, None, None, 0, 0, 0, 1, 1, 16, dtype="f32")
    assert (d.out.bits() == before).all()
    keyless = Case(21, "f32", 16, 1, 1, [(4, 0)])
    d = OnDevice(ctx, keyless)
    d.k = d.v = None
    d.forward()
    assert (d.out.get() == 0).all() and np.isneginf(d.lse.get()).all()


def test_refusals(ctx):
    from ferrograd_b200.backend import FgError
    c = Case(22, "bf16", 64, 4, 2, SELF(16))
    d = OnDevice(ctx, c)
    t = Placed(ctx, c.dout, "bf16"), Placed(ctx, np.zeros((4, 16))), Placed(ctx, c.dout, "bf16")

    def fwd(q=d.q, k=d.k, v=d.v, out=d.out, qs=d.q_starts, ks=d.k_starts, sizes=d.sizes, **more):
        ctx.attention_fwd(q, k, v, out, qs, ks, *sizes, **{**d.more, **more})

    def bwd(out=t[0], lse=t[1], dout=t[2], sizes=d.sizes, dq=d.dq, dk=d.dk, dv=d.dv, **more):
        ctx.attention_bwd(d.q, d.k, d.v, out, lse, dout, d.q_starts, d.k_starts, *sizes, dq=dq, dk=dk, dv=dv, **{**d.more, **more})

    fwd()
    bwd()
    s = d.sizes
    bad = [lambda: fwd(q=None), lambda: fwd(k=None), lambda: fwd(v=None), lambda: fwd(out=None), lambda: fwd(qs=None), lambda: fwd(ks=None),
           lambda: fwd(sizes=(*s[:3], 4, 3, 64)), lambda: fwd(sizes=(*s[:3], 4, 0, 64)), lambda: fwd(sizes=(*s[:3], 0, 1, 64)),
           lambda: fwd(sizes=(*s[:3], 4, 2, 0)), lambda: fwd(sizes=(*s[:3], 4, 2, 257)), lambda: fwd(sizes=(1, 1 << 31, 16, 4, 2, 64)),
           lambda: fwd(sizes=(1, 16, 1 << 31, 4, 2, 64)), lambda: fwd(scale=float("nan")), lambda: fwd(scale=float("inf")),
           lambda: fwd(q_stride=255), lambda: fwd(k_stride=127), lambda: fwd(v_stride=1), lambda: fwd(q_stride=1 << 40), lambda: fwd(q=d.q + 1),
           lambda: fwd(out=d.q), lambda: fwd(out=d.v), lambda: fwd(out=d.k + 64), lambda: fwd(lse=d.q), lambda: fwd(lse=d.out.ptr), lambda: fwd(out=d.q_starts),
           lambda: bwd(out=None), lambda: bwd(lse=None), lambda: bwd(dout=None), lambda: bwd(dq=None, dk=None, dv=None), lambda: bwd(dk=None),
           lambda: bwd(dv=None), lambda: bwd(dq=d.q), lambda: bwd(dk=d.v), lambda: bwd(dv=t[2].ptr), lambda: bwd(dk=d.dq), lambda: bwd(dv=d.dk + 2),
           lambda: bwd(dv=d.dk)]
    for i, f in enumerate(bad):
        with pytest.raises(FgError) as e:
            f()
        assert e.value.kind == "FG_ERR_INVALID_ARGUMENT", i
    with pytest.raises(KeyError):
        fwd(dtype="f64")
    assert ctx.device_status() == 0
