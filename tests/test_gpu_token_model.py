"""The token operators together, as a program uses them: a model of tokens (lookup, layer norm, a dense layer, softmax and cross-entropy) trained
step by step, eager and recorded, and its next tokens drawn.  Tolerance: that of the matrix products, 1e-4 of the value and the rms."""
import numpy as np
import pytest

from conftest import rel_err_ok
from test_gpu_sample import definition
from token_ops import empty, Placed

pytestmark = pytest.mark.gpu
TOL = 1e-4
SCALE, EPS, LR = 2.0, 1e-5, 0.05


class Model:
    def __init__(self, ctx, vocab, dim, tokens, seed=0):
        r = np.random.Generator(np.random.Philox(seed))
        self.ctx, self.vocab, self.dim, self.tokens = ctx, vocab, dim, tokens
        self.p = {"E": 0.5 * r.standard_normal((vocab, dim)), "g": 1 + 0.1 * r.standard_normal(dim), "b": 0.1 * r.standard_normal(dim),
                  "W": r.standard_normal((dim, vocab)) * dim ** -0.5, "c": 0.1 * r.standard_normal(vocab)}
        self.p = {k: v.astype(np.float32) for k, v in self.p.items()}
        self.d = {k: ctx.init_tensor_f32(v.shape, v) for k, v in self.p.items()}
        self.grad = {k: ctx.init_tensor_f32(v.shape, np.zeros_like(v)) for k, v in self.p.items()}
        self.ids, self.labels = (ctx.init_tensor_u32((tokens,), np.zeros(tokens, np.uint32)) for _ in range(2))
        new = lambda *s: ctx.new_tensor(s)   # noqa: E731
        self.x, self.h, self.dh, self.dx = (new(tokens, dim) for _ in range(4))
        self.mean, self.rstd, self.loss, self.loss_mean = new(tokens), new(tokens), new(tokens), new(1)
        self.logits, self.dlogits = new(tokens, vocab), new(tokens, vocab)

    def feed(self, ids, labels):
        self.ctx.upload(self.ids.data, ids)
        self.ctx.upload(self.labels.data, labels)

    def forward(self, tokens=None):
        c, n = self.ctx, tokens or self.tokens
        c.embedding_fwd(self.d["E"], self.ids, self.x, n, self.vocab, self.dim, scale=SCALE)
        c.layernorm_fwd(self.x, self.d["g"], self.d["b"], self.h, n, self.dim, eps=EPS, mean=self.mean, rstd=self.rstd)
        c.gemm(self.h, self.d["W"], self.logits, n, self.vocab, self.dim, bias=self.d["c"])

    def backward(self):
        c, n = self.ctx, self.tokens
        c.softmax_ce(self.logits, self.labels, n, self.vocab, grad_scale=1.0 / n, loss_row=self.loss, loss_mean=self.loss_mean, dlogits=self.dlogits)
        c.gemm_bwd(self.h, self.d["W"], self.dlogits, n, self.vocab, self.dim, dA=self.dh, dB=self.grad["W"], dbias=self.grad["c"])
        c.layernorm_bwd(self.x, self.dh, self.d["g"], self.mean, self.rstd, n, self.dim, dx=self.dx, dgamma=self.grad["g"], dbeta=self.grad["b"])
        c.embedding_bwd(self.ids, self.dx, self.grad["E"], n, self.vocab, self.dim, scale=SCALE, accumulate=True)

    def update(self):
        self.ctx.sgd_step_multi([{"w": self.d[k], "g": self.grad[k], "n": v.size} for k, v in self.p.items()], LR)      # leaves the gradients at zero

    def numpy(self, tensors):
        return {k: self.ctx.to_numpy(v) for k, v in tensors.items()}


def step64(p, ids, labels):
    """Loss, logits and gradients in 64 bits."""
    p = {k: v.astype(np.float64) for k, v in p.items()}
    n, inside = len(ids), ids < p["E"].shape[0]
    x = np.where(inside[:, None], SCALE * p["E"][np.where(inside, ids, 0)], 0.0)
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + EPS)
    xh = (x - mean) * rstd
    h = xh * p["g"] + p["b"]
    z = h @ p["W"] + p["c"]
    logp = z - z.max(1, keepdims=True)
    logp -= np.log(np.exp(logp).sum(1, keepdims=True))
    dz = np.exp(logp)
    dz[np.arange(n), labels] -= 1
    dz /= n
    dh = dz @ p["W"].T
    gh = dh * p["g"]
    dx = rstd * (gh - gh.mean(1, keepdims=True) - xh * (gh * xh).mean(1, keepdims=True))
    dE = np.zeros_like(p["E"])
    np.add.at(dE, ids[inside], SCALE * dx[inside])
    return -logp[np.arange(n), labels].mean(), z, {"E": dE, "g": (dh * xh).sum(0), "b": dh.sum(0), "W": h.T @ dz, "c": dz.sum(0)}


@pytest.fixture()
def ctx():
    from ferrograd_b200 import GpuContext
    c = GpuContext(0)
    yield c
    assert c.device_status() == 0
    c.destroy()


def batch(r, tokens, vocab):
    ids = np.minimum(np.exp(r.random(tokens) * np.log(vocab + 1)) - 1, vocab - 1).astype(np.uint32)
    labels = ((ids * 7 + 3) % vocab).astype(np.uint32)
    ids[tokens - tokens // 8:] = 0xffffffff          # the end of the batch is padding
    return ids, labels


@pytest.mark.parametrize("vocab,dim,tokens", [(50, 48, 96), (1000, 256, 640), (333, 77, 1500)])
def test_training_steps(ctx, vocab, dim, tokens):
    r = np.random.Generator(np.random.Philox(vocab))
    m, recorded = Model(ctx, vocab, dim, tokens), Model(ctx, vocab, dim, tokens)
    batches = [batch(r, tokens, vocab) for _ in range(4)]
    for m_ in (m, recorded):          # one step each, which also sizes the arena
        m_.feed(*batches[0])
        m_.forward()
        m_.backward()
        loss, z, want = step64(m_.p, *batches[0])
        for name, got, ref in [("loss", ctx.to_numpy(m_.loss_mean), [loss]), ("logits", ctx.to_numpy(m_.logits), z)] + \
                [("grad " + k, v, want[k]) for k, v in m_.numpy(m_.grad).items()]:
            ok, worst = rel_err_ok(got, ref, TOL)
            assert ok, f"{name}: {worst:.3g}"
        m_.update()
        got = m_.numpy(m_.d)
        for k, v in want.items():
            ok, worst = rel_err_ok(got[k], m_.p[k] - LR * v, TOL)
            assert ok, f"{k}: {worst:.3g}"
        assert all(not g.any() for g in m_.numpy(m_.grad).values())
    ctx.plan_begin()
    recorded.forward()
    recorded.backward()
    recorded.update()
    plan = ctx.plan_end()
    for ids, labels in batches[1:]:
        for m_ in (m, recorded):
            m_.feed(ids, labels)
        m.forward()
        m.backward()
        m.update()
        plan.launch()
    a, b = m.numpy(m.d), recorded.numpy(recorded.d)
    plan.destroy()
    for k in a:
        ok, worst = rel_err_ok(b[k], a[k], 1e-6)          # (small sums add in another order in a plan)
        assert ok, f"{k}: {worst:.3g}"


def test_generating(ctx):
    # token by token: one row through the model, the next token drawn and fed back on the device
    vocab, dim = 400, 64
    r = np.random.Generator(np.random.Philox(3))
    m = Model(ctx, vocab, dim, 1)
    u = r.random(12).astype(np.float32)
    params = {"temperature": np.full(1, 0.8, np.float32), "top_k": np.full(1, 40, np.uint32), "top_p": np.full(1, 0.9, np.float32), "min_p": np.full(1, 0.02, np.float32)}
    dev = {k: Placed(ctx, v, "u32" if k == "top_k" else "f32") for k, v in params.items()}
    draws, drawn = Placed(ctx, u), empty(ctx, (12,), "u32")
    m.feed(np.array([5], np.uint32), np.zeros(1, np.uint32))
    rows = []
    for i in range(12):
        m.forward(1)
        rows.append(ctx.to_numpy(m.logits)[0])
        ctx.sample(m.logits, draws.ptr + 4 * i, m.ids, 1, vocab, **dev)
        ctx.copy_dev_async(drawn.ptr + 4 * i, m.ids, 4)
    got = drawn.get()
    for i in range(12):
        assert got[i] == definition(rows[i], u[i], params["temperature"][0], int(params["top_k"][0]), params["top_p"][0], params["min_p"][0])[0]


def test_two_contexts_at_once():
    # two streams, each with a workspace of its own, work without waiting for each other
    from ferrograd_b200 import GpuContext
    r = np.random.Generator(np.random.Philox(9))
    vocab, dim, tokens = 700, 128, 3000
    models = [Model(GpuContext(0), vocab, dim, tokens, seed) for seed in (1, 2)]
    data = [batch(r, tokens, vocab) for _ in models]
    for m, d in zip(models, data):
        m.feed(*d)
    for _ in range(3):
        for m in models:
            m.forward()
        for m in models:
            m.backward()
    for m, d in zip(models, data):
        want = step64(m.p, *d)[2]
        for k, v in m.numpy(m.grad).items():
            ok, worst = rel_err_ok(v, 3 * want[k] if k == "E" else want[k], TOL)          # the table's gradient adds up
            assert ok, f"{k}: {worst:.3g}"
        assert m.ctx.device_status() == 0
        m.ctx.destroy()
