"""The operators of a decoder block together, as a program uses them: lookup, root-mean-square norm, attention over packed sequences, the residual's addition with
the next norm, the head and its log probabilities, trained by a policy's loss and generating token by token over a cache.  Tolerance: that of the matrix
products, 1e-4 of the value and the rms."""
import numpy as np
import pytest
import torch

from conftest import rel_err_ok

pytestmark = pytest.mark.gpu
TOL = 1e-4
EPS, SCALE = 1e-5, 1.25


def rng(*key):
    return np.random.Generator(np.random.Philox(key))


class Block:
    def __init__(self, ctx, vocab, dim, heads, kv, tokens, lens, seed=0):
        r = rng(seed)
        self.ctx, self.vocab, self.dim, self.heads, self.kv, self.tokens, self.lens = ctx, vocab, dim, heads, kv, tokens, lens
        self.hd = dim // heads
        self.row = (heads + 2 * kv) * self.hd
        self.p = {"E": r.standard_normal((vocab, dim)), "g1": 1 + 0.1 * r.standard_normal(dim), "Wqkv": 1.5 * r.standard_normal((dim, self.row)) * dim ** -0.5,
                  "Wo": r.standard_normal((dim, dim)) * dim ** -0.5, "g2": 1 + 0.1 * r.standard_normal(dim), "Wu": 2 * r.standard_normal((dim, vocab)) * dim ** -0.5}
        self.p = {k: v.astype(np.float32) for k, v in self.p.items()}
        self.d = {k: ctx.init_tensor_f32(v.shape, v) for k, v in self.p.items()}
        self.grad = {k: ctx.init_tensor_f32(v.shape, np.zeros_like(v)) for k, v in self.p.items()}
        new = lambda *s: ctx.new_tensor(s)   # noqa: E731
        u32 = lambda a: ctx.init_tensor_u32((len(a),), np.asarray(a, np.uint32))   # noqa: E731
        self.ids, self.targets = u32(np.zeros(tokens)), u32(np.zeros(tokens))
        self.starts = u32(np.concatenate([[0], np.cumsum(lens)]))
        self.x0, self.h1, self.a, self.o, self.x1, self.h2 = (new(tokens, dim) for _ in range(6))
        self.qkv, self.dqkv = new(tokens, self.row), new(tokens, self.row)
        self.r1, self.r2, self.logp, self.ent, self.lz = (new(tokens) for _ in range(5))
        self.lse, self.logits, self.dlogits = new(heads, tokens), new(tokens, vocab), new(tokens, vocab)
        self.dh2, self.dx1, self.da, self.dh1, self.dx0 = (new(tokens, dim) for _ in range(5))
        self.gl, self.ge = new(tokens), new(tokens)

    def parts(self, t):
        return t.ptr, t.ptr + 4 * self.heads * self.hd, t.ptr + 4 * (self.heads + self.kv) * self.hd

    def sizes(self):
        return len(self.lens), self.tokens, self.tokens, self.heads, self.kv, self.hd

    def forward(self):
        c, n, dim, s = self.ctx, self.tokens, self.dim, dict(q_stride=self.row, k_stride=self.row, v_stride=self.row, dtype="f32")
        c.embedding_fwd(self.d["E"], self.ids, self.x0, n, self.vocab, dim)
        c.rmsnorm_fwd(self.x0, self.d["g1"], self.h1, n, dim, eps=EPS, rstd=self.r1)
        c.gemm(self.h1, self.d["Wqkv"], self.qkv, n, self.row, dim)
        q, k, v = self.parts(self.qkv)
        c.attention_fwd(q, k, v, self.a, self.starts, self.starts, *self.sizes(), lse=self.lse, **s)
        c.gemm(self.a, self.d["Wo"], self.o, n, dim, dim)
        c.rmsnorm_fwd(self.o, self.d["g2"], self.h2, n, dim, eps=EPS, residual=self.x0, sum=self.x1, rstd=self.r2)
        c.gemm(self.h2, self.d["Wu"], self.logits, n, self.vocab, dim)
        c.logprobs_fwd(self.logits, self.targets, self.logp, n, self.vocab, scale=SCALE, entropy=self.ent, lse=self.lz)

    def backward(self):
        c, n, dim, s = self.ctx, self.tokens, self.dim, dict(q_stride=self.row, k_stride=self.row, v_stride=self.row, dtype="f32")
        c.logprobs_bwd(self.logits, self.targets, self.lz, n, self.vocab, self.dlogits, scale=SCALE, dlogprob=self.gl, entropy=self.ent, dentropy=self.ge)
        c.gemm_bwd(self.h2, self.d["Wu"], self.dlogits, n, self.vocab, dim, dA=self.dh2, dB=self.grad["Wu"])
        c.rmsnorm_bwd(self.x1, self.dh2, self.d["g2"], self.r2, n, dim, dx=self.dx1, dgamma=self.grad["g2"])
        c.gemm_bwd(self.a, self.d["Wo"], self.dx1, n, dim, dim, dA=self.da, dB=self.grad["Wo"])
        (q, k, v), (dq, dk, dv) = self.parts(self.qkv), self.parts(self.dqkv)
        c.attention_bwd(q, k, v, self.a, self.lse, self.da, self.starts, self.starts, *self.sizes(), dq=dq, dk=dk, dv=dv, **s)
        c.gemm_bwd(self.h1, self.d["Wqkv"], self.dqkv, n, self.row, dim, dA=self.dh1, dB=self.grad["Wqkv"])
        c.rmsnorm_bwd(self.x0, self.dh1, self.d["g1"], self.r1, n, dim, dx=self.dx0, dgamma=self.grad["g1"], dsum=self.dx1)
        c.embedding_bwd(self.ids, self.dx0, self.grad["E"], n, self.vocab, dim)

    def feed(self, ids, targets, gl, ge):
        for t, v in ((self.ids, ids), (self.targets, targets), (self.gl, gl), (self.ge, ge)):
            self.ctx.upload(t.data, v)


def block64(p, b, ids, targets, gl, ge):
    """Log probabilities, entropies and gradients in 64 bits, by differentiation."""
    t = {k: torch.tensor(v, dtype=torch.float64, requires_grad=True) for k, v in p.items()}
    norm = lambda h, g: h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * g   # noqa: E731
    x0 = t["E"][torch.tensor(ids.astype(np.int64))]
    qkv = norm(x0, t["g1"]) @ t["Wqkv"]
    q, k, v = qkv.split((b.heads * b.hd, b.kv * b.hd, b.kv * b.hd), 1)
    out, at = [], 0
    for n in b.lens:
        i = slice(at, at + n)
        at += n
        heads = lambda x, h: x[i].reshape(n, h, b.hd).transpose(0, 1).repeat_interleave(b.heads // h, 0)   # noqa: E731
        s = heads(q, b.heads) @ heads(k, b.kv).transpose(1, 2) * b.hd ** -0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -torch.inf)
        out.append((torch.softmax(s, 2) @ heads(v, b.kv)).transpose(0, 1).reshape(n, -1))
    x1 = x0 + torch.cat(out) @ t["Wo"]
    logp = torch.log_softmax(SCALE * (norm(x1, t["g2"]) @ t["Wu"]), 1)
    there = torch.tensor(targets < b.vocab)
    pick = torch.where(there, logp[torch.arange(len(ids)), torch.tensor(np.where(targets < b.vocab, targets, 0).astype(np.int64))], 0.0)
    ent = torch.where(there, -(logp.exp() * logp).sum(1), 0.0)
    ((pick * torch.tensor(gl)).sum() + (ent * torch.tensor(ge)).sum()).backward()
    return pick.detach().numpy(), ent.detach().numpy(), {k: x.grad.numpy() for k, x in t.items()}


@pytest.fixture()
def ctx():
    from ferrograd_b200 import GpuContext
    c = GpuContext(0)
    yield c
    assert c.device_status() == 0
    c.destroy()


def batch(r, b):
    ids = r.integers(0, b.vocab, b.tokens).astype(np.uint32)
    targets = np.roll(ids, -1)
    targets[np.cumsum(b.lens) - 1] = 0xffffffff          # the last token of a sequence has no next one
    return ids, targets, r.standard_normal(b.tokens).astype(np.float32), (0.1 * r.standard_normal(b.tokens)).astype(np.float32)


@pytest.mark.parametrize("vocab,dim,heads,kv,lens", [(101, 64, 4, 2, (40, 1, 70)), (500, 256, 8, 1, (300, 33)), (77, 96, 3, 3, (129,))])
def test_policy_step(ctx, vocab, dim, heads, kv, lens):
    eager, recorded = (Block(ctx, vocab, dim, heads, kv, sum(lens), lens) for _ in range(2))
    r = rng(vocab)
    data = batch(r, eager)
    for b in (eager, recorded):          # one step each, which also sizes the arena
        b.feed(*data)
        b.forward()
        b.backward()
    logp, ent, want = block64(eager.p, eager, *data)
    for name, got, ref in [("logprob", ctx.to_numpy(eager.logp), logp), ("entropy", ctx.to_numpy(eager.ent), ent)] + [("grad " + k, ctx.to_numpy(eager.grad[k]), v) for k, v in want.items()]:
        ok, worst = rel_err_ok(got, ref, TOL)
        assert ok, f"{name}: {worst:.3g}"
    ctx.plan_begin()
    recorded.forward()
    recorded.backward()
    plan = ctx.plan_end()
    for _ in range(2):
        data = batch(r, eager)
        for b in (eager, recorded):
            b.feed(*data)
        eager.forward()
        eager.backward()
        plan.launch()
    for k in want:
        ok, worst = rel_err_ok(ctx.to_numpy(recorded.grad[k]), ctx.to_numpy(eager.grad[k]), 1e-5)          # (small sums add in another order in a plan)
        assert ok, f"{k}: {worst:.3g}"
    plan.destroy()


def test_generating_over_a_cache(ctx):
    # the same tokens one at a time for two requests, their keys in slots of a cache: the log probabilities of the whole pass
    lens = (23, 23)
    whole = Block(ctx, 150, 64, 4, 2, 46, lens)
    r = rng(7)
    ids, targets, gl, ge = batch(r, whole)
    whole.feed(ids, targets, gl, ge)
    whole.forward()
    want = ctx.to_numpy(whole.logp).reshape(2, 23)
    step = Block(ctx, 150, 64, 4, 2, 2, (1, 1))
    step.d = whole.d
    slot, line = 30, 2 * 16
    cache = [ctx.init_tensor_f32((2 * slot, line), np.full((2 * slot, line), np.nan, np.float32)) for _ in range(2)]
    starts = ctx.init_tensor_u32((3,), np.array([0, slot, 2 * slot], np.uint32))
    used = ctx.init_tensor_u32((2,), np.zeros(2, np.uint32))
    ids, targets = ids.reshape(2, 23), targets.reshape(2, 23)
    for i in range(23):
        step.feed(ids[:, i], targets[:, i], gl[:2], ge[:2])
        ctx.upload(used.data, np.full(2, i + 1, np.uint32))
        c, dim = ctx, 64
        c.embedding_fwd(step.d["E"], step.ids, step.x0, 2, 150, dim)
        c.rmsnorm_fwd(step.x0, step.d["g1"], step.h1, 2, dim, eps=EPS)
        c.gemm(step.h1, step.d["Wqkv"], step.qkv, 2, step.row, dim)
        q, k, v = step.parts(step.qkv)
        for b in range(2):
            for t, at in zip(cache, (k, v)):
                c.copy_dev_async(t.ptr + 4 * line * (b * slot + i), at + 4 * step.row * b, 4 * line)
        c.attention_fwd(q, cache[0], cache[1], step.a, step.starts, starts, 2, 2, 2 * slot, 4, 2, 16, q_stride=step.row, k_lengths=used, dtype="f32")
        c.gemm(step.a, step.d["Wo"], step.o, 2, dim, dim)
        c.rmsnorm_fwd(step.o, step.d["g2"], step.h2, 2, dim, eps=EPS, residual=step.x0)
        c.gemm(step.h2, step.d["Wu"], step.logits, 2, 150, dim)
        c.logprobs_fwd(step.logits, step.targets, step.logp, 2, 150, scale=SCALE)
        ok, worst = rel_err_ok(c.to_numpy(step.logp), want[:, i], TOL)
        assert ok, f"token {i}: {worst:.3g}"
