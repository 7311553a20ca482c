"""A decoder block's operators where an element's offset passes 32 bits: the same calls on the same numbers, near and far, give the same bits."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ctx():
    import torch
    from ferrograd_b200 import GpuContext
    c = GpuContext(0)
    yield c
    assert c.device_status() == 0
    c.destroy()
    torch.cuda.empty_cache()


def ready(ctx, run):
    import torch
    torch.cuda.synchronize()
    run()
    ctx.sync()


def normal(*shape, seed, dtype="bfloat16"):
    import torch
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(getattr(torch, dtype)).cuda()


# The keys' tokens lie 2^21 elements apart, 2200 of them: the last starts at 4.6e9.
@pytest.mark.parametrize("dtype,name", [("bf16", "bfloat16"), ("f32", "float32")])
@pytest.mark.parametrize("queries", [1, 300])
def test_attention(ctx, dtype, name, queries):
    import torch
    keys, heads, kv, dim, stride = 2200, 4, 2, 64, 1 << 21
    line = kv * dim
    near = {n: normal(keys, line, seed=s, dtype=name) for s, n in enumerate("kv")}
    q, dout = (normal(queries, heads * dim, seed=s, dtype=name) for s in (7, 8))
    starts = torch.tensor([0, queries, 0, keys], dtype=torch.int32).cuda()
    sizes = (starts.data_ptr(), starts.data_ptr() + 8, 1, queries, keys, heads, kv, dim)
    far, grads = (torch.empty((keys - 1) * stride + 2 * line, dtype=near["k"].dtype, device="cuda") for _ in range(2))
    columns = lambda t: t.as_strided((keys, 2 * line), (stride, 1))   # noqa: E731
    columns(far).copy_(torch.cat([near["k"], near["v"]], 1))
    size, got = q.element_size(), {}
    for where in ("near", "far"):
        out, dq = torch.empty_like(q), torch.empty_like(q)
        lse = torch.empty(heads, queries, device="cuda")
        dk, dv = torch.empty_like(near["k"]), torch.empty_like(near["v"])
        if where == "near":
            k, v, gk, gv, extra = near["k"].data_ptr(), near["v"].data_ptr(), dk.data_ptr(), dv.data_ptr(), {}
        else:
            k, gk = far.data_ptr(), grads.data_ptr()
            v, gv, extra = k + line * size, gk + line * size, dict(k_stride=stride, v_stride=stride)
        ready(ctx, lambda: ctx.attention_fwd(q.data_ptr(), k, v, out.data_ptr(), *sizes, lse=lse.data_ptr(), dtype=dtype, **extra))
        ready(ctx, lambda: ctx.attention_bwd(q.data_ptr(), k, v, out.data_ptr(), lse.data_ptr(), dout.data_ptr(), *sizes, dq=dq.data_ptr(), dk=gk, dv=gv,
                                             dtype=dtype, **extra))
        if where == "far":
            dk, dv = columns(grads)[:, :line], columns(grads)[:, line:]
        got[where] = (out, lse, dq, dk, dv)
    for a, b in zip(got["near"], got["far"]):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())


# The last rows of 2^20 + 5 of 4096 columns, and of 70001 of 65551 (which no thread group holds).
@pytest.mark.parametrize("rows,cols", [((1 << 20) + 5, 4096), (70001, 65551)])
def test_rmsnorm(ctx, rows, cols):
    import torch
    tail = 1000
    last, dlast = (normal(tail, cols, seed=s) for s in (1, 2))
    gamma = normal(cols, seed=3)
    far, dfar = (torch.ones(rows, cols, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    far[-tail:], dfar[-tail:] = last, dlast
    got = []
    for n, x, dy in ((tail, last, dlast), (rows, far, dfar)):
        rstd, y = torch.empty(n, device="cuda"), torch.empty_like(x)
        ready(ctx, lambda: ctx.rmsnorm_fwd(x.data_ptr(), gamma.data_ptr(), y.data_ptr(), n, cols, rstd=rstd.data_ptr(), dtype="bf16"))
        got.append((rstd[-tail:], y[-tail:].clone()))
        ready(ctx, lambda: ctx.rmsnorm_bwd(x.data_ptr(), dy.data_ptr(), gamma.data_ptr(), rstd.data_ptr(), n, cols, dx=y.data_ptr(), dtype="bf16"))
        got[-1] += (y[-tail:],)
    for a, b in zip(*got):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())


# 140001 rows of 32001: the last rows; few of them would be shared out differently.
def test_logprobs(ctx):
    import torch
    rows, cols, tail = 140001, 32001, 1200
    last = normal(tail, cols, seed=1)
    far = torch.ones(rows, cols, dtype=torch.bfloat16, device="cuda")
    far[-tail:] = last
    got = []
    for n, x in ((tail, last), (rows, far)):
        t = (torch.arange(n, dtype=torch.int32) - n + tail).remainder(cols).to(torch.int32).cuda()
        logprob, lse, entropy, g = (torch.empty(n, device="cuda") for _ in range(4))
        g.fill_(0.5)
        dx = torch.empty_like(x)
        ready(ctx, lambda: ctx.logprobs_fwd(x.data_ptr(), t.data_ptr(), logprob.data_ptr(), n, cols, entropy=entropy.data_ptr(), lse=lse.data_ptr(), dtype="bf16"))
        ready(ctx, lambda: ctx.logprobs_bwd(x.data_ptr(), t.data_ptr(), lse.data_ptr(), n, cols, dx.data_ptr(), dlogprob=g.data_ptr(), entropy=entropy.data_ptr(),
                                            dentropy=g.data_ptr(), dtype="bf16"))
        got.append((logprob[-tail:], lse[-tail:], entropy[-tail:], dx[-tail:]))
    # The rows start at other distances from 16-byte boundaries, so the sums are of other parts.  With n = cols / 32 + 64 additions in a chain and U = 2^-24, n U is
    # 6.4e-5; lse is off by n U and entropy by (1 + 2 * 5) n U at most (the mean distance from the largest is below 5), on either side: 1.4e-3 < 2^-9.  A gradient:
    # a rounding to bf16 on either side, and of the largest probability, 1.7e-3, half of 1.4e-3: 1.2e-6 < 2^-18.
    for a, b in zip(got[0][:3], got[1][:3]):
        assert bool(((a - b).abs() <= 2.0 ** -9).all())
    assert bool(((got[0][3].float() - got[1][3].float()).abs() <= 2.0 ** -7 * got[0][3].float().abs() + 2.0 ** -18).all())


# As many rows of one column as there are numbers for: a log probability of one choice is zero.
def test_rows_to_the_last_number(ctx):
    import torch
    rows = (1 << 32) - 3
    x = torch.full((rows,), -1.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(rows, device="cuda")
    ready(ctx, lambda: ctx.logprobs_fwd(x.data_ptr(), None, None, rows, 1, lse=lse.data_ptr(), dtype="bf16"))
    assert bool((lse[-1000:] == -1.0).all()) and bool((lse[:1000] == -1.0).all()) and float(lse.min()) == float(lse.max()) == -1.0
