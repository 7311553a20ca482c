"""The largest scales of attention and of log probabilities: the powers of two that the exponentials are made of have to stay numbers."""
import numpy as np
import pytest

from token_ops import empty, Placed

pytestmark = pytest.mark.gpu
LARGEST, BEYOND = float(np.float32(2.0 ** 127)), (float(np.nextafter(np.float32(2.0 ** 127), np.float32(np.inf))), 2.4e38, 3.4028234e38)


@pytest.fixture()
def ctx():
    from ferrograd_b200 import GpuContext
    c = GpuContext(0)
    yield c
    assert c.device_status() == 0
    c.destroy()


def refused(f):
    from ferrograd_b200.backend import FgError
    with pytest.raises(FgError) as e:
        f()
    assert e.value.kind == "FG_ERR_INVALID_ARGUMENT"


@pytest.mark.parametrize("rows,cols,top", [(2, 40, 3), (2, 9000, 0), (700, 64, 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_logprobs(ctx, rows, cols, top, dtype):
    # the largest logit has all of the weight
    x = -np.ones((rows, cols))
    x[:, 7] = 0.0
    d, t = Placed(ctx, x, dtype), Placed(ctx, np.where(np.arange(rows) % 2, 7, 8).astype(np.uint32), "u32")
    logp, ent, lse = (empty(ctx, (rows,)) for _ in range(3))
    ids, lps = (empty(ctx, (rows, top), "u32"), empty(ctx, (rows, top))) if top else (None, None)

    def forward(scale):
        ctx.logprobs_fwd(d, t, logp, rows, cols, scale=scale, entropy=ent, lse=lse, top=top, top_ids=ids, top_logprobs=lps, dtype=dtype)

    forward(LARGEST)
    assert (lse.get() == 0).all() and (ent.get() == 0).all()
    assert np.array_equal(logp.get(), np.where(np.arange(rows) % 2, 0.0, -LARGEST).astype(np.float32))
    if top:
        assert (ids.get()[:, 0] == 7).all() and (lps.get()[:, 0] == 0).all() and (lps.get()[:, 1:] == -LARGEST).all()
    g, one = empty(ctx, (rows, cols), dtype), Placed(ctx, np.full(rows, 2.0 ** -127))

    def backward(scale):
        ctx.logprobs_bwd(d, t, lse, rows, cols, g, scale=scale, dlogprob=one, dtype=dtype)

    backward(LARGEST)
    want = np.zeros((rows, cols))
    want[::2, 8], want[::2, 7] = 1, -1
    assert np.array_equal(g.get(), want)
    for scale in BEYOND:
        refused(lambda: forward(scale))
        refused(lambda: backward(scale))


@pytest.mark.parametrize("dtype,dim", [("f32", 32), ("f16", 64), ("bf16", 128), ("bf16", 36)])
@pytest.mark.parametrize("queries", [1, 200])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention(ctx, dtype, dim, queries, sign):
    # key 3 has a score of zero, the others one far below: its value comes out
    r = np.random.Generator(np.random.Philox(dim))
    q, k = np.ones((queries, dim)), np.full((60, dim), -1.0 * sign)
    k[3] = 0.0
    v = r.integers(-9, 10, (60, dim))
    starts = Placed(ctx, np.array([0, queries, 0, 60]), "u32")
    t = [Placed(ctx, x, dtype) for x in (q, k, v)]
    out, lse = empty(ctx, (queries, dim), dtype), empty(ctx, (1, queries))

    def forward(scale):
        ctx.attention_fwd(*t, out, starts.ptr, starts.ptr + 8, 1, queries, 60, 1, 1, dim, scale=scale, causal=False, lse=lse, dtype=dtype)

    forward(sign * LARGEST)
    assert (out.get() == v[3]).all() and (lse.get() == 0).all()
    for scale in BEYOND:
        refused(lambda: forward(sign * scale))
