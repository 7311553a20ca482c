"""The 8-bit form of the root-mean-square norm: its bytes as they are defined, and more rows than 31 bits count."""
import numpy as np
import pytest

from test_gpu_rmsnorm import Bytes, e4m3_values
from token_ops import empty, Placed

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ctx():
    from ferrograd_b200 import GpuContext
    c = GpuContext(0)
    yield c
    assert c.device_status() == 0
    c.destroy()


def test_rows_beyond_31_bits(ctx):
    # one column: y is 1 / sqrt(1 + eps / 4) with the sign of x, its own largest, so 448 in its bytes
    import torch
    rows = (1 << 31) + 5
    x = torch.full((rows,), -2.0, dtype=torch.bfloat16, device="cuda")
    x[-3:] = 2.0
    y = torch.zeros(rows, dtype=torch.uint8, device="cuda")
    scale = torch.zeros(rows, device="cuda")
    torch.cuda.synchronize()
    ctx.rmsnorm_fwd_e4m3(x.data_ptr(), None, y.data_ptr(), scale.data_ptr(), rows, 1, eps=1e-5, dtype="bf16")
    ctx.sync()
    byte = {v: b for b, v in enumerate(e4m3_values().tolist())}
    assert int(y[:-3].min()) == int(y[:-3].max()) == byte[-448.0] and y[-3:].tolist() == [byte[448.0]] * 3
    want = (1 + 1e-5 / 4) ** -0.5 / 448          # (off by less than 16 steps of 2^-24)
    assert abs(float(scale.min()) / want - 1) <= 2.0 ** -20 and float(scale.min()) == float(scale.max())
    del x, y, scale
    torch.cuda.empty_cache()


def from_quotients(q):
    """The bytes of f32 numbers, to nearest even (no larger than 448 after it)."""
    import torch
    return torch.tensor(np.minimum(np.maximum(q, -448), 448)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


# The forms: packs held by threads, by elements (a warp a row, a block a row), read once per sum.
@pytest.mark.parametrize("cols", [4096, 96, 1001, 3999, 20000, 70001])
@pytest.mark.parametrize("group", [0, 32, 128, 256])
def test_borders_between_bytes(ctx, cols, group):
    # x is 1 everywhere, so y is gamma times the row's rstd, rounded once.  gamma places y / scale on the borders between neighbouring bytes, and two steps of f32 on either side.
    rows = 3
    r = np.random.Generator(np.random.Philox([cols, group]))
    values = e4m3_values()[:127]
    borders = np.concatenate([(values[:-1] + values[1:]) / 2] * 2)
    groups = -(-cols // group) if group else 1
    each = group or cols
    x = Placed(ctx, np.ones((rows, cols)))
    gamma = np.ones(cols, np.float32)
    for eps in (1e-5, 0.3, 2.7):
        def run():
            q, scale, rstd = Bytes(ctx, rows * cols, 0), empty(ctx, (rows, groups)), empty(ctx, (rows,))
            ctx.rmsnorm_fwd_e4m3(x, Placed(ctx, gamma), q, scale, rows, cols, group=group, eps=eps, rstd=rstd, dtype="f32")
            return q.get().reshape(rows, cols), scale.get(), rstd.get()
        rstd = run()[2][0]
        for g in range(groups):
            c0, c1 = g * each, min(cols, (g + 1) * each)
            largest = np.float32(1 + 3 * r.random())
            scale = np.float32(np.float32(largest * rstd) / np.float32(448))
            at = np.float32(r.choice(borders, c1 - c0) * float(scale) / float(rstd) * r.choice((-1, 1), c1 - c0))
            at = (at.view(np.int32) + r.integers(-2, 3, c1 - c0).astype(np.int32)).view(np.float32)
            gamma[c0:c1] = np.where(np.abs(at) < largest, at, 1.0)
            gamma[c0] = largest
        bytes_, scale, rstd = run()
        y = gamma * rstd[:, None]
        assert y.dtype == np.float32
        most = np.stack([np.abs(y[:, c:c + each]).max(1) for c in range(0, cols, each)], 1)
        assert np.array_equal(scale, most / np.float32(448))
        want = from_quotients(y / np.repeat(scale, each, 1)[:, :cols])
        assert np.array_equal(bytes_ & 0x7f, want & 0x7f), f"{(bytes_ != want).sum()} of {want.size} bytes"
        assert np.array_equal(bytes_[want != 0x80], want[want != 0x80])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", [4096, 64, 1001, 3999, 20000])
def test_zeros_of_both_signs(ctx, dtype, cols):
    # groups of zeros have bytes of 0, whatever the zeros' signs and those of gamma are; a NaN stays one
    x = np.zeros((4, cols), np.float32)
    x[1] = -0.0
    x[2, ::2] = -0.0
    x[3] = np.nan
    gamma = np.where(np.arange(cols) % 3 == 0, -1.0, 1.0)
    for group in (0, 64):
        groups = -(-cols // group) if group else 1
        for g in (None, Placed(ctx, gamma, dtype)):
            q, scale = Bytes(ctx, 4 * cols, 0), empty(ctx, (4, groups))
            ctx.rmsnorm_fwd_e4m3(Placed(ctx, x, dtype), g, q, scale, 4, cols, group=group, dtype=dtype)
            b = q.get().reshape(4, cols)
            assert (b[:3] == 0).all() and (scale.get()[:3] == 0).all()
            assert ((b[3] & 0x7f) == 0x7f).all()
