"""The 8-bit form of the root-mean-square norm: its bytes as they are defined, and more rows than 31 bits count."""
import numpy as np
import pytest

from test_gpu_rmsnorm import e4m3_values

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
