"""Storage types, placement off 16-byte boundaries with guards on both sides, and 64-bit formulas for the tests of the token operators."""
import numpy as np

HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}        # half a subnormal step, or less than one
U = 2.0 ** -24
GUARD = 37          # elements behind a tensor that must stay as they were


def bits(a, dtype):
    from ferrograd_b200.backend import to_bf16_bits
    a = np.ascontiguousarray(a, np.float32)
    return a.view(np.uint32) if dtype == "f32" else a.astype(np.float16).view(np.uint16) if dtype == "f16" else to_bf16_bits(a)


def values(b, dtype):
    from ferrograd_b200.backend import from_bf16_bits
    return b.view(np.float32) if dtype == "f32" else b.view(np.float16).astype(np.float32) if dtype == "f16" else from_bf16_bits(b)


def rounded(a, dtype):
    """The values that a tensor of this type holds, as f32."""
    return values(bits(a, dtype), dtype).reshape(np.shape(a))


class Placed:
    """An array on the device `shift` elements behind a 256-byte boundary, a pattern before and behind it."""

    def __init__(self, ctx, a, dtype="f32", shift=0):
        self.ctx, self.dtype, self.shape, self.shift = ctx, dtype, np.shape(a), shift
        word = np.uint32 if dtype in ("f32", "u32") else np.uint16
        b = np.ascontiguousarray(a, np.uint32) if dtype == "u32" else bits(a, dtype)
        self.n = b.size
        self.fill = word(0x7eadbeef & np.iinfo(word).max)
        whole = np.full(shift + self.n + GUARD, self.fill, word)
        whole[shift:shift + self.n] = b.ravel()
        self.t = ctx.new_tensor(whole.shape, word)
        ctx.upload(self.t.data, whole)
        self.ptr = self.t.ptr + shift * word().itemsize

    def bits(self):
        b = self.ctx.to_numpy(self.t)
        assert (b[:self.shift] == self.fill).all() and (b[self.shift + self.n:] == self.fill).all(), "written outside the tensor"
        return b[self.shift:self.shift + self.n].reshape(self.shape)

    def get(self):
        b = self.bits()
        return b if self.dtype == "u32" else values(b, self.dtype).reshape(self.shape)


def empty(ctx, shape, dtype="f32", shift=0):
    """An output: NaN everywhere, so that what is not written shows."""
    if dtype == "u32":
        return Placed(ctx, np.full(shape, 0xabcdabcd, np.uint32), dtype, shift)
    return Placed(ctx, np.full(shape, np.nan, np.float32), dtype, shift)


def check(got, want, bound, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert np.isfinite(got).all(), f"{what}: not finite"
    over = np.abs(got - want) - bound
    i = np.unravel_index(np.argmax(over), over.shape)
    assert over[i] <= 0, f"{what}: {got[i]} for {want[i]} at {i}, off by {abs(got[i] - want[i]):.3g} of {np.broadcast_to(bound, over.shape)[i]:.3g}"
