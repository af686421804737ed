"""Shared by the tests of the training operators: 16-bit types in numpy, device
copies of arrays with a row stride and an offset, and roundings as tolerances."""
import numpy as np

U32 = 2.0**-24  # half a step of fp32, relative
HALF = {"fp32": 2.0**-24, "bf16": 2.0**-8, "fp16": 2.0**-11}  # half a step: torch.finfo(t).eps / 2
TINY = {"fp32": 2.0**-149, "bf16": 2.0**-133, "fp16": 2.0**-24}  # the smallest step
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def encode(a, kind):
    """float64 values rounded once to `kind`, as the bytes a kernel reads."""
    if kind == "fp16":
        return np.asarray(a, np.float64).astype(np.float16)
    f = np.asarray(a, np.float64).astype(np.float32)
    if kind == "fp32":
        return f
    u = f.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(f), np.uint16(0x7FC0), r)


def decode(a, kind):
    if kind == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def storage(kind):
    return {"fp32": np.float32, "bf16": np.uint16, "fp16": np.float16}[kind]


class Rows:
    """A [rows][cols] array on the device with a row stride and `offset` elements
    before it; the padding and 64 elements behind hold a pattern that must stay."""

    FILL = 0x5A

    def __init__(self, mg, values, kind, ld=0, offset=0, shape=None):
        self.kind = kind
        self.rows, self.cols = shape if values is None else values.shape
        self.ld, self.offset = ld or self.cols, offset
        self.count = offset + max(0, self.rows - 1) * self.ld + (self.cols if self.rows else 0) + 64
        host = np.full(self.count * SIZE[kind], self.FILL, np.uint8).view(storage(kind))
        if values is not None:
            self.view(host)[:] = encode(values, kind)
        self.buf = mg.DeviceBuffer.from_array(host)

    def view(self, host):
        s = host.itemsize
        return np.lib.stride_tricks.as_strided(host[self.offset:], (self.rows, self.cols), (self.ld * s, s))

    @property
    def ptr(self):
        return self.buf.ptr + self.offset * SIZE[self.kind]

    def get(self):
        """The values, after checking that nothing around them was written."""
        host = self.buf.download(storage(self.kind), (self.count,))
        inside = np.zeros(self.count, bool)
        if self.rows:
            self.view(inside.view(np.uint8))[:] = 1
        rest = host[~inside].view(np.uint8)
        assert (rest == self.FILL).all(), "elements outside the array were written"
        return decode(self.view(host).copy(), self.kind)


def assert_within(got, want, tol, what):
    bad = ~(np.abs(got - want) <= tol) & ~(np.isnan(got) & np.isnan(want)) & ~(got == want)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, np.abs(got - want) - tol, -np.inf)), got.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} outside; at {i} got {got[i]!r} want {want[i]!r} "
                             f"tolerance {np.broadcast_to(tol, got.shape)[i]!r}")
