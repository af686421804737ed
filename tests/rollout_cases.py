"""Shared by the tests of the operators over rollouts: rows of (step, sequence) on the device in any
order, and values in 64 bits that carry a bound of what fp32 arithmetic may be off by."""
import numpy as np

from operator_cases import HALF, TINY, U32, Rows, decode, encode, storage


# The instruction for 2^x gives 0 for a result under fp32's normal range (2^x < 2^-126): it is off by
# less than that, whatever the argument.
FLUSH = 2.0**-126


class V:
    """A value in 64 bits and how far an fp32 computation of it may be off (to first order):
    every operation adds half a step of its result, a sum one for each of its terms."""

    def __init__(self, v, err=0.0):
        self.v = np.asarray(v, np.float64)
        self.e = np.broadcast_to(np.asarray(err, np.float64), self.v.shape)

    def __mul__(self, o):
        o = o if isinstance(o, V) else V(o)
        v = self.v * o.v
        return V(v, np.abs(self.v) * o.e + np.abs(o.v) * self.e + U32 * np.abs(v))

    def __add__(self, o):
        o = o if isinstance(o, V) else V(o)
        v = self.v + o.v
        return V(v, self.e + o.e + U32 * np.abs(v))

    def __getitem__(self, k):
        return V(self.v[k], self.e[k])

    def sum(self, axis):
        n = np.prod([self.v.shape[a] for a in np.atleast_1d(axis)])
        return V(self.v.sum(axis), self.e.sum(axis) + n * U32 * np.abs(self.v).sum(axis))

    def where(self, keep):
        return V(np.where(keep, self.v, 0.0), np.where(keep, self.e, 0.0))

    def tolerance(self, kind):
        """Rounded once to `kind`; twice the bound for what is of second order."""
        return 2 * self.e + (np.abs(self.v) + self.e) * HALF[kind] + TINY[kind]


def stack(vs, axis=0):
    return V(np.stack([v.v for v in vs], axis), np.stack([v.e for v in vs], axis))


def sigmoid(v):
    """exp2 takes the rounding of its argument along: 2 |v|; itself, the sum, the reciprocal and a product: 8."""
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-v.v))
        rest = 1 / (1 + np.exp(v.v))
    off = (2 * np.abs(v.v) + 8) * U32
    return V(s, s * off + s * rest * v.e + FLUSH), V(rest, rest * off + s * rest * v.e + FLUSH)


def silu(v):
    return v * sigmoid(v)[0]


def silu_slope(v):
    s, rest = sigmoid(v)
    return s * (V(np.ones_like(v.v)) + v * rest)


def softplus(v):
    """Exponential 4 half steps, its sum with 1 what is made good again but for a share t, the
    logarithm's instruction 2, its product and sums 4, then a sum."""
    with np.errstate(over="ignore"):
        log = np.log1p(np.exp(-np.abs(v.v)))
        slope = 1 / (1 + np.exp(-v.v))
    r = np.maximum(v.v, 0) + log
    return V(r, 15 * U32 * log + U32 * r + slope * v.e + FLUSH)


class Shape:
    """How the rows of `steps` x `seqs` lie: "steps" [steps][seqs], "seqs" [seqs][steps], "apart" with
    rows between them that belong to nothing."""

    def __init__(self, steps, seqs, order="steps"):
        self.steps, self.seqs = steps, seqs
        self.strides = {"steps": (0, 0), "seqs": (1, steps), "apart": (seqs + 2, 1)}[order]
        a, b = self.strides if order != "steps" else (seqs, 1)
        self.index = np.arange(steps)[:, None] * a + np.arange(seqs)[None] * b
        self.rows = int(self.index.max()) + 1 if self.index.size else 0

    def args(self):
        return dict(step_rows=self.strides[0], seq_rows=self.strides[1])

    def rows_of(self, a, fill=0.0):
        """[steps][seqs][...] as [rows][...], what lies between them `fill`."""
        out = np.full((self.rows,) + a.shape[2:], fill, a.dtype)
        out[self.index] = a
        return out


class Operand:
    """Rows on the device; `ld` columns more than they are wide, from `offset` elements on."""

    def __init__(self, mg, shape, values, kind, cols=None, pad=0, offset=0):
        self.shape, self.kind = shape, kind
        cols = values.shape[2] if values is not None else cols
        v = None if values is None else shape.rows_of(values, np.nan)
        self.rows = Rows(mg, v, kind, ld=cols + pad, offset=offset, shape=(shape.rows, cols))
        self.ld, self.ptr = cols + pad, self.rows.ptr

    def get(self, live):
        """[steps][seqs][cols]; rows that are not `live` must hold what they held."""
        got = self.rows.get()
        mark = decode(np.full(8, Rows.FILL, np.uint8).view(storage(self.kind))[:1], self.kind)[0]
        rest = np.ones(self.shape.rows, bool)
        rest[self.shape.index[live]] = False
        assert (got[rest] == mark).all(), "rows behind a sequence were written"
        return got[self.shape.index]


class Held:
    """A packed array with a margin on either side that must stay."""

    def __init__(self, mg, values, kind="fp32", shape=None):
        self.kind = kind
        self.values = values
        self.shape = shape if values is None else values.shape
        flat = None if values is None else np.asarray(values, np.float64).reshape(1, -1)
        self.rows = Rows(mg, flat, kind, offset=64, shape=(1, int(np.prod(self.shape))))
        self.ptr = self.rows.ptr

    def get(self):
        return self.rows.get().reshape(self.shape)


def rounded(a, kind):
    return decode(encode(a, kind), kind)


def bytes_of(mg, a):
    return mg.DeviceBuffer.from_array(np.ascontiguousarray(a))
