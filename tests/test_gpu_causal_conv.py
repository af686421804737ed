"""mg_causal_conv and mg_causal_conv_backward against 64 bits."""
import numpy as np
import pytest

from operator_cases import assert_within
from rollout_cases import Held, Operand, Shape, V, bytes_of, rounded, silu, silu_slope

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, steps, seqs, channels, taps, kind, seed=0, order="steps", act=True, carry=True, resets=0.2,
                 lengths=None, bias=True):
        r = np.random.RandomState(seed)
        self.steps, self.seqs, self.channels, self.taps, self.kind, self.act = steps, seqs, channels, taps, kind, act
        self.shape = Shape(steps, seqs, order)
        q = lambda *s: rounded(r.normal(0, 1, s), kind)  # noqa: E731
        self.x, self.dy = q(steps, seqs, channels), q(steps, seqs, channels)
        self.weight = rounded(r.normal(0, 1, (channels, taps)), "fp32")
        self.bias = rounded(r.normal(0, 1, channels), "fp32") if bias else None
        self.initial = q(seqs, taps - 1, channels) if carry else None
        self.dfinal = q(seqs, taps - 1, channels) if carry else None
        self.reset = (r.rand(steps, seqs) < resets).astype(np.uint8) * r.randint(1, 256, (steps, seqs)).astype(
            np.uint8) if resets else None
        self.lengths = None if lengths is None else np.array(lengths, np.uint32)
        self.live = np.arange(steps)[:, None] < (np.full(seqs, steps) if lengths is None else self.lengths)[None]

    def length(self, n):
        return self.steps if self.lengths is None else min(self.steps, int(self.lengths[n]))

    def reference(self):
        """Sequence by sequence with the window as it stands: y, final, and the gradients."""
        steps, taps, seqs, C = self.steps, self.taps, self.seqs, self.channels
        z = lambda *s: (np.zeros(s), np.zeros(s))  # noqa: E731
        y, dx, final, dinitial = z(steps, seqs, C), z(steps, seqs, C), z(seqs, taps - 1, C), z(seqs, taps - 1, C)
        dw, db, count = z(C, taps), z(C), 0
        put = lambda to, at, v: (to[0].__setitem__(at, v.v), to[1].__setitem__(at, v.e))  # noqa: E731
        add = lambda to, at, v: (to[0].__setitem__(at, to[0][at] + v.v),  # noqa: E731
                                 to[1].__setitem__(at, to[1][at] + v.e + np.abs(v.v) * 2e-7))
        size = np.zeros((C, taps)), np.zeros(C)
        for n in range(seqs):
            window = [self.initial[n, k] if self.initial is not None else np.zeros(C) for k in range(taps - 1)]
            places = [("i", n, k) for k in range(taps - 1)]
            grad = lambda at, v: add(dinitial, at[1:], v) if at[0] == "i" else add(dx, at[1:], v)  # noqa: E731
            for t in range(self.length(n)):
                if self.reset is not None and self.reset[t, n]:
                    window, places = [np.zeros(C)] * (taps - 1), [None] * (taps - 1)
                window, places = window + [self.x[t, n]], places + [("x", t, n)]
                terms = [V(self.weight[:, k]) * V(window[k]) for k in range(taps)]
                pre = V(self.bias) if self.bias is not None else V(np.zeros(C))
                for term in terms:
                    pre = pre + term
                put(y, (t, n), silu(pre) if self.act else pre)
                d = V(self.dy[t, n]) * silu_slope(pre) if self.act else V(self.dy[t, n])
                count += 1
                add(db, slice(None), d)
                size[1][:] += np.abs(d.v)
                for k in range(taps):
                    v = d * V(window[k])
                    add(dw, (slice(None), k), v)
                    size[0][:, k] += np.abs(v.v)
                    if places[k]:
                        grad(places[k], d * V(self.weight[:, k]))
                window, places = window[1:], places[1:]
            for k in range(taps - 1):
                final[0][n, k] = window[k]
                if places[k] and self.dfinal is not None:
                    grad(places[k], V(self.dfinal[n, k]))
        # sums over rows: a half step of their size for each term
        dw, db = (V(s[0], s[1] + count * 6e-8 * z) for s, z in zip((dw, db), size))
        return dict(y=V(*y), final=final[0], dx=V(*dx), dweight=dw, dbias=db, dinitial=V(*dinitial))

    def inputs(self, mg, pad, offset):
        op = lambda a: Operand(mg, self.shape, a, self.kind, pad=pad, offset=offset)  # noqa: E731
        self.keep = dict(x=op(self.x), dy=op(self.dy), weight=Held(mg, self.weight))
        p = dict(self.shape.args(), silu=self.act, x_ld=self.keep["x"].ld)
        for k, v, kind in (("bias", self.bias, "fp32"), ("initial", self.initial, self.kind)):
            if v is not None:
                self.keep[k] = Held(mg, v, kind)
                p[k] = self.keep[k].ptr
        if self.reset is not None:
            self.keep["reset"] = bytes_of(mg, self.shape.rows_of(self.reset, 1))
            p["reset"] = self.keep["reset"].ptr
        if self.lengths is not None:
            self.keep["lengths"] = bytes_of(mg, self.lengths)
            p["lengths"] = self.keep["lengths"].ptr
        return p

    def dims(self):
        return self.steps, self.seqs, self.channels, self.taps, self.kind

    def check(self, mg, pad=0, offset=0, in_place=False):
        want, p = self.reference(), self.inputs(mg, pad, offset)
        out = lambda: Operand(mg, self.shape, None, self.kind, self.channels, pad, offset)  # noqa: E731
        held = lambda *s: Held(mg, None, self.kind, s)  # noqa: E731
        y, dx = out(), out()
        x, w = self.keep["x"].ptr, self.keep["weight"].ptr
        window = (self.seqs, self.taps - 1, self.channels)
        dweight, dbias = Held(mg, None, shape=self.weight.shape), Held(mg, None, shape=(self.channels,))
        dinitial = held(*window)
        space = mg.DeviceBuffer(mg.causal_conv_backward_workspace(*self.dims()[:4]) + 256)
        b = dict(p)
        if self.dfinal is not None:
            self.keep["dfinal"] = Held(mg, self.dfinal, self.kind)
            b["dfinal"] = self.keep["dfinal"].ptr
        mg.causal_conv_backward(x, w, self.keep["dy"].ptr, dx.ptr, *self.dims(), dweight=dweight.ptr, dbias=dbias.ptr,
                                dinitial=dinitial.ptr, dy_ld=dx.ld, dx_ld=dx.ld, workspace=space.ptr,
                                workspace_bytes=space.nbytes, **b)
        final = self.keep["initial"] if in_place else held(*window)
        mg.causal_conv(x, w, y.ptr, *self.dims(), final=final.ptr, y_ld=y.ld, **p)
        mg._capi.check(mg.lib().mg_synchronize())
        got = y.get(self.live)
        assert_within(got[self.live], want["y"].v[self.live], want["y"].tolerance(self.kind)[self.live], "y")
        np.testing.assert_array_equal(final.get(), want["final"])
        got = dx.get(self.live)
        assert_within(got[self.live], want["dx"].v[self.live], want["dx"].tolerance(self.kind)[self.live], "dx")
        for name, h, kind in (("dweight", dweight, "fp32"), ("dbias", dbias, "fp32"), ("dinitial", dinitial, self.kind)):
            assert_within(h.get(), want[name].v, want[name].tolerance(kind), name)


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("taps", [2, 3, 4])
@pytest.mark.parametrize("steps,seqs,channels", [(1, 5, 128), (2, 3, 7), (3, 4, 1), (8, 2, 64), (9, 3, 33), (33, 2, 130),
                                                 (70, 1, 12)])
def test_causal_conv(mg, kind, taps, steps, seqs, channels):
    Case(steps, seqs, channels, taps, kind, seed=steps).check(mg)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("order", ["steps", "seqs", "apart"])
@pytest.mark.parametrize("pad,offset", [(0, 1), (3, 5), (8, 0)])
def test_causal_conv_strides(mg, kind, order, pad, offset):
    Case(21, 3, 37, 4, kind, seed=1, order=order).check(mg, pad, offset)


@pytest.mark.parametrize("kind", ["fp32", "fp16"])
@pytest.mark.parametrize("lengths", [[0, 1, 2, 3, 40], [40, 39, 8, 9, 33], [100, 0, 0, 7, 2**31]])
@pytest.mark.parametrize("carry,resets", [(True, 0.0), (False, 0.3)])
def test_causal_conv_lengths(mg, kind, lengths, carry, resets):
    Case(40, 5, 24, 4, kind, seed=2, lengths=lengths, carry=carry, resets=resets, order="seqs").check(mg)


@pytest.mark.parametrize("steps", [0, 1, 2, 50])
@pytest.mark.parametrize("act,bias", [(False, True), (True, False)])
def test_causal_conv_final_in_place(mg, steps, act, bias):
    Case(steps, 6, 20, 4, "bf16", seed=3, act=act, bias=bias).check(mg, in_place=True)


def test_causal_conv_every_step_begins(mg):
    c = Case(30, 2, 16, 3, "fp32", seed=4)
    c.reset[:] = 1
    c.check(mg)


@pytest.mark.parametrize("steps,seqs,channels", [(32, 1030, 130), (5000, 2, 200), (1, 70000, 5)])
def test_causal_conv_many_rows(mg, steps, seqs, channels):
    """Over many workgroups, against the same in numpy over whole arrays."""
    taps, kind = 4, "fp32"
    c = Case(steps, seqs, channels, taps, kind, seed=5, carry=False, resets=0.0)
    p = c.inputs(mg, 0, 0)
    y, dx = (Operand(mg, c.shape, None, kind, channels) for _ in range(2))
    dweight, dbias = Held(mg, None, shape=c.weight.shape), Held(mg, None, shape=(channels,))
    space = mg.DeviceBuffer(mg.causal_conv_backward_workspace(steps, seqs, channels, taps) + 256)
    a = (c.keep["x"].ptr, c.keep["weight"].ptr)
    mg.causal_conv(*a, y.ptr, *c.dims(), **p)
    mg.causal_conv_backward(*a, c.keep["dy"].ptr, dx.ptr, *c.dims(), dweight=dweight.ptr, dbias=dbias.ptr,
                            workspace=space.ptr, workspace_bytes=space.nbytes, **p)
    long = np.concatenate([np.zeros((taps - 1, seqs, channels)), c.x])
    pre, size = c.bias + np.zeros_like(c.x), np.abs(c.bias) + np.zeros_like(c.x)
    for k in range(taps):
        pre = pre + c.weight[:, k] * long[k:k + steps]
        size = size + np.abs(c.weight[:, k] * long[k:k + steps])
    v = V(pre, 5 * 6e-8 * size)
    want = silu(v)
    assert_within(y.get(c.live), want.v, want.tolerance(kind), "y")
    d = V(c.dy) * silu_slope(v)
    dlong, off = np.zeros_like(long), np.zeros_like(long)
    for k in range(taps):
        dlong[k:k + steps] += c.weight[:, k] * d.v
        off[k:k + steps] += np.abs(c.weight[:, k]) * (d.e + 5 * 6e-8 * np.abs(d.v))
    assert_within(dx.get(c.live), dlong[taps - 1:], V(dlong, off).tolerance(kind)[taps - 1:], "dx")
    # sums in chains of a thread's rows, a workgroup's threads and 32 slices of the parts
    chain = 64 + 32 + 64 * steps * seqs // (1024 * 8)
    want = V(d.v.sum((0, 1)), d.e.sum((0, 1)) + chain * 6e-8 * np.abs(d.v).sum((0, 1)))
    assert_within(dbias.get(), want.v, want.tolerance(kind), "dbias")
    for k in range(taps):
        t = d.v * long[k:k + steps]
        off = (d.e * np.abs(long[k:k + steps])).sum((0, 1)) + (chain + 1) * 6e-8 * np.abs(t).sum((0, 1))
        assert_within(dweight.get()[:, k], t.sum((0, 1)), V(t.sum((0, 1)), off).tolerance(kind), f"dweight {k}")


def test_causal_conv_nan_stays_in_its_episode(mg):
    c = Case(40, 3, 16, 4, "fp32", seed=6, resets=0.0)
    c.reset = np.zeros((40, 3), np.uint8)
    c.reset[20, 1] = 1
    bad = Case(40, 3, 16, 4, "fp32", seed=6, resets=0.0)
    bad.reset = c.reset
    bad.x[19, 1] = np.nan
    bad.x[5, 2] = np.inf
    outs = []
    for v in (c, bad):
        p = v.inputs(mg, 0, 0)
        y = Operand(mg, v.shape, None, "fp32", 16)
        mg.causal_conv(v.keep["x"].ptr, v.keep["weight"].ptr, y.ptr, *v.dims(), **p)
        outs.append(y.get(v.live))
    touched = np.zeros((40, 3), bool)
    touched[19, 1] = True
    touched[5:9, 2] = True
    np.testing.assert_array_equal(outs[0][~touched], outs[1][~touched])
    assert np.isnan(outs[1][19, 1]).all() and not np.isfinite(outs[1][5, 2]).any()


def test_causal_conv_a_step_at_a_time(mg):
    """Steps of their own, with the window carried on, give the whole call's bits."""
    c = Case(20, 7, 33, 4, "bf16", seed=7)
    p = c.inputs(mg, 0, 0)
    y, single = (Operand(mg, c.shape, None, "bf16", 33) for _ in range(2))
    final = Held(mg, None, "bf16", c.initial.shape)
    mg.causal_conv(c.keep["x"].ptr, c.keep["weight"].ptr, y.ptr, *c.dims(), final=final.ptr, **p)
    window = Held(mg, c.initial, "bf16")
    row, reset = 7 * 33 * 2, p.pop("reset")
    p.pop("initial"), p.pop("step_rows"), p.pop("seq_rows")
    for t in range(20):
        mg.causal_conv(c.keep["x"].ptr + t * row, c.keep["weight"].ptr, single.ptr + t * row, 1, 7, 33, 4, "bf16",
                       reset=reset + t * 7, initial=window.ptr, final=window.ptr, **p)
    np.testing.assert_array_equal(y.get(c.live), single.get(c.live))
    np.testing.assert_array_equal(final.get(), window.get())
