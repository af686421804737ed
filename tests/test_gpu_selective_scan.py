"""mg_selective_scan and mg_selective_scan_backward against 64 bits."""
import numpy as np
import pytest

from operator_cases import U32, assert_within
from rollout_cases import FLUSH, Held, Operand, Shape, V, bytes_of, rounded, sigmoid, silu, silu_slope, softplus, stack

pytestmark = pytest.mark.gpu

ROWS = ("x", "dt", "b", "c", "z", "dy")
CHUNK = 64


class Case:
    def __init__(self, steps, seqs, channels, states, kind, seed=0, groups=1, order="steps", gate=True, carry=True,
                 resets=0.1, lengths=None, vectors=True, slow=False):
        r = np.random.RandomState(seed)
        self.steps, self.seqs, self.channels, self.states, self.kind = steps, seqs, channels, states, kind
        self.groups = groups
        self.shape = Shape(steps, seqs, order)
        q = lambda *s: rounded(r.normal(0, 1, s), kind)  # noqa: E731
        self.x, self.dt, self.dy = (q(steps, seqs, channels) for _ in range(3))
        self.b, self.c = q(steps, seqs, groups * states), q(steps, seqs, groups * states)
        self.z = q(steps, seqs, channels) if gate else None
        f = lambda a: rounded(a, "fp32")  # noqa: E731
        self.a = f(-np.exp(r.normal(0, 1, (channels, states))) * (0.02 if slow else 1))
        if not slow:
            self.a[::3, 0] = 0  # a state that never fades
        self.d = f(r.normal(0, 1, channels)) if vectors else None
        self.dt_bias = f(r.normal(-2, 2, channels)) if vectors else None
        held = lambda: f(r.normal(0, 1, (seqs, channels, states))) if carry else None  # noqa: E731
        self.initial, self.dfinal = held(), held()
        self.reset = (r.rand(steps, seqs) < resets).astype(np.uint8) * 3 if resets else None
        self.lengths = None if lengths is None else np.array(lengths, np.uint32)
        self.live = np.arange(steps)[:, None] < (np.full(seqs, steps) if lengths is None else self.lengths)[None]

    def reference(self):
        steps, seqs, C, S, G = self.steps, self.seqs, self.channels, self.states, self.groups
        group = np.arange(C) // (C // G)
        each = lambda a: V(a.reshape(seqs, G, S)[:, group])  # noqa: E731
        zero = V(np.zeros((seqs, C, S)))
        skip = V(self.d) if self.d is not None else V(np.zeros(C))
        h = V(self.initial) if self.initial is not None else zero
        hs, before, decays, deltas, raws, ys, pres, kept = [], [], [], [], [], [], [], []
        long = 2 * CHUNK < steps
        for t in range(steps):
            live = self.live[t][:, None, None]
            if t % CHUNK == 0:
                kept.append(h)
            fresh = np.zeros((seqs, 1, 1), bool) if self.reset is None else (self.reset[t] != 0)[:, None, None]
            raw = V(self.dt[t]) + V(self.dt_bias) if self.dt_bias is not None else V(self.dt[t])
            delta = softplus(raw)
            arg = delta.v[..., None] * self.a
            # exp(delta A): 3 roundings of the argument, 2 of the result; a split's decay is that
            # of the sum of its steps' delta, each of which may round the whole sum
            off = (3 + (steps if long else 0)) * np.abs(arg) + 2
            decay = V(np.exp(arg), np.exp(arg) * (off * U32 + np.abs(self.a) * delta.e[..., None]) + FLUSH).where(~fresh)
            x = V(self.x[t])
            prev = h.where(~fresh)
            new = decay * prev + (delta * x)[..., None] * each(self.b[t])
            before.append(prev), decays.append(decay), deltas.append(delta), raws.append(raw)
            hs.append(new)
            pre = (new * each(self.c[t])).sum(-1) + skip * x
            pres.append(pre)
            ys.append(pre * silu(V(self.z[t])) if self.z is not None else pre)
            h = V(np.where(live, new.v, h.v), np.where(live, new.e, h.e))
        out = {"final": h}
        if steps:
            out["y"], out["checkpoints"] = stack(ys), stack(kept)
        # and back
        g = V(self.dfinal) if self.dfinal is not None else zero
        rows = {k: [None] * steps for k in ("dx", "ddt", "db", "dc", "dz")}
        sums = {"da": [], "dd": [], "ddt_bias": []}
        for t in reversed(range(steps)):
            live = self.live[t]
            x, dy = V(self.x[t]), V(self.dy[t])
            if self.z is not None:
                rows["dz"][t] = dy * pres[t] * silu_slope(V(self.z[t]))
                dy = dy * silu(V(self.z[t]))
            gt = g + each(self.c[t]) * dy[..., None]
            over = lambda v: V(v.v.reshape(seqs, G, C // G, S), v.e.reshape(seqs, G, C // G, S)).sum(2)  # noqa: E731
            flat = lambda v: V(v.v.reshape(seqs, G * S), v.e.reshape(seqs, G * S))  # noqa: E731
            rows["dc"][t] = flat(over(hs[t] * dy[..., None]))
            rows["db"][t] = flat(over(gt * (deltas[t] * x)[..., None]))
            gb = (gt * each(self.b[t])).sum(-1)
            rows["dx"][t] = dy * skip + deltas[t] * gb
            back = gt * decays[t]
            via = back * before[t]
            # a log2(e) stands for a: one rounding more, and one back
            ddelta = x * gb + (via * V(self.a, 3 * U32 * np.abs(self.a))).sum(-1)
            ddt = ddelta * sigmoid(raws[t])[0]
            rows["ddt"][t] = ddt
            sums["da"].append((via * deltas[t][..., None]).where(live[:, None, None]))
            sums["dd"].append((dy * x).where(live[:, None]))
            sums["ddt_bias"].append(ddt.where(live[:, None]))
            fresh = np.zeros(seqs, bool) if self.reset is None else self.reset[t] != 0
            back = back.where(~fresh[:, None, None])
            keep = live[:, None, None]
            g = V(np.where(keep, back.v, g.v), np.where(keep, back.e, g.e))
        out["dinitial"] = g
        for k, v in rows.items():
            if steps and v[0] is not None:
                out[k] = stack(v)
        for k, v in sums.items():
            out[k] = stack(v).sum((0, 1)) if v else V(np.zeros({"da": (C, S)}.get(k, (C,))))
        return out

    def dims(self):
        return self.steps, self.seqs, self.channels, self.states, self.kind

    def inputs(self, mg, pad=0, offset=0):
        self.keep = {k: Operand(mg, self.shape, getattr(self, k), self.kind, pad=pad, offset=offset) for k in ROWS
                     if getattr(self, k) is not None}
        p = dict(self.shape.args(), groups=self.groups)
        for k in ("b", "c", "z"):
            if k in self.keep:
                p[k] = self.keep[k].ptr
        for k in self.keep:
            if k != "dy":
                p[k + "_ld"] = self.keep[k].ld
        for k in ("a", "d", "dt_bias", "initial"):
            if getattr(self, k) is not None:
                self.keep[k] = Held(mg, getattr(self, k))
                p[k] = self.keep[k].ptr
        if self.reset is not None:
            self.keep["reset"] = bytes_of(mg, self.shape.rows_of(self.reset, 1))
            p["reset"] = self.keep["reset"].ptr
        if self.lengths is not None:
            self.keep["lengths"] = bytes_of(mg, self.lengths)
            p["lengths"] = self.keep["lengths"].ptr
        return p

    def forward(self, mg, pad=0, offset=0, in_place=False):
        p = self.inputs(mg, pad, offset)
        state = (self.seqs, self.channels, self.states)
        y = Operand(mg, self.shape, None, self.kind, self.channels, pad, offset)
        final = self.keep["initial"] if in_place else Held(mg, None, shape=state)
        chunks = (self.steps + CHUNK - 1) // CHUNK
        kept = Held(mg, None, shape=(max(1, chunks),) + state)
        space = mg.DeviceBuffer(mg.selective_scan_workspace(*self.dims()[:4]) + 256)
        mg.selective_scan(self.keep["x"].ptr, self.keep["dt"].ptr, y.ptr, *self.dims(), final=final.ptr,
                          checkpoints=kept.ptr, y_ld=y.ld, workspace=space.ptr, workspace_bytes=space.nbytes, **p)
        mg._capi.check(mg.lib().mg_synchronize())
        return dict(y=y, final=final, checkpoints=kept)

    def backward(self, mg, kept, pad=0, offset=0):
        p = self.inputs(mg, pad, offset)
        C, w = self.channels, self.groups * self.states
        row = lambda cols: Operand(mg, self.shape, None, self.kind, cols, pad, offset)  # noqa: E731
        out = dict(dx=row(C), ddt=row(C), db=row(w), dc=row(w))
        if self.z is not None:
            out["dz"] = row(C)
        for k in list(out):
            p[k + "_ld"] = out[k].ld
        out.update(da=Held(mg, None, shape=self.a.shape), dd=Held(mg, None, shape=(C,)),
                   ddt_bias=Held(mg, None, shape=(C,)), dinitial=Held(mg, None, shape=(self.seqs, C, self.states)))
        if self.dfinal is not None:
            self.keep["dfinal"] = Held(mg, self.dfinal)
            p["dfinal"] = self.keep["dfinal"].ptr
        space = mg.DeviceBuffer(mg.selective_scan_backward_workspace(*self.dims()[:4], self.groups) + 256)
        mg.selective_scan_backward(self.keep["x"].ptr, self.keep["dt"].ptr, self.keep["dy"].ptr, *self.dims(),
                                   dy_ld=self.keep["dy"].ld, checkpoints=kept.ptr if kept else None,
                                   workspace=space.ptr, workspace_bytes=space.nbytes,
                                   **{k: v.ptr for k, v in out.items()}, **p)
        mg._capi.check(mg.lib().mg_synchronize())
        return out

    def check(self, mg, pad=0, offset=0, in_place=False, need_kept=True):
        want = self.reference()
        o = self.forward(mg, pad, offset)
        if in_place:
            again = self.forward(mg, pad, offset, in_place=True)
            np.testing.assert_array_equal(o["final"].get(), again["final"].get())
        o.update(self.backward(mg, o["checkpoints"] if need_kept else None, pad, offset))
        for k, v in o.items():
            if k == "checkpoints":
                if not self.steps:
                    continue
                got, w = v.get(), want[k]
                reached = self.live[::CHUNK]
                assert_within(got[reached], w.v[reached], w.tolerance("fp32")[reached], k)
            elif isinstance(v, Operand):
                if self.steps:
                    got, w = v.get(self.live), want[k]
                    assert_within(got[self.live], w.v[self.live], w.tolerance(self.kind)[self.live], k)
            else:
                assert_within(v.get(), want[k].v, want[k].tolerance("fp32"), k)


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("steps,seqs,channels,states", [(1, 5, 128, 16), (2, 3, 7, 16), (8, 2, 64, 16), (9, 3, 65, 16),
                                                        (33, 2, 130, 16), (65, 2, 40, 16)])
def test_selective_scan(mg, kind, steps, seqs, channels, states):
    Case(steps, seqs, channels, states, kind, seed=steps).check(mg)


@pytest.mark.parametrize("states", [1, 2, 3, 4, 5, 8, 13, 31, 32, 33, 64, 100, 128, 200, 256])
@pytest.mark.parametrize("steps", [1, 19])
def test_selective_scan_states(mg, states, steps):
    Case(steps, 2, 37, states, "fp32", seed=states, groups=1).check(mg)


@pytest.mark.parametrize("channels,groups", [(8, 8), (96, 2), (192, 3), (520, 4), (1, 1)])
@pytest.mark.parametrize("steps", [1, 17])
def test_selective_scan_groups(mg, channels, groups, steps):
    Case(steps, 2, channels, 16, "bf16", seed=groups, groups=groups).check(mg)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("order", ["steps", "seqs", "apart"])
@pytest.mark.parametrize("pad,offset", [(0, 1), (3, 5), (8, 0)])
def test_selective_scan_strides(mg, kind, order, pad, offset):
    Case(21, 3, 37, 12, kind, seed=1, order=order).check(mg, pad, offset)


@pytest.mark.parametrize("lengths", [[0, 1, 2, 63, 130], [64, 65, 128, 129, 127], [200, 0, 0, 7, 2**31]])
@pytest.mark.parametrize("carry,resets,gate", [(True, 0.0, True), (False, 0.05, False)])
def test_selective_scan_lengths(mg, lengths, carry, resets, gate):
    Case(130, 5, 24, 16, "fp32", seed=2, lengths=lengths, carry=carry, resets=resets, gate=gate, order="seqs").check(mg)


@pytest.mark.parametrize("steps", [0, 1, 2, 70, 400])
def test_selective_scan_final_in_place(mg, steps):
    Case(steps, 3, 20, 16, "fp32", seed=3, vectors=False).check(mg, in_place=True)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("steps,seqs,channels,states,resets", [(385, 1, 40, 16, 0.0), (500, 2, 70, 16, 0.004),
                                                              (641, 1, 9, 64, 0.0), (1030, 1, 20, 4, 0.002)])
def test_selective_scan_split_steps(mg, kind, steps, seqs, channels, states, resets):
    """Few sequences of many steps: several splits, which have to carry a state a long way."""
    lengths = None if seqs == 1 else [steps, steps - 200]
    Case(steps, seqs, channels, states, kind, seed=4, resets=resets, slow=True, lengths=lengths).check(mg)


def test_selective_scan_split_states_never_fading(mg):
    """States that keep all they take in, over several splits."""
    c = Case(513, 1, 16, 8, "fp32", seed=5, slow=True, resets=0.0)
    c.a[:] = 0
    c.check(mg)


def test_selective_scan_every_step_begins(mg):
    c = Case(140, 2, 16, 16, "fp32", seed=6)
    c.reset[:] = 1
    c.check(mg)


def test_selective_scan_without_checkpoints(mg):
    Case(64, 3, 50, 16, "bf16", seed=7).check(mg, need_kept=False)


def test_selective_scan_far_rates(mg):
    """Rates that softplus leaves as they are, or makes next to nothing."""
    c = Case(12, 2, 32, 16, "fp32", seed=8, resets=0.0)
    r = np.random.RandomState(9)
    c.dt[:] = rounded(r.choice([-90.0, -30.0, -8.0, 0.0, 8.0, 30.0, 100.0], c.dt.shape), "fp32")
    c.dt_bias[:] = 0
    c.check(mg)


@pytest.mark.parametrize("steps", [130, 500])
def test_selective_scan_nan_stays_in_its_episode(mg, steps):
    outs = []
    for spoil in (False, True):
        c = Case(steps, 3, 16, 16, "fp32", seed=10, resets=0.0, slow=True)
        c.reset = np.zeros((steps, 3), np.uint8)
        c.reset[100, 1] = 1
        if spoil:
            c.x[99, 1] = np.nan
            c.initial[1] = np.inf
        f = c.forward(mg)
        b = c.backward(mg, f["checkpoints"])
        outs.append((f["y"].get(c.live), f["final"].get(), b["dx"].get(c.live), b["db"].get(c.live)))
    clean = np.ones((steps, 3), bool)
    clean[:100, 1] = False
    for k in (0, 2, 3):
        np.testing.assert_array_equal(outs[0][k][clean], outs[1][k][clean])
    np.testing.assert_array_equal(outs[0][1], outs[1][1])
    assert not np.isfinite(outs[1][0][99, 1]).any()


def test_selective_scan_a_step_at_a_time(mg):
    """Steps of their own, with the state carried on, against the whole call."""
    c = Case(20, 7, 33, 16, "bf16", seed=11)
    whole = c.forward(mg)
    p = c.inputs(mg)
    y = Operand(mg, c.shape, None, "bf16", 33)
    state = c.keep["initial"]
    for k in ("step_rows", "seq_rows"):
        p.pop(k)
    wide, narrow = 7 * 33 * 2, 7 * 16 * 2
    at = {k: p.pop(k) for k in ("b", "c", "z", "reset")}
    for t in range(20):
        mg.selective_scan(c.keep["x"].ptr + t * wide, c.keep["dt"].ptr + t * wide, y.ptr + t * wide, 1, 7, 33, 16,
                          "bf16", b=at["b"] + t * narrow, c=at["c"] + t * narrow, z=at["z"] + t * wide,
                          reset=at["reset"] + t * 7, final=state.ptr, **p)
    want = c.reference()
    assert_within(y.get(c.live), want["y"].v, want["y"].tolerance("bf16"), "y")
    assert_within(state.get(), whole["final"].get(), 2 * want["final"].tolerance("fp32"), "state")


@pytest.mark.parametrize("steps", [9, 200])
def test_selective_scan_gradient_against_differences(mg, steps):
    """The loss sum(y R) + sum(final Q) in 64 bits, moved along a direction of each input."""
    c = Case(steps, 2, 12, 8, "fp32", seed=12, slow=True, resets=0.02)
    f = c.forward(mg)
    g = c.backward(mg, f["checkpoints"])

    def loss():
        o = c.reference()
        return (o["y"].v * c.dy).sum() + (o["final"].v * c.dfinal).sum()

    r, h = np.random.RandomState(13), 1e-4
    for name in ("x", "dt", "b", "c", "z", "a", "d", "dt_bias", "initial"):
        value = getattr(c, name)
        along = r.normal(0, 1, value.shape) * (np.abs(value) if name == "a" else 1)
        ends = []
        for sign in (1, -1):
            setattr(c, name, value + sign * h * along)
            ends.append(loss())
        setattr(c, name, value)
        got = g["d" + name]
        got = got.get(c.live) if isinstance(got, Operand) else got.get()
        # h^2 of the differences (third derivatives of a few), fp32's sums of terms that cancel
        assert abs((got * along).sum() - (ends[0] - ends[1]) / (2 * h)) <= 2e-5 * np.abs(got * along).sum() + 1e-4, name


def test_selective_scan_rows_far_apart(mg):
    """Steps 192 MB apart, every array a column panel of the same rows: past what 31 bits hold in
    eight steps, and past 32 in all."""
    c = Case(27, 2, 20, 16, "fp32", seed=14)
    near_f = c.forward(mg)
    near_b = c.backward(mg, None)
    ld, wide = 1 << 24, 64
    p = {k: v for k, v in c.inputs(mg).items() if not k.endswith("_ld")}
    p.update(step_rows=3, seq_rows=1, **{k + "_ld": ld for k in ("x", "dt", "b", "c", "z")})
    whole = mg.DeviceBuffer((27 * 3 * ld) * 4)
    names = ("x", "dt", "b", "c", "z", "dy", "y", "dx", "ddt", "db", "dc", "dz")
    at = {k: whole.ptr + 4 * wide * i for i, k in enumerate(names)}
    row = lambda t, n: 4 * (3 * t + n) * ld  # noqa: E731
    reset = np.zeros(27 * 3, np.uint8)
    for t in range(27):
        for n in range(2):
            for k in ("x", "dt", "b", "c", "z", "dy"):
                mg.h2d(at[k] + row(t, n), getattr(c, k)[t, n].astype(np.float32))
            reset[3 * t + n] = c.reset[t, n]
    resets = bytes_of(mg, reset)
    state = (2, 20, 16)
    final, kept = Held(mg, None, shape=state), Held(mg, None, shape=(1,) + state)
    p.update(reset=resets.ptr, b=at["b"], c=at["c"], z=at["z"])
    mg.selective_scan(at["x"], at["dt"], at["y"], *c.dims(), y_ld=ld, final=final.ptr, checkpoints=kept.ptr, **p)
    sums = dict(da=Held(mg, None, shape=c.a.shape), dd=Held(mg, None, shape=(20,)),
                ddt_bias=Held(mg, None, shape=(20,)), dinitial=Held(mg, None, shape=state))
    space = mg.DeviceBuffer(mg.selective_scan_backward_workspace(*c.dims()[:4]) + 256)
    grads = {k: at[k] for k in ("dx", "ddt", "db", "dc", "dz")}
    dfinal = Held(mg, c.dfinal)
    mg.selective_scan_backward(at["x"], at["dt"], at["dy"], *c.dims(), dfinal=dfinal.ptr, workspace=space.ptr,
                               workspace_bytes=space.nbytes, dy_ld=ld, **{k + "_ld": ld for k in grads}, **grads,
                               **{k: v.ptr for k, v in sums.items()}, **p)
    mg._capi.check(mg.lib().mg_synchronize())
    want = c.reference()
    assert_within(final.get(), want["final"].v, want["final"].tolerance("fp32"), "final")
    for k in ("y",) + tuple(grads):
        w = want[k]
        got = np.array([[mg.d2h(at[k] + row(t, n), np.float32, (w.v.shape[2],)) for n in range(2)] for t in range(27)])
        assert_within(got.astype(np.float64), w.v, w.tolerance("fp32"), k)
    for k, v in sums.items():
        assert_within(v.get(), want[k].v, want[k].tolerance("fp32"), k)
    assert_within(near_f["final"].get(), final.get(), 2 * want["final"].tolerance("fp32"), "near and far")
    assert_within(near_b["da"].get(), sums["da"].get(), 2 * want["da"].tolerance("fp32"), "near and far")
