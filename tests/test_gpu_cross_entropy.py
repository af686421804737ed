"""mg_cross_entropy and mg_cross_entropy_backward against 64 bits."""
import numpy as np
import pytest

from operator_cases import HALF, TINY, U32, Rows, assert_within
from rollout_cases import Held, bytes_of, rounded

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, rows, classes, width, kind, seed=0, entropy=True, pad=0, offset=0, spread=1.5, out=0.1):
        r = np.random.RandomState(seed)
        self.rows, self.classes, self.width, self.kind = rows, classes, width, kind
        self.x = rounded(r.normal(0, 1, (rows, width)), kind)
        self.w = rounded(r.normal(0, spread * width**-0.5, (classes, width)), kind)
        self.targets = r.randint(0, classes, rows).astype(np.int32)
        self.targets[r.rand(rows) < out] = r.choice([-1, classes, 2**31 - 1, -(2**31)])
        self.dloss = rounded(r.normal(0, 1, rows) / max(1, rows), "fp32")
        self.dentropy = rounded(r.normal(0, 0.1, rows) / max(1, rows), "fp32") if entropy else None
        self.pad, self.offset = pad, offset

    @property
    def live(self):
        return (self.targets >= 0) & (self.targets < self.classes)

    def dims(self):
        return self.rows, self.classes, self.width, self.kind

    def reference(self):
        """The results, and what fp32 sums of exact 16-bit products may be off by: an instruction adds 16
        products to its sum and may cut off what is under the sum's last place (a whole step, 2 u);
        pairs take three instructions, leave out 2^-22 of a factor on either side and the product of
        the low halves, and nothing finer than 2^-39 of an array's largest."""
        x, w, K = self.x, self.w, self.width
        pairs = self.kind == "fp32"
        s = x @ w.T
        size = np.abs(x) @ np.abs(w).T
        chain = 2 * U32 * (16 + K / 16 * (3 if pairs else 1))
        es = size * (chain + 2 * U32)
        if pairs:
            # a row of x is scaled by itself, w as a whole
            xm, wm = np.abs(x).max(1, keepdims=True), np.abs(w).max()
            es = es + size * 3 * 2.0**-22 + 2.0**-39 * (xm * np.abs(w).sum(1) + wm * np.abs(x).sum(1, keepdims=True))
        top = s.max(1)
        d = s - top[:, None]
        e = np.exp(d)
        total = e.sum(1)
        lse = top + np.log(total)
        p = e / total[:, None]
        rows = np.arange(self.rows)
        hit = np.where(self.live, self.targets, 0)
        loss = np.where(self.live, lse - s[rows, hit], 0.0)
        entropy = lse - (p * s).sum(1)
        # exp2: half a step of its argument, one of the result; sums of 64 terms in a row, then of two and
        # of a wave's and a tile's, each with a factor of that kind; a logarithm; a product by log 2
        terms = 64 + 2 + 8 + (self.classes + 255) // 256 / 64 + 6 * 3
        rel = (p * (np.abs(d) * 4 * U32 + es)).sum(1) + (terms + 4) * U32 + U32 * 2.0
        ends = 4 * U32 * (np.abs(top) + np.abs(np.log(total)) + np.abs(s[rows, hit]) + 1)
        worst = es.max(1)
        self.err = dict(lse=rel + worst + ends, loss=np.where(self.live, rel + worst + es[rows, hit] + ends, 0.0),
                        entropy=(p * np.abs(d)).sum(1) * (terms + 8) * U32 + rel * (1 + (p * np.abs(d)).sum(1)) + ends
                        + (p * (1 + np.abs(d)) * es).sum(1) + worst * 2 * p.max(1))
        self.s, self.es, self.p = s, es, p
        return dict(loss=loss, lse=lse, entropy=entropy)

    def gradients(self, lse, entropy):
        """From the statistics that the call is given."""
        x, w, kind = self.x, self.w, self.kind
        log = self.s - lse[:, None]
        p = np.exp(log)
        off = self.es + 4 * U32 * (np.abs(self.s) + np.abs(lse)[:, None] + 1)  # of log p
        rows = np.flatnonzero(self.live)
        g = self.dloss[:, None] * p
        eg = np.abs(g) * (off + 4 * U32)
        if self.dentropy is not None:
            more = self.dentropy[:, None] * p * (log + entropy[:, None])
            g = g - more
            eg = eg + np.abs(more) * (off + 6 * U32) + np.abs(self.dentropy[:, None]) * p * (
                off + 4 * U32 * np.abs(entropy)[:, None])
        g[rows, self.targets[rows]] -= self.dloss[rows]
        eg = eg + U32 * np.abs(g)
        g[~self.live], eg[~self.live] = 0, 0
        pairs = kind == "fp32"
        eg = eg + np.abs(g) * (2.0**-22 if pairs else HALF[kind])  # rounded for the products
        if kind != "bf16" and rows.size:
            most = np.abs(self.dloss[rows])
            if self.dentropy is not None:
                most = most + (np.log(self.classes) + 1) * np.abs(self.dentropy[rows])
            eg[rows] += most.max() * 2.0**-38
        mult = 3 if pairs else 1
        rep = 2.0**-21 if pairs else 0.0

        def product(a, ea, b):
            v, size = a @ b, np.abs(a) @ np.abs(b)
            n = a.shape[1]
            chain = 2 * U32 * (16 + n / 16 * mult) + U32 * (n / 2048 + 2)  # and the parts' sums
            err = ea @ np.abs(b) + size * (chain + rep)
            if pairs:
                err = err + 2.0**-38 * (np.abs(a).sum(1, keepdims=True) * np.abs(b).max()
                                        + np.abs(b).sum(0) * np.abs(a).max())
            return v, 2 * err + (np.abs(v) + err) * HALF[kind] + TINY[kind]

        xl = np.where(self.live[:, None], x, 0.0)
        return dict(dx=product(g, eg, w), dw=product(g.T, eg.T, xl))

    def upload(self, mg):
        rows = lambda v: Rows(mg, v, self.kind, self.width + self.pad, self.offset)  # noqa: E731
        self.dev = dict(x=rows(self.x), w=rows(self.w), targets=bytes_of(mg, self.targets), dloss=Held(mg, self.dloss))
        if self.dentropy is not None:
            self.dev["dentropy"] = Held(mg, self.dentropy)
        self.at = (self.dev["x"].ptr, self.dev["w"].ptr, self.dev["targets"].ptr)
        self.ld = dict(x_ld=self.width + self.pad, w_ld=self.width + self.pad)

    def forward(self, mg):
        out = {k: Held(mg, None, shape=(self.rows,)) for k in ("loss", "lse", "entropy")}
        space = mg.DeviceBuffer(mg.cross_entropy_workspace(*self.dims()) + 256)
        mg.cross_entropy(*self.at, *self.dims(), workspace=space.ptr, workspace_bytes=space.nbytes, **self.ld,
                         **{k: v.ptr for k, v in out.items()})
        mg._capi.check(mg.lib().mg_synchronize())
        return {k: v.get() for k, v in out.items()}

    def backward(self, mg, lse, entropy):
        out = {k: Rows(mg, None, self.kind, self.width + self.pad, self.offset, shape=(n, self.width))
               for k, n in (("dx", self.rows), ("dw", self.classes))}
        self.dev["lse"], self.dev["entropy"] = Held(mg, lse), Held(mg, entropy)
        space = mg.DeviceBuffer(mg.cross_entropy_backward_workspace(*self.dims()) + 256)
        more = {}
        if self.dentropy is not None:
            more = dict(dentropy=self.dev["dentropy"].ptr, entropy=self.dev["entropy"].ptr)
        mg.cross_entropy_backward(*self.at, *self.dims(), lse=self.dev["lse"].ptr, dloss=self.dev["dloss"].ptr,
                                  dx_ld=self.ld["x_ld"], dw_ld=self.ld["w_ld"], workspace=space.ptr,
                                  workspace_bytes=space.nbytes, **self.ld, **more,
                                  **{k: v.ptr for k, v in out.items()})
        mg._capi.check(mg.lib().mg_synchronize())
        return {k: v.get() for k, v in out.items()}

    def check(self, mg):
        want = self.reference()
        self.upload(mg)
        got = self.forward(mg)
        for k in want:
            assert_within(got[k], want[k], 2 * self.err[k], k)
        lse, entropy = rounded(want["lse"], "fp32"), rounded(want["entropy"], "fp32")
        got = self.backward(mg, lse, entropy)
        for k, (v, tol) in self.gradients(lse, entropy).items():
            assert_within(got[k], v, tol, k)


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,classes,width", [(1, 1, 1), (1, 2, 8), (3, 255, 16), (64, 256, 32), (65, 257, 33),
                                                (255, 100, 128), (257, 513, 130), (31, 1000, 40), (300, 300, 300)])
def test_cross_entropy(mg, kind, rows, classes, width):
    Case(rows, classes, width, kind, seed=rows).check(mg)


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("pad,offset", [(0, 1), (3, 5), (8, 8), (8, 0), (1, 0)])
def test_cross_entropy_strides(mg, kind, pad, offset):
    Case(70, 130, 64, kind, seed=1, pad=pad, offset=offset, entropy=pad == 8).check(mg)


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
def test_cross_entropy_pieces(mg, kind):
    """More classes than a piece has, more rows than a range, and a last piece of few."""
    Case(8300, 4200, 24, kind, seed=2).check(mg)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_cross_entropy_long_contractions(mg, kind):
    Case(40, 20011, 520, kind, seed=3).check(mg)


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,classes,width", [(32, 4100, 1030), (33, 4100, 1030), (700, 1100, 1100), (513, 9000, 129),
                                                (1030, 300, 72), (2, 70000, 16), (260, 270, 4104)])
def test_cross_entropy_either_way(mg, kind, rows, classes, width):
    """Sizes around those where small products take over, each with tiles that stick out."""
    Case(rows, classes, width, kind, seed=12).check(mg)


@pytest.mark.parametrize("kind", ["fp32", "fp16"])
def test_cross_entropy_sharp_rows(mg, kind):
    """Logits of a spread of 40: most probabilities are under fp32's range."""
    Case(66, 700, 64, kind, seed=4, spread=40).check(mg)


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("classes,width", [(300, 48), (30011, 200)])
def test_cross_entropy_rows_left_out(mg, kind, classes, width):
    """Rows without a target hold NaN, infinity and large numbers, and reach nothing."""
    c = Case(80, classes, width, kind, seed=5)
    c.targets[10:14] = [-1, classes, -5, 2**31 - 1]
    want = c.reference()
    lse, entropy = rounded(want["lse"], "fp32"), rounded(want["entropy"], "fp32")
    grads = c.gradients(lse, entropy)
    c.x[10], c.x[11, 3], c.x[12] = np.nan, np.inf, rounded(np.full(width, 3e4), kind)
    c.dloss[10], c.dloss[12], c.dentropy[13] = np.nan, 1e30, np.inf
    lse[10], entropy[11] = np.nan, np.inf
    c.upload(mg)
    got = c.forward(mg)
    others = np.ones(80, bool)
    others[10:13] = False
    for k in want:
        assert_within(got[k][others], want[k][others], 2 * c.err[k][others], k)
    assert (got["loss"][~c.live] == 0).all()
    got = c.backward(mg, lse, entropy)
    for k, (v, tol) in grads.items():
        assert_within(got[k], v, tol, k)
    assert (got["dx"][~c.live] == 0).all()


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("classes,width", [(300, 32), (30000, 520)])
def test_cross_entropy_not_finite(mg, kind, classes, width):
    """A row's NaN is its own, forward; minus infinity as a logit is a class that is never taken."""
    c = Case(70, classes, width, kind, seed=6, out=0)
    want = c.reference()
    clean = want["loss"].copy()
    c.x[7, 5] = np.nan
    c.upload(mg)
    got = c.forward(mg)
    others = np.arange(70) != 7
    assert np.isnan(got["lse"][7]) and np.isnan(got["loss"][7]) and np.isnan(got["entropy"][7])
    assert_within(got["loss"][others], clean[others], 2 * c.err["loss"][others], "loss")
    c = Case(70, classes, width, kind, seed=6, out=0)
    c.x = np.abs(c.x) + rounded(np.full(c.x.shape, 0.0078125), kind)
    c.x = rounded(c.x, kind)
    c.targets[c.targets == 9] = 8
    without = Case(70, classes - 1, width, kind, seed=6, out=0)
    without.x, without.w = c.x, np.delete(c.w, 9, 0)
    without.targets = np.where(c.targets > 9, c.targets - 1, c.targets).astype(np.int32)
    want = without.reference()
    c.w[9] = -np.inf
    c.upload(mg)
    got = c.forward(mg)
    for k in want:
        assert_within(got[k], want[k], 2 * without.err[k], k)


@pytest.mark.parametrize("kind", ["fp32", "fp16"])
@pytest.mark.parametrize("size", [1e-30, 1e30])
@pytest.mark.parametrize("rows,classes,width", [(50, 260, 40), (300, 5000, 264)])
def test_cross_entropy_gradients_of_any_size(mg, kind, size, rows, classes, width):
    c = Case(rows, classes, width, kind, seed=7)
    c.dloss, c.dentropy = rounded(c.dloss * size, "fp32"), rounded(c.dentropy * size, "fp32")
    if kind == "fp16":  # a result's own range
        c.dloss, c.dentropy = rounded(c.dloss / size * 1e-3, "fp32"), rounded(c.dentropy / size * 1e-3, "fp32")
    c.check(mg)


@pytest.mark.parametrize("classes,width", [(200, 40), (40000, 264)])
def test_cross_entropy_rows_of_different_sizes(mg, classes, width):
    """fp32 rows of x over twenty powers of ten: each keeps its own accuracy."""
    c = Case(64, classes, width, "fp32", seed=8)
    c.x = rounded(c.x * 10.0 ** np.linspace(-20, 0.5, 64)[:, None], "fp32")
    want = c.reference()
    c.upload(mg)
    got = c.forward(mg)
    for k in want:
        assert_within(got[k], want[k], 2 * c.err[k], k)


@pytest.mark.parametrize("dx,dw", [(True, False), (False, True)])
@pytest.mark.parametrize("rows,classes,width", [(60, 500, 72), (600, 5000, 136)])
def test_cross_entropy_one_gradient(mg, dx, dw, rows, classes, width):
    c = Case(rows, classes, width, "bf16", seed=9)
    want = c.reference()
    c.upload(mg)
    lse, entropy = rounded(want["lse"], "fp32"), rounded(want["entropy"], "fp32")
    both = c.backward(mg, lse, entropy)
    out = Rows(mg, None, "bf16", shape=(rows if dx else classes, width))
    space = mg.DeviceBuffer(mg.cross_entropy_backward_workspace(*c.dims()) + 256)
    mg.cross_entropy_backward(*c.at, *c.dims(), lse=c.dev["lse"].ptr, dloss=c.dev["dloss"].ptr,
                              dentropy=c.dev["dentropy"].ptr, entropy=c.dev["entropy"].ptr, workspace=space.ptr,
                              workspace_bytes=space.nbytes, **{"dx" if dx else "dw": out.ptr}, **c.ld)
    mg._capi.check(mg.lib().mg_synchronize())
    np.testing.assert_array_equal(out.get(), both["dx" if dx else "dw"])


def test_cross_entropy_of_no_rows(mg):
    mg.cross_entropy(None, None, None, 0, 10, 16)
    out = Rows(mg, None, "fp32", shape=(10, 16))
    space = mg.DeviceBuffer(mg.cross_entropy_backward_workspace(0, 10, 16) + 256)
    mg.cross_entropy_backward(None, None, None, 0, 10, 16, lse=None, dloss=None, dw=out.ptr, workspace=space.ptr,
                              workspace_bytes=space.nbytes)
    mg._capi.check(mg.lib().mg_synchronize())
    assert (out.get() == 0).all()


def test_cross_entropy_gradient_against_differences(mg):
    """sum(loss a) + sum(entropy b) in 64 bits, moved along a direction of x and of w."""
    c = Case(30, 120, 24, "fp32", seed=10)

    def value():
        o = c.reference()
        return (o["loss"] * c.dloss).sum() + np.where(c.live, o["entropy"] * c.dentropy, 0).sum()

    want = c.reference()
    c.upload(mg)
    got = c.backward(mg, rounded(want["lse"], "fp32"), rounded(want["entropy"], "fp32"))
    r, h = np.random.RandomState(11), 1e-5
    for k, grad in (("x", got["dx"]), ("w", got["dw"])):
        v = getattr(c, k)
        along = r.normal(0, 1, v.shape)
        ends = []
        for sign in (1, -1):
            setattr(c, k, v + sign * h * along)
            ends.append(value())
        setattr(c, k, v)
        # h^2 of the differences, fp32's sums of terms that cancel
        assert abs((grad * along).sum() - (ends[0] - ends[1]) / (2 * h)) <= 1e-5 * np.abs(grad * along).sum(), k
