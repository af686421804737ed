"""The partial sums of the cross entropy's gradients: a last range of classes that ends before what a piece is
filled up to. New device memory is NaN (conftest.py), so a sum of what nothing wrote shows."""
import numpy as np
import pytest

from operator_cases import HALF, TINY, U32, assert_within
from rollout_cases import rounded
from test_gpu_cross_entropy import Case

pytestmark = pytest.mark.gpu


def statistics(c):
    """lse and entropy about as a forward pass leaves them for logits of a spread of 1.5: the gradients are those of
    whatever statistics the call is given."""
    r = np.random.RandomState(6)
    most = np.log(c.classes)
    return (rounded(most + 1.125 + r.normal(0, 0.1, c.rows), "fp32"), rounded(most - 1.125 + r.normal(0, 0.1, c.rows), "fp32"))


def some_gradients(c, lse, entropy, rows, classes, held=None):
    """dX of some rows and dW of some classes, with the bounds of Case.gradients; `held`: half a step of what the
    logits' gradient is kept in, where that is less than the type's."""
    pairs = c.kind == "fp32"
    live = c.live
    most = np.abs(c.dloss[live])
    if c.dentropy is not None:
        most = most + (np.log(c.classes) + 1) * np.abs(c.dentropy[live])
    width = c.width

    def of(R, C):
        x, w = c.x[R], c.w[C]
        s, size = x @ w.T, np.abs(x) @ np.abs(w).T
        es = size * 2 * U32 * (17 + width / 16 * (3 if pairs else 1))
        if pairs:
            xm, wm = np.abs(x).max(1, keepdims=True), np.abs(c.w).max()
            es = es + size * 3 * 2.0**-22 + 2.0**-39 * (xm * np.abs(w).sum(1) + wm * np.abs(x).sum(1, keepdims=True))
        log = s - lse[R][:, None]
        p = np.exp(log)
        off = es + 4 * U32 * (np.abs(s) + np.abs(lse[R])[:, None] + 1)
        g = c.dloss[R][:, None] * p
        eg = np.abs(g) * (off + 4 * U32)
        if c.dentropy is not None:
            more = c.dentropy[R][:, None] * p * (log + entropy[R][:, None])
            g = g - more
            eg = eg + np.abs(more) * (off + 6 * U32) + np.abs(c.dentropy[R])[:, None] * p * (
                off + 4 * U32 * np.abs(entropy[R])[:, None])
        g = g - np.where(c.targets[R][:, None] == C[None], c.dloss[R][:, None], 0)
        eg = eg + U32 * np.abs(g)
        eg = eg + np.abs(g) * (held or (2.0**-22 if pairs else HALF[c.kind]))
        if c.kind != "bf16":
            eg = eg + most.max() * 2.0**-38
        g[~live[R]], eg[~live[R]] = 0, 0
        return g, eg

    def product(a, ea, b):
        v, size = a @ b, np.abs(a) @ np.abs(b)
        n = a.shape[1]
        # the parts' sums, and where pieces add to them a rounding for each
        chain = 2 * U32 * (16 + n / 16 * (3 if pairs else 1)) + U32 * (n / 256 + 16)
        err = ea @ np.abs(b) + size * (chain + (2.0**-21 if pairs else 0.0))
        if pairs:
            err = err + 2.0**-38 * (np.abs(a).sum(1, keepdims=True) * np.abs(b).max()
                                    + np.abs(b).sum(0) * np.abs(a).max())
        return v, 2 * err + (np.abs(v) + err) * HALF[c.kind] + TINY[c.kind]

    g, eg = of(rows, np.arange(c.classes))
    dx = product(g, eg, c.w)
    g, eg = of(np.arange(c.rows), classes)
    return dx, product(g.T, eg.T, np.where(live[:, None], c.x, 0.0))


def check_some(c, mg, rows, classes, held=None):
    lse, entropy = statistics(c)
    c.upload(mg)
    got = c.backward(mg, lse, entropy)
    dx, dw = some_gradients(c, lse, entropy, rows, classes, held)
    assert_within(got["dx"][rows], *dx, "dx")
    assert_within(got["dw"][classes], *dw, "dw")
    assert np.isfinite(got["dx"]).all() and np.isfinite(got["dw"]).all()
    return lse, entropy, got


@pytest.mark.parametrize("kind,rows,classes,width", [
    ("bf16", 512, 50000, 128), ("fp32", 512, 50000, 128), ("bf16", 1024, 9250, 128), ("fp32", 1024, 9250, 256),
    ("bf16", 512, 9250, 512), ("fp16", 512, 9250, 512), ("bf16", 743, 14141, 128), ("fp32", 282, 25354, 165),
    ("fp16", 388, 27767, 128), ("bf16", 4, 41171, 128)])
def test_last_range_of_padding(mg, kind, rows, classes, width):
    c = Case(rows, classes, width, kind, seed=1)
    r = np.random.RandomState(2)
    some = np.unique(np.r_[0, rows - 1, r.randint(0, rows, 30)])
    few = np.unique(np.r_[0, classes - 1, c.targets[c.live][:10], r.randint(0, classes, 40)])
    lse, entropy, got = check_some(c, mg, some, few)

    # whatever the workspace held
    make = mg.DeviceBuffer.__init__

    def zeros(self, nbytes):
        make(self, nbytes)
        self.zero()

    mg.DeviceBuffer.__init__ = zeros
    try:
        again = c.backward(mg, lse, entropy)
    finally:
        mg.DeviceBuffer.__init__ = make
    for k in got:
        np.testing.assert_array_equal(again[k], got[k])
