"""Rows and matrices that lie more than 2^32 elements apart, and the same values at
ordinary strides: the same bits."""
import numpy as np
import pytest

from operator_cases import SIZE, decode, encode, storage

pytestmark = pytest.mark.gpu


class Far:
    """`count` blocks of rows x cols elements, `stride` apart, their rows `ld` apart, in an
    allocation that is written and read only there."""

    def __init__(self, mg, values, kind, ld, stride):
        self.mg, self.kind, self.ld, self.stride = mg, kind, ld, stride
        self.shape = values.shape
        count, rows, cols = values.shape
        self.buf = mg.DeviceBuffer(((count - 1) * stride + (rows - 1) * ld + cols) * SIZE[kind])
        for k in range(count):
            for i in range(rows):
                a = np.ascontiguousarray(encode(values[k, i], kind))
                mg._capi.check(mg.lib().mg_memcpy_h2d(self.at(k, i), a.ctypes.data, a.nbytes))

    @property
    def ptr(self):
        return self.buf.ptr

    def at(self, k, i):
        return self.buf.ptr + (k * self.stride + i * self.ld) * SIZE[self.kind]

    def matrices(self):
        return self.mg.matrices(self.ptr, *self.shape, self.kind, self.ld, self.stride)

    def get(self):
        count, rows, cols = self.shape
        return np.stack([np.stack([decode(self.mg._capi.d2h(self.at(k, i), storage(self.kind), (cols,)), self.kind)
                                   for i in range(rows)]) for k in range(count)])


def floats(mg, n):
    return mg.DeviceBuffer.from_array(np.zeros(n, np.float32))


@pytest.mark.parametrize("cols", [40, 20001])
def test_layernorm_rows_far_apart(mg, cols):
    r = np.random.RandomState(0)
    rows, far = 3, (1 << 31) + 8
    x, dy = r.normal(1, 2, (1, rows, cols)), r.normal(0, 1, (1, rows, cols))
    out = []
    for ld in (far, cols):
        X, DY = Far(mg, x, "bf16", ld, 0), Far(mg, dy, "bf16", ld, 0)
        mean, rstd, dg, db = (floats(mg, n) for n in (rows, rows, cols, cols))
        y = floats(mg, rows * cols)
        n = mg.layernorm_backward_workspace(rows, cols)
        ws = mg.DeviceBuffer(max(n, 16))
        mg.layernorm(X.ptr, y.ptr, rows, cols, "bf16", x_ld=ld, mean=mean.ptr, rstd=rstd.ptr)
        mg.layernorm_backward(X.ptr, DY.ptr, mean.ptr, rstd.ptr, DY.ptr, rows, cols, "bf16", x_ld=ld, dy_ld=ld, dx_ld=ld,
                              dgamma=dg.ptr, dbeta=db.ptr, workspace=ws.ptr, workspace_bytes=n)
        mg.layernorm(X.ptr, X.ptr, rows, cols, "bf16", x_ld=ld, y_ld=ld)
        mg._capi.check(mg.lib().mg_synchronize())
        out.append([X.get(), DY.get(), y.download(np.uint16, (rows, cols)), dg.download(np.float32, (cols,)),
                    db.download(np.float32, (cols,))])
    for a, b in zip(*out):
        np.testing.assert_array_equal(a, b)
    assert np.isfinite(out[0][0]).all() and np.abs(out[0][1]).any(axis=2).all()


@pytest.mark.parametrize("rows,cols", [(4, 50), (140, 150)])
def test_matrices_far_apart(mg, rows, cols):
    r = np.random.RandomState(1)
    w, m, g = r.normal(0, 1, (2, rows, cols)), r.normal(0, 1e-3, (2, rows, cols)), r.normal(0, 1e-3, (2, rows, cols))
    out = []
    far_ld = (1 << 31) - 1 if rows == 4 else cols
    for ld, stride in ((far_ld, (rows - 1) * far_ld + (1 << 32)), (cols, rows * cols)):
        W, G = Far(mg, w, "bf16", ld, stride), Far(mg, g, "fp16", ld, stride)
        M = Far(mg, m, "fp32", cols, (1 << 32) + 8 if stride > rows * cols else stride)
        n = mg.orthogonalize_workspace(2, rows, cols)
        ws = mg.DeviceBuffer(n)
        mg.muon_step(W.matrices(), M.matrices(), G.matrices(), lr=0.1, workspace=ws.ptr, workspace_bytes=n)
        mg.orthogonalize(G.matrices(), G.matrices(), workspace=ws.ptr, workspace_bytes=n)
        mg._capi.check(mg.lib().mg_synchronize())
        out.append([W.get(), M.get(), G.get()])
    for a, b in zip(*out):
        np.testing.assert_array_equal(a, b)
    assert (out[0][0] != decode(encode(w, "bf16"), "bf16")).any() and np.abs(out[0][2]).max() > 0.01
