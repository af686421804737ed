"""mg_layernorm and mg_layernorm_backward against float64 numpy.

Tolerances count roundings (u = 2^-24). A row's sums are chains of at most 16
terms a lane, 6 lane exchanges and 16 waves (D = 38; past 16384 columns the lane
chains grow by cols / 1024), so a mean is off by D u mean|x|, a second moment by
(D + 4) u of itself, an output by half a step of its type more. A gradient of a
vector is a chain of the rows of a group, the groups of a workgroup and the
partial rows."""
import numpy as np
import pytest

from operator_cases import HALF, TINY, U32, Rows, assert_within, decode, encode

pytestmark = pytest.mark.gpu

COLS = [1, 2, 3, 7, 8, 31, 32, 33, 64, 100, 127, 128, 129, 256, 257, 500, 512, 513, 1000, 1024, 1025, 2048, 2049, 4096,
        5000, 8192, 8193, 16384, 16385, 40001]


def rows_of(r, rows, cols, kind):
    x = r.normal(0, 1, (rows, cols)) * np.exp(0.5 * r.normal(0, 1, cols)) + r.normal(0, 2, (rows, 1))
    return decode(encode(x, kind), kind)


def chain(cols):
    return 38 + (cols / 1024 if cols > 16384 else 0)


def forward64(s, gamma, beta, eps):
    mean = s.mean(1)
    d = s - mean[:, None]
    rstd = 1 / np.sqrt((d * d).mean(1) + eps)
    return d * rstd[:, None] * gamma + beta, mean, rstd


def check_forward(got, s, gamma, beta, eps, kind):
    y, mean, rstd = got
    want, m64, r64 = forward64(s, gamma, beta, eps)
    cols = s.shape[1]
    D = chain(cols)
    off = D * U32 * np.abs(s).mean(1)
    if mean is not None:
        assert_within(mean, m64, off + U32 * np.abs(m64), "mean")
    # the second moment about a mean that is off by e grows by e^2
    rel = (D + 8) * U32 + (off * r64) ** 2
    if rstd is not None:
        assert_within(rstd, r64, r64 * rel, "rstd")
    xn = np.abs(s - m64[:, None]) * r64[:, None]
    tol = np.abs(gamma) * (xn * (rel[:, None] + 4 * U32) + (off * r64)[:, None]) + 2 * U32 * (np.abs(want) + np.abs(beta))
    assert_within(y, want, tol + HALF[kind] * (np.abs(want) + tol) + TINY[kind], "y")


def run_forward(mg, x, kind, gamma=None, beta=None, residual=None, eps=1e-5, stats=True, ld=0, offset=0, alias=None,
                stream=None):
    """y, mean, rstd and the stored sum. alias: the operand whose place y takes."""
    rows, cols = x.shape
    X = Rows(mg, x, kind, ld, offset)
    R = Rows(mg, residual, kind, ld, offset) if residual is not None else None
    S = Rows(mg, None, kind, ld, offset, x.shape) if residual is not None else None
    Y = {"x": X, "residual": R, "sum": S}.get(alias) or Rows(mg, None, kind, ld, offset, x.shape)
    vec = [mg.DeviceBuffer.from_array(v.astype(np.float32)) if v is not None else None for v in (gamma, beta)]
    st = [mg.DeviceBuffer(4 * max(1, rows)) if stats else None for _ in range(2)]
    ptr = lambda b: b.ptr if b is not None else None  # noqa: E731
    mg.layernorm(X.ptr, Y.ptr, rows, cols, kind, gamma=ptr(vec[0]), beta=ptr(vec[1]), eps=eps, residual=ptr(R),
                 sum=ptr(S), mean=ptr(st[0]), rstd=ptr(st[1]), x_ld=ld, residual_ld=ld, sum_ld=ld, y_ld=ld,
                 stream=stream)
    mg._capi.check(mg.lib().mg_synchronize())
    m, v = [b.download(np.float32, (rows,)).astype(np.float64) if b is not None else None for b in st]
    return Y.get(), m, v, S.get() if S is not None and alias != "sum" else None


def vectors(r, cols):
    return (r.normal(1, 0.2, cols).astype(np.float32).astype(np.float64),
            r.normal(0, 0.2, cols).astype(np.float32).astype(np.float64))


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("cols", COLS)
def test_forward_widths(mg, cols, kind):
    r = np.random.RandomState(cols)
    rows = 37 if cols < 5000 else 3
    x, (g, b) = rows_of(r, rows, cols, kind), vectors(r, cols)
    y, m, v, _ = run_forward(mg, x, kind, g, b)
    check_forward((y, m, v), x, g, b, 1e-5, kind)
    branch = decode(encode(r.normal(0, 1, x.shape), kind), kind)
    y, m, v, s = run_forward(mg, x, kind, g, b, residual=branch)
    np.testing.assert_array_equal(s, decode(encode((x + branch).astype(np.float32), kind), kind))
    check_forward((y, m, v), s, g, b, 1e-5, kind)


@pytest.mark.parametrize("rows", [0, 1, 2, 15, 16, 17, 63, 1000, 40000, 70001])
def test_forward_row_counts(mg, rows):
    r = np.random.RandomState(rows)
    x, (g, b) = rows_of(r, rows, 128, "fp32"), vectors(r, 128)
    y, m, v, _ = run_forward(mg, x, "fp32", g, b)
    if rows:
        check_forward((y, m, v), x, g, b, 1e-5, "fp32")


@pytest.mark.parametrize("kind,cols,ld,offset", [("fp32", 128, 131, 1), ("bf16", 128, 129, 3), ("fp16", 1001, 1003, 5),
                                                 ("fp32", 30, 200, 7), ("bf16", 20000, 20001, 1), ("fp32", 2000, 2048, 2)])
def test_strides_and_offsets(mg, kind, cols, ld, offset):
    r = np.random.RandomState(1)
    x, (g, b) = rows_of(r, 21, cols, kind), vectors(r, cols)
    branch = rows_of(r, 21, cols, kind)
    y, m, v, s = run_forward(mg, x, kind, g, b, residual=branch, ld=ld, offset=offset)
    check_forward((y, m, v), s, g, b, 1e-5, kind)


@pytest.mark.parametrize("cols", [128, 1000, 3000, 20000])
@pytest.mark.parametrize("alias", ["x", "residual", "sum"])
def test_forward_in_place(mg, cols, alias):
    r = np.random.RandomState(2)
    x, (g, b) = rows_of(r, 19, cols, "bf16"), vectors(r, cols)
    branch = rows_of(r, 19, cols, "bf16")
    want, m0, v0, _ = run_forward(mg, x, "bf16", g, b, residual=branch)
    y, m, v, _ = run_forward(mg, x, "bf16", g, b, residual=branch, alias=alias)
    np.testing.assert_array_equal(y, want)
    np.testing.assert_array_equal(m, m0)
    if alias == "x":
        np.testing.assert_array_equal(run_forward(mg, x, "bf16", g, b, alias="x")[0], run_forward(mg, x, "bf16", g, b)[0])


def test_forward_without_vectors_or_statistics(mg):
    x = rows_of(np.random.RandomState(3), 33, 100, "fp32")
    y, m, v, _ = run_forward(mg, x, "fp32", stats=False)
    assert m is None and v is None
    check_forward((y, None, None), x, np.ones(100), np.zeros(100), 1e-5, "fp32")


@pytest.mark.parametrize("cols", [128, 5000, 20000])
def test_forward_special_rows(mg, cols):
    """A constant row gives beta; a row that holds NaN or infinity gives NaN and
    leaves the others alone; a large offset keeps the deviations."""
    r = np.random.RandomState(4)
    x, (g, b) = rows_of(r, 6, cols, "fp32"), vectors(r, cols)
    x[1] = 0.0
    x[2, cols // 2] = np.nan
    x[4, 0] = np.inf
    y, m, v, _ = run_forward(mg, x, "fp32", g, b)
    np.testing.assert_array_equal(y[1], b)
    assert np.isnan(y[2]).all() and np.isnan(y[4]).all()
    keep = [0, 3, 5]
    check_forward((y[keep], m[keep], v[keep]), x[keep], g, b, 1e-5, "fp32")


# ---- backward -------------------------------------------------------------------------------------


def backward64(x, dy, gamma, mean, rstd, dsum):
    xn = (x - mean[:, None]) * rstd[:, None]
    d = dy * gamma
    n = x.shape[1]
    dx = rstd[:, None] * (d - d.sum(1, keepdims=True) / n - xn * ((d * xn).sum(1, keepdims=True) / n))
    return dx + (dsum if dsum is not None else 0), (dy * xn).sum(0), dy.sum(0)


def run_backward(mg, x, dy, kind, gamma, mean, rstd, dsum=None, sums=(True, True), ld=0, offset=0, alias=None,
                 stream=None):
    rows, cols = x.shape
    X, D = Rows(mg, x, kind, ld, offset), Rows(mg, dy, kind, ld, offset)
    S = Rows(mg, dsum, kind, ld, offset) if dsum is not None else None
    O = {"x": X, "dy": D, "dsum": S}.get(alias) or Rows(mg, None, kind, ld, offset, x.shape)
    f = lambda v: mg.DeviceBuffer.from_array(v.astype(np.float32)) if v is not None else None  # noqa: E731
    G, M, V = f(gamma), f(np.append(mean, 0)), f(np.append(rstd, 0))
    out = [Rows(mg, None, "fp32", shape=(1, cols)) if want else None for want in sums]
    need = mg.layernorm_backward_workspace(rows, cols)
    W = Rows(mg, None, "fp32", shape=(1, max(1, need // 4)))
    ptr = lambda b: b.ptr if b is not None else None  # noqa: E731
    mg.layernorm_backward(X.ptr, D.ptr, M.ptr, V.ptr, O.ptr, rows, cols, kind, gamma=ptr(G), dsum=ptr(S),
                          dgamma=ptr(out[0]), dbeta=ptr(out[1]), x_ld=ld, dy_ld=ld, dsum_ld=ld, dx_ld=ld,
                          workspace=W.ptr if need else None, workspace_bytes=need, stream=stream)
    mg._capi.check(mg.lib().mg_synchronize())
    W.get()  # nothing behind the workspace
    return (O.get(),) + tuple(o.get()[0] if o is not None else None for o in out)


def check_backward(got, x, dy, kind, gamma, mean, rstd, dsum):
    dx, dg, db = got
    want, g64, b64 = backward64(x, dy, gamma, mean, rstd, dsum)
    rows, cols = x.shape
    D = chain(cols)
    xn = np.abs(x - mean[:, None]) * rstd[:, None]
    d = np.abs(dy * gamma)
    m0, m1 = d.mean(1, keepdims=True), (d * xn).mean(1, keepdims=True)
    tol = (D + 12) * U32 * rstd[:, None] * (d + m0 + xn * m1)
    if dsum is not None:
        tol = tol + 2 * U32 * np.abs(dsum)
    assert_within(dx, want, tol + HALF[kind] * (np.abs(want) + tol) + TINY[kind], "dx")
    # rows of a group (at least 256 groups of a large grid), 6 + 16 in a workgroup, 16 + 32 partial rows
    terms = rows / 256 + 80
    if dg is not None:
        assert_within(dg, g64, (terms + 4) * U32 * np.abs(dy * xn).sum(0), "dgamma")
    if db is not None:
        assert_within(db, b64, terms * U32 * np.abs(dy).sum(0), "dbeta")


def backward_case(r, rows, cols, kind):
    x = rows_of(r, rows, cols, kind)
    dy = decode(encode(r.normal(0, 1, (rows, cols)), kind), kind)
    g, _ = vectors(r, cols)
    _, mean, rstd = forward64(x, g, 0, 1e-5) if rows else (0, np.zeros(0), np.zeros(0))
    return x, dy, g, mean.astype(np.float32).astype(np.float64), rstd.astype(np.float32).astype(np.float64)


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("cols", COLS)
def test_backward_widths(mg, cols, kind):
    r = np.random.RandomState(cols)
    x, dy, g, m, v = backward_case(r, 37 if cols < 5000 else 3, cols, kind)
    check_backward(run_backward(mg, x, dy, kind, g, m, v), x, dy, kind, g, m, v, None)
    dsum = decode(encode(r.normal(0, 1, x.shape), kind), kind)
    check_backward(run_backward(mg, x, dy, kind, g, m, v, dsum), x, dy, kind, g, m, v, dsum)


@pytest.mark.parametrize("rows,cols", [(0, 128), (1, 128), (2, 128), (31, 128), (32, 128), (33, 128), (1000, 128),
                                       (16384, 128), (40001, 128), (70000, 16), (3000, 1500), (600, 20000), (0, 20000)])
def test_backward_row_counts(mg, rows, cols):
    x, dy, g, m, v = backward_case(np.random.RandomState(rows), rows, cols, "fp32")
    got = run_backward(mg, x, dy, "fp32", g, m, v)
    if rows:
        check_backward(got, x, dy, "fp32", g, m, v, None)
    else:
        assert not got[1].any() and not got[2].any()


@pytest.mark.parametrize("sums", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("rows,cols", [(5, 100), (3000, 100), (7, 3000), (3, 20000)])
def test_backward_some_sums(mg, rows, cols, sums):
    x, dy, g, m, v = backward_case(np.random.RandomState(5), rows, cols, "fp32")
    check_backward(run_backward(mg, x, dy, "fp32", g, m, v, sums=sums), x, dy, "fp32", g, m, v, None)


@pytest.mark.parametrize("kind,cols,ld,offset", [("fp32", 128, 131, 1), ("bf16", 128, 129, 3), ("fp16", 1001, 1003, 5),
                                                 ("bf16", 20000, 20001, 1), ("fp32", 2000, 2048, 2)])
def test_backward_strides_and_offsets(mg, kind, cols, ld, offset):
    r = np.random.RandomState(6)
    x, dy, g, m, v = backward_case(r, 45, cols, kind)
    dsum = decode(encode(r.normal(0, 1, x.shape), kind), kind)
    got = run_backward(mg, x, dy, kind, g, m, v, dsum, ld=ld, offset=offset)
    check_backward(got, x, dy, kind, g, m, v, dsum)


@pytest.mark.parametrize("rows,cols", [(77, 128), (9, 3000), (5, 20000)])
@pytest.mark.parametrize("alias", ["x", "dy", "dsum"])
def test_backward_in_place(mg, rows, cols, alias):
    r = np.random.RandomState(7)
    x, dy, g, m, v = backward_case(r, rows, cols, "fp32")
    dsum = decode(encode(r.normal(0, 1, x.shape), "fp32"), "fp32")
    for a, b in zip(run_backward(mg, x, dy, "fp32", g, m, v, dsum, alias=alias),
                    run_backward(mg, x, dy, "fp32", g, m, v, dsum)):
        np.testing.assert_array_equal(a, b)


def test_backward_is_the_forwards_gradient(mg):
    """Central differences of the float64 forward, in the direction of random dx."""
    r = np.random.RandomState(8)
    x, dy, g, m, v = backward_case(r, 12, 96, "fp32")
    dx, dg, db = run_backward(mg, x, dy, "fp32", g, m, v)
    h = 1e-5
    along = r.normal(0, 1, x.shape)
    loss = lambda x, g, b: (forward64(x, g, b, 1e-5)[0] * dy).sum()  # noqa: E731
    num = (loss(x + h * along, g, 0) - loss(x - h * along, g, 0)) / (2 * h)
    # differences lose h^2 and 1e-16 / h, the fp32 gradient 60 u of its terms
    assert abs((dx * along).sum() - num) <= 1e-5 * np.abs(dx * along).sum()
    av = r.normal(0, 1, 96)
    assert abs((dg * av).sum() - (loss(x, g + h * av, 0) - loss(x, g - h * av, 0)) / (2 * h)) <= 1e-5 * np.abs(dg * av).sum()
    assert abs((db * av).sum() - (loss(x, g, h * av) - loss(x, g, -h * av)) / (2 * h)) <= 1e-5 * np.abs(db * av).sum()


def test_a_nan_row_stays_in_its_row(mg):
    x, dy, g, m, v = backward_case(np.random.RandomState(9), 50, 128, "fp32")
    dy[7, 3] = np.nan
    dx, dg, db = run_backward(mg, x, dy, "fp32", g, m, v)
    assert np.isnan(dx[7]).all() and np.isfinite(np.delete(dx, 7, 0)).all()
    assert np.isnan(dg[3]) and np.isfinite(np.delete(dg, 3)).all() and np.isfinite(np.delete(db, 3)).all()


def test_reruns_have_the_same_bits(mg):
    x, dy, g, m, v = backward_case(np.random.RandomState(10), 20000, 128, "bf16")
    first = run_backward(mg, x, dy, "bf16", g, m, v)
    for a, b in zip(first, run_backward(mg, x, dy, "bf16", g, m, v)):
        np.testing.assert_array_equal(a, b)
