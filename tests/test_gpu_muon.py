"""mg_orthogonalize and mg_muon_step against float64 numpy.

Tolerance of an orthogonalised matrix, in the Frobenius norm: the kernels' operands
keep 22 bits where fp32 keeps 24, so four times the error that the plain iteration
in fp32 (numpy) has on the same matrix, and half a step of the result's type. On a
matrix of few elements fp32's own error may be small by chance; what the products
may lose in any case is 12 u each (u = 2^-24): the halves' remainders are at most
2^-11 and 2^-22 of an element, so each operand is off by 4 u, and the product of the
low halves, left out, is 4 u. One such loss a step is the least allowed."""
import numpy as np
import pytest

from operator_cases import HALF, TINY, U32, Rows, assert_within, decode, encode

pytestmark = pytest.mark.gpu

COEFFS = (3.4445, -4.7750, 2.0315)


def iterate(g, dtype, steps=5, coeffs=COEFFS, eps=1e-7):
    a, b, c = (dtype(np.float32(k)) for k in coeffs)
    x = g.astype(dtype)
    tall = x.shape[0] > x.shape[1]
    x = x.T.copy() if tall else x
    x = x / (dtype(np.sqrt((x * x).sum())) + dtype(np.float32(eps)))
    for _ in range(steps):
        gram = x @ x.T
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.T if tall else x).astype(np.float64)


def tolerance(g, want, kind, **kw):
    own = np.linalg.norm(iterate(g, np.float32, **kw) - want)
    least = 12 * U32 * kw.get("steps", 5) * np.linalg.norm(want)
    return max(4 * own, least) + HALF[kind] * np.linalg.norm(want) + TINY[kind] * want.size**0.5


def check_orthogonal(got, g, kind, **kw):
    want = iterate(g, np.float64, **kw)
    off = np.linalg.norm(got - want)
    tol = tolerance(g, want, kind, **kw)
    assert off <= tol, f"off by {off:.3e}, tolerance {tol:.3e}, norm {np.linalg.norm(want):.3e}"


def gradients(r, count, rows, cols, kind="gauss"):
    m = min(rows, cols)
    if kind == "gauss":
        g = r.normal(0, 1e-3, (count, rows, cols))
    else:  # a few strong directions over a floor
        rank = max(1, m // 8)
        g = r.normal(0, 1, (count, rows, rank)) * np.logspace(0, -2, rank) @ r.normal(0, 1, (count, rank, cols))
        g = 1e-3 * (g + 0.1 * r.normal(0, 1, (count, rows, cols)))
    return g


def stack(mg, values, kind, ld=0, gap=0, offset=0):
    """A batch as rows of a Rows array: matrices follow each other with `gap` rows between."""
    count, rows, cols = values.shape
    ld = ld or cols
    full = np.zeros((count, rows + gap, cols))
    full[:, :rows] = values
    R = Rows(mg, full.reshape(-1, cols), kind, ld, offset)
    desc = mg.matrices(R.ptr, count, rows, cols, kind, ld, (rows + gap) * ld)
    return R, desc, lambda: R.get().reshape(count, rows + gap, cols)[:, :rows]


def space(mg, count, rows, cols, ns=None):
    """A workspace whose words are NaN, so that one that is read unwritten shows."""
    n = mg.orthogonalize_workspace(count, rows, cols, ns)
    guard = 4096
    b = mg.DeviceBuffer.from_array(np.full(n + guard, 0xFF, np.uint8))

    def untouched():
        assert (b.download(np.uint8, (n + guard,))[n:] == 0xFF).all(), "written behind the workspace"

    return b, n, untouched


def run_orth(mg, g, kind="fp32", out_kind=None, ns=None, ld=0, gap=0, offset=0, in_place=False, stream=None):
    count, rows, cols = g.shape
    A, a, _ = stack(mg, g, kind, ld, gap, offset)
    out_kind = out_kind or kind
    B, b, get = (A, a, lambda: A.get().reshape(count, rows + gap, cols)[:, :rows]) if in_place else stack(
        mg, np.zeros_like(g), out_kind, ld, gap, offset)
    w, n, untouched = space(mg, count, rows, cols, ns)
    mg.orthogonalize(a, b, ns=ns, workspace=w.ptr, workspace_bytes=n, stream=stream)
    mg._capi.check(mg.lib().mg_synchronize())
    untouched()
    return get()


SHAPES = [(1, 1), (1, 5), (7, 1), (2, 3), (16, 16), (31, 33), (32, 64), (65, 64), (64, 200), (100, 128), (127, 129),
          (128, 128), (128, 512), (512, 128), (129, 128), (130, 1000), (256, 256), (257, 1000), (1000, 257), (300, 301),
          (128, 2500), (20, 4001), (640, 700)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("spectrum", ["gauss", "strong"])
def test_shapes(mg, rows, cols, spectrum):
    g = decode(encode(gradients(np.random.RandomState(rows + cols), 1, rows, cols, spectrum), "fp32"), "fp32")
    check_orthogonal(run_orth(mg, g)[0], g[0], "fp32")


@pytest.mark.parametrize("kind,out_kind", [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "fp32"), ("fp32", "bf16")])
@pytest.mark.parametrize("rows,cols", [(128, 512), (100, 77), (400, 150)])
def test_types(mg, kind, out_kind, rows, cols):
    g = decode(encode(gradients(np.random.RandomState(1), 2, rows, cols, "strong"), kind), kind)
    got = run_orth(mg, g, kind, out_kind)
    for k in range(2):
        check_orthogonal(got[k], g[k], out_kind)


@pytest.mark.parametrize("count,rows,cols", [(3, 128, 256), (16, 40, 50), (2, 200, 150), (33, 8, 8)])
def test_batches_with_strides(mg, count, rows, cols):
    g = decode(encode(gradients(np.random.RandomState(2), count, rows, cols), "bf16"), "bf16")
    got = run_orth(mg, g, "bf16", ld=cols + 3, gap=2, offset=5)
    for k in range(count):
        check_orthogonal(got[k], g[k], "bf16")


@pytest.mark.parametrize("rows,cols", [(128, 512), (150, 140)])
def test_in_place(mg, rows, cols):
    g = decode(encode(gradients(np.random.RandomState(3), 2, rows, cols), "fp32"), "fp32")
    np.testing.assert_array_equal(run_orth(mg, g, in_place=True), run_orth(mg, g))


@pytest.mark.parametrize("count,rows,cols", [(4, 1000, 1100), (4, 1100, 1000), (2, 1400, 2000), (9, 600, 1100)])
def test_larger_batches(mg, count, rows, cols):
    """Batches that take 128 x 128 tiles, with and without segments of two steps."""
    g = decode(encode(gradients(np.random.RandomState(11), count, rows, cols, "strong"), "bf16"), "bf16")
    got = run_orth(mg, g, "bf16", "fp32")
    for k in {0, count - 1}:
        check_orthogonal(got[k], g[k], "fp32")
    np.testing.assert_array_equal(got, run_orth(mg, g, "bf16", "fp32"))


@pytest.mark.parametrize("kind,powers", [("bf16", (110, 60, 0, -12)), ("fp16", (14, 6, 0, -4))])
@pytest.mark.parametrize("rows,cols", [(200, 333), (500, 150), (90, 200), (170, 180)])
def test_half_width_sources_of_any_scale(mg, kind, powers, rows, cols):
    """A batch whose matrices differ by powers of two, from beyond fp32's squares to near
    eps, with entries over a wide range; in fp32, so that the result's own rounding hides
    nothing. The formula is taken without the power, which the plain iteration needs."""
    r = np.random.RandomState(9)
    g = gradients(r, len(powers), rows, cols, "strong") * np.exp(r.normal(0, 1.5, (1, rows, 1)))
    g = decode(encode(g * 2.0 ** np.array(powers)[:, None, None], kind), kind)
    assert np.isfinite(g).all()
    got = run_orth(mg, g, kind, "fp32")
    for k, power in enumerate(powers):
        check_orthogonal(got[k], g[k] / 2.0**power, "fp32", eps=1e-7 / 2.0**power)


def test_an_empty_batch_is_nothing(mg):
    mg.orthogonalize(mg.matrices(None, 0, 4, 4), mg.matrices(None, 0, 4, 4))


@pytest.mark.parametrize("rows,cols", [(96, 300), (200, 170)])
def test_a_matrix_and_its_transpose(mg, rows, cols):
    g = gradients(np.random.RandomState(4), 1, rows, cols).astype(np.float32).astype(np.float64)
    np.testing.assert_array_equal(run_orth(mg, g)[0], run_orth(mg, np.ascontiguousarray(g.transpose(0, 2, 1)))[0].T)


@pytest.mark.parametrize("steps,coeffs", [(1, COEFFS), (2, COEFFS), (3, COEFFS), (4, COEFFS), (6, COEFFS), (7, COEFFS),
                                          (12, (1.875, -1.25, 0.375)), (20, (1.5, -0.5, 0.0)), (3, (1.0, 0.0, 0.0))])
@pytest.mark.parametrize("rows,cols", [(64, 200), (150, 160), (140, 400)])
def test_steps_and_polynomials(mg, steps, coeffs, rows, cols):
    g = gradients(np.random.RandomState(5), 1, rows, cols).astype(np.float32).astype(np.float64)
    ns = mg.NewtonSchulz(steps, *coeffs, 1e-7)
    check_orthogonal(run_orth(mg, g, ns=ns)[0], g[0], "fp32", steps=steps, coeffs=coeffs)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,cols", [(60, 200), (200, 333), (500, 140)])
def test_special_half_width_matrices(mg, kind, rows, cols):
    """As below for 16-bit sources, whose norms go from eps to past fp32's range."""
    r = np.random.RandomState(10)
    g = gradients(r, 5, rows, cols)
    g[0] = 0
    g[1, rows // 2, 3] = np.nan
    g[2, rows - 1, cols - 1] = -np.inf
    g[3] = np.sign(g[3]) * (3e38 if kind == "bf16" else 65000.0)
    g = decode(encode(g, kind), kind)
    got = run_orth(mg, g, kind, "fp32")
    assert not got[0].any()
    assert np.isnan(got[1]).all() and np.isnan(got[2]).all()
    check_orthogonal(got[3], np.sign(g[3]), "fp32", eps=0.0)
    check_orthogonal(got[4], g[4], "fp32")


@pytest.mark.parametrize("count,rows,cols", [(300, 70, 200), (130, 128, 520), (40, 1300, 96), (260, 200, 20)])
def test_batches_of_more_matrices_than_fit_at_once(mg, count, rows, cols):
    """Workgroups that take one, several or all slabs of a matrix."""
    g = gradients(np.random.RandomState(11), count, rows, cols).astype(np.float32).astype(np.float64)
    got = run_orth(mg, g)
    for k in range(count):
        check_orthogonal(got[k], g[k], "fp32")


@pytest.mark.parametrize("kind", ["fp32", "fp16"])
@pytest.mark.parametrize("count,rows,cols", [(1, 250, 8230), (1, 8230, 250), (3, 250, 2800), (1, 500, 4100)])
def test_long_matrices(mg, kind, count, rows, cols):
    """Squares in smaller tiles than the products with X."""
    g = decode(encode(gradients(np.random.RandomState(12), count, rows, cols), kind), kind)
    got = run_orth(mg, g, kind)
    for k in range(count):
        check_orthogonal(got[k], g[k], kind)


@pytest.mark.parametrize("rows,cols", [(60, 200), (200, 170)])
def test_special_matrices(mg, rows, cols):
    """Zeros give zeros, a NaN or an infinity gives NaN throughout, huge and tiny
    entries scale away, and eps keeps a vanishing matrix small."""
    r = np.random.RandomState(6)
    g = gradients(r, 6, rows, cols).astype(np.float32).astype(np.float64)
    g[0] = 0
    g[1, rows // 2, 3] = np.nan
    g[2, 0, cols - 1] = np.inf
    g[3] = (g[3] * 1e40).astype(np.float32)  # squares beyond fp32
    g[4] = (g[4] * 1e-18).astype(np.float32)  # under eps
    got = run_orth(mg, g)
    assert not got[0].any()
    assert np.isnan(got[1]).all() and np.isnan(got[2]).all()
    big = g[3] / 2.0**100  # a power of two: the same bits but for eps
    check_orthogonal(got[3], big, "fp32", eps=0.0)
    check_orthogonal(got[5], g[5], "fp32")
    assert np.isfinite(got[4]).all() and np.linalg.norm(got[4]) < 1e-9


def test_reruns_have_the_same_bits(mg):
    g = gradients(np.random.RandomState(7), 2, 300, 500)
    np.testing.assert_array_equal(run_orth(mg, g), run_orth(mg, g))


# ---- the optimiser's step ---------------------------------------------------------------------------


def run_muon(mg, w, m, g, kind, grad, ld=0, gap=0, **kw):
    count, rows, cols = w.shape
    _, a, get_w = stack(mg, w, kind, ld, gap)
    _, b, get_m = stack(mg, m, "fp32", ld, gap)
    _, c, _ = stack(mg, g, grad, ld, gap)
    buf, n, untouched = space(mg, count, rows, cols)
    mg.muon_step(a, b, c, workspace=buf.ptr, workspace_bytes=n, **kw)
    mg._capi.check(mg.lib().mg_synchronize())
    untouched()
    return get_w(), get_m()


def check_muon(got, w, m, g, kind, lr=0.02, momentum=0.95, weight_decay=0.0, scale=0.0, nesterov=True):
    f = lambda x: float(np.float32(x))  # noqa: E731
    beta = f(momentum)
    m1 = m + (1 - beta) * (g - m)
    u = g + beta * (m1 - g) if nesterov else m1
    rows, cols = w.shape[1:]
    rate = f(lr) * (f(scale) if scale else np.sqrt(max(1, cols / rows)))
    keep = 1 - f(lr) * f(weight_decay)
    # 1 - beta is one rounding of fp32, the difference and the two steps to M one each
    assert_within(got[1], m1, 4 * U32 * (np.abs(m) + np.abs(g)), "momentum")
    for k in range(len(w)):
        o = iterate(u[k], np.float64)
        want = keep * w[k] - rate * o
        # U is a few roundings off, which the iteration takes as it takes its operands'
        tol = 2 * rate * tolerance(u[k], o, "fp32") + (4 * U32 + HALF[kind]) * np.linalg.norm(np.abs(w[k]) + rate * np.abs(o))
        off = np.linalg.norm(got[0][k] - want)
        assert off <= tol, f"matrix {k}: off by {off:.3e}, tolerance {tol:.3e}"


@pytest.mark.parametrize("kind,grad", [("fp32", "fp32"), ("fp32", "bf16"), ("bf16", "bf16"), ("fp16", "fp32")])
@pytest.mark.parametrize("rows,cols", [(128, 512), (512, 128), (200, 333)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step(mg, kind, grad, rows, cols, nesterov):
    r = np.random.RandomState(8)
    q = lambda x, t: decode(encode(x, t), t)  # noqa: E731
    w, m = q(r.normal(0, rows**-0.5, (2, rows, cols)), kind), q(gradients(r, 2, rows, cols), "fp32")
    g = q(gradients(r, 2, rows, cols, "strong"), grad)
    kw = dict(lr=0.05, momentum=0.9, weight_decay=0.1, nesterov=nesterov)
    check_muon(run_muon(mg, w, m, g, kind, grad, **kw), w, m, g, kind, **kw)


@pytest.mark.parametrize("count,rows,cols", [(2, 128, 1500), (1, 2100, 60), (300, 40, 200), (1, 250, 8230), (2, 1100, 1300)])
def test_muon_step_of_several_slabs_and_tiles(mg, count, rows, cols):
    """Sources that are read twice, the momentum's update between."""
    r = np.random.RandomState(13)
    q = lambda x, t: decode(encode(x, t), t)  # noqa: E731
    w, m = q(r.normal(0, rows**-0.5, (count, rows, cols)), "fp32"), q(gradients(r, count, rows, cols), "fp32")
    g = q(gradients(r, count, rows, cols, "strong"), "bf16")
    check_muon(run_muon(mg, w, m, g, "fp32", "bf16"), w, m, g, "fp32")


def test_muon_scale_strides_and_no_rate(mg):
    r = np.random.RandomState(9)
    w, m, g = (gradients(r, 3, 50, 70).astype(np.float32).astype(np.float64) for _ in range(3))
    kw = dict(lr=0.1, scale=0.2, momentum=0.0)
    check_muon(run_muon(mg, w, m, g, "fp32", "fp32", ld=75, gap=1, **kw), w, m, g, "fp32", **kw)
    got_w, got_m = run_muon(mg, w, m, g, "fp32", "fp32", lr=0.0)
    np.testing.assert_array_equal(got_w, w)
    check_muon((got_w, got_m), w, m, g, "fp32", lr=0.0)


def test_muon_steps_lead_to_an_orthogonal_direction(mg):
    """The same gradient again and again: the weights move along one direction whose
    singular values lie between 0.68 and 1.21 times the rate, the polynomial's range
    over [1e-2, 1] (128 alike singular values are 0.09 of the norm each)."""
    r = np.random.RandomState(10)
    q1 = np.linalg.qr(r.normal(0, 1, (128, 128)))[0]
    q2 = np.linalg.qr(r.normal(0, 1, (256, 128)))[0]
    g = (q1 * r.uniform(0.5, 1.5, 128) @ q2.T)[None]
    w, m = np.zeros_like(g), np.zeros_like(g)
    for _ in range(3):
        w, m = run_muon(mg, w, m, g, "fp32", "fp32", lr=1.0, scale=1.0)
    s = np.linalg.svd(w[0], compute_uv=False)
    assert 3 * 0.68 < s.min() and s.max() < 3 * 1.21
