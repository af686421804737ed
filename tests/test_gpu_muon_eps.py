"""Matrices whose norm is far under eps: X starts at |G| / eps and the result stays small,
but it is the formula's result to as many bits as any other's.

The tolerance is test_gpu_muon's relative one: four times plain fp32's error, or 12 u a
step (u = 2^-24)."""
import numpy as np
import pytest

from operator_cases import decode, encode
from test_gpu_muon import COEFFS, check_orthogonal, gradients, run_muon, run_orth, tolerance

pytestmark = pytest.mark.gpu

SHAPES = [(60, 200), (128, 512), (300, 20), (200, 170), (150, 900), (1000, 257)]


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_vanishing_matrices(mg, rows, cols, kind):
    """A batch whose norms go from eps to 1e-27 of it, in binary steps."""
    powers = np.array([0, -3, -6, -9, -12, -15, -20, -30, -50, -90])
    g = gradients(np.random.RandomState(20), len(powers), rows, cols)
    g /= np.linalg.norm(g, axis=(1, 2), keepdims=True) / 1e-7
    g = decode(encode(g * 2.0 ** powers[:, None, None], kind), kind)
    got = run_orth(mg, g, kind, "fp32")
    for k, power in enumerate(powers):
        print(power, flush=True)
        # the same singular values with the power taken out of both, as fp32's squares need
        check_orthogonal(got[k], g[k] / 2.0**power, "fp32", eps=1e-7 / 2.0**power)


@pytest.mark.parametrize("eps", [1e-3, 1.0, 1e3, 1e8])
@pytest.mark.parametrize("steps,coeffs", [(5, COEFFS), (1, COEFFS), (12, (1.875, -1.25, 0.375)), (3, (1.0, 0.0, 0.0)),
                                          (7, (-1.5, 0.5, 0.0))])
@pytest.mark.parametrize("rows,cols", [(60, 200), (200, 170), (140, 500)])
def test_large_eps(mg, rows, cols, steps, coeffs, eps):
    g = gradients(np.random.RandomState(21), 2, rows, cols).astype(np.float32).astype(np.float64)
    ns = mg.NewtonSchulz(steps, *coeffs, eps)
    got = run_orth(mg, g, ns=ns)
    for k in range(2):
        check_orthogonal(got[k], g[k], "fp32", steps=steps, coeffs=coeffs, eps=eps)


@pytest.mark.parametrize("rows,cols", [(60, 200), (200, 170)])
def test_the_largest_growth(mg, rows, cols):
    """0.998 of Chebyshev's polynomial (itself takes 1 + 2^-52 out of [-2, 2] in 13 steps)
    makes up to 4.99^32 = 2e22 of a singular value: from 2^-80 and less it stays a power,
    and then is bounded by the polynomial alone."""
    coeffs = (4.99, -19.96, 15.968)
    ns = mg.NewtonSchulz(32, *coeffs, 1e-7)
    g = gradients(np.random.RandomState(23), 3, rows, cols)
    g /= np.linalg.norm(g, axis=(1, 2), keepdims=True)
    g = decode(encode(g * 2.0 ** np.array([-80.0, -126.0, -138.0])[:, None, None], "fp32"), "fp32")
    got = run_orth(mg, g, ns=ns)
    assert np.isfinite(got).all()
    assert all(np.linalg.svd(x, compute_uv=False).max() < 1.1 for x in got)


@pytest.mark.parametrize("rows,cols", [(128, 512), (200, 170)])
def test_a_step_by_a_vanishing_gradient(mg, rows, cols):
    from test_gpu_muon import iterate

    g = gradients(np.random.RandomState(22), 2, rows, cols)
    g = (1e-15 * g / np.linalg.norm(g, axis=(1, 2), keepdims=True)).astype(np.float32).astype(np.float64)
    z = np.zeros_like(g)
    w, m = run_muon(mg, z, z, g, "fp32", "fp32", lr=1.0, scale=1.0, momentum=0.0)
    np.testing.assert_array_equal(m, g)
    for k in range(2):
        want = iterate(g[k], np.float64)
        assert np.linalg.norm(-w[k] - want) <= tolerance(g[k], want, "fp32")
