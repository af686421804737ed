"""mg_muon_step on fp32 weights orthogonalises as accurately as mg_orthogonalize does."""
import numpy as np
import pytest

from test_gpu_muon import gradients, run_muon, run_orth

pytestmark = pytest.mark.gpu


def step_of_zeros(mg, g, grad="fp32"):
    """The Muon step of W = 0 and M = 0 that is minus the orthogonalised gradient."""
    z = np.zeros_like(g)
    w, m = run_muon(mg, z, z, g, "fp32", grad, lr=1.0, scale=1.0, momentum=0.0)
    np.testing.assert_array_equal(m, g)
    return -w


def f32(a):
    return a.astype(np.float32).astype(np.float64)


@pytest.mark.parametrize("count,rows,cols", [(2, 128, 512), (1, 512, 128), (3, 72, 56), (2, 40, 90), (1, 20, 33),
                                             (1, 200, 900), (2, 300, 257), (1, 1000, 257), (1, 2100, 60)])
def test_a_step_of_fp32_weights_has_the_bits_of_the_result(mg, count, rows, cols):
    """No weight is there whose rounding, and no rate under 1 that could hide fewer bits."""
    g = f32(gradients(np.random.RandomState(rows + cols), count, rows, cols, "strong"))
    np.testing.assert_array_equal(step_of_zeros(mg, g), run_orth(mg, g))
