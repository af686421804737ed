"""mg_layernorm_backward of rows whose mean times rstd passes fp32's range: what lies
past a row's end in its last vector and its lanes must not reach the row's sums."""
import numpy as np
import pytest

from operator_cases import decode, encode
from test_gpu_layernorm import backward64, check_backward, run_backward, vectors

pytestmark = pytest.mark.gpu


def constant_row_case(rows, cols, kind, size):
    """Ordinary rows, and a constant one of +-2^120 whose rstd is that of eps 1e-5: each of
    its (x - mean) rstd is 0, while mean rstd is 2^128.3."""
    r = np.random.RandomState(cols)
    x = decode(encode(r.normal(0, 1, (rows, cols)), kind), kind)
    dy = decode(encode(r.normal(0, 1, (rows, cols)), kind), kind)
    mean, rstd = x.mean(1).astype(np.float32), (1 / np.sqrt(x.var(1) + 1e-5)).astype(np.float32)
    x[rows // 2], mean[rows // 2], rstd[rows // 2] = size, size, np.float32(1e-5) ** np.float32(-0.5)
    return x, dy, vectors(r, cols)[0], mean.astype(np.float64), rstd.astype(np.float64)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("cols", [3, 7, 17, 100, 127, 128, 300, 600, 1001, 1500, 3001, 8000, 12001, 20000, 20001])
def test_a_large_constant_row(mg, cols, kind):
    rows = 9 if cols < 5000 else 3
    for size in (2.0**120, -(2.0**120)):
        x, dy, g, m, v = constant_row_case(rows, cols, kind, size)
        got = run_backward(mg, x, dy, kind, g, m, v)
        assert np.isfinite(backward64(x, dy, g, m, v, None)[0]).all()
        check_backward(got, x, dy, kind, g, m, v, None)
