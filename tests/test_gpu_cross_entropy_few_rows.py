"""Gradients of 16-bit heads with few rows, whose logits' gradient is kept as two halves: their error is the results'
own rounding, with what fp32 sums are off by, and nothing of 16 bits before it."""
import numpy as np
import pytest

from operator_cases import HALF, Rows, assert_within
from rollout_cases import rounded
from test_gpu_cross_entropy import Case
from test_gpu_cross_entropy_parts import check_some, some_gradients, statistics

pytestmark = pytest.mark.gpu

# a row or a few, an odd last block of 32 and a full one, the most; one piece's classes and two pieces'
SHAPES = [(1, 25032, 368), (2, 60760, 128), (7, 13566, 1016), (30, 27257, 348), (33, 9329, 4104), (64, 9250, 520),
          (96, 30000, 129), (97, 20011, 264), (128, 50000, 128), (3, 1 << 20, 64)]


def picked(c, seed):
    r = np.random.RandomState(seed)
    live = c.targets[c.live]
    return np.arange(c.rows), np.unique(np.r_[0, c.classes - 1, live, r.randint(0, c.classes, 60)])


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,classes,width", SHAPES)
def test_gradients_of_few_rows(mg, kind, rows, classes, width):
    """Two halves, each rounded: HALF squared."""
    c = Case(rows, classes, width, kind, seed=rows, out=0.1 if rows > 3 else 0)
    check_some(c, mg, *picked(c, 1), held=HALF[kind] ** 2)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 5)])
def test_strided_rows(mg, kind, pad, offset):
    c = Case(45, 20011, 520, kind, seed=2, pad=pad, offset=offset, entropy=False)
    check_some(c, mg, *picked(c, 3), held=HALF[kind] ** 2)


@pytest.mark.parametrize("dx", [True, False])
def test_one_gradient(mg, dx):
    c = Case(40, 20011, 520, "bf16", seed=4)
    rows, classes = picked(c, 5)
    lse, entropy, both = check_some(c, mg, rows, classes, held=HALF["bf16"] ** 2)
    out = Rows(mg, None, "bf16", shape=(c.rows if dx else c.classes, c.width))
    space = mg.DeviceBuffer(mg.cross_entropy_backward_workspace(*c.dims()) + 256)
    mg.cross_entropy_backward(*c.at, *c.dims(), lse=c.dev["lse"].ptr, dloss=c.dev["dloss"].ptr,
                              dentropy=c.dev["dentropy"].ptr, entropy=c.dev["entropy"].ptr, workspace=space.ptr,
                              workspace_bytes=space.nbytes, **{"dx" if dx else "dw": out.ptr}, **c.ld)
    mg._capi.check(mg.lib().mg_synchronize())
    np.testing.assert_array_equal(out.get(), both["dx" if dx else "dw"])


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_rows_left_out_hold_anything(mg, kind):
    c = Case(60, 30011, 200, kind, seed=6)
    c.targets[10:14] = [-1, c.classes, -5, 2**31 - 1]
    lse, entropy = statistics(c)
    rows, classes = picked(c, 7)
    dx, dw = some_gradients(c, lse, entropy, rows, classes, HALF[kind] ** 2)
    c.x[10], c.x[11, 3], c.x[12] = np.nan, np.inf, rounded(np.full(c.width, 3e4), kind)
    c.dloss[10], c.dloss[12], c.dentropy[13] = np.nan, 1e30, np.inf
    lse[10], entropy[11] = np.nan, np.inf
    c.upload(mg)
    got = c.backward(mg, lse, entropy)
    assert_within(got["dx"], *dx, "dx")
    assert_within(got["dw"][classes], *dw, "dw")
    assert (got["dx"][~c.live] == 0).all()
