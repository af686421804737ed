"""Groups that take several rows: grids of workgroups smaller than the rows, at every
width class whose group is a workgroup, and the wide kernels. The reduction sets in LDS
and the grid stride are used again and again here.

Statistics and outputs are held to the tolerances of test_gpu_layernorm. dgamma and
dbeta have their own: a group's chain is its rows (rows / groups + 1), then partial rows
are added in 32 slices (chains of groups / 32 + 1) and the slices in order (32), with the
lanes' and waves' sums before (6 + 16)."""
import numpy as np
import pytest

from operator_cases import U32, assert_within, decode, encode
from test_gpu_layernorm import (backward64, backward_case, check_backward, check_forward, rows_of, run_backward, run_forward,
                                vectors)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols,kind,residual", [
    (2100, 1500, "fp32", False), (2100, 1500, "bf16", True), (1100, 3000, "fp16", False), (1100, 3000, "fp32", True),
    (1100, 8192, "bf16", True), (1100, 8000, "fp32", False), (600, 16384, "fp32", False), (600, 12001, "bf16", True),
    (600, 16385, "fp32", False), (600, 20001, "fp16", True), (9000, 1025, "bf16", False), (20000, 1000, "fp16", True)])
def test_forward(mg, rows, cols, kind, residual):
    r = np.random.RandomState(rows + cols)
    x, (g, b) = rows_of(r, rows, cols, kind), vectors(r, cols)
    branch = decode(encode(r.normal(0, 1, x.shape), kind), kind) if residual else None
    y, m, v, s = run_forward(mg, x, kind, g, b, residual=branch)
    if residual:
        np.testing.assert_array_equal(s, decode(encode((x + branch).astype(np.float32), kind), kind))
    check_forward((y, m, v), s if residual else x, g, b, 1e-5, kind)


@pytest.mark.parametrize("rows,cols,kind,groups", [
    (8200, 1100, "fp32", 1024), (8191, 1100, "bf16", 512), (8192, 1025, "fp16", 1024), (1100, 3000, "fp32", 512),
    (1100, 4096, "bf16", 512), (600, 8192, "fp32", 256), (600, 5001, "fp16", 256), (600, 16384, "bf16", 256),
    (600, 12001, "fp32", 256), (600, 16385, "fp32", 64), (20000, 1000, "bf16", 512)])
def test_backward(mg, rows, cols, kind, groups):
    x, dy, g, m, v = backward_case(np.random.RandomState(rows + cols), rows, cols, kind)
    dx, dg, db = got = run_backward(mg, x, dy, kind, g, m, v)
    check_backward((dx, None, None), x, dy, kind, g, m, v, None)
    _, g64, b64 = backward64(x, dy, g, m, v, None)
    terms = rows / groups + 1 + groups / 32 + 1 + 32 + 6 + 16
    xn = np.abs(x - m[:, None]) * v[:, None]
    assert_within(dg, g64, (terms + 4) * U32 * np.abs(dy * xn).sum(0), "dgamma")
    assert_within(db, b64, terms * U32 * np.abs(dy).sum(0), "dbeta")
    for a, b in zip(got, run_backward(mg, x, dy, kind, g, m, v)):
        np.testing.assert_array_equal(a, b)
