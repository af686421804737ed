"""Classes that are masked by the type's lowest value: a column of ones in x, and in w that value for the classes
that cannot be taken. They are as if they were not there."""
import numpy as np
import pytest

from operator_cases import assert_within
from rollout_cases import rounded
from test_gpu_cross_entropy import Case

pytestmark = pytest.mark.gpu

LOWEST = {"fp32": -np.finfo(np.float32).max, "bf16": -(2.0 - 2.0**-7) * 2.0**127, "fp16": -65504.0}


@pytest.mark.parametrize("kind,rows,classes,width", [
    ("fp32", 70, 300, 48), ("bf16", 70, 300, 48), ("fp16", 70, 300, 48), ("bf16", 300, 20011, 200), ("fp16", 300, 20011, 200),
    ("bf16", 300, 20011, 520), ("bf16", 1025, 9001, 264)])
def test_masked_classes(mg, kind, rows, classes, width):
    c = Case(rows, classes, width, kind, seed=1)
    gone = np.zeros(classes, bool)
    gone[32:classes // 3] = gone[classes // 2:classes // 2 + 90] = gone[-70:] = True
    kept = np.flatnonzero(~gone)
    c.targets[c.live] = kept[c.targets[c.live] % kept.size]
    c.x[:, 0] = 1
    c.w[gone, 0] = rounded(LOWEST[kind], kind)
    without = Case(rows, kept.size, width, kind, seed=1)
    place = np.full(classes, -1)
    place[kept] = np.arange(kept.size)
    without.x, without.w, without.dloss, without.dentropy = c.x, c.w[kept], c.dloss, c.dentropy
    without.targets = np.where(c.live, place[np.where(c.live, c.targets, 0)], -1).astype(np.int32)
    want = without.reference()
    c.upload(mg)
    got = c.forward(mg)
    for k in want:
        assert_within(got[k], want[k], 2 * without.err[k], k)
    lse, entropy = rounded(want["lse"], "fp32"), rounded(want["entropy"], "fp32")
    got = c.backward(mg, lse, entropy)
    grads = without.gradients(lse, entropy)
    assert_within(got["dx"], *grads["dx"], "dx")
    assert_within(got["dw"][kept], *grads["dw"], "dw")
    assert (got["dw"][gone] == 0).all()
