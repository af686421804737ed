"""Matrices that are column panels of one array: the bits of the same matrices one after
another, and nothing between or behind the panels written."""
import numpy as np
import pytest

from operator_cases import Rows, decode, encode
from test_gpu_muon import gradients, space

pytestmark = pytest.mark.gpu


class Panels:
    """[count][rows][cols] side by side in an array of rows, `gap` elements between them."""

    def __init__(self, mg, values, kind, gap):
        self.shape = count, rows, cols = values.shape
        wide = np.zeros((rows, count, cols + gap))
        wide[:, :, :cols] = values.transpose(1, 0, 2)
        self.gap, self.kind = gap, kind
        self.wide = decode(encode(wide, kind), kind)
        self.rows = Rows(mg, wide.reshape(rows, -1), kind)
        self.desc = mg.matrices(self.rows.ptr, count, rows, cols, kind, count * (cols + gap), cols + gap)

    def get(self):
        count, rows, cols = self.shape
        got = self.rows.get().reshape(rows, count, cols + self.gap)
        np.testing.assert_array_equal(got[:, :, cols:], self.wide[:, :, cols:])
        return got[:, :, :cols].transpose(1, 0, 2)


class Stacked:
    def __init__(self, mg, values, kind, gap):
        self.shape = values.shape
        self.rows = Rows(mg, values.reshape(-1, values.shape[2]), kind)
        self.desc = mg.matrices(self.rows.ptr, *values.shape, kind)

    def get(self):
        return self.rows.get().reshape(self.shape)


@pytest.mark.parametrize("count,rows,cols,gap", [(3, 128, 256, 0), (5, 40, 50, 3), (4, 300, 7, 1), (2, 200, 150, 0),
                                                 (3, 170, 333, 5), (1, 150, 140, 0)])
def test_panels_give_the_bits_of_a_stack(mg, count, rows, cols, gap):
    r = np.random.RandomState(count + cols)
    w, m, g = r.normal(0, rows**-0.5, (count, rows, cols)), gradients(r, count, rows, cols), gradients(r, count, rows, cols)
    out = []
    for kind in (Panels, Stacked):
        W, M, G = kind(mg, w, "bf16", gap), kind(mg, m, "fp32", gap), kind(mg, g, "fp16", gap)
        buf, n, untouched = space(mg, count, rows, cols)
        mg.muon_step(W.desc, M.desc, G.desc, lr=0.1, weight_decay=0.1, workspace=buf.ptr, workspace_bytes=n)
        mg.orthogonalize(G.desc, G.desc, workspace=buf.ptr, workspace_bytes=n)
        mg._capi.check(mg.lib().mg_synchronize())
        untouched()
        out.append((W.get(), M.get(), G.get()))
    for a, b in zip(*out):
        np.testing.assert_array_equal(a, b)
    assert np.abs(out[0][2]).max() > 0.01
