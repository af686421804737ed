"""The cross entropy's gradients over several pieces of the classes, and of fp32 rows of different sizes."""
import numpy as np
import pytest

from rollout_cases import rounded
from test_gpu_cross_entropy import Case
from test_gpu_cross_entropy_parts import check_some

pytestmark = pytest.mark.gpu

# two pieces of the classes, three, and 17, the last of which has one range where the others have two
PIECES = [(9000, 24001, 24), (8200, 40500, 24), (16384, 139310, 16)]


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,classes,width", PIECES)
def test_pieces_of_classes(mg, kind, rows, classes, width):
    # the gradient of all logits at once would not fit: there are several pieces
    planes = 2 if kind == "fp32" else 1
    assert mg.cross_entropy_backward_workspace(rows, classes, width, kind) < 2 * planes * rows * classes
    c = Case(rows, classes, width, kind, seed=3)
    r = np.random.RandomState(4)
    some = np.unique(np.r_[0, rows - 1, r.randint(0, rows, 20)])
    few = np.unique(np.r_[0, classes // 3, classes // 2, classes - 1, c.targets[c.live][:10], r.randint(0, classes, 40)])
    check_some(c, mg, some, few)


@pytest.mark.parametrize("rows,classes,width", [(64, 200, 40), (600, 9000, 130)])
def test_gradients_of_rows_of_different_sizes(mg, rows, classes, width):
    """fp32 rows of x, and of dloss the other way round, over eight powers of ten: pairs at a power of two for
    each array keep 2^-38 of its largest."""
    c = Case(rows, classes, width, "fp32", seed=5)
    size = 10.0 ** np.linspace(-8, 0.5, rows)
    c.x = rounded(c.x * size[:, None], "fp32")
    c.dloss, c.dentropy = rounded(c.dloss * size[::-1], "fp32"), rounded(c.dentropy * size[::-1], "fp32")
    c.check(mg)
