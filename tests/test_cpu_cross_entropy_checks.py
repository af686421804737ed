"""The cross entropy operators refuse bad arguments before any device work."""
import ctypes as C

import pytest

from metalgym_amd._capi import CapiError, CrossEntropyArgs, CrossEntropyBackwardArgs
from test_cpu_operator_checks import AT, refused


def forward(mg, **kw):
    a = dict(x=AT, w=AT, targets=AT, rows=4, classes=10, width=8, dtype="fp32", loss=AT, workspace=1 << 20,
             workspace_bytes=1 << 40)
    mg.cross_entropy(**dict(a, **kw))


def backward(mg, **kw):
    a = dict(x=AT, w=AT, targets=AT, rows=4, classes=10, width=8, dtype="fp32", lse=AT, dloss=AT, dx=AT, dw=AT,
             workspace=1 << 20, workspace_bytes=1 << 40)
    mg.cross_entropy_backward(**dict(a, **kw))


@pytest.mark.parametrize("call", [forward, backward])
@pytest.mark.parametrize("kw,needle", [
    (dict(rows=(1 << 20) + 1), "rows"),
    (dict(classes=0), "classes"),
    (dict(classes=(1 << 20) + 1), "classes"),
    (dict(width=0), "width"),
    (dict(width=65537), "width"),
    (dict(x=None), "x is NULL"),
    (dict(w=None), "w is NULL"),
    (dict(targets=None), "targets is NULL"),
    (dict(x=AT + 2), "x is not aligned"),
    (dict(w=AT + 1, dtype="bf16"), "w is not aligned"),
    (dict(targets=AT + 2), "targets is not aligned"),
    (dict(x_ld=7), "x_ld"),
    (dict(w_ld=(1 << 24) + 1), "w_ld"),
    (dict(lse=AT + 2), "lse is not aligned"),
    (dict(entropy=AT + 1, dentropy=AT), "entropy is not aligned"),
    (dict(workspace=None), "workspace needs"),
    (dict(workspace_bytes=100), "workspace needs"),
    (dict(workspace=(1 << 20) + 16), "256-byte"),
])
def test_refusals(mg, call, kw, needle):
    if call is forward:
        kw = {k: v for k, v in kw.items() if k != "dentropy"}
    refused(lambda: call(mg, **kw), needle)


@pytest.mark.parametrize("kw,needle", [
    (dict(lse=None), "lse is NULL"),
    (dict(dloss=None), "dloss is NULL"),
    (dict(dloss=AT + 2), "dloss is not aligned"),
    (dict(dentropy=AT), "entropy is NULL"),
    (dict(entropy=AT, dentropy=AT + 2), "dentropy is not aligned"),
    (dict(dx=AT + 2), "dx is not aligned"),
    (dict(dw=AT + 2), "dw is not aligned"),
    (dict(dx_ld=3), "dx_ld"),
    (dict(dw_ld=3), "dw_ld"),
])
def test_backward_refusals(mg, kw, needle):
    refused(lambda: backward(mg, **kw), needle)


def test_unknown_types_and_null_arguments(mg):
    L = mg.lib()
    for fn, args in ((L.mg_cross_entropy, CrossEntropyArgs), (L.mg_cross_entropy_backward, CrossEntropyBackwardArgs)):
        assert fn(None, None) == -1
        assert fn(None, C.byref(args(rows=1, classes=2, width=8, type=3))) == -1 and b"type" in L.mg_last_error()
    assert L.mg_cross_entropy_workspace(1, 2, 8, 0, None) == -1
    assert L.mg_cross_entropy_backward_workspace(1, 2, 8, 0, None) == -1


def test_nothing_to_do(mg):
    mg.cross_entropy(None, None, None, 0, 10, 8)
    space = dict(workspace=1 << 20, workspace_bytes=1 << 40)
    mg.cross_entropy_backward(None, None, None, 0, 10, 8, lse=None, dloss=None, **space)
    mg.cross_entropy_backward(AT, AT, AT, 4, 10, 8, lse=AT, dloss=AT, **space)


def test_workspaces(mg):
    """A few copies of the operands and two pieces' gradients, never the logits."""
    assert mg.cross_entropy_workspace(0, 10, 8) == 0
    for rows, classes, width in ((4096, 65536, 1024), (16384, 131072, 512), (1, 1 << 20, 64)):
        for dtype, size in (("bf16", 2), ("fp32", 4)):
            once = (rows + classes) * width * size
            assert mg.cross_entropy_workspace(rows, classes, width, dtype) <= 1.1 * once + (1 << 27)
            back = mg.cross_entropy_backward_workspace(rows, classes, width, dtype)
            assert back <= 4 * once + (1 << 30)
    with pytest.raises(CapiError):
        mg.cross_entropy_workspace(1, 0, 8)


def test_wide_heads_of_few_rows(mg):
    """Past 2^33 elements of W small tiles are too many for a launch: pairs of halves take their place."""
    classes, width = 1 << 18, 1 << 15
    assert mg.cross_entropy_workspace(8, classes, width, "fp32") < 1 << 30
    assert mg.cross_entropy_workspace(8, classes + 1, width, "fp32") > 4 * classes * width
