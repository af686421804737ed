"""Batches whose matrices are column panels of a wider array (ld over the whole, stride
from panel to panel) are batches like others: only what overlaps is refused."""
import pytest

from metalgym_amd._capi import CapiError

AT = 0x1000  # an address that is never read: every call here is refused


def message(call):
    with pytest.raises(CapiError) as e:
        call()
    assert e.value.rc == -1
    return str(e.value)


def calls(mg, count, rows, cols, ld, stride):
    a = mg.matrices(AT, count, rows, cols, "fp32", ld, stride)
    small = dict(workspace=1 << 20, workspace_bytes=16)
    return [lambda: mg.orthogonalize(a, a, **small), lambda: mg.muon_step(a, a, a, **small)]


# panels that touch, that lie apart, of one column, and the first shape of matrices one after another
FINE = [(3, 8, 16, 48, 16), (3, 8, 16, 60, 20), (3, 8, 16, 56, 20), (5, 4, 1, 5, 1), (2, 1, 16, 100, 16),
        (65535, 2, 7, 7 * 65535, 7), (2, 8, 16, 16, 128), (2, 8, 16, 24, 7 * 24 + 16), (1, 8, 16, 16, 3)]
OVERLAP = [(3, 8, 16, 47, 16), (3, 8, 16, 48, 15), (4, 8, 16, 48, 16), (2, 8, 16, 24, 7 * 24 + 15), (2, 8, 16, 24, 24),
           (65535, 2, 7, 7 * 65535 - 1, 7)]


@pytest.mark.parametrize("count,rows,cols,ld,stride", FINE)
def test_panels_are_taken(mg, count, rows, cols, ld, stride):
    for call in calls(mg, count, rows, cols, ld, stride):
        assert "workspace needs" in message(call)


@pytest.mark.parametrize("count,rows,cols,ld,stride", OVERLAP)
def test_overlapping_batches_are_refused(mg, count, rows, cols, ld, stride):
    for call in calls(mg, count, rows, cols, ld, stride):
        assert "overlap" in message(call)
