import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs the HIP kernels through the C ABI)")


@pytest.fixture(scope="session")
def orc():
    import oracle

    oracle.lib()
    return oracle


@pytest.fixture(scope="session")
def mg():
    import metalgym_amd

    metalgym_amd.lib()
    fill_new_memory(metalgym_amd)
    return metalgym_amd


def fill_new_memory(mg):
    """Device memory that a test asks for holds 0xFF bytes, NaN in every float type: fresh memory is often zeros,
    which hide what is read before it is written (a workspace needs no clearing)."""
    make = mg.DeviceBuffer.__init__

    def filled(self, nbytes):
        make(self, nbytes)
        mg._capi.check(mg.lib().mg_memset(self.ptr, 0xFF, self.nbytes))
        mg._capi.check(mg.lib().mg_synchronize())

    mg.DeviceBuffer.__init__ = filled
