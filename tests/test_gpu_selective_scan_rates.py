"""States that keep nothing (a of -infinity, or so low that a log2(e) passes fp32's range) in scans whose steps end
before a round of eight does, in splits that a sequence does not reach, and a step at a time."""
import numpy as np
import pytest

from test_gpu_selective_scan import Case

pytestmark = pytest.mark.gpu


class Forgetful(Case):
    def __init__(self, *args, rate, **kw):
        super().__init__(*args, **kw)
        self.gone = np.zeros(self.a.shape, bool)
        self.gone[1::2, 0] = self.gone[::3, -1] = True
        self.a[self.gone] = rate

    def reference(self):
        # in 64 bits a rate whose every decay is 0 too, but with products that are numbers
        given, self.a = self.a, np.where(self.gone, -1e30, self.a)
        try:
            return super().reference()
        finally:
            self.a = given


@pytest.mark.parametrize("rate", [-np.inf, -3e38])
@pytest.mark.parametrize("steps,channels,states,lengths", [
    (13, 20, 16, [13, 5, 0]), (13, 20, 5, [13, 5, 0]), (13, 6, 100, [13, 5, 0]), (9, 20, 40, None), (1, 20, 16, [1, 0, 1]),
    (1, 20, 3, [1, 0, 1]), (400, 12, 16, [400, 70, 0]), (400, 12, 4, [400, 70, 1]), (400, 12, 50, None)])
def test_states_that_keep_nothing(mg, rate, steps, channels, states, lengths):
    Forgetful(steps, 3, channels, states, "fp32", seed=states, lengths=lengths, slow=steps > 100, rate=rate).check(mg)


def test_pairs_of_channels(mg):
    Forgetful(9, 1030, 67, 13, "bf16", seed=1, rate=-np.inf).check(mg)


def test_a_rate_that_is_no_number_shows(mg):
    c = Case(9, 2, 20, 16, "fp32", seed=2, resets=0.0)
    c.a[3, 2] = np.nan
    y = c.forward(mg)["y"].get(c.live)
    assert np.isnan(y[:, :, 3]).all() and np.isfinite(np.delete(y, 3, 2)).all()
