"""The selective scan of many sequences, where each quad of lanes has two channels, against 64 bits."""
import numpy as np
import pytest

from test_gpu_selective_scan import Case

pytestmark = pytest.mark.gpu

# steps, sequences, channels, states, groups; how many channels a quad has forwards and backwards: an odd last
# channel, groups of one workgroup and of two, 161 channels of which the gradient alone takes two
SHAPES = [(9, 1030, 67, 13, 1, "22"), (8, 257, 260, 16, 4, "22"), (5, 257, 400, 16, 2, "22"), (5, 512, 161, 16, 1, "12"),
          (66, 1024, 65, 13, 1, "22"), (2, 1024, 128, 16, 1, "22")]


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("steps,seqs,channels,states,groups,_", SHAPES[:4])
def test_pairs(mg, kind, steps, seqs, channels, states, groups, _):
    Case(steps, seqs, channels, states, kind, seed=steps, groups=groups).check(mg)


@pytest.mark.parametrize("kind,carry,gate", [("fp32", True, True), ("bf16", False, False)])
def test_pairs_over_chunks_of_any_length(mg, kind, carry, gate):
    """Past the first kept state, with resets, and sequences of no step, of a few and of all."""
    steps, seqs, channels, states, groups, _ = SHAPES[4]
    lengths = np.random.RandomState(2).randint(0, steps + 1, seqs)
    lengths[:6] = [0, 1, steps, steps - 1, 64, 65]
    Case(steps, seqs, channels, states, kind, seed=1, groups=groups, lengths=lengths, carry=carry, gate=gate,
         vectors=carry).check(mg)


@pytest.mark.parametrize("kind,order,pad,offset", [("bf16", "seqs", 0, 1), ("fp32", "apart", 3, 5), ("fp16", "seqs", 8, 0)])
def test_pairs_of_strided_rows(mg, kind, order, pad, offset):
    steps, seqs, channels, states, groups, _ = SHAPES[0]
    Case(steps, seqs, channels, states, kind, seed=3, groups=groups, order=order).check(mg, pad, offset, in_place=True)


def test_gradient_of_single_steps(mg):
    """One step, whose gradient alone is of pairs."""
    Case(1, 1030, 67, 16, "fp32", seed=4).check(mg)


@pytest.mark.parametrize("at", [0, 8])
def test_pairs_keep_what_is_not_finite_apart(mg, at):
    """NaN in one channel of a quad reaches neither the other, nor other sequences, nor the next episode."""
    outs = []
    steps, seqs, channels, states = 19, 1030, 67, 16
    for spoil in (False, True):
        c = Case(steps, seqs, channels, states, "bf16", seed=5, resets=0.0)
        c.reset = np.zeros((steps, seqs), np.uint8)
        c.reset[at + 3, 7] = 1
        if spoil:
            c.x[at, 7, 4] = np.nan
        f = c.forward(mg)
        b = c.backward(mg, f["checkpoints"])
        outs.append([f["y"].get(c.live), f["final"].get()] + [b[k].get(c.live) for k in ("dx", "db", "dc")])
    same = np.ones((steps, seqs, channels), bool)
    same[at:at + 3, 7, 4] = False
    np.testing.assert_array_equal(outs[0][0][same], outs[1][0][same])
    np.testing.assert_array_equal(outs[0][1], outs[1][1])
    np.testing.assert_array_equal(outs[0][2][same], outs[1][2][same])
    rows = np.ones((steps, seqs), bool)
    rows[at:at + 3, 7] = False
    for k in (3, 4):
        np.testing.assert_array_equal(outs[0][k][rows], outs[1][k][rows])
    assert np.isnan(outs[1][0][at:at + 3, 7, 4]).all()
