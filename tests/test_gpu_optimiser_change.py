"""Adam on the block matrices after a change from Muon in mid-training: their moments
start from 0 again, so their bias correction does too, while the vector parameters and
the head go on.

Each update is checked against the stored moments in float64: lr mHat / (sqrt(vHat) + eps).
Powers of beta are off by half a step of 1, which 1 - beta^k takes as u / (1 - beta^k)
(u = 2^-24), half of it under the root; ten roundings more, and the parameter's own."""
import numpy as np
import pytest

from operator_cases import U32
from test_gpu_ppo_muon import blocks, rest, twins

pytestmark = pytest.mark.gpu

B1, B2 = float(np.float32(0.9)), float(np.float32(0.999))


def check_adam(before, after, m, v, lr, step, what):
    before, after, m, v = (a.astype(np.float64) for a in (before, after, m, v))
    c1, c2 = 1 - B1**step, 1 - B2**step
    move = lr * (m / c1) / (np.sqrt(v / c2) + float(np.float32(1e-8)))
    tol = np.abs(move) * U32 * (10 + 1 / c1 + 0.5 / c2) + 2 * U32 * (np.abs(before) + np.abs(move))
    bad = np.abs(after - (before - move)) > tol
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off at step {step}; moves of {np.abs(after - before).max() / lr} lr"


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
@pytest.mark.parametrize("noalloc", [False, True])
def test_adam_starts_anew_on_the_block_matrices(mg, precision, noalloc):
    (gym, model), = twins(mg, precision=precision, count=1)
    lr = float(np.float32(model.cfg.lr))
    total = 0

    def train(block):
        model.train_block_noalloc(block) if noalloc else model.train_block(block)
        gym.sync()

    for k in range(12):
        train(k % 4)
        total += 1
    for _ in range(2):
        model.set_muon(lr=0.01)
        train(0)
        total += 1
        model.set_adam()
        for step in (1, 2, 3):
            p0 = model.params()
            train(step)
            total += 1
            p1, (m, v, count) = model.params(), model.adam_state()
            assert count == total
            check_adam(rest(model, p0), rest(model, p1), rest(model, m), rest(model, v), lr, total, "the rest")
            for (name, a), (_, b), (_, mm), (_, vv) in zip(*(blocks(model, x) for x in (p0, p1, m, v))):
                check_adam(a, b, mm, vv, lr, step, name)
                if step == 1:  # a fresh Adam moves an element by lr at most, as far as the bias correction is exact
                    assert np.abs(b - a).max() <= lr * 1.001 + 2 * U32 * np.abs(a).max(), name
