"""mg_ppo_set_muon: the block matrices of a model on Muon, everything else on Adam.

A twin on Adam, alike up to the update, gives the clipped gradient (its first moment
after one step from 0 is (1 - 0.9) g) and what must stay the same to the bit: the
LossStats, the vector parameters and the head."""
import numpy as np
import pytest

from operator_cases import U32
from parity import ENVS, assert_bit_exact, assert_close
from test_gpu_muon import check_muon

pytestmark = pytest.mark.gpu


def twins(mg, env="cartpole", n=1024, B=512, layers=2, scale=4, precision="fp32", count=2):
    out = []
    for _ in range(count):
        gym = mg.Gym(ENVS[env][1], n, 0)
        model = mg.PPOModel(gym, scale=scale, layers=layers, horizon=2, seed=0, minibatch=B, precision=precision)
        model.collect()
        out.append((gym, model))
    return out


def blocks(model, arena):
    pv = model.pv
    E, H = pv.embed, pv.hidden
    for l in range(pv.layers):
        yield f"up{l}", arena[pv.off_up[l]:][:E * H].reshape(1, E, H).astype(np.float64)
        yield f"down{l}", arena[pv.off_down[l]:][:E * H].reshape(1, H, E).astype(np.float64)


def rest(model, arena):
    pv = model.pv
    return np.concatenate([arena[:pv.float_group], arena[pv.off_head:]])


CASES = [("cartpole", 2, 4, "fp32"), ("cartpole", 1, 1, "fp32"), ("cartpole", 5, 2, "fp32"), ("cartpole", 8, 1, "fp32"),
         ("cartpole", 2, 8, "fp32"), ("cartpole_continuous", 2, 4, "fp32"), ("voxelnav16", 2, 4, "fp32"),
         ("cartpole", 2, 4, "bf16")]


@pytest.mark.parametrize("env,layers,scale,precision", CASES)
def test_one_minibatch(mg, env, layers, scale, precision):
    (_, adam), (_, muon) = twins(mg, env, layers=layers, scale=scale, precision=precision)
    kw = dict(lr=0.02, momentum=0.9, weight_decay=0.1)
    muon.set_muon(**kw)
    p0 = muon.params()
    assert_bit_exact(p0, adam.params(), "initial parameters")
    adam.train_block(1)
    muon.train_block(1)
    assert_bit_exact(np.array(muon.last_stats().as_tuple(), np.float32),
                     np.array(adam.last_stats().as_tuple(), np.float32), "LossStats")
    assert_bit_exact(rest(muon, muon.params()), rest(adam, adam.params()), "vector parameters and head")
    (m_a, v_a, _), (m_m, v_m, _) = adam.adam_state(), muon.adam_state()
    assert_bit_exact(rest(muon, m_m), rest(adam, m_a), "their first moments")
    assert_bit_exact(rest(muon, v_m), rest(adam, v_a), "their second moments")
    g = m_a.astype(np.float64) / float(np.float32(1) - np.float32(0.9))
    p1 = muon.params()
    for (name, w), (_, m), (_, u), (_, got) in zip(blocks(muon, p0), blocks(muon, m_m), blocks(muon, g), blocks(muon, p1)):
        print(name, flush=True)
        assert np.abs(u).max() > 0
        # g itself is known to two roundings (the product with 0.1 and Adam's own clip)
        assert np.all(np.abs(m - (1 - float(np.float32(0.9))) * u) <= 6 * U32 * np.abs(u))
        check_muon((got, m), w, np.zeros_like(w), u, "fp32", **kw)
    for _, v in blocks(muon, v_m):
        assert not v.any()


@pytest.mark.parametrize("env,layers,scale,precision", CASES)
def test_the_copies_follow_the_weights(mg, env, layers, scale, precision):
    """After three updates a model given the same parameters computes the same heads and,
    in its next minibatch, the same losses."""
    (_, muon), (_, fresh) = twins(mg, env, layers=layers, scale=scale, precision=precision)
    muon.set_muon(lr=0.05)
    for b in (0, 1, 2):
        muon.train_block(b)
    obs = muon.download_slots()["obs"][0]
    fresh.set_params(muon.params())
    assert_close(muon.forward(obs), fresh.forward(obs), 1e-5, "head")
    muon.train_block(3)
    fresh.train_block(3)
    got, want = (np.array(m.last_stats().as_tuple()) for m in (muon, fresh))
    # clip_frac counts rows, of which one may lie at the edge
    assert_close(got[[0, 1, 2, 3, 5]], want[[0, 1, 2, 3, 5]], 1e-4 if precision == "fp32" else 1e-3, "LossStats")
    assert abs(got[4] - want[4]) * 512 <= 1.001


def test_noalloc_and_reruns_have_the_same_bits(mg):
    (_, a), (gym, b), (_, c) = twins(mg, count=3)
    for m in (a, b, c):
        m.set_muon(lr=0.03)
    for block in (0, 3):
        a.train_block(block)
        b.train_block_noalloc(block)
        c.train_block(block)
    gym.sync()
    assert_bit_exact(b.params(), a.params(), "no-alloc parameters")
    assert_bit_exact(b.adam_state()[0], a.adam_state()[0], "no-alloc momentum")
    assert_bit_exact(c.params(), a.params(), "a rerun's parameters")


def test_a_change_of_optimiser_clears_the_blocks_moments(mg):
    (_, model), (_, adam) = twins(mg)
    model.train_block(0)
    model.set_muon(lr=0.02)
    for arena in model.adam_state()[:2]:
        assert all(not x.any() for _, x in blocks(model, arena)) and rest(model, arena).any()
    model.train_block(1)
    kept = model.adam_state()[0]
    model.set_muon(lr=0.01, momentum=0.8)  # another configuration of the same: nothing is cleared
    assert_bit_exact(model.adam_state()[0], kept, "momentum")
    model.set_adam()
    for arena in model.adam_state()[:2]:
        assert all(not x.any() for _, x in blocks(model, arena))
    model.train_block(2)
    assert np.isfinite(model.params()).all()
    # set and taken back before any update: Adam as if nothing had been
    adam.set_muon()
    adam.set_adam()
    (_, plain), = twins(mg, count=1)
    adam.train_block(0)
    plain.train_block(0)
    assert_bit_exact(adam.params(), plain.params(), "parameters")


def test_training_runs(mg):
    (_, model), = twins(mg, n=2048, B=1024, count=1)
    model.set_muon(lr=0.02, weight_decay=0.01)
    for _ in range(3):
        model.train(2)
        model.collect()
    assert np.isfinite(model.params()).all() and np.isfinite(model.train_stats()).all()
    for name, w in blocks(model, model.params()):
        assert np.linalg.svd(w[0], compute_uv=False).max() < 100, name


def test_refusals_leave_the_model_alone(mg):
    from metalgym_amd._capi import CapiError

    (_, a), (_, b) = twins(mg)
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(lr=2.0, weight_decay=1.0), dict(ns=mg.NewtonSchulz(40, 1, 0, 0, 1e-7))):
        with pytest.raises(CapiError):
            a.set_muon(**kw)
    a.train_block(0)
    b.train_block(0)
    assert_bit_exact(a.params(), b.params(), "parameters")
