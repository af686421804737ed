"""The training operators as a program uses them: one after the other in a training
step of a residual block, on streams of their own, and captured into HIP graphs that
are replayed with eager work between the replays."""
import ctypes as C

import numpy as np
import pytest

from operator_cases import U32, assert_within, decode, encode
from test_gpu_layernorm import check_backward, check_forward, forward64
from test_gpu_muon import check_muon

pytestmark = pytest.mark.gpu


class Hip:
    """The few HIP calls that a capture takes, from the runtime the library is linked with."""

    def __init__(self, mg):
        self.L = mg.lib()

    def __call__(self, name, *args):
        fn = getattr(self.L, name)
        fn.restype = C.c_int
        rc = fn(*args)
        assert rc == 0, f"{name}: {rc}"

    def stream(self):
        s = C.c_void_p()
        self("hipStreamCreate", C.byref(s))
        return s

    def capture(self, stream, work):
        graph, exe = C.c_void_p(), C.c_void_p()
        self("hipStreamBeginCapture", stream, C.c_int(2))  # relaxed
        work()
        self("hipStreamEndCapture", stream, C.byref(graph))
        self("hipGraphInstantiate", C.byref(exe), graph, None, None, C.c_size_t(0))
        self("hipGraphDestroy", graph)
        return exe

    def launch(self, exe, stream):
        self("hipGraphLaunch", exe, stream)

    def sync(self, stream):
        self("hipStreamSynchronize", stream)


class Step:
    """The device side of one training step: sum = x + branch, y = norm(sum); then, from dy, the
    gradients of the norm, and from `grad` the Muon step of a batch of matrices."""

    def __init__(self, mg, seed, rows, cols, mats, kind="bf16"):
        self.mg, self.rows, self.cols, self.mats, self.kind = mg, rows, cols, mats, kind
        r = np.random.RandomState(seed)
        q = lambda a, t: decode(encode(a, t), t)  # noqa: E731
        self.x, self.branch, self.dy, self.dsum = (q(r.normal(0, 1, (rows, cols)), kind) for _ in range(4))
        self.gamma, self.beta = q(r.normal(1, 0.1, cols), "fp32"), q(r.normal(0, 0.1, cols), "fp32")
        self.w, self.m, self.g = (q(r.normal(0, 0.05, mats), "fp32") for _ in range(3))
        up = lambda a, t: mg.DeviceBuffer.from_array(encode(a, t))  # noqa: E731
        self.d = {k: up(getattr(self, k), kind) for k in ("x", "branch", "dy", "dsum")}
        self.d.update({k: up(getattr(self, k), "fp32") for k in ("gamma", "beta", "w", "m", "g")})
        size = rows * cols * (4 if kind == "fp32" else 2)
        for k in ("sum", "y", "dx"):
            self.d[k] = mg.DeviceBuffer(size)
        for k, n in (("mean", rows), ("rstd", rows), ("dgamma", cols), ("dbeta", cols)):
            self.d[k] = mg.DeviceBuffer(4 * n)
        self.ws_norm = mg.DeviceBuffer(max(256, mg.layernorm_backward_workspace(rows, cols)))
        self.ws_muon = mg.DeviceBuffer(mg.orthogonalize_workspace(*mats))

    def forward(self, stream=None):
        p = {k: b.ptr for k, b in self.d.items()}
        self.mg.layernorm(p["x"], p["y"], self.rows, self.cols, self.kind, gamma=p["gamma"], beta=p["beta"],
                          residual=p["branch"], sum=p["sum"], mean=p["mean"], rstd=p["rstd"], stream=stream)

    def backward(self, stream=None):
        p = {k: b.ptr for k, b in self.d.items()}
        self.mg.layernorm_backward(p["sum"], p["dy"], p["mean"], p["rstd"], p["dx"], self.rows, self.cols, self.kind,
                                   gamma=p["gamma"], dsum=p["dsum"], dgamma=p["dgamma"], dbeta=p["dbeta"],
                                   workspace=self.ws_norm.ptr, workspace_bytes=self.ws_norm.nbytes, stream=stream)

    def update(self, stream=None):
        a = [self.mg.matrices(self.d[k].ptr, *self.mats) for k in ("w", "m", "g")]
        self.mg.muon_step(*a, workspace=self.ws_muon.ptr, workspace_bytes=self.ws_muon.nbytes, stream=stream)

    def run(self, stream=None):
        self.forward(stream)
        self.backward(stream)
        self.update(stream)

    def get(self, name):
        kind = self.kind if name in ("sum", "y", "dx", "dy") else "fp32"
        shape = {"w": self.mats, "m": self.mats, "g": self.mats, "mean": (self.rows,), "rstd": (self.rows,),
                 "dgamma": (self.cols,), "dbeta": (self.cols,)}.get(name, (self.rows, self.cols))
        from operator_cases import storage
        return decode(self.d[name].download(storage(kind), shape), kind)

    OUT = ("sum", "y", "mean", "rstd", "dx", "dgamma", "dbeta", "w", "m")

    def outputs(self):
        return {k: self.get(k) for k in self.OUT}

    def restore(self):
        self.d["w"].upload(encode(self.w, "fp32"))
        self.d["m"].upload(encode(self.m, "fp32"))
        for k in ("sum", "y", "dx", "mean", "rstd", "dgamma", "dbeta"):
            self.d[k].upload(np.full(self.d[k].nbytes, 0x7F, np.uint8))


def same(a, b, what):
    for k in a:
        np.testing.assert_array_equal(a[k], b[k], err_msg=f"{what}: {k}")


def sync(mg):
    mg._capi.check(mg.lib().mg_synchronize())


CASES = [(37, 128, (2, 128, 512)), (1000, 1001, (1, 200, 300)), (300, 3000, (3, 64, 40)), (5, 20000, (1, 512, 640))]


@pytest.mark.parametrize("rows,cols,mats", CASES)
def test_a_block_of_matrices_and_its_norm_train(mg, rows, cols, mats):
    """The whole step against float64, each operator on what the one before it stored."""
    s = Step(mg, 1, rows, cols, mats)
    s.run()
    sync(mg)
    o = s.outputs()
    np.testing.assert_array_equal(o["sum"], decode(encode((s.x + s.branch).astype(np.float32), "bf16"), "bf16"))
    check_forward((o["y"], o["mean"], o["rstd"]), o["sum"], s.gamma, s.beta, 1e-5, "bf16")
    check_backward((o["dx"], o["dgamma"], o["dbeta"]), o["sum"], s.dy, "bf16", s.gamma, o["mean"], o["rstd"], s.dsum)
    check_muon((o["w"], o["m"]), s.w, s.m, s.g, "fp32")


def test_gradients_through_a_linear_layer(mg):
    """z = norm(x + branch) W with the loss sum(z R): the operators' gradients of x and of
    the vectors against differences of the loss, and W's gradient into a Muon step."""
    s = Step(mg, 2, 24, 96, (1, 96, 160), "fp32")
    R = np.random.RandomState(3).normal(0, 1, (24, 160))
    s.forward()
    sync(mg)
    y = s.get("y")
    s.dy = decode(encode(R @ s.w[0].T, "fp32"), "fp32")
    s.d["dy"].upload(encode(s.dy, "fp32"))
    s.dsum[:] = 0
    s.d["dsum"].upload(encode(s.dsum, "fp32"))
    s.g = decode(encode(y.T @ R, "fp32"), "fp32")[None]
    s.d["g"].upload(encode(s.g, "fp32"))
    s.backward()
    s.update()
    sync(mg)
    o = s.outputs()
    loss = lambda x, g, b: ((forward64(x + s.branch, g, b, 1e-5)[0] @ s.w[0]) * R).sum()  # noqa: E731
    r, h = np.random.RandomState(4), 1e-5
    for grad, along, f in ((o["dx"], r.normal(0, 1, s.x.shape), lambda t: loss(s.x + t, s.gamma, s.beta)),
                           (o["dgamma"], r.normal(0, 1, 96), lambda t: loss(s.x, s.gamma + t, s.beta)),
                           (o["dbeta"], r.normal(0, 1, 96), lambda t: loss(s.x, s.gamma, s.beta + t))):
        num = (f(h * along) - f(-h * along)) / (2 * h)
        # h^2 of the differences, and fp32's sums (60 u) of terms that cancel
        assert abs((grad * along).sum() - num) <= 1e-5 * np.abs(grad * along).sum()
    check_muon((o["w"], o["m"]), s.w, s.m, s.g, "fp32")


@pytest.mark.parametrize("rows,cols,mats", CASES)
def test_captured_steps_replay(mg, rows, cols, mats):
    """Replays of one graph, with the same buffers' eager step and other eager work between
    them: each replay moves the weights as an eager step does."""
    hip = Hip(mg)
    stream = hip.stream()
    ref, s, other = (Step(mg, 5, rows, cols, mats) for _ in range(3))
    exe = hip.capture(stream, lambda: s.run(stream))
    for turn in range(4):
        print("replay", turn, flush=True)
        ref.run()
        sync(mg)
        if turn == 2:  # an eager step of the captured buffers counts like a replay
            s.run(stream)
        else:
            hip.launch(exe, stream)
        hip.sync(stream)
        same(s.outputs(), ref.outputs(), f"turn {turn}")
        other.run()
        sync(mg)
    s.restore()
    ref.restore()
    hip.launch(exe, stream)
    hip.launch(exe, stream)
    hip.sync(stream)
    ref.run()
    ref.run()
    sync(mg)
    same(s.outputs(), ref.outputs(), "two replays in a row")
    hip("hipGraphExecDestroy", exe)
    hip("hipStreamDestroy", stream)


def test_two_streams_at_once(mg):
    """Steps of two programs, each with its own buffers and workspaces, queued on two streams."""
    hip = Hip(mg)
    streams = [hip.stream(), hip.stream()]
    shapes = [(1000, 1001, (1, 200, 300)), (700, 128, (4, 128, 512))]
    steps = [Step(mg, 6 + k, *shapes[k]) for k in range(2)]
    refs = [Step(mg, 6 + k, *shapes[k]) for k in range(2)]
    for _ in range(5):
        for s, st in zip(steps, streams):
            s.run(st)
    for st in streams:
        hip.sync(st)
    for ref in refs:
        for _ in range(5):
            ref.run()
        sync(mg)
    for k in range(2):
        same(steps[k].outputs(), refs[k].outputs(), f"stream {k}")
    for st in streams:
        hip("hipStreamDestroy", st)


def test_the_operators_on_a_models_stream(mg):
    """Between a model's own calls on the gym's stream: the norm of its last block's input
    rows is what the fused update captured."""
    gym = mg.Gym("rollout_cartpole", 256, 0)
    model = mg.PPOModel(gym, horizon=2, minibatch=256)
    model.collect()
    p0 = model.params()
    model.train_block(0)
    ln = model.train_capture(0)[0]  # the first block's LN output
    obs = model.download_slots()["obs"][0]
    pv = model.pv
    w = p0[pv.off_in_w:][:pv.obs_dim * 128].reshape(pv.obs_dim, 128).astype(np.float64)
    h = decode(encode(obs.astype(np.float64) @ w + p0[pv.off_in_b:][:128], "fp32"), "fp32")
    gamma, beta = p0[pv.off_ln_gamma[0]:][:128], p0[pv.off_ln_beta[0]:][:128]
    x, y = mg.DeviceBuffer.from_array(encode(h, "fp32")), mg.DeviceBuffer(h.size * 4)
    vec = [mg.DeviceBuffer.from_array(np.ascontiguousarray(v, np.float32)) for v in (gamma, beta)]
    mg.layernorm(x.ptr, y.ptr, 256, 128, "fp32", gamma=vec[0].ptr, beta=vec[1].ptr, stream=gym.buf.stream)
    gym.sync()
    got = y.download(np.float32, (256, 128)).astype(np.float64)
    # both sides round the embedding (a chain of obs_dim + 1 products) and the norm's sums (38 u)
    std = h.std(1, keepdims=True)
    tol = 2 * 60 * U32 * (np.abs(got) + np.abs(gamma) * (1 + np.abs(h).max(1, keepdims=True) / std))
    assert_within(got, ln.astype(np.float64), tol, "LN output")


def test_captured_model_updates_replay(mg):
    """mg_ppo_train_block_noalloc with Muon in a graph: replays take the captured minibatch
    with the captured Adam step count, as eager calls of another model from the same state."""
    hip = Hip(mg)

    def model():
        gym = mg.Gym("rollout_cartpole", 256, 0)
        m = mg.PPOModel(gym, horizon=2, minibatch=256)
        m.set_muon(lr=0.02)
        m.collect()
        return gym, m

    (gym, m), (ref_gym, ref) = model(), model()
    stats = mg.DeviceBuffer(24)
    m.train_block_noalloc(0, stats.ptr)  # eager once: modules are loaded and pages placed
    ref.train_block_noalloc(0, stats.ptr)
    gym.sync()
    exe = hip.capture(C.c_void_p(gym.buf.stream), lambda: m.train_block_noalloc(1, stats.ptr))
    hip.launch(exe, C.c_void_p(gym.buf.stream))
    gym.sync()
    ref.train_block_noalloc(1, stats.ptr)
    ref_gym.sync()
    np.testing.assert_array_equal(m.params(), ref.params())
    np.testing.assert_array_equal(m.adam_state()[0], ref.adam_state()[0])
    for turn in range(3):  # the block matrices' own step does not depend on a step count
        print("replay", turn, flush=True)
        before = m.params()
        hip.launch(exe, C.c_void_p(gym.buf.stream))
        gym.sync()
        other = mg.DeviceBuffer.from_array(np.ones(1000, np.float32))
        other.zero()
        after = m.params()
        assert np.isfinite(after).all() and (after != before).mean() > 0.5
    hip("hipGraphExecDestroy", exe)
