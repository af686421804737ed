"""The operators of a policy with memory as a program uses them: a block of causal convolution,
scan, layer norm and cross entropy over a rollout, forward and backward; a step at a time against
the whole; on streams and in graphs that are replayed with eager work between the replays."""
import ctypes as C

import numpy as np
import pytest

from operator_cases import decode, encode, storage
from test_gpu_operator_runs import Hip, same, sync

pytestmark = pytest.mark.gpu

T, N, D, S, V, TAPS = 12, 6, 48, 16, 1000, 4


def sigmoid(v):
    return 1 / (1 + np.exp(-v))


class Block:
    """x -> conv (SiLU) -> scan with rates, B and C from the conv's output by matrices, gated by x ->
    layer norm -> cross entropy over V actions. Rollout rows [T][N], resets where episodes begin."""

    def __init__(self, mg, seed, kind="fp32", steps=T, classes=V):
        self.mg, self.kind, self.steps, self.classes = mg, kind, steps, classes
        r = np.random.RandomState(seed)
        q = lambda a, t=kind: decode(encode(a, t), t)  # noqa: E731
        f = lambda a: q(a, "fp32")  # noqa: E731
        rows = steps * N
        self.v = dict(
            x=q(r.normal(0, 1, (rows, D))), taps=f(r.normal(0, 0.5, (D, TAPS))), tap_bias=f(r.normal(0, 0.1, D)),
            a=f(-np.exp(r.normal(0, 0.5, (D, S)))), d=f(r.normal(1, 0.1, D)), dt_bias=f(r.normal(-2, 1, D)),
            window=q(r.normal(0, 1, (N, TAPS - 1, D))), state=f(r.normal(0, 1, (N, D, S))),
            dt=q(r.normal(0, 1, (rows, D))), b=q(r.normal(0, 1, (rows, S))), c=q(r.normal(0, 1, (rows, S))),
            gamma=f(r.normal(1, 0.1, D)), beta=f(r.normal(0, 0.1, D)),
            w=q(r.normal(0, 1.5 * D**-0.5, (classes, D))))
        self.reset = (r.rand(rows) < 0.15).astype(np.uint8)
        self.targets = r.randint(0, classes, rows).astype(np.int32)
        self.targets[::7] = -1
        self.v["dloss"], self.v["dentropy"] = f(r.normal(0, 1, rows) / rows), f(np.full(rows, -0.01 / rows))
        rowwise = ("x", "window", "dt", "b", "c", "w")
        self.d = {k: mg.DeviceBuffer.from_array(encode(v, kind if k in rowwise else "fp32")) for k, v in self.v.items()}
        self.d["reset"] = mg.DeviceBuffer.from_array(self.reset)
        self.d["targets"] = mg.DeviceBuffer.from_array(self.targets)
        size = 4 if kind == "fp32" else 2
        self.shape = {}

        def out(name, shape, t=kind):
            self.shape[name] = (shape, t)
            self.d[name] = mg.DeviceBuffer(int(np.prod(shape)) * (4 if t == "fp32" else size))

        for k in ("u", "s", "y", "dy", "ds", "du", "dx", "ddt", "dz"):
            out(k, (rows, D))
        for k in ("db", "dc"):
            out(k, (rows, S))
        for k in ("mean", "rstd", "loss", "lse", "entropy"):
            out(k, (rows,), "fp32")
        out("final_window", (N, TAPS - 1, D))
        out("final_state", (N, D, S), "fp32")
        out("kept", ((steps + 63) // 64, N, D, S), "fp32")
        out("dw", (classes, D))
        for k, s in (("dgamma", (D,)), ("dbeta", (D,)), ("da", (D, S)), ("dd", (D,)), ("ddt_bias", (D,)),
                     ("dtaps", (D, TAPS)), ("dtap_bias", (D,)), ("dstate", (N, D, S))):
            out(k, s, "fp32")
        out("dwindow", (N, TAPS - 1, D))
        space = lambda n: mg.DeviceBuffer(n + 256)  # noqa: E731
        self.ws = dict(scan=space(mg.selective_scan_workspace(steps, N, D, S)),
                       scan_back=space(mg.selective_scan_backward_workspace(steps, N, D, S)),
                       conv_back=space(mg.causal_conv_backward_workspace(steps, N, D, TAPS)),
                       norm=space(mg.layernorm_backward_workspace(rows, D)),
                       loss=space(mg.cross_entropy_workspace(rows, classes, D, kind)),
                       loss_back=space(mg.cross_entropy_backward_workspace(rows, classes, D, kind)))

    def space(self, k):
        return dict(workspace=self.ws[k].ptr, workspace_bytes=self.ws[k].nbytes)

    def forward(self, stream=None):
        mg, p, kind, rows = self.mg, {k: b.ptr for k, b in self.d.items()}, self.kind, self.steps * N
        on = dict(stream=stream)
        mg.causal_conv(p["x"], p["taps"], p["u"], self.steps, N, D, TAPS, kind, bias=p["tap_bias"], silu=True,
                       reset=p["reset"], initial=p["window"], final=p["final_window"], **on)
        mg.selective_scan(p["u"], p["dt"], p["s"], self.steps, N, D, S, kind, a=p["a"], b=p["b"], c=p["c"], d=p["d"],
                          dt_bias=p["dt_bias"], z=p["x"], reset=p["reset"], initial=p["state"],
                          final=p["final_state"], checkpoints=p["kept"], **self.space("scan"), **on)
        mg.layernorm(p["s"], p["y"], rows, D, kind, gamma=p["gamma"], beta=p["beta"], mean=p["mean"], rstd=p["rstd"],
                     **on)
        mg.cross_entropy(p["y"], p["w"], p["targets"], rows, self.classes, D, kind, loss=p["loss"], lse=p["lse"],
                         entropy=p["entropy"], **self.space("loss"), **on)

    def backward(self, stream=None):
        mg, p, kind, rows = self.mg, {k: b.ptr for k, b in self.d.items()}, self.kind, self.steps * N
        on = dict(stream=stream)
        mg.cross_entropy_backward(p["y"], p["w"], p["targets"], rows, self.classes, D, kind, lse=p["lse"],
                                  dloss=p["dloss"], entropy=p["entropy"], dentropy=p["dentropy"], dx=p["dy"],
                                  dw=p["dw"], **self.space("loss_back"), **on)
        mg.layernorm_backward(p["s"], p["dy"], p["mean"], p["rstd"], p["ds"], rows, D, kind, gamma=p["gamma"],
                              dgamma=p["dgamma"], dbeta=p["dbeta"], **self.space("norm"), **on)
        mg.selective_scan_backward(p["u"], p["dt"], p["ds"], self.steps, N, D, S, kind, a=p["a"], b=p["b"], c=p["c"],
                                   d=p["d"], dt_bias=p["dt_bias"], z=p["x"], reset=p["reset"], initial=p["state"],
                                   checkpoints=p["kept"], dx=p["du"], ddt=p["ddt"], db=p["db"], dc=p["dc"],
                                   dz=p["dz"], da=p["da"], dd=p["dd"], ddt_bias=p["ddt_bias"],
                                   dinitial=p["dstate"], **self.space("scan_back"), **on)
        mg.causal_conv_backward(p["x"], p["taps"], p["du"], p["dx"], self.steps, N, D, TAPS, kind,
                                bias=p["tap_bias"], silu=True, reset=p["reset"], initial=p["window"],
                                dweight=p["dtaps"], dbias=p["dtap_bias"], dinitial=p["dwindow"],
                                **self.space("conv_back"), **on)

    def run(self, stream=None):
        self.forward(stream)
        self.backward(stream)

    def get(self, name):
        shape, t = self.shape[name]
        return decode(self.d[name].download(storage(t), shape), t)

    def outputs(self):
        return {k: self.get(k) for k in self.shape}

    def spoil(self):
        for k in self.shape:
            self.d[k].upload(np.full(self.d[k].nbytes, 0x7F, np.uint8))

    def loss64(self, v):
        """sum(loss dloss) + sum(entropy dentropy), all of it in 64 bits."""
        steps = self.steps
        x = v["x"].reshape(steps, N, D)
        reset = self.reset.reshape(steps, N)
        window, h, out = v["window"].copy(), v["state"].copy(), []
        for t in range(steps):
            keep = (reset[t] == 0)[:, None]
            window, h = window * keep[..., None], h * keep[..., None]
            seen = np.concatenate([window, x[t][:, None]], 1)
            pre = (seen * v["taps"].T).sum(1) + v["tap_bias"]
            u, window = pre * sigmoid(pre), seen[:, 1:]
            row = lambda k: v[k].reshape(steps, N, -1)[t]  # noqa: E731
            delta = np.logaddexp(0, row("dt") + v["dt_bias"])
            h = np.exp(delta[..., None] * v["a"]) * h + (delta * u)[..., None] * row("b")[:, None]
            s = (h * row("c")[:, None]).sum(-1) + v["d"] * u
            out.append(s * x[t] * sigmoid(x[t]))
        s = np.concatenate(out)
        c = s - s.mean(1, keepdims=True)
        y = c / np.sqrt((c * c).mean(1, keepdims=True) + 1e-5) * v["gamma"] + v["beta"]
        logits = y @ v["w"].T
        top = logits.max(1, keepdims=True)
        e = np.exp(logits - top)
        lse = top[:, 0] + np.log(e.sum(1))
        live = self.targets >= 0
        entropy = lse - (e * logits).sum(1) / e.sum(1)
        loss = np.where(live, lse - logits[np.arange(len(s)), np.where(live, self.targets, 0)], 0)
        return (loss * v["dloss"]).sum() + np.where(live, entropy * v["dentropy"], 0).sum()


@pytest.mark.parametrize("classes", [1000, 20000])
def test_gradients_of_the_whole_block(mg, classes):
    """Every gradient along a direction against differences of the loss in 64 bits."""
    b = Block(mg, 1, classes=classes)
    b.run()
    sync(mg)
    o = b.outputs()
    # x reaches the loss through the convolution and as the gate
    grads = dict(x=o["dx"] + o["dz"], taps=o["dtaps"], tap_bias=o["dtap_bias"], a=o["da"], d=o["dd"],
                 dt_bias=o["ddt_bias"], window=o["dwindow"], state=o["dstate"], dt=o["ddt"], b=o["db"], c=o["dc"],
                 gamma=o["dgamma"], beta=o["dbeta"], w=o["dw"])
    r, h = np.random.RandomState(2), 1e-5
    for k, g in grads.items():
        along = r.normal(0, 1, g.shape) * (np.abs(b.v[k]) if k == "a" else 1)
        ends = []
        for sign in (1, -1):
            v = dict(b.v)
            v[k] = v[k] + sign * h * along
            ends.append(b.loss64(v))
        # fp32 through four operators, each with sums of some tens of terms that cancel
        assert abs((g * along).sum() - (ends[0] - ends[1]) / (2 * h)) <= 3e-5 * np.abs(g * along).sum() + 1e-9, k


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_acting_a_step_at_a_time(mg, kind):
    """Window and state carried on in place: the same rows as the whole rollout's."""
    b = Block(mg, 3, kind)
    b.forward()
    sync(mg)
    want = b.outputs()
    size = 4 if kind == "fp32" else 2
    p = {k: x.ptr for k, x in b.d.items()}
    for k in ("u", "s", "y", "loss"):
        b.d[k].upload(np.full(b.d[k].nbytes, 0x7F, np.uint8))
    row = N * D * size
    for t in range(T):
        reset = p["reset"] + t * N
        mg.causal_conv(p["x"] + t * row, p["taps"], p["u"] + t * row, 1, N, D, TAPS, kind, bias=p["tap_bias"], silu=True,
                       reset=reset, initial=p["window"], final=p["window"])
        mg.selective_scan(p["u"] + t * row, p["dt"] + t * row, p["s"] + t * row, 1, N, D, S, kind, a=p["a"],
                          b=p["b"] + t * N * S * size, c=p["c"] + t * N * S * size, d=p["d"], dt_bias=p["dt_bias"],
                          z=p["x"] + t * row, reset=reset, initial=p["state"], final=p["state"])
        mg.layernorm(p["s"] + t * row, p["y"] + t * row, N, D, kind, gamma=p["gamma"], beta=p["beta"])
        mg.cross_entropy(p["y"] + t * row, p["w"], p["targets"] + 4 * t * N, N, V, D, kind, loss=p["loss"] + 4 * t * N,
                         **b.space("loss"))
    sync(mg)
    np.testing.assert_array_equal(b.get("u"), want["u"])  # the same products in the same order
    # sums over states in the same order; decays that are exponentials of the same arguments
    np.testing.assert_array_equal(b.get("s"), want["s"])
    np.testing.assert_allclose(b.get("loss"), want["loss"], rtol=1e-5, atol=1e-5 if kind == "fp32" else 2e-2)
    np.testing.assert_array_equal(decode(b.d["window"].download(storage(kind), (N, TAPS - 1, D)), kind),
                                  want["final_window"])
    np.testing.assert_array_equal(b.d["state"].download(np.float32, (N, D, S)), want["final_state"])


@pytest.mark.parametrize("kind,steps,classes", [("fp32", 12, 1000), ("bf16", 12, 30000), ("fp32", 12, 30000),
                                                ("fp16", 400, 300), ("fp32", 400, 3000)])
def test_captured_blocks_replay(mg, kind, steps, classes):
    """Replays with the same buffers' eager pass and other eager work between them."""
    hip = Hip(mg)
    stream = hip.stream()
    ref, b, other = (Block(mg, 4, kind, steps, classes) for _ in range(3))
    ref.run()
    sync(mg)
    want = ref.outputs()
    exe = hip.capture(stream, lambda: b.run(stream))
    for turn in range(4):
        print("replay", turn, flush=True)
        b.spoil()
        if turn == 2:
            b.run(stream)
        else:
            hip.launch(exe, stream)
        hip.sync(stream)
        same(b.outputs(), want, f"turn {turn}")
        other.run()
        sync(mg)
    hip.launch(exe, stream)
    hip.launch(exe, stream)
    hip.sync(stream)
    same(b.outputs(), want, "two replays in a row")
    hip("hipGraphExecDestroy", exe)
    hip("hipStreamDestroy", stream)


def test_two_blocks_on_two_streams(mg):
    """Each with its own buffers and workspaces, queued at the same time."""
    hip = Hip(mg)
    streams = [hip.stream(), hip.stream()]
    sizes = [("fp32", 12, 1000), ("bf16", 70, 9000)]
    blocks = [Block(mg, 5 + k, *sizes[k]) for k in range(2)]
    refs = [Block(mg, 5 + k, *sizes[k]) for k in range(2)]
    for _ in range(4):
        for b, st in zip(blocks, streams):
            b.run(st)
    for st in streams:
        hip.sync(st)
    for ref in refs:
        ref.run()
        sync(mg)
    for k in range(2):
        same(blocks[k].outputs(), refs[k].outputs(), f"stream {k}")
    for st in streams:
        hip("hipStreamDestroy", st)


def test_resets_of_a_gym(mg):
    """A gym's done flags, as they are before a step, are the resets: the state of every env that
    starts anew is what its first step alone gives."""
    gym = mg.Gym("rollout_cartpole", 256, 0)
    r = np.random.RandomState(6)
    d, s = 32, 16
    f = lambda *k: r.normal(0, 1, k).astype(np.float32)  # noqa: E731
    up = mg.DeviceBuffer.from_array
    a = -np.exp(f(d, s))
    mats = f(4, d)
    state, fresh = up(f(256, d, s)), up(np.zeros((256, d, s), np.float32))
    dev = {k: up(v) for k, v in dict(a=a, dt=f(256, d), b=f(256, s), c=f(256, s)).items()}
    y, alone = mg.DeviceBuffer(256 * d * 4), mg.DeviceBuffer(256 * d * 4)
    begun = 0
    for t in range(40):
        done = gym.done()
        x = up(gym.obs() @ mats + np.float32(t))
        args = dict(a=dev["a"].ptr, b=dev["b"].ptr, c=dev["c"].ptr, stream=gym.buf.stream)
        mg.selective_scan(x.ptr, dev["dt"].ptr, y.ptr, 1, 256, d, s, reset=gym.buf.done, initial=state.ptr,
                          final=state.ptr, **args)
        mg.selective_scan(x.ptr, dev["dt"].ptr, alone.ptr, 1, 256, d, s, final=fresh.ptr, **args)
        gym.set_actions(np.full(256, t % 3 == 0, np.int32))
        gym.run()
        new = done != 0
        begun += int(new.sum())
        np.testing.assert_array_equal(state.download(np.float32, (256, d, s))[new],
                                      fresh.download(np.float32, (256, d, s))[new])
        np.testing.assert_array_equal(y.download(np.float32, (256, d))[new], alone.download(np.float32, (256, d))[new])
    assert begun > 256  # every env's first, and some that fell
