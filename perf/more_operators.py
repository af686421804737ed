"""The operators of a policy with memory and a head over many actions, as cases that can be timed
and compared.

* ``conv``       a short causal convolution of each channel over the steps of an episode, with SiLU.
* ``conv_grad``  its gradients.
* ``scan``       a selective state space scan: each channel keeps a few states that decay and take in
                 the channel's input at rates of their own each step.
* ``scan_grad``  its gradients.
* ``loss``       minus the log-probability of a taken action under softmax(x W'), with the log of the
                 softmax's sum and, where asked for, the entropy; the logits are not kept.
* ``loss_grad``  the gradients of x and W.

Rows of the first four are a rollout's: (step, sequence), either of which may come first in memory.
``reset`` is set where a sequence's next episode begins. ``run`` computes them with elementary torch
operations in 32 bits, or, where ``own`` is set, through metalgym_amd. ``exact`` has them in 64 bits.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
CHUNK = 64  # steps between the states that the scan keeps for its gradient

MOST_CELLS = 32 * 4096 * 256 * 16          # states updated by the largest scan
MOST_FLOPS = 4096 * 65536 * 1024           # multiply-adds of the largest product
MOST_LOGITS = 4096 * 65536


def listed():
    def rollout(name, kind, steps, seqs, channels, dtype, **more):
        return dict({"name": name, "kind": kind, "steps": steps, "seqs": seqs, "channels": channels, "type": dtype,
                     "by_seq": False, "resets": True, "carry": True}, **more)

    return [
        # acting: one step of 4096 envs, each with the window of its last inputs
        rollout("conv_step_4096x512", "conv", 1, 4096, 512, "bf16", taps=4),
        # the update of a rollout of 4096 envs and 32 steps
        rollout("conv_grad_32x4096x256", "conv_grad", 32, 4096, 256, "fp32", taps=4),
        # acting with a handful of envs: latency is all
        rollout("scan_step_64x256", "scan", 1, 64, 256, "fp32", states=16, groups=1, gate=True, keep=False),
        # acting with 65536 envs: the states' way to memory and back
        rollout("scan_step_65536x128", "scan", 1, 65536, 128, "bf16", states=16, groups=1, gate=True, keep=False),
        # the forward pass of an update over a whole rollout, episodes ending anywhere
        rollout("scan_32x4096x256", "scan", 32, 4096, 256, "bf16", states=16, groups=1, gate=True, keep=True),
        # one long history, of an odd length, through a wide state
        rollout("scan_16001x1x512", "scan", 16001, 1, 512, "fp16", states=64, groups=1, gate=False, keep=False,
                by_seq=True, resets=False, carry=False),
        # the gradient of the rollout
        rollout("scan_grad_32x4096x256", "scan_grad", 32, 4096, 256, "bf16", states=16, groups=1, gate=True),
        # the gradient of a few long episodes, sequence after sequence
        rollout("scan_grad_2049x3x384", "scan_grad", 2049, 3, 384, "fp32", states=16, groups=2, gate=False,
                by_seq=True, carry=False),
        # acting: the log-probabilities of 64 envs' actions at the default policy's width
        {"name": "loss_64x1000x128", "kind": "loss", "rows": 64, "classes": 1000, "width": 128, "type": "fp32",
         "entropy": True},
        # a large vocabulary of no round size
        {"name": "loss_4095x50001x1024", "kind": "loss", "rows": 4095, "classes": 50001, "width": 1024,
         "type": "bf16", "entropy": True},
        # a minibatch of the default policy's rows over ten thousand actions
        {"name": "loss_grad_4096x10007x128", "kind": "loss_grad", "rows": 4096, "classes": 10007, "width": 128,
         "type": "fp32", "entropy": True},
        # the largest: a minibatch over 65536 tokens
        {"name": "loss_grad_4096x65536x1024", "kind": "loss_grad", "rows": 4096, "classes": 65536, "width": 1024,
         "type": "bf16", "entropy": False},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(["conv", "conv_grad", "scan", "scan", "scan_grad", "scan_grad", "loss", "loss_grad"])
    dtype = rng.choice(list(TYPES))
    if kind in ("loss", "loss_grad"):
        width = rng.choice([128, _spread(rng, 16, 4096), 8 * _spread(rng, 2, 512)])
        classes = _spread(rng, 2, 131072)
        rows = _spread(rng, 1, min(16384, MOST_LOGITS // classes, MOST_FLOPS // (classes * width)))
        return {"kind": kind, "rows": rows, "classes": classes, "width": width, "type": dtype,
                "entropy": rng.random() < 0.5}
    scan = kind.startswith("scan")
    states = rng.choice([16, 16, _spread(rng, 1, 128)]) if scan else 1
    groups = rng.choice([1, 1, 2, 4]) if scan else 1
    channels = groups * max(1, rng.choice([128, 256, _spread(rng, 8, 2048)]) // groups)
    most = (MOST_CELLS if scan else 32 * 4096 * 256) // (channels * states)
    steps = rng.choice([1, 32, _spread(rng, 2, 16384)]) if not kind.endswith("grad") else rng.choice(
        [32, _spread(rng, 1, 16384)])
    steps = min(steps, most)
    seqs = _spread(rng, 1, max(1, min(65536, most // steps)))
    case = {"kind": kind, "steps": steps, "seqs": seqs, "channels": channels, "type": dtype,
            "by_seq": rng.random() < 0.5, "resets": rng.random() < 0.7, "carry": rng.random() < 0.7}
    if not scan:
        return dict(case, taps=rng.choice([2, 3, 4, 4]))
    case.update(states=states, groups=groups, gate=rng.random() < 0.5)
    if kind == "scan":
        case["keep"] = rng.random() < 0.5
    return case


# ---- what a program holds before the call ---------------------------------------------------------


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _uniform(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _logits_in_parts(x, w):
    """(first class, logits in 64 bits) of a few thousand classes at a time."""
    x = x.double()
    part = max(1, (1 << 26) // max(1, x.shape[0]))
    for at in range(0, w.shape[0], part):
        yield at, x @ w[at:at + part].double().T.contiguous()


def _statistics(x, w):
    """The log of the softmax's sum and the entropy, as the forward pass leaves them."""
    top = torch.full((x.shape[0],), -math.inf, dtype=torch.float64, device="cuda")
    total, weighted = torch.zeros_like(top), torch.zeros_like(top)
    for _, s in _logits_in_parts(x, w):
        most = torch.maximum(top, s.amax(1))
        keep = torch.exp(top - most)
        e = torch.exp(s - most[:, None])
        total, weighted, top = total * keep + e.sum(1), weighted * keep + (e * s).sum(1), most
    lse = top + total.log()
    return lse.float(), (lse - weighted / total).float()


def _prepare_loss(case, s, g):
    rows, classes, width, kind = case["rows"], case["classes"], case["width"], TYPES[case["type"]]
    s["x"] = _normal(g, rows, width).to(kind)  # as a layer norm leaves them
    s["w"] = (1.5 * width ** -0.5 * _normal(g, classes, width)).to(kind)
    s["targets"] = torch.randint(classes, (rows,), generator=g, device="cuda", dtype=torch.int32)
    s["targets"][_uniform(g, rows) < 0.03] = -1  # rows that took no action
    if case["kind"] == "loss":
        return s
    s["lse"], entropy = _statistics(s["x"], s["w"])
    s["entropy_of"] = entropy if case["entropy"] else None
    s["dloss"] = _normal(g, rows) / rows  # advantages over the minibatch
    s["dentropy"] = torch.full((rows,), -0.01 / rows, device="cuda") if case["entropy"] else None
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["kind"] in ("loss", "loss_grad"):
        return _prepare_loss(case, s, g)
    steps, seqs, channels, kind = case["steps"], case["seqs"], case["channels"], TYPES[case["type"]]
    lead = (seqs, steps) if case["by_seq"] else (steps, seqs)
    s["reset"] = (_uniform(g, *lead) < 0.02).to(torch.uint8) if case["resets"] else None
    s["x"] = _normal(g, *lead, channels).to(kind)
    if case["kind"].endswith("grad"):
        s["dy"] = (1e-2 * _normal(g, *lead, channels)).to(kind)
    if case["kind"].startswith("conv"):
        taps = case["taps"]
        s["weight"] = _normal(g, channels, taps) * taps ** -0.5
        s["bias"] = 0.1 * _normal(g, channels)
        s["initial"] = _normal(g, seqs, taps - 1, channels).to(kind) if case["carry"] else None
        return s
    states, groups = case["states"], case["groups"]
    s["dt"] = (0.5 * _normal(g, *lead, channels)).to(kind)
    s["b"] = _normal(g, *lead, groups, states).to(kind)
    s["c"] = _normal(g, *lead, groups, states).to(kind)
    s["z"] = _normal(g, *lead, channels).to(kind) if case["gate"] else None
    s["a"] = -torch.arange(1, states + 1, device="cuda") * (0.9 + 0.2 * _uniform(g, channels, states))
    s["d"] = 1 + 0.1 * _normal(g, channels)
    rate = torch.exp(math.log(1e-3) + math.log(100) * _uniform(g, channels))  # of 0.001 to 0.1
    s["dt_bias"] = rate + torch.log(-torch.expm1(-rate))
    s["initial"] = 0.5 * _normal(g, seqs, channels, states) if case["carry"] else None
    if case["kind"] == "scan_grad":
        s["dfinal"] = 1e-2 * _normal(g, seqs, channels, states) if case["carry"] else None
        s["checkpoints"] = _checkpoints(s) if steps > CHUNK else None
    return s


def _by_step(s, t):
    """The array with its steps first."""
    return t if t is None or not s["by_seq"] else t.transpose(0, 1)


def _checkpoints(s):
    """The states before every CHUNK steps, as the forward pass leaves them."""
    t = {k: _by_step(s, s[k]) for k in ("x", "dt", "b", "reset")}
    h = s["initial"] if s["initial"] is not None else torch.zeros(s["seqs"], s["channels"], s["states"], device="cuda")
    h, kept = h.double(), []
    for at in range(0, s["steps"], CHUNK):
        kept.append(h.float())
        decay, gain = _terms(s, *(t[k][at:at + CHUNK] if t[k] is not None else None for k in ("x", "dt", "b", "reset")),
                             torch.float64)
        gain[0] += decay[0] * h
        h = _recur(decay, gain)[-1]
    return torch.stack(kept)


# ---- the operators in plain form --------------------------------------------------------------------


def _recur(decay, gain):
    """h[t] = decay[t] h[t - 1] + gain[t] along the first axis, by doubling the span that each takes in."""
    span = 1
    while span < len(gain):
        gain = torch.cat([gain[:span], gain[span:] + decay[span:] * gain[:-span]])
        decay = torch.cat([decay[:span], decay[span:] * decay[:-span]])
        span *= 2
    return gain


def _each(s, t):
    """[..., groups, states] for every channel: [..., channels, states]."""
    return t.repeat_interleave(s["channels"] // s["groups"], -2)


def _softplus(v):
    return v.clamp_min(0) + torch.log1p(torch.exp(-v.abs()))


def _terms(s, x, dt, b, reset, kind):
    delta = _softplus(dt.to(kind) + s["dt_bias"].to(kind))
    decay = torch.exp(delta[..., None] * s["a"].to(kind))
    if reset is not None:
        decay *= (reset == 0)[..., None, None]
    return decay, (delta * x.to(kind))[..., None] * _each(s, b.to(kind))


def _scan(s):
    kind = TYPES[s["type"]]
    x, dt, b, c, z, reset = (_by_step(s, s[k]) for k in ("x", "dt", "b", "c", "z", "reset"))
    decay, gain = _terms(s, x, dt, b, reset, torch.float32)
    if s["initial"] is not None:
        gain[0] += decay[0] * s["initial"]
    h = _recur(decay, gain)
    y = (h * _each(s, c.float())).sum(-1) + s["d"] * x.float()
    if z is not None:
        z = z.float()
        y = y * (z * torch.sigmoid(z))
    out = {"y": _by_step(s, y.to(kind)).contiguous()}
    if s["carry"]:
        out["final"] = h[-1].contiguous()
    if s["keep"]:
        first = s["initial"] if s["initial"] is not None else torch.zeros_like(h[0])
        out["checkpoints"] = torch.cat([first[None], h[CHUNK - 1:-1:CHUNK]])
    return out


def _over_channels(s, t):
    """[..., channels, states] summed over each group's channels."""
    return t.unflatten(-2, (s["groups"], -1)).sum(-2)


def _scan_grad(s):
    kind = TYPES[s["type"]]
    x, dt, b, c, z, reset, dy = (_by_step(s, s[k]) for k in ("x", "dt", "b", "c", "z", "reset", "dy"))
    decay, gain = _terms(s, x, dt, b, reset, torch.float32)
    first = s["initial"] if s["initial"] is not None else torch.zeros_like(gain[0])
    gain[0] += decay[0] * first
    h = _recur(decay, gain)
    del gain
    x, dy, ec, out = x.float(), dy.float(), _each(s, c.float()), {}
    if z is not None:
        z = z.float()
        sig = torch.sigmoid(z)
        y = (h * ec).sum(-1) + s["d"] * x
        out["dz"] = dy * y * (sig * (1 + z * (1 - sig)))
        dy = dy * (z * sig)
    g = ec * dy[..., None]
    if s["dfinal"] is not None:
        g[-1] += s["dfinal"]
    g = _recur(torch.cat([torch.zeros_like(first)[None], decay[1:].flip(0)]), g.flip(0)).flip(0)
    raw = dt.float() + s["dt_bias"]
    delta = _softplus(raw)
    gb = (g * _each(s, b.float())).sum(-1)
    out["dx"] = dy * s["d"] + delta * gb
    out["dc"] = _over_channels(s, h * dy[..., None])
    out["db"] = _over_channels(s, g * (delta * x)[..., None])
    if s["carry"]:
        out["dinitial"] = decay[0] * g[0]
    g = g * decay * torch.cat([first[None], h[:-1]])
    ddt = (x * gb + (g * s["a"]).sum(-1)) * torch.sigmoid(raw)
    out["ddt"] = ddt
    for k in ("dx", "ddt", "dz", "db", "dc"):
        if k in out:
            out[k] = _by_step(s, out[k].to(kind)).contiguous()
    out["da"] = (g * delta[..., None]).sum((0, 1))
    out["dd"] = (dy * x).sum((0, 1))
    out["ddt_bias"] = ddt.sum((0, 1))
    return out


def _windows(s, x):
    """[taps][steps][seqs][channels]: the inputs that each step sees, the oldest first."""
    taps, steps = s["taps"], s["steps"]
    first = s["initial"].float().transpose(0, 1) if s["initial"] is not None else x.new_zeros(taps - 1, *x.shape[1:])
    long = torch.cat([first, x])
    seen = torch.stack([long[k:k + steps] for k in range(taps)])
    if s["reset"] is None:
        return seen, None
    reset = torch.cat([x.new_zeros(taps - 1, s["seqs"]), _by_step(s, s["reset"]).float()])
    # episodes begun up to each place: a step sees the places of its own episode
    count = reset.cumsum(0)
    same = torch.stack([count[k:k + steps] == count[taps - 1:] for k in range(taps)])[..., None]
    return seen.where(same, 0.0), same


def _conv(s):
    kind, taps = TYPES[s["type"]], s["taps"]
    x = _by_step(s, s["x"]).float()
    seen, _ = _windows(s, x)
    pre = (seen * s["weight"].T[:, None, None]).sum(0) + s["bias"]
    out = {"y": _by_step(s, (pre * torch.sigmoid(pre)).to(kind)).contiguous()}
    if s["carry"]:
        out["final"] = _last_inputs(s, seen).to(kind)
    return out


def _last_inputs(s, seen):
    """The window that the next step would see: what the last step saw but for the oldest."""
    return seen[1:, -1].transpose(0, 1).contiguous()


def _conv_grad(s):
    kind, taps, steps = TYPES[s["type"]], s["taps"], s["steps"]
    x, dy = _by_step(s, s["x"]).float(), _by_step(s, s["dy"]).float()
    seen, same = _windows(s, x)
    w = s["weight"].T[:, None, None]
    pre = (seen * w).sum(0) + s["bias"]
    sig = torch.sigmoid(pre)
    dpre = dy * (sig * (1 + pre * (1 - sig)))
    each = dpre * w
    if same is not None:
        each = each.where(same, 0.0)
    dlong = x.new_zeros(taps - 1 + steps, *x.shape[1:])
    for k in range(taps):
        dlong[k:k + steps] += each[k]
    out = {"dx": _by_step(s, dlong[taps - 1:].to(kind)).contiguous(),
           "dweight": (seen * dpre).sum((1, 2)).T.contiguous(), "dbias": dpre.sum((0, 1))}
    if s["carry"]:
        out["dinitial"] = dlong[:taps - 1].transpose(0, 1).to(kind).contiguous()
    return out


def _loss(s):
    logits = s["x"].float() @ s["w"].float().T
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1)
    lse = total.log() + top.squeeze(1)
    took = s["targets"] >= 0
    of = logits.gather(1, s["targets"].clamp_min(0).long()[:, None]).squeeze(1)
    out = {"loss": torch.where(took, lse - of, 0.0), "lse": lse}
    if s["entropy"]:
        out["entropy"] = total.log() - (e * (logits - top)).sum(1) / total
    return out


def _loss_grad(s):
    kind = TYPES[s["type"]]
    x, w = s["x"].float(), s["w"].float()
    took = (s["targets"] >= 0)[:, None]
    logp = x @ w.T - s["lse"][:, None]
    p = torch.exp(logp)
    d = p * s["dloss"][:, None]
    if s["entropy"]:
        d -= s["dentropy"][:, None] * p * (logp + s["entropy_of"][:, None])
    del logp, p
    d.scatter_add_(1, s["targets"].clamp_min(0).long()[:, None], -s["dloss"][:, None])
    d *= took
    return {"dx": (d @ w).to(kind), "dw": (d.T @ x).to(kind)}


# ---- the same through the framework -----------------------------------------------------------------


def _at(t):
    return None if t is None else t.data_ptr()


def _space(n):
    return torch.empty(n, dtype=torch.uint8, device="cuda")


def _own_rollout(s, mg, stream):
    steps, seqs, channels = s["steps"], s["seqs"], s["channels"]
    order = {"step_rows": 1, "seq_rows": steps} if s["by_seq"] else {}
    order.update(reset=_at(s["reset"]), initial=_at(s["initial"]), stream=stream)
    kind, x = s["kind"], s["x"]
    if kind == "conv":
        out = {"y": torch.empty_like(x)}
        if s["carry"]:
            out["final"] = torch.empty_like(s["initial"])
        mg.causal_conv(_at(x), _at(s["weight"]), _at(out["y"]), steps, seqs, channels, s["taps"], s["type"],
                       bias=_at(s["bias"]), silu=True, final=_at(out.get("final")), **order)
        return out
    if kind == "conv_grad":
        out = {"dx": torch.empty_like(x), "dweight": torch.empty_like(s["weight"]),
               "dbias": torch.empty_like(s["bias"])}
        if s["carry"]:
            out["dinitial"] = torch.empty_like(s["initial"])
        space = _space(mg.causal_conv_backward_workspace(steps, seqs, channels, s["taps"]))
        mg.causal_conv_backward(_at(x), _at(s["weight"]), _at(s["dy"]), _at(out["dx"]), steps, seqs, channels,
                                s["taps"], s["type"], bias=_at(s["bias"]), silu=True, dweight=_at(out["dweight"]),
                                dbias=_at(out["dbias"]), dinitial=_at(out.get("dinitial")), workspace=_at(space),
                                workspace_bytes=space.numel(), **order)
        return out
    states, groups = s["states"], s["groups"]
    inputs = dict(a=_at(s["a"]), b=_at(s["b"]), c=_at(s["c"]), d=_at(s["d"]), dt_bias=_at(s["dt_bias"]), z=_at(s["z"]))
    if kind == "scan":
        out = {"y": torch.empty_like(x)}
        if s["carry"]:
            out["final"] = torch.empty(seqs, channels, states, device="cuda")
        if s["keep"]:
            out["checkpoints"] = torch.empty((steps + CHUNK - 1) // CHUNK, seqs, channels, states, device="cuda")
        space = _space(mg.selective_scan_workspace(steps, seqs, channels, states))
        mg.selective_scan(_at(x), _at(s["dt"]), _at(out["y"]), steps, seqs, channels, states, s["type"],
                          groups=groups, final=_at(out.get("final")), checkpoints=_at(out.get("checkpoints")),
                          workspace=_at(space), workspace_bytes=space.numel(), **inputs, **order)
        return out
    out = {k: torch.empty_like(s[k[1:]]) for k in ("dx", "ddt", "db", "dc", "da", "dd", "ddt_bias")}
    if s["gate"]:
        out["dz"] = torch.empty_like(x)
    if s["carry"]:
        out["dinitial"] = torch.empty_like(s["initial"])
    space = _space(mg.selective_scan_backward_workspace(steps, seqs, channels, states, groups))
    mg.selective_scan_backward(_at(x), _at(s["dt"]), _at(s["dy"]), steps, seqs, channels, states, s["type"],
                               groups=groups, checkpoints=_at(s["checkpoints"]), dfinal=_at(s["dfinal"]),
                               workspace=_at(space), workspace_bytes=space.numel(),
                               **{k: _at(v) for k, v in out.items()}, **inputs, **order)
    return out


def _own(s):
    import metalgym_amd as mg

    stream = torch.cuda.current_stream().cuda_stream
    if not s["kind"].startswith("loss"):
        return _own_rollout(s, mg, stream)
    shape = (s["rows"], s["classes"], s["width"])
    if s["kind"] == "loss":
        out = {"loss": torch.empty(s["rows"], device="cuda"), "lse": torch.empty(s["rows"], device="cuda")}
        if s["entropy"]:
            out["entropy"] = torch.empty(s["rows"], device="cuda")
        space = _space(mg.cross_entropy_workspace(*shape, s["type"]))
        mg.cross_entropy(_at(s["x"]), _at(s["w"]), _at(s["targets"]), *shape, s["type"], loss=_at(out["loss"]),
                         lse=_at(out["lse"]), entropy=_at(out.get("entropy")), workspace=_at(space),
                         workspace_bytes=space.numel(), stream=stream)
        return out
    out = {"dx": torch.empty_like(s["x"]), "dw": torch.empty_like(s["w"])}
    space = _space(mg.cross_entropy_backward_workspace(*shape, s["type"]))
    mg.cross_entropy_backward(_at(s["x"]), _at(s["w"]), _at(s["targets"]), *shape, s["type"], lse=_at(s["lse"]),
                              dloss=_at(s["dloss"]), entropy=_at(s["entropy_of"]), dentropy=_at(s["dentropy"]),
                              dx=_at(out["dx"]), dw=_at(out["dw"]), workspace=_at(space),
                              workspace_bytes=space.numel(), stream=stream)
    return out


PLAIN = {"conv": _conv, "conv_grad": _conv_grad, "scan": _scan, "scan_grad": _scan_grad, "loss": _loss,
         "loss_grad": _loss_grad}


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------


def work(case):
    kind, b = case["kind"], BYTES[case["type"]]
    if kind.startswith("loss"):
        rows, classes, width = case["rows"], case["classes"], case["width"]
        once = (rows + classes) * width * b
        if kind == "loss":  # x, W, a target and two or three results a row; one product
            return {"bytes": once + rows * (16 if case["entropy"] else 12), "flops": 2 * rows * classes * width}
        # x and W and their gradients; the product for the logits and one for each gradient
        return {"bytes": 2 * once + rows * (20 if case["entropy"] else 12), "flops": 6 * rows * classes * width}
    rows, channels = case["steps"] * case["seqs"], case["channels"]
    cells = rows * channels
    resets = rows if case["resets"] else 0
    if kind.startswith("conv"):
        taps = case["taps"]
        window = 2 * case["seqs"] * (taps - 1) * channels * b if case["carry"] else 0
        if kind == "conv":  # x and y, and the window in and out
            return {"bytes": 2 * cells * b + window + resets + 4 * channels * (taps + 1),
                    "flops": cells * (2 * taps + 5)}
        # x, dy and dx
        return {"bytes": 3 * cells * b + window + resets + 8 * channels * (taps + 1), "flops": cells * (6 * taps + 9)}
    states, gate = case["states"], int(case["gate"])
    held = case["seqs"] * channels * states * 4
    vectors = 4 * channels * (states + 2)
    shared = 2 * rows * case["groups"] * states * b  # B and C
    if kind == "scan":  # x, dt, the gate and y; the states in and out, and those that are kept
        kept = held * -(-case["steps"] // CHUNK) if case["keep"] else 0
        return {"bytes": (3 + gate) * cells * b + shared + resets + vectors + kept + (2 * held if case["carry"] else 0),
                "flops": cells * (7 * states + 8 + 5 * gate)}
    # x, dt, dy, the gate and the gradients of all but dy; the states that were kept; the states' gradients
    kept = held * -(-case["steps"] // CHUNK) if case["steps"] > CHUNK or case["carry"] else 0
    return {"bytes": (5 + 2 * gate) * cells * b + 2 * shared + resets + 2 * vectors + kept
            + (2 * held if case["carry"] else 0), "flops": cells * (22 * states + 12 + 12 * gate)}


# ---- the same in 64 bits ----------------------------------------------------------------------------


def _exact_conv(case, s):
    """Step by step: the window as it stands, emptied where an episode begins."""
    steps, taps, carry = case["steps"], case["taps"], case["carry"]
    pick = (lambda t, i: t[:, i]) if case["by_seq"] else (lambda t, i: t[i])
    w, bias = s["weight"].double(), s["bias"].double()
    x = s["x"].double()
    past = [torch.zeros_like(pick(x, 0)) for _ in range(taps - 1)]
    if s["initial"] is not None:
        past = [s["initial"][:, k].double() for k in range(taps - 1)]
    y = torch.empty_like(x)
    grad = case["kind"] == "conv_grad"
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(bias)
    first = [torch.zeros_like(p) for p in past]  # the gradients of the inputs from before the call
    one = torch.ones(case["seqs"], 1, dtype=torch.float64, device="cuda")
    lives = [one] * (taps - 1)  # whether a place of the window is of this episode
    for i in range(steps):
        new = pick(x, i)
        if s["reset"] is not None:
            live = (pick(s["reset"], i) == 0).double()[:, None]
            past, lives = [p * live for p in past], [v * live for v in lives]
        window = past + [new]
        pre = bias + sum(window[k] * w[:, k] for k in range(taps))
        sig = 1 / (1 + torch.exp(-pre))
        pick(y, i).copy_(pre * sig)
        if grad:
            d = pick(s["dy"], i).double() * (sig + pre * sig * (1 - sig))
            db += d.sum(0)
            for k in range(taps):
                dw[:, k] += (d * window[k]).sum(0)
                mine = d * w[:, k] * (lives[k] if k < taps - 1 else 1.0)
                at = i - (taps - 1) + k
                if at >= 0:
                    pick(dx, at).add_(mine)
                else:
                    first[at + taps - 1] += mine
        past, lives = window[1:], lives[1:] + [one]
    if grad:
        out = {"dx": dx, "dweight": dw, "dbias": db}
        return dict(out, dinitial=torch.stack(first, 1)) if carry else out
    return dict({"y": y}, final=torch.stack(past, 1)) if carry else {"y": y}


def _exact_scan(case, s):
    """Step by step forwards, with every state kept for the way back."""
    steps, seqs, channels, states = (case[k] for k in ("steps", "seqs", "channels", "states"))
    pick = (lambda t, i: t[:, i]) if case["by_seq"] else (lambda t, i: t[i])
    group = torch.arange(channels, device="cuda") // (channels // case["groups"])
    a, skip, bias = s["a"].double(), s["d"].double(), s["dt_bias"].double()
    grad = case["kind"] == "scan_grad"
    h = torch.zeros(seqs, channels, states, dtype=torch.float64, device="cuda")
    if s["initial"] is not None:
        h = h + s["initial"]
    y = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda")
    kept, all_h = [], [h]
    live = lambda i: 1.0 if s["reset"] is None else (pick(s["reset"], i) == 0).double()[:, None, None]  # noqa: E731
    for i in range(steps):
        if i % CHUNK == 0:
            kept.append(h)
        raw = pick(s["dt"], i).double() + bias
        delta = torch.logaddexp(raw, torch.zeros_like(raw))
        x = pick(s["x"], i).double()
        b, c = (pick(s[k], i).double()[:, group] for k in ("b", "c"))
        h = torch.exp(delta[..., None] * a) * h * live(i) + b * (delta * x)[..., None]
        v = (h * c).sum(-1) + skip * x
        if s["z"] is not None and not grad:
            z = pick(s["z"], i).double()
            v = v * z / (1 + torch.exp(-z))
        pick(y, i).copy_(v)
        if grad:
            all_h.append(h)
    if not grad:
        out = {"y": y}
        if case["carry"]:
            out["final"] = h
        if case["keep"]:
            out["checkpoints"] = torch.stack(kept)
        return out
    new = lambda k: torch.zeros(s[k].shape, dtype=torch.float64, device="cuda")  # noqa: E731
    out = {"dx": new("x"), "ddt": new("dt"), "db": new("b"), "dc": new("c"), "da": new("a"), "dd": new("d"),
           "ddt_bias": new("dt_bias")}
    if case["gate"]:
        out["dz"] = new("z")
    g = torch.zeros_like(h) if s["dfinal"] is None else s["dfinal"].double()
    for i in reversed(range(steps)):
        raw = pick(s["dt"], i).double() + bias
        delta = torch.logaddexp(raw, torch.zeros_like(raw))
        x, dy = pick(s["x"], i).double(), pick(s["dy"], i).double()
        b, c = (pick(s[k], i).double()[:, group] for k in ("b", "c"))
        if s["z"] is not None:
            z = pick(s["z"], i).double()
            sig = 1 / (1 + torch.exp(-z))
            pick(out["dz"], i).copy_(dy * pick(y, i) * (sig + z * sig * (1 - sig)))
            dy = dy * z * sig
        g = g + c * dy[..., None]
        to = torch.zeros(seqs, case["groups"], states, dtype=torch.float64, device="cuda")
        pick(out["dc"], i).copy_(to.index_add(1, group, all_h[i + 1] * dy[..., None]))
        pick(out["db"], i).copy_(to.index_add(1, group, g * (delta * x)[..., None]))
        gb = (g * b).sum(-1)
        pick(out["dx"], i).copy_(gb * delta + dy * skip)
        out["dd"] += (dy * x).sum(0)
        g = g * torch.exp(delta[..., None] * a) * live(i)
        via = g * all_h[i]
        out["da"] += (via * delta[..., None]).sum(0)
        ddt = (gb * x + (via * a).sum(-1)) / (1 + torch.exp(-raw))
        pick(out["ddt"], i).copy_(ddt)
        out["ddt_bias"] += ddt.sum(0)
    if case["carry"]:
        out["dinitial"] = g
    return out


def _exact_loss(case, s):
    if case["kind"] == "loss":
        n = case["rows"]
        lse = torch.full((n,), -math.inf, dtype=torch.float64, device="cuda")
        of, mean = torch.zeros_like(lse), torch.zeros_like(lse)
        rows = torch.arange(n, device="cuda")
        for at, part in _logits_in_parts(s["x"], s["w"]):
            here = torch.logsumexp(part, 1)
            both = torch.logaddexp(lse, here)
            mean = mean * torch.exp(lse - both) + (torch.exp(part - both[:, None]) * part).sum(1)
            lse = both
            inside = (s["targets"] >= at) & (s["targets"] < at + part.shape[1])
            of[inside] = part[rows[inside], (s["targets"][inside] - at).long()]
        out = {"loss": (lse - of) * (s["targets"] >= 0), "lse": lse}
        return dict(out, entropy=lse - mean) if case["entropy"] else out
    dx = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
    dw = torch.empty(s["w"].shape, dtype=torch.float64, device="cuda")
    x, lse = s["x"].double(), s["lse"].double()[:, None]
    scale = (s["dloss"].double() * (s["targets"] >= 0))[:, None]
    for at, part in _logits_in_parts(s["x"], s["w"]):
        p = torch.exp(part - lse)
        hit = torch.arange(at, at + part.shape[1], device="cuda") == s["targets"][:, None]
        d = scale * (p - hit.double())
        if case["entropy"]:
            more = s["dentropy"].double()[:, None] * (s["targets"] >= 0)[:, None]
            d = d - more * p * (part - lse + s["entropy_of"].double()[:, None])
        dx += d @ s["w"][at:at + part.shape[1]].double()
        dw[at:at + part.shape[1]] = d.T.contiguous() @ x
    return {"dx": dx, "dw": dw}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"].startswith("loss"):
        return _exact_loss(case, s)
    if case["steps"] * (3 if case["kind"].endswith("grad") else 1) > 40000:
        return None  # too many single steps
    return _exact_conv(case, s) if case["kind"].startswith("conv") else _exact_scan(case, s)
