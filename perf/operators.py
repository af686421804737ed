"""The training operators beside the fused update, as cases that can be timed and compared.

A policy is a stack of residual blocks: a layer norm with two vectors, then two matrices. These
operators train such blocks of any width outside the fused update, which is for blocks of 128:

* ``norm``   layer norm forward: rows of a residual stream, with the branch's output added first
             where ``residual`` is set; the mean and 1 / deviation of each row for the backward pass.
* ``grad``   its backward pass: the rows' gradient (plus the residual stream's own, where
             ``residual`` is set) and the gradients of the two vectors, sums over all rows.
* ``orth``   a batch of matrices orthogonalised by five Newton-Schulz steps.
* ``muon``   an optimiser step on a batch of matrices: momentum, the orthogonalised update, decay.

``run`` computes them with elementary torch operations in 32 bits, or, where ``own`` is set,
through metalgym_amd. ``exact`` has them in 64 bits.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5                       # layer norm's
STEPS = 5                        # Newton-Schulz steps
COEFFS = (3.4445, -4.7750, 2.0315)
FLOOR = 1e-7                     # added to a matrix's norm
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01

MOST_CELLS = 1 << 25             # elements of the largest layer norm
MOST_FLOPS = (3 * 8192 + 17 * 2048) * 2048 ** 2  # of the largest batch of matrices


def listed():
    return [
        # acting: the rows of a handful of envs through the policy's width; launch latency is all
        {"name": "norm_64x128", "kind": "norm", "rows": 64, "cols": 128, "type": "fp32", "residual": False},
        # every row of a rollout of 4096 envs and 32 steps through a block's entry
        {"name": "norm_131072x128", "kind": "norm", "rows": 131072, "cols": 128, "type": "fp32", "residual": True},
        # a wide torso in bfloat16, an odd number of rows
        {"name": "norm_bf16_4095x8192", "kind": "norm", "rows": 4095, "cols": 8192, "type": "bf16", "residual": True},
        # one minibatch of the default policy
        {"name": "grad_4096x128", "kind": "grad", "rows": 4096, "cols": 128, "type": "fp32", "residual": True},
        # as many rows as the largest run has envs, in one minibatch
        {"name": "grad_262144x128", "kind": "grad", "rows": 262144, "cols": 128, "type": "fp32", "residual": True},
        # an odd width in binary16, whose rows begin at any alignment
        {"name": "grad_fp16_10007x1001", "kind": "grad", "rows": 10007, "cols": 1001, "type": "fp16",
         "residual": False},
        # the down matrices of the default policy's two blocks (hidden 512)
        {"name": "orth_2x512x128", "kind": "orth", "count": 2, "rows": 512, "cols": 128, "type": "fp32"},
        # all matrices of the deepest and widest policy (8 blocks, hidden 1024) in bfloat16
        {"name": "orth_bf16_16x128x1024", "kind": "orth", "count": 16, "rows": 128, "cols": 1024, "type": "bf16"},
        # an encoder's matrix of no round size
        {"name": "orth_fp16_1000x257", "kind": "orth", "count": 1, "rows": 1000, "cols": 257, "type": "fp16"},
        # a wide torso's matrix
        {"name": "orth_bf16_2048x8192", "kind": "orth", "count": 1, "rows": 2048, "cols": 8192, "type": "bf16"},
        # the optimiser's step on the up matrices of the default policy
        {"name": "muon_2x128x512", "kind": "muon", "count": 2, "rows": 128, "cols": 512, "type": "fp32",
         "grad": "fp32", "nesterov": True},
        # and on a few matrices of a wide torso, with 16-bit gradients
        {"name": "muon_4x1024x2048", "kind": "muon", "count": 4, "rows": 1024, "cols": 2048, "type": "fp32",
         "grad": "bf16", "nesterov": True},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "grad", "orth", "muon"])
    kinds = ["fp32", "bf16", "fp16"]
    if kind in ("norm", "grad"):
        cols = rng.choice([128, _spread(rng, 8, 8192), _spread(rng, 64, 8192)])
        rows = _spread(rng, 1, min(262144, MOST_CELLS // cols))
        return {"kind": kind, "rows": rows, "cols": cols, "type": rng.choice(kinds), "residual": rng.random() < 0.5}
    short = rng.choice([128, _spread(rng, 1, 256), _spread(rng, 128, 2048)])
    long = short * rng.choice([1, 2, 4, 8]) if rng.random() < 0.5 else _spread(rng, short, 8 * short)
    long = min(long, 8192)
    most = MOST_FLOPS // max(1, (3 * long + 17 * short) * short * short)
    count = _spread(rng, 1, max(1, min(16, most)))
    rows, cols = (short, long) if rng.random() < 0.5 else (long, short)
    case = {"kind": kind, "count": count, "rows": rows, "cols": cols, "type": rng.choice(kinds)}
    if kind == "muon":
        case.update(grad=rng.choice(kinds), nesterov=rng.random() < 0.75)
    return case


# ---- what a program holds before the call ---------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _stream_rows(g, rows, cols):
    """Rows of a residual stream: unit-sized features, some of which run larger, and an offset of
    each row."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda"))
    return x.add_(torch.randn(rows, 1, generator=g, device="cuda"))


def _gradients(g, count, rows, cols):
    """Gradients of a layer's matrix: few strong directions over a noise floor, small entries."""
    rank = max(1, min(rows, cols) // 8)
    left = torch.randn(count, rows, rank, generator=g, device="cuda")
    left *= torch.logspace(0, -2, rank, device="cuda")
    right = torch.randn(count, rank, cols, generator=g, device="cuda")
    noise = torch.randn(count, rows, cols, generator=g, device="cuda")
    return 1e-3 * (torch.bmm(left, right) + 0.3 * noise)


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    if case["kind"] in ("norm", "grad"):
        rows, cols, kind = case["rows"], case["cols"], TYPES[case["type"]]
        s["x"] = _stream_rows(g, rows, cols).to(kind)
        s["gamma"] = 1 + 0.1 * torch.randn(cols, generator=g, device="cuda")
        s["beta"] = 0.05 * torch.randn(cols, generator=g, device="cuda")
        if case["kind"] == "norm":
            s["branch"] = torch.randn(rows, cols, generator=g, device="cuda").to(kind) if case["residual"] else None
            return s
        s["dy"] = (1e-2 * torch.randn(rows, cols, generator=g, device="cuda")).to(kind)
        s["dsum"] = (1e-2 * torch.randn(rows, cols, generator=g, device="cuda")).to(kind) if case["residual"] else None
        wide = s["x"].double()
        mean = wide.mean(1, keepdim=True)
        s["mean"] = mean.squeeze(1).float()
        s["rstd"] = (wide.sub_(mean).square_().mean(1) + EPS).rsqrt().float()
        return s
    count, rows, cols = case["count"], case["rows"], case["cols"]
    grad = _gradients(g, count, rows, cols)
    if case["kind"] == "orth":
        s["g"] = grad.to(TYPES[case["type"]])
        return s
    s["g"] = grad.to(TYPES[case["grad"]])
    s["w"] = (torch.randn(count, rows, cols, generator=g, device="cuda") * rows ** -0.5).to(TYPES[case["type"]])
    # the mean of earlier gradients, which this one resembles
    s["m"] = (0.8 * grad + 2e-4 * torch.randn(count, rows, cols, generator=g, device="cuda")).contiguous()
    return s


# ---- the operators in plain form --------------------------------------------------------------------


def _norm(s):
    kind = TYPES[s["type"]]
    x = s["x"]
    out = {}
    if s["branch"] is not None:
        out["sum"] = x = (x.float() + s["branch"].float()).to(kind)  # stored in the stream's type, and normalised as stored
    x = x.float()
    mean = x.mean(1, keepdim=True)
    x = x - mean
    rstd = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    out["y"] = (x * rstd * s["gamma"] + s["beta"]).to(kind)
    out["mean"], out["rstd"] = mean.squeeze(1), rstd.squeeze(1)
    return out


def _grad(s):
    dy, rstd = s["dy"].float(), s["rstd"].unsqueeze(1)
    xn = (s["x"].float() - s["mean"].unsqueeze(1)) * rstd
    d = dy * s["gamma"]
    dx = rstd * (d - d.mean(1, keepdim=True) - xn * (d * xn).mean(1, keepdim=True))
    if s["dsum"] is not None:
        dx = dx + s["dsum"].float()
    return {"dx": dx.to(TYPES[s["type"]]), "dgamma": (dy * xn).sum(0), "dbeta": dy.sum(0)}


def _orthogonal(u):
    """Five Newton-Schulz steps on each matrix over its norm, on the short side's products."""
    a, b, c = COEFFS
    tall = u.shape[1] > u.shape[2]
    x = u.mT.contiguous() if tall else u
    x = x / (torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True) + FLOOR)
    for _ in range(STEPS):
        gram = torch.bmm(x, x.mT.contiguous())
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    return x.mT if tall else x


def _momentum(s, m, g):
    m = m + (1 - MOMENTUM) * (g - m)
    return m, g + MOMENTUM * (m - g) if s["nesterov"] else m


def _muon(s):
    m, u = _momentum(s, s["m"], s["g"].float())
    scale = math.sqrt(max(1.0, s["cols"] / s["rows"]))
    w = s["w"].float() * (1 - LR * DECAY) - LR * scale * _orthogonal(u)
    s["m"].copy_(m)
    s["w"].copy_(w)
    return {"w": s["w"], "m": s["m"]}


# ---- the same through the framework -----------------------------------------------------------------


def _at(t):
    return None if t is None else t.data_ptr()


def _own(s):
    import metalgym_amd as mg

    stream = torch.cuda.current_stream().cuda_stream
    kind = s["kind"]
    if kind == "norm":
        x, rows, cols = s["x"], s["rows"], s["cols"]
        out = {}
        if s["branch"] is not None:
            out["sum"] = torch.empty_like(x)
        out["y"] = torch.empty_like(x)
        out["mean"] = torch.empty(rows, device="cuda")
        out["rstd"] = torch.empty(rows, device="cuda")
        mg.layernorm(_at(x), _at(out["y"]), rows, cols, s["type"], gamma=_at(s["gamma"]), beta=_at(s["beta"]), eps=EPS,
                     residual=_at(s["branch"]), sum=_at(out.get("sum")), mean=_at(out["mean"]), rstd=_at(out["rstd"]),
                     stream=stream)
        return out
    if kind == "grad":
        x, rows, cols = s["x"], s["rows"], s["cols"]
        out = {"dx": torch.empty_like(x), "dgamma": torch.empty(cols, device="cuda"),
               "dbeta": torch.empty(cols, device="cuda")}
        space = torch.empty(mg.layernorm_backward_workspace(rows, cols), dtype=torch.uint8, device="cuda")
        mg.layernorm_backward(_at(x), _at(s["dy"]), _at(s["mean"]), _at(s["rstd"]), _at(out["dx"]), rows, cols,
                              s["type"], gamma=_at(s["gamma"]), dsum=_at(s["dsum"]), dgamma=_at(out["dgamma"]),
                              dbeta=_at(out["dbeta"]), workspace=_at(space), workspace_bytes=space.numel(),
                              stream=stream)
        return out
    ns = mg.NewtonSchulz(STEPS, *COEFFS, FLOOR)
    shape = (s["count"], s["rows"], s["cols"])
    space = torch.empty(mg.orthogonalize_workspace(*shape, ns=ns), dtype=torch.uint8, device="cuda")
    if kind == "orth":
        out = torch.empty_like(s["g"])
        mg.orthogonalize(mg.matrices(_at(s["g"]), *shape, s["type"]), mg.matrices(_at(out), *shape, s["type"]), ns=ns,
                         workspace=_at(space), workspace_bytes=space.numel(), stream=stream)
        return out
    mg.muon_step(mg.matrices(_at(s["w"]), *shape, s["type"]), mg.matrices(_at(s["m"]), *shape, "fp32"),
                 mg.matrices(_at(s["g"]), *shape, s["grad"]), lr=LR, momentum=MOMENTUM, weight_decay=DECAY,
                 nesterov=s["nesterov"], ns=ns, workspace=_at(space), workspace_bytes=space.numel(), stream=stream)
    return {"w": s["w"], "m": s["m"]}


def run(state):
    if own:
        return _own(state)
    kind = state["kind"]
    if kind == "norm":
        return _norm(state)
    if kind == "grad":
        return _grad(state)
    if kind == "orth":
        return _orthogonal(state["g"].float()).to(TYPES[state["type"]])
    return _muon(state)


# ---- what a pass cannot do without ------------------------------------------------------------------

_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def work(case):
    kind, b = case["kind"], _BYTES[case["type"]]
    rows, cols = case["rows"], case["cols"]
    if kind == "norm":  # x and y, with the branch and the sum; two vectors; two statistics a row
        return {"bytes": rows * cols * b * (4 if case["residual"] else 2) + 8 * (rows + cols),
                "flops": 8 * rows * cols}
    if kind == "grad":  # x, dy and dx, with the stream's gradient; gamma and two sums
        return {"bytes": rows * cols * b * (4 if case["residual"] else 3) + 8 * rows + 12 * cols,
                "flops": 12 * rows * cols}
    # The steps as products of symmetric matrices: one Gram product (half of it is enough) and one
    # product with the update; between them a square, two products for the next Gram matrix and one
    # for the polynomials so far, half of each; or, where the sides are alike, every step by itself.
    count, m, n = case["count"], min(rows, cols), max(rows, cols)
    flops = count * m * m * min(3 * n + (4 * STEPS - 3) * m, STEPS * (3 * n + m))
    if kind == "orth":
        return {"bytes": 2 * count * rows * cols * b, "flops": flops}
    return {"bytes": count * rows * cols * (2 * b + 8 + _BYTES[case["grad"]]), "flops": flops}


# ---- the same in 64 bits ----------------------------------------------------------------------------


def _exact_orthogonal(u):
    """Each matrix's p(p(...p(u / |u|))) with p(x) = (a + b x x' + c x x' x x') x."""
    a, b, c = (float(k) for k in COEFFS)
    out = torch.empty_like(u)
    for k, each in enumerate(u):
        x = each if each.shape[0] <= each.shape[1] else each.T.contiguous()
        x = x / (x.square().sum().sqrt() + FLOOR)
        eye = torch.eye(x.shape[0], dtype=x.dtype, device=x.device)
        for _ in range(STEPS):
            gram = x @ x.T.contiguous()
            x = (a * eye + gram @ (b * eye + c * gram)) @ x
        out[k] = x if each.shape[0] <= each.shape[1] else x.T
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        x, out = s["x"].double(), {}
        if s["branch"] is not None:
            x = (x + s["branch"].double()).to(TYPES[case["type"]]).double()
            out["sum"] = s["x"].double() + s["branch"].double()
        mean = x.sum(1) / case["cols"]
        var = (x - mean[:, None]).square().sum(1) / case["cols"]
        rstd = 1 / torch.sqrt(var + EPS)
        out["y"] = (x - mean[:, None]) * rstd[:, None] * s["gamma"].double() + s["beta"].double()
        out["mean"], out["rstd"] = mean, rstd
        return out
    if kind == "grad":
        x, dy, r = s["x"].double(), s["dy"].double(), s["rstd"].double()[:, None]
        hat = (x - s["mean"].double()[:, None]) * r
        d = dy * s["gamma"].double()
        n = case["cols"]
        dx = (d - (d.sum(1) / n)[:, None] - hat * ((d * hat).sum(1) / n)[:, None]) * r
        if s["dsum"] is not None:
            dx += s["dsum"].double()
        return {"dx": dx, "dgamma": (dy * hat).sum(0), "dbeta": dy.sum(0)}
    if kind == "orth":
        return _exact_orthogonal(s["g"].double())
    m0, g = s["m"].double(), s["g"].double()
    m = MOMENTUM * m0 + (1 - MOMENTUM) * g
    u = MOMENTUM * m + (1 - MOMENTUM) * g if case["nesterov"] else m
    step = LR * math.sqrt(max(1.0, case["cols"] / case["rows"]))
    return {"w": (1 - LR * DECAY) * s["w"].double() - step * _exact_orthogonal(u), "m": m}
