"""Arrays past 2^32 bytes and elements: what lies at their far ends comes out as it should."""
import numpy as np
import pytest

from operator_cases import decode, encode
from rollout_cases import rounded

pytestmark = pytest.mark.gpu


def sync(mg):
    mg._capi.check(mg.lib().mg_synchronize())


def zeros(mg, nbytes):
    b = mg.DeviceBuffer(nbytes)
    b.zero()
    return b


def test_rows_past_32_bits(mg):
    """66000 steps of 65536 channels in bfloat16: 4.3e9 elements an array, all 0 but the last few
    steps' last channels."""
    steps, channels, last, some = 66000, 65536, 5, 64
    x, dt, y = (zeros(mg, steps * channels * 2) for _ in range(3))
    r = np.random.RandomState(0)
    vals = rounded(r.normal(0, 1, (last, some)), "bf16")
    place = lambda t: ((steps - last + t) * channels + channels - some) * 2  # noqa: E731
    for t in range(last):
        mg.h2d(x.ptr + place(t), encode(vals[t], "bf16"))
    get = lambda b, t: decode(mg.d2h(b.ptr + place(t), np.uint16, (some,)), "bf16")  # noqa: E731
    weight = rounded(r.normal(0, 1, (channels, 4)), "fp32")
    w = mg.DeviceBuffer.from_array(weight.astype(np.float32))
    mg.causal_conv(x.ptr, w.ptr, y.ptr, steps, 1, channels, 4, "bf16", step_rows=1, seq_rows=steps)
    sync(mg)
    seen = np.concatenate([np.zeros((3, some)), vals])
    for t in range(last):
        want = (seen[t:t + 4].T * weight[-some:]).sum(1)
        size = (np.abs(seen[t:t + 4].T * weight[-some:])).sum(1)
        assert (np.abs(get(y, t) - want) <= 2.0**-8 * np.abs(want) + 8 * 2.0**-24 * size).all()
    a = mg.DeviceBuffer.from_array(np.full((channels, 1), -1, np.float32))
    ones = mg.DeviceBuffer.from_array(np.full(steps, 0x3F80, np.uint16))
    space = mg.DeviceBuffer(mg.selective_scan_workspace(steps, 1, channels, 1) + 256)
    mg.selective_scan(x.ptr, dt.ptr, y.ptr, steps, 1, channels, 1, "bf16", a=a.ptr, b=ones.ptr, c=ones.ptr, step_rows=1,
                      seq_rows=steps, workspace=space.ptr, workspace_bytes=space.nbytes)
    sync(mg)
    delta, h, size = np.log(2.0), np.zeros(some), np.zeros(some)
    for t in range(last):
        h, size = 0.5 * h + delta * vals[t], 0.5 * size + delta * np.abs(vals[t])
        assert (np.abs(get(y, t) - h) <= 2.0**-8 * np.abs(h) + 60 * 2.0**-24 * size).all()


@pytest.mark.parametrize("kind,rows,classes,width", [("bf16", 8, 600000, 4096), ("fp32", 8, 600000, 2048),
                                                     ("fp32", 40, 600000, 2048)])
def test_classes_past_32_bits(mg, kind, rows, classes, width):
    """W of 4.9 GB, 0 but for a few classes at its ends: every other logit is 0."""
    size = 2 if kind == "bf16" else 4
    r = np.random.RandomState(1)
    special = np.array([0, 1, classes - 3, classes - 1])
    x = rounded(r.normal(0, 1, (rows, width)), kind)
    ws = rounded(r.normal(0, 3 * width**-0.5, (len(special), width)), kind)
    w, dw = zeros(mg, classes * width * size), mg.DeviceBuffer(classes * width * size)
    for k, c in enumerate(special):
        mg.h2d(w.ptr + int(c) * width * size, encode(ws[k], kind))
    targets = r.choice(np.append(special, classes - 2), rows).astype(np.int32)
    dloss = rounded(r.normal(0, 1, rows), "fp32")
    up = mg.DeviceBuffer.from_array
    dx_, dt_, dl = up(encode(x, kind)), up(targets), up(dloss.astype(np.float32))
    loss, lse, dx = mg.DeviceBuffer(4 * rows), mg.DeviceBuffer(4 * rows), mg.DeviceBuffer(rows * width * size)
    space = mg.DeviceBuffer(max(mg.cross_entropy_workspace(rows, classes, width, kind),
                                mg.cross_entropy_backward_workspace(rows, classes, width, kind)) + 256)
    use = dict(workspace=space.ptr, workspace_bytes=space.nbytes)
    mg.cross_entropy(dx_.ptr, w.ptr, dt_.ptr, rows, classes, width, kind, loss=loss.ptr, lse=lse.ptr, **use)
    mg.cross_entropy_backward(dx_.ptr, w.ptr, dt_.ptr, rows, classes, width, kind, lse=lse.ptr, dloss=dl.ptr, dx=dx.ptr,
                              dw=dw.ptr, **use)
    sync(mg)
    s = x @ ws.T
    want = np.log(classes - len(special) + np.exp(s).sum(1))
    of = np.array([s[i, np.flatnonzero(special == t)[0]] if t in special else 0.0 for i, t in enumerate(targets)])
    # logits are off by at most 2 (16 + width / 16) half steps of their products' size, 1e-4 here
    got = lse.download(np.float32, (rows,)).astype(np.float64)
    assert (np.abs(got - want) <= 2e-4).all()
    assert (np.abs(loss.download(np.float32, (rows,)) - (want - of)) <= 4e-4).all()
    p = np.exp(s - want[:, None])
    hit = targets[:, None] == special
    g = dloss[:, None] * (p - hit)
    near = 2.0**-7 if kind == "bf16" else 1e-3  # g and the result rounded; probabilities off by their logits'
    d = decode(dx.download(np.uint16 if kind == "bf16" else np.float32, (rows, width)), kind)
    assert np.linalg.norm(d - g @ ws) <= near * np.linalg.norm(g @ ws)
    row = lambda c: decode(mg.d2h(dw.ptr + int(c) * width * size, np.uint16 if size == 2 else np.float32, (width,)),  # noqa: E731
                           kind)
    for k, c in enumerate(special):
        ref = g[:, k] @ x
        assert np.linalg.norm(row(c) - ref) <= near * (np.linalg.norm(ref) + np.linalg.norm(g[:, k]) * width**0.5), c
    for c in (2, classes // 2, classes - 2):
        ref = (dloss * (np.exp(-want) - (targets == c))) @ x
        assert np.linalg.norm(row(c) - ref) <= near * (np.linalg.norm(ref) + 1e-5), c


def test_more_tiles_than_a_launch_takes(mg):
    """2^20 rows of 262444 classes: 2^22 tiles of logits and more, whose threads pass 32 bits."""
    rows, classes, width, kind = 1 << 20, (1 << 18) + 300, 16, "bf16"
    r = np.random.RandomState(2)
    x = rounded(r.standard_normal((rows, width)).astype(np.float32), kind)
    w = rounded(r.standard_normal((classes, width)).astype(np.float32) * 0.5, kind)
    targets = r.randint(0, classes, rows).astype(np.int32)
    targets[:8] = classes - 1 - np.arange(8)
    targets[8] = -1
    dloss = rounded(r.standard_normal(rows).astype(np.float32), "fp32")
    up = mg.DeviceBuffer.from_array
    dx_, dw_, dt, dl = up(encode(x, kind)), up(encode(w, kind)), up(targets), up(dloss.astype(np.float32))
    loss, lse, entropy = (mg.DeviceBuffer(4 * rows) for _ in range(3))
    dx, dw = mg.DeviceBuffer(2 * rows * width), mg.DeviceBuffer(2 * classes * width)
    space = mg.DeviceBuffer(max(mg.cross_entropy_workspace(rows, classes, width, kind),
                                mg.cross_entropy_backward_workspace(rows, classes, width, kind)) + 256)
    use = dict(workspace=space.ptr, workspace_bytes=space.nbytes)
    mg.cross_entropy(dx_.ptr, dw_.ptr, dt.ptr, rows, classes, width, kind, loss=loss.ptr, lse=lse.ptr,
                     entropy=entropy.ptr, **use)
    mg.cross_entropy_backward(dx_.ptr, dw_.ptr, dt.ptr, rows, classes, width, kind, lse=lse.ptr, dloss=dl.ptr, dx=dx.ptr,
                              dw=dw.ptr, **use)
    sync(mg)
    got = [mg.d2h(b.ptr, np.float32, (rows,)).astype(np.float64) for b in (loss, lse, entropy)]
    some = np.concatenate([np.arange(12), [rows // 2, rows - 2, rows - 1]])
    s = x[some] @ w.T
    want_lse = np.log(np.exp(s).sum(1))
    p = np.exp(s - want_lse[:, None])
    live = targets[some] >= 0
    want_loss = np.where(live, want_lse - s[np.arange(len(some)), np.maximum(targets[some], 0)], 0)
    want_entropy = want_lse - (p * s).sum(1)
    # logits: 32 products in turn, at the size of the largest row's; a lane's sums have 128 terms and
    # meet in 20 joins; each exponential, logarithm and difference from the maximum adds a few steps of |s|
    size = (np.abs(x[some])[:, None, :] * np.abs(w[None, :, :])).sum(2).max(1)
    tol = 2.0**-24 * (2 * 40 * size + 256 + 16 * np.abs(want_lse))
    assert (np.abs(got[1][some] - want_lse) <= tol).all()
    assert (np.abs(got[0][some] - want_loss) <= 2 * tol).all()
    # the entropy is a mean of (lse - s), off by twice as much and by its weights' relative error of `tol`
    assert (np.abs(got[2][some] - want_entropy) <= 2 * tol * (2 + np.abs(want_entropy))).all()
    # gradients: each g rounded to bfloat16, and the result; 2^-11 stands for the fp32 sums (4096
    # terms at a time) and for the probabilities' own errors
    share = 2.0**-8 + 2.0**-11
    g = p * dloss[some][:, None]
    g[np.arange(len(some))[live], targets[some][live]] -= dloss[some][live]
    g[~live] = 0
    want = g @ w
    have = decode(mg.d2h(dx.ptr, np.uint16, (rows, width)), kind)[some]
    assert (np.abs(have - want) <= share * (np.abs(g) @ np.abs(w)) + 2.0**-8 * np.abs(want)).all()
    ends = np.array([0, 255, (1 << 18) - 1, 1 << 18, classes - 1])
    p = np.exp(x @ w[ends].T - got[1][:, None])
    g = p * dloss[:, None]
    for k, c in enumerate(ends):
        g[targets == c, k] -= dloss[targets == c]
    g[targets < 0] = 0
    want = g.T @ x
    have = decode(mg.d2h(dw.ptr, np.uint16, (classes, width)), kind)[ends]
    assert (np.abs(have - want) <= share * (np.abs(g).T @ np.abs(x)) + 2.0**-8 * np.abs(want)).all()
