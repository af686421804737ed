"""The training operators refuse bad arguments before any device work."""
import ctypes as C

import pytest

from metalgym_amd._capi import CapiError

AT = 0x1000  # an address that is never read: every call here is refused


def refused(call, needle):
    with pytest.raises(CapiError) as e:
        call()
    assert e.value.rc == -1 and needle in str(e.value), e.value


@pytest.mark.parametrize("kw,needle", [
    (dict(cols=0), "cols"),
    (dict(cols=(1 << 24) + 1), "cols"),
    (dict(x=None), "x is NULL"),
    (dict(y=None), "y is NULL"),
    (dict(x=AT + 2), "x is not aligned"),
    (dict(y=AT + 1, dtype="bf16"), "y is not aligned"),
    (dict(gamma=AT + 2), "gamma is not aligned"),
    (dict(rstd=AT + 1), "rstd is not aligned"),
    (dict(x_ld=7), "x_ld"),
    (dict(y_ld=1 << 41), "y_ld"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"),
    (dict(residual=AT), "residual and sum"),
    (dict(sum=AT), "residual and sum"),
    (dict(residual=AT, sum=AT, sum_ld=3), "sum_ld"),
])
def test_layernorm_refusals(mg, kw, needle):
    a = dict(x=AT, y=AT, rows=4, cols=8, dtype="fp32")
    a.update(kw)
    refused(lambda: mg.layernorm(**a), needle)


def test_layernorm_unknown_type(mg):
    from metalgym_amd._capi import LayernormArgs

    a = LayernormArgs(x=AT, y=AT, rows=1, cols=8, type=3, eps=1e-5)
    assert mg.lib().mg_layernorm(None, C.byref(a)) == -1 and b"type" in mg.lib().mg_last_error()
    assert mg.lib().mg_layernorm(None, None) == -1


def test_layernorm_of_no_rows_is_nothing(mg):
    mg.layernorm(None, None, 0, 128)
    mg.layernorm_backward(None, None, None, None, None, 0, 128)


@pytest.mark.parametrize("kw,needle", [
    (dict(cols=0), "cols"),
    (dict(dy=None), "dy is NULL"),
    (dict(dx=AT + 2), "dx is not aligned"),
    (dict(mean=None), "mean and rstd"),
    (dict(rstd=None), "mean and rstd"),
    (dict(dsum=AT, dsum_ld=5), "dsum_ld"),
    (dict(dgamma=AT + 2), "dgamma is not aligned"),
    (dict(dgamma=AT, workspace=AT, workspace_bytes=16), "workspace needs"),
    (dict(dbeta=AT, workspace=None, workspace_bytes=1 << 30), "workspace needs"),
    (dict(dbeta=AT, workspace=AT + 4, workspace_bytes=1 << 30), "16-byte"),
])
def test_layernorm_backward_refusals(mg, kw, needle):
    a = dict(x=AT, dy=AT, mean=AT, rstd=AT, dx=AT, rows=4096, cols=128, dtype="fp32")
    a.update(kw)
    refused(lambda: mg.layernorm_backward(**a), needle)


def test_layernorm_backward_workspace(mg):
    assert mg.layernorm_backward_workspace(0, 128) == 0
    assert mg.layernorm_backward_workspace(1, 128) == 0
    most = mg.layernorm_backward_workspace(1 << 31, 128)
    assert 0 < most <= 1 << 20 and mg.layernorm_backward_workspace(4096, 128) <= most
    assert mg.lib().mg_layernorm_backward_workspace(1, 128, None) == -1
    with pytest.raises(CapiError):
        mg.layernorm_backward_workspace(1, 0)


def batch(mg, data=AT, count=2, rows=8, cols=16, dtype="fp32", ld=0, stride=0):
    return mg.matrices(data, count, rows, cols, dtype, ld, stride)


@pytest.mark.parametrize("kw,needle", [
    (dict(rows=0), "sides"),
    (dict(cols=65537), "sides"),
    (dict(rows=8193, cols=8193), "smaller side"),
    (dict(count=65536), "count"),
    (dict(data=None), "no data"),
    (dict(data=AT + 2), "not aligned"),
    (dict(ld=15), "ld"),
    (dict(stride=127), "overlap"),
    (dict(stride=8 * 20, ld=24), "overlap"),
])
def test_matrix_batch_refusals(mg, kw, needle):
    full = dict(workspace=1 << 20, workspace_bytes=1 << 40)
    refused(lambda: mg.orthogonalize(batch(mg, **kw), batch(mg, **kw), **full), needle)
    ok = batch(mg, **{k: v for k, v in kw.items() if k in ("count", "rows", "cols")})
    refused(lambda: mg.muon_step(batch(mg, **kw), ok, ok, **full), needle)


def test_matrix_batches_differ(mg):
    full = dict(workspace=1 << 20, workspace_bytes=1 << 40)
    for other in (dict(count=3), dict(rows=9), dict(cols=15)):
        refused(lambda: mg.orthogonalize(batch(mg), batch(mg, **other), **full), "differ in shape")
        refused(lambda: mg.muon_step(batch(mg), batch(mg), batch(mg, **other), **full), "differ in shape")
    refused(lambda: mg.muon_step(batch(mg), batch(mg, dtype="bf16"), batch(mg), **full), "momentum must be fp32")


@pytest.mark.parametrize("space,size,needle", [(None, 1 << 40, "workspace needs"), (1 << 20, 100, "workspace needs"),
                                               ((1 << 20) + 16, 1 << 40, "256-byte")])
def test_matrix_workspace_refusals(mg, space, size, needle):
    refused(lambda: mg.orthogonalize(batch(mg), batch(mg), workspace=space, workspace_bytes=size), needle)
    refused(lambda: mg.muon_step(batch(mg), batch(mg), batch(mg), workspace=space, workspace_bytes=size), needle)


@pytest.mark.parametrize("ns,needle", [
    ((0, 3.4445, -4.7750, 2.0315, 1e-7), "steps"),
    ((33, 3.4445, -4.7750, 2.0315, 1e-7), "steps"),
    ((5, 3.4445, -4.7750, 2.0315, 0.0), "eps"),
    ((5, 3.4445, -4.7750, 2.0315, float("nan")), "eps"),
    ((5, 3.0, 0.0, 0.0, 1e-7), "leaves"),          # grows threefold
    ((2, 65.0, -64.0, 0.0, 1e-7), "leaves"),
    ((5, float("nan"), 0.0, 0.0, 1e-7), "leaves"),
    ((5, float("inf"), 0.0, 0.0, 1e-7), "leaves"),
    ((5, 1.0, float("inf"), float("-inf"), 1e-7), "leaves"),
])
def test_newton_schulz_refusals(mg, ns, needle):
    ns = mg.NewtonSchulz(*ns)
    refused(lambda: mg.orthogonalize_workspace(1, 8, 8, ns), needle)
    refused(lambda: mg.orthogonalize(batch(mg), batch(mg), ns=ns, workspace=1 << 20, workspace_bytes=1 << 40), needle)


def test_newton_schulz_accepts_what_stays_in_range(mg):
    for ns in ((5, 3.4445, -4.7750, 2.0315, 1e-7), (32, 1.5, -0.5, 0.0, 1e-6), (12, 1.875, -1.25, 0.375, 1e-7),
               (1, 2.0, 0.0, 0.0, 1e-7), (5, 1.0, 0.0, 0.0, 1e-7)):
        assert mg.orthogonalize_workspace(1, 8, 8, mg.NewtonSchulz(*ns)) >= 0
    refused(lambda: mg.orthogonalize_workspace(1, 8, 8, mg.NewtonSchulz(2, 2.0, 0.0, 0.0, 1e-7)), "leaves")


@pytest.mark.parametrize("kw,needle", [(dict(lr=-1.0), "lr"), (dict(lr=float("inf")), "lr"),
                                       (dict(weight_decay=float("nan")), "lr"), (dict(scale=-0.1), "lr"),
                                       (dict(momentum=1.0), "momentum"), (dict(momentum=-0.1), "momentum"),
                                       (dict(momentum=float("nan")), "momentum")])
def test_muon_refusals(mg, kw, needle):
    full = dict(workspace=1 << 20, workspace_bytes=1 << 40)
    refused(lambda: mg.muon_step(batch(mg), batch(mg), batch(mg), **kw, **full), needle)


def test_matrix_null_arguments(mg):
    L = mg.lib()
    ok = C.byref(batch(mg))
    assert L.mg_orthogonalize(None, None, None, ok, None, 0) == -1
    assert L.mg_orthogonalize(None, None, ok, None, None, 0) == -1
    assert L.mg_muon_step(None, None, ok, ok, ok, None, 0) == -1
    assert L.mg_orthogonalize_workspace(None, 1, 8, 8, None) == -1
    mg.orthogonalize(batch(mg, count=0, data=None), batch(mg, count=0, data=None))
    mg.muon_step(*(batch(mg, count=0, data=None) for _ in range(3)))


def test_muon_decay_is_bounded(mg):
    full = dict(workspace=1 << 20, workspace_bytes=1 << 40)
    refused(lambda: mg.muon_step(batch(mg), batch(mg), batch(mg), lr=2.0, weight_decay=0.6, **full), "at most 1")


@pytest.mark.parametrize("kw", [dict(lr=1e30, scale=1e30), dict(lr=3e38, scale=0.0)])
def test_muon_rate_is_finite(mg, kw):
    full = dict(workspace=1 << 20, workspace_bytes=1 << 40)
    refused(lambda: mg.muon_step(batch(mg), batch(mg), batch(mg), **kw, **full), "lr * scale")


def test_set_muon_needs_a_model(mg):
    assert mg.lib().mg_ppo_set_muon(None, None) == -1
