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
