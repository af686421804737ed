"""The operators over rollouts refuse bad arguments before any device work."""
import ctypes as C

import pytest

from metalgym_amd._capi import CapiError
from test_cpu_operator_checks import AT, refused

ROLLOUT = [
    (dict(dtype="fp32", channels=0), "channels"),
    (dict(channels=65537), "channels"),
    (dict(steps=(1 << 30) + 1), "steps and seqs"),
    (dict(seqs=(1 << 30) + 1), "steps and seqs"),
    (dict(step_rows=1, seq_rows=1), "overlap"),
    (dict(step_rows=2, seq_rows=1), "overlap"),  # three sequences
    (dict(step_rows=1, seq_rows=3), "overlap"),  # four steps
    (dict(step_rows=1, seq_rows=0), "overlap"),
    (dict(step_rows=0, seq_rows=1), "overlap"),
    (dict(step_rows=(1 << 32) + 1, seq_rows=1), "2^32"),
    (dict(lengths=AT + 2), "lengths is not aligned"),
    (dict(x=None), "x is NULL"),
    (dict(x=AT + 2), "x is not aligned"),
    (dict(x=AT + 1, dtype="bf16"), "x is not aligned"),
    (dict(x_ld=7), "x_ld"),
    (dict(x_ld=(1 << 24) + 1), "x_ld"),
]


def conv(mg, **kw):
    a = dict(x=AT, weight=AT, y=AT, steps=4, seqs=3, channels=8, taps=4, dtype="fp32")
    mg.causal_conv(**dict(a, **kw))


def conv_backward(mg, **kw):
    a = dict(x=AT, weight=AT, dy=AT, dx=AT, steps=4, seqs=3, channels=8, taps=4, dtype="fp32", dweight=AT,
             workspace=1 << 20, workspace_bytes=1 << 40)
    mg.causal_conv_backward(**dict(a, **kw))


def scan(mg, **kw):
    p = dict(x=AT, dt=AT, y=AT, steps=4, seqs=3, channels=8, states=16, dtype="fp32", a=AT, b=AT, c=AT)
    mg.selective_scan(**dict(p, **kw))


def scan_backward(mg, **kw):
    p = dict(x=AT, dt=AT, dy=AT, steps=4, seqs=3, channels=8, states=16, dtype="fp32", a=AT, b=AT, c=AT, dx=AT, ddt=AT,
             db=AT, dc=AT, da=AT, workspace=1 << 20, workspace_bytes=1 << 40)
    mg.selective_scan_backward(**dict(p, **kw))


@pytest.mark.parametrize("call", [conv, conv_backward, scan, scan_backward])
@pytest.mark.parametrize("kw,needle", ROLLOUT)
def test_rollout_refusals(mg, call, kw, needle):
    refused(lambda: call(mg, **kw), needle)


@pytest.mark.parametrize("kw,needle", [
    (dict(taps=1), "taps"),
    (dict(taps=5), "taps"),
    (dict(y=None), "y is NULL"),
    (dict(weight=None), "weight is NULL"),
    (dict(weight=AT + 2), "weight is not aligned"),
    (dict(bias=AT + 1), "bias is not aligned"),
    (dict(initial=AT + 1), "initial is not aligned"),
    (dict(final=AT + 1, dtype="bf16"), "final is not aligned"),
    (dict(y_ld=3), "y_ld"),
])
def test_causal_conv_refusals(mg, kw, needle):
    refused(lambda: conv(mg, **kw), needle)


@pytest.mark.parametrize("kw,needle", [
    (dict(taps=0), "taps"),
    (dict(dy=None), "dy is NULL"),
    (dict(dx=None), "dx is NULL"),
    (dict(dx_ld=1), "dx_ld"),
    (dict(dbias=AT + 2), "dbias is not aligned"),
    (dict(dfinal=AT + 2), "dfinal is not aligned"),
    (dict(dinitial=AT + 1), "dinitial is not aligned"),
    (dict(workspace=None), "workspace needs"),
    (dict(workspace_bytes=16), "workspace needs"),
    (dict(workspace=(1 << 20) + 16), "256-byte"),
])
def test_causal_conv_backward_refusals(mg, kw, needle):
    refused(lambda: conv_backward(mg, **kw), needle)


@pytest.mark.parametrize("kw,needle", [
    (dict(states=0), "states"),
    (dict(states=257), "states"),
    (dict(groups=0), "groups"),
    (dict(groups=3), "groups"),
    (dict(y=None), "y is NULL"),
    (dict(dt=None), "dt is NULL"),
    (dict(b=None), "b is NULL"),
    (dict(c=AT + 2), "c is not aligned"),
    (dict(c_ld=15), "c_ld"),
    (dict(z=AT, z_ld=2), "z_ld"),
    (dict(a=None), "a is NULL"),
    (dict(d=AT + 2), "d is not aligned"),
    (dict(dt_bias=AT + 2), "dt_bias is not aligned"),
    (dict(initial=AT + 2), "initial is not aligned"),
    (dict(final=AT + 2), "final is not aligned"),
    (dict(checkpoints=AT + 2), "checkpoints is not aligned"),
    (dict(steps=4096, seqs=1), "workspace needs"),
])
def test_selective_scan_refusals(mg, kw, needle):
    refused(lambda: scan(mg, **kw), needle)


@pytest.mark.parametrize("kw,needle", [
    (dict(states=300), "states"),
    (dict(groups=5), "groups"),
    (dict(dy=None), "dy is NULL"),
    (dict(dx=None), "dx is NULL"),
    (dict(ddt=None), "ddt is NULL"),
    (dict(db=AT + 2), "db is not aligned"),
    (dict(dc_ld=3), "dc_ld"),
    (dict(dz=AT), "dz without z"),
    (dict(z=AT), "dz is NULL"),
    (dict(steps=65), "checkpoints is NULL"),
    (dict(dd=AT + 1), "dd is not aligned"),
    (dict(ddt_bias=AT + 1), "ddt_bias is not aligned"),
    (dict(dinitial=AT + 1), "dinitial is not aligned"),
    (dict(workspace_bytes=16), "workspace needs"),
    (dict(workspace=(1 << 20) + 16), "256-byte"),
])
def test_selective_scan_backward_refusals(mg, kw, needle):
    refused(lambda: scan_backward(mg, **kw), needle)


def test_unknown_types_and_null_arguments(mg):
    L = mg.lib()
    from metalgym_amd import _capi

    for fn, args in ((L.mg_causal_conv, _capi.CausalConvArgs), (L.mg_causal_conv_backward, _capi.CausalConvBackwardArgs),
                     (L.mg_selective_scan, _capi.SelectiveScanArgs),
                     (L.mg_selective_scan_backward, _capi.SelectiveScanBackwardArgs)):
        assert fn(None, None) == -1
        assert fn(None, C.byref(args(steps=1, seqs=1, channels=8, type=3))) == -1 and b"type" in L.mg_last_error()
    assert L.mg_causal_conv_backward_workspace(1, 1, 8, 4, None) == -1
    assert L.mg_selective_scan_workspace(1, 1, 8, 16, None) == -1
    assert L.mg_selective_scan_backward_workspace(1, 1, 8, 16, 1, None) == -1


def test_no_sequences_are_nothing(mg):
    none = dict(x=None, weight=None, steps=4, seqs=0, channels=8, taps=4)
    mg.causal_conv(y=None, **none)
    mg.causal_conv_backward(dy=None, dx=None, **none)
    none = dict(x=None, dt=None, steps=4, seqs=0, channels=8, states=16, a=None, b=None, c=None)
    mg.selective_scan(y=None, **none)
    mg.selective_scan_backward(dy=None, dx=None, ddt=None, db=None, dc=None, **none)


def test_workspaces(mg):
    assert mg.selective_scan_workspace(1, 1, 128, 16) == 0
    assert mg.selective_scan_workspace(32, 4096, 256, 16) == 0  # enough sequences: nothing is split
    long = mg.selective_scan_workspace(16384, 1, 512, 64)
    assert 0 < long <= 1 << 28
    assert mg.selective_scan_backward_workspace(0, 0, 128, 16) == 0
    assert mg.causal_conv_backward_workspace(1 << 30, 1, 128, 4) <= 1 << 24
    with pytest.raises(CapiError):
        mg.selective_scan_backward_workspace(1, 1, 10, 16, 3)
    # groups make more blocks of channels and no more splits: one size serves them all
    for channels in (4, 96, 512, 2048):
        for groups in (2, 4):
            for steps in (1000, 16384):  # always split
                assert split_space(mg, steps, channels, groups) <= mg.selective_scan_workspace(steps, 2, channels, 16)


def split_space(mg, steps, channels, groups):
    """What the call itself asks for, from its refusal."""
    try:
        scan(mg, steps=steps, seqs=2, channels=channels, groups=groups, workspace_bytes=1, workspace=1 << 20)
    except CapiError as e:
        return int(str(e).split("needs ")[1].split()[0])
    raise AssertionError("not refused")
