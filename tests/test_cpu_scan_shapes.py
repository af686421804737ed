"""Which selective scans take two channels a quad of lanes, from the dispatch's own rule compiled for the host
(tests/native/scan_shapes.hip): not those that leave most lanes without a channel, and those that
tests/test_gpu_selective_scan_pairs.py is there for."""
import os
import subprocess

import pytest

from test_gpu_selective_scan_pairs import SHAPES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.fixture(scope="module")
def shapes(tmp_path_factory):
    at = str(tmp_path_factory.mktemp("scan_shapes"))
    obj, exe = os.path.join(at, "scan_shapes.o"), os.path.join(at, "scan_shapes")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "--offload-host-only", "-O1", "-std=c++17", "-Wno-unused-function",
                    "-I", os.path.join(ROOT, "include"), "-c", os.path.join(ROOT, "tests", "native", "scan_shapes.hip"),
                    "-o", obj], check=True)
    subprocess.run([HIPCC, obj, "-o", exe], check=True)

    def run(asked):
        text = "".join("%d %d %d %d %d %d\n" % a for a in asked)
        out = subprocess.run([exe], input=text, capture_output=True, text=True, timeout=120, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]

    return run


def test_two_channels_a_quad_fill_their_lanes(shapes):
    asked = [(steps, seqs, per * groups, states, groups, backward) for steps in (9, 32, 400) for seqs in (1, 300, 5000)
             for per in list(range(1, 400, 7)) + [64, 128, 192, 256] for groups in (1, 2, 4) for states in (13, 16)
             for backward in (0, 1)]
    pairs = 0
    for (steps, seqs, channels, states, groups, backward), (wide, apiece, splits) in zip(asked, shapes(asked)):
        per = channels // groups
        if wide == 2:
            pairs += 1
            assert splits == 1 and apiece == -(-per // 128)
            # lanes, in channels, of workgroups of two channels a quad and of one
            assert 128 * -(-per // 128) <= (64 * -(-per // 64)) * (4 / 3 if backward else 1), (per, backward)
    assert pairs > 100
    assert [s[0] for s in shapes([(32, 4096, 64, 16, 1, 0), (32, 4096, 256, 16, 4, 1), (32, 4096, 256, 16, 1, 0)])] == [1, 1, 2]


def test_shapes_of_the_gpu_tests(shapes):
    for *shape, ways in SHAPES:
        got = shapes([(*shape, 0), (*shape, 1)])
        assert ["%d" % s[0] for s in got] == list(ways), shape
