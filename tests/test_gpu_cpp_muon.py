"""PPOModel::useMuon and useAdam from C++."""
import math
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu

BUILD = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "build")


def test_a_training_loop_with_muon_runs():
    path = os.path.join(BUILD, "cartpole_muon")
    assert os.path.exists(path), f"{path} missing: run __graft_entry__.build()"
    p = subprocess.run([path], capture_output=True, text=True, timeout=100)
    print(p.stdout, p.stderr)
    assert p.returncode == 0
    lines = [line.split() for line in p.stdout.splitlines() if line.startswith("iter")]
    assert [int(w[1]) for w in lines] == [4, 9, 14, 19]
    assert all(math.isfinite(float(w[3])) and math.isfinite(float(w[5])) for w in lines)
