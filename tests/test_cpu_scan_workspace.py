"""The selective scan's gradient for more rows than any memory has parts of dB and dC for (lengths may leave most of
them out) is refused: the workspace's size must not wrap around in 64 bits."""
import pytest

from test_cpu_operator_checks import refused
from test_cpu_rollout_checks import scan_backward

SIZES = [(1 << 30, 1 << 30, 65536, 256, 1), (1 << 30, 512, 65536, 256, 1), (1 << 30, 1 << 24, 4096, 16, 2),
         (1 << 30, 1 << 9, 65536, 256, 4), (1 << 28, 1 << 12, 512, 20, 1)]


@pytest.mark.parametrize("steps,seqs,channels,states,groups", SIZES)
def test_sizes_past_any_memory(mg, steps, seqs, channels, states, groups):
    refused(lambda: mg.selective_scan_backward_workspace(steps, seqs, channels, states, groups), "2^48")
    refused(lambda: scan_backward(mg, steps=steps, seqs=seqs, channels=channels, states=states, groups=groups,
                                  workspace_bytes=(1 << 64) - 1, checkpoints=1 << 20), "2^48")


@pytest.mark.parametrize("steps,seqs,channels,states", [(1 << 20, 64, 65536, 16), (1 << 30, 1, 65536, 16), (4096, 8192, 2048, 64)])
def test_sizes_grow_with_the_rows(mg, steps, seqs, channels, states):
    one = mg.selective_scan_backward_workspace(steps, seqs, channels, states)
    two = mg.selective_scan_backward_workspace(steps, 2 * seqs, channels, states) if seqs > 1 else 2 * one
    assert one >= steps * seqs * 2 * states * 4 and 1.9 * one <= two <= 2.1 * one


def test_one_workgroup_a_group_keeps_no_parts(mg):
    assert mg.selective_scan_backward_workspace(1 << 30, 1 << 30, 16, 16, 1) < 1 << 30
