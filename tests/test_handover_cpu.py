"""What the CTAs of a pair hand to each other, read off the kernels' source.

An arrive on the other CTA's barrier that names no scope releases to the
arriving CTA's own threads.  It may say that an accumulator has been read (the
loads from tensor memory are complete, and a tcgen05 fence is before it); memory
that was written goes with a release of cluster scope, such as the completion of
a copy that was issued behind it.  Nothing on a GPU fails reliably where these
are missing, so this looks for the calls."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qauntrunner_b200", "csrc")


def source(name):
    """A file's statements, without comments, one to a line."""
    with open(os.path.join(CSRC, name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    return [line.strip() for line in text.replace("{", "{\n").replace(";", ";\n").split("\n") if line.strip()]


@pytest.mark.parametrize("name", ["fp4.cuh", "fp8.cuh"])
def test_arrives_without_a_scope_follow_reads_of_tensor_memory(name):
    lines = source(name)
    calls = [i for i, line in enumerate(lines) if "bar_arrive_cluster(" in line]
    assert calls
    for i in calls:
        before = lines[i - 2:i]
        assert before == ["tc_fence_before();", "__syncwarp();"], (lines[i], before)


def test_scales_of_the_second_cta_come_ahead_of_its_copies():
    """fp4_pair_kernel: the thread that issues a stage's copies waits for its scales, and the MMAs' thread acquires
    what the copies' completion releases."""
    lines = source("fp4.cuh")
    first_copy = next(i for i, line in enumerate(lines) if line.startswith("tma_pair_2d(st, &x_map"))
    wait = next(line for line in reversed(lines[:first_copy]) if "bar_wait" in line)
    assert "bar_wait(x_full0" in wait
    mma = next(i for i, line in enumerate(lines) if line.startswith("umma_mxf4<2>(d,"))
    wait = next(line for line in reversed(lines[:mma]) if "bar_wait" in line)
    assert "bar_wait_cluster(full0" in wait
    shared = "\n".join(source("umma_sync.cuh"))
    assert "mbarrier.try_wait.parity.acquire.cluster" in shared.split("bool bar_try_cluster(")[1].split("return")[0]
