"""qrm_sort_tokens where its shared memory is just below and above what a kernel
has without asking: 48 KB, the kernel's own 128 bytes of it included.  Each case is a
process of its own, with counts of experts in ascending order, because asking once
for more holds for the rest of a process."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import sys, torch
import qauntrunner_b200 as Q
from tests import fp8_plain as F
T, k, *counts = (int(a) for a in sys.argv[1:])
for experts in counts:
    g = torch.Generator()
    g.manual_seed(experts)
    idx = torch.randint(-1, experts, (T, k), generator=g, dtype=torch.int32)
    perm, pos = (torch.empty(T * k, dtype=torch.int32).cuda() for _ in range(2))
    off = torch.empty(experts + 1, dtype=torch.int32).cuda()
    Q.sort_tokens(idx.cuda(), T, k, experts, perm, pos, off)
    assert (perm.tolist(), pos.tolist(), off.tolist()) == F.order(idx, 0, experts)
"""


# (2 + warps) experts 4 bytes: 8 warps up to 256 assignments, 8 more for each 256 more, 32 from 769 on; more than
# 4096 assignments take the cluster.  49024 bytes are the most that need no asking.
@pytest.mark.parametrize("T,k,experts", [
    (100, 8, [360, 361, 362]),    # 34 experts 4: 48960, 49096, 49232
    (1000, 8, [360, 361, 362]),   # the same in the cluster
    (75, 8, [471, 472, 473]),     # 26 experts 4: 48984, 49088, 49192
    (50, 8, [680, 681]),          # 18 experts 4: 48960, 49032
    (50, 8, [682, 683])])         # 49104, 49176
def test_sort_tokens_around_the_default_limit(T, k, experts):
    r = subprocess.run([sys.executable, "-c", CHILD, str(T), str(k), *map(str, experts)], cwd=ROOT, capture_output=True,
                       text=True, timeout=300, env={**os.environ, "PYTHONPATH": ROOT})
    assert r.returncode == 0, r.stderr[-2000:]
