"""Every bounded wait of the 4-bit products says when it gave up, read off the
source: it is not something that a GPU test can bring about."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qauntrunner_b200", "csrc")


def statements(name):
    with open(os.path.join(CSRC, name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    return [" ".join(s.split()) for s in re.split(r"[;{}]", text)]


def test_no_answer_of_a_wait_is_dropped():
    """Waits are conditions.  Those with (void) run where a wait gave up before, and the error is raised."""
    waits = [s for s in statements("fp4.cuh") if re.search(r"\b(mbar_wait|bar_wait|bar_wait_both|bar_wait_cluster)\(", s)]
    waits = [s for s in waits if not s.startswith("__device__")]   # definitions
    assert len(waits) >= 10
    dropped = [s for s in waits if not re.search(r"(if|while) ?\(+!?|return |= |\(void\)", s.split("bar_wait")[0])]
    assert dropped == []
    assert sorted(s for s in waits if "(void)" in s) == ["(void)mbar_wait(&full[slot], parity)",
                                                        "if (lane == 0) (void)mbar_wait(left_bar, 0u)"]


def test_a_split_cta_whose_mmas_did_not_end_writes_nothing():
    s = statements("fp4.cuh")
    i = next(i for i, line in enumerate(s) if line == "if (!mbar_wait(done_bar, 0u))")
    assert s[i + 1:i + 3] == ["*abort_flag = 1", "atomicOr(p.err, (int)ERR_TIMEOUT)"]
    assert any("items = *abort_flag ? 0 :" in line for line in s[i:])
