"""How a pair of CTAs leaves when a wait gave up (csrc/pair_drain.h), on the CPU:
the header's own loop against a model of the barriers, for every point at which
one CTA, or both, can have stopped issuing and every order in which the copies
land.  No GPU: the model says where a wait would not end and which copies would
still be in flight."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

MODEL = r"""
#include <string.h>
#include "pair_drain.h"
// Barriers of `stages` slots, one arrival and 2 shares of bytes a phase.  A phase is over when its arrival came and
// the shares expected have landed; shares may land before they are expected.
constexpr int kMost = 8;
struct Model {
    int stages, phase[kMost], pending[kMost], bytes[kMost];   // bytes: expected less landed
    int in_flight[kMost][2];                                  // shares of each CTA not landed yet, at a slot
    int stuck, wrong;
    void close(int s) {
        if (pending[s] == 0 && bytes[s] == 0) {
            phase[s]++;
            pending[s] = 1;
        }
    }
    void arrive(int s, int shares) {
        if (pending[s] == 0) wrong = 1;   // a second arrival in one phase
        pending[s] = 0;
        bytes[s] += shares;
        close(s);
    }
    void land(int s, int cta) {
        in_flight[s][cta] = 0;
        bytes[s]--;
        close(s);
    }
    // what the loop does
    void expect(uint32_t s) { arrive((int)s, 1); }
    void complete(uint32_t s) {
        bytes[s]--;
        close((int)s);
    }
    void wait(uint32_t s, uint32_t parity) {
        // copies in flight land sooner or later; the wait is over when the phase is
        for (int c = 0; c < 2 && (uint32_t)(phase[s] & 1) == parity; c++)
            if (in_flight[s][c]) land((int)s, c);
        if ((uint32_t)(phase[s] & 1) == parity) stuck = 1;
    }
};
// Both CTAs issue stages, at most `stages` apart; the copies of all but the last `stages` have landed.  early: the copies in flight that have landed before the drain, as bits.
// Result: 1 a wait that does not end, 2 copies left in flight, 4 the model was misused.
extern "C" int run(int mine, int peer, int stages, unsigned early, int old_way) {
    Model m;
    memset(&m, 0, sizeof m);
    m.stages = stages;
    for (int i = 0; i < kMost; i++) m.pending[i] = 1;
    const int most = mine > peer ? mine : peer;
    for (int j = 0; j < most; j++) {
        const int s = j % stages;
        if (j < peer) m.in_flight[s][1] = 1;
        if (j < mine) {
            m.in_flight[s][0] = 1;
            m.arrive(s, 2);
        }
        const bool last = j >= most - stages;   // the others were waited for before their slot was used again
        for (int c = 0; c < 2; c++)
            if (m.in_flight[s][c] && (!last || (early >> (2 * s + c) & 1))) m.land(s, c);
        if (!last && m.phase[s] != j / stages + 1) return 4;
    }
    if (old_way) {   // the first CTA waits for what it issued itself
        for (int j = mine > stages ? mine - stages : 0; j < mine; j++) m.wait(j % stages, (j / stages) & 1);
    } else {
        qrm::drain_pair(mine, peer, stages, m);
    }
    int left = 0;
    for (int s = 0; s < stages; s++) left |= m.in_flight[s][0] | m.in_flight[s][1];
    return (m.stuck ? 1 : 0) | (left ? 2 : 0) | (m.wrong ? 4 : 0);
}
"""


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    d = tmp_path_factory.mktemp("drain")
    src, so = d / "model.cpp", d / "libmodel.so"
    src.write_text(MODEL)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC",
                    "-I", os.path.join(ROOT, "qauntrunner_b200", "csrc"), str(src), "-o", str(so)], check=True)
    return C.CDLL(str(so)).run


def counts(stages):
    """What two producers can have issued: at most `stages` apart, the slower one's stages waited for."""
    return [(a, b) for a in range(0, 3 * stages + 2) for b in range(max(0, a - stages), a + stages + 1)]


@pytest.mark.parametrize("stages", [1, 2, 3])
def test_every_copy_has_landed_and_every_wait_ends(model, stages):
    for mine, peer in counts(stages):
        for early in range(1 << (2 * stages)):
            assert model(mine, peer, stages, early, 0) == 0, (mine, peer, early)


def test_six_stages(model):
    for mine, peer in counts(6):
        for early in (0, 0xFFF, 0x555, 0xAAA, 0x0F3):
            assert model(mine, peer, 6, early, 0) == 0, (mine, peer, early)


def test_the_model_sees_what_counting_one_cta_misses(model):
    """The first CTA waiting for its own issues only: stuck where the other issued fewer, copies left in flight where
    it issued more."""
    assert model(4, 4, 2, 0, 1) == 0
    assert model(4, 3, 2, 0, 1) & 1
    assert model(3, 4, 2, 0, 1) & 2
