"""How a pair of CTAs of the 4-bit product leaves when a wait gave up
(csrc/pair_drain.h), on the CPU: as test_fp8_give_up.py, but with stages of
different numbers of bytes, which tiles with and without a few rows behind them
have.  Each CTA keeps the share of the stage that it issued last in each slot."""
import ctypes as C
import os
import subprocess

import pytest

from tests.test_fp8_give_up import ROOT, counts

MODEL = r"""
#include <string.h>
#include "pair_drain.h"
// Barriers of `stages` slots, one arrival a phase, which expects both CTAs' shares of its stage; a phase is over when it
// came and the bytes expected have landed.
constexpr int kMost = 8;
struct Model {
    int stages, phase[kMost], pending[kMost], bytes[kMost];   // bytes: expected less landed
    int flying[kMost][2];                                     // bytes of each CTA's copy not landed yet, at a slot
    int last[2][kMost];                                       // share of the stage that a CTA issued last in a slot
    int stuck, wrong;
    void close(int s) {
        if (pending[s] == 0 && bytes[s] == 0) {
            phase[s]++;
            pending[s] = 1;
        }
    }
    void arrive(int s, int expected) {
        if (pending[s] == 0) wrong = 1;   // a second arrival in one phase
        pending[s] = 0;
        bytes[s] += expected;
        close(s);
    }
    void land(int s, int cta) {
        bytes[s] -= flying[s][cta];
        flying[s][cta] = 0;
        close(s);
    }
    // what the loop does, with what the kernel knows: its own shares, and the other CTA's by reading its memory
    void expect(uint32_t s) { arrive((int)s, last[1][s]); }
    void complete(uint32_t s) {
        bytes[s] -= last[0][s];
        close((int)s);
    }
    void wait(uint32_t s, uint32_t parity) {
        for (int c = 0; c < 2 && (uint32_t)(phase[s] & 1) == parity; c++)
            if (flying[s][c]) land((int)s, c);
        if ((uint32_t)(phase[s] & 1) == parity) stuck = 1;
    }
};
// Both CTAs issue stages, at most `stages` apart, of share[j] bytes each; the copies of all but the last `stages` have
// landed, and of those the ones in `early`.  equal: the drain takes every stage to be as large as the first (what it
// must not do).  Result: 1 a wait that does not end, 2 copies left in flight, 4 the model was misused, 8 bytes left over.
extern "C" int run(int mine, int peer, int stages, unsigned early, const int* share, int equal) {
    Model m;
    memset(&m, 0, sizeof m);
    m.stages = stages;
    for (int i = 0; i < kMost; i++) m.pending[i] = 1;
    const int most = mine > peer ? mine : peer;
    for (int j = 0; j < most; j++) {
        const int s = j % stages;
        if (j < peer) m.flying[s][1] = m.last[1][s] = share[j];
        if (j < mine) {
            m.flying[s][0] = m.last[0][s] = share[j];
            m.arrive(s, 2 * share[j]);
        }
        const bool late = j >= most - stages;   // the others were waited for before their slot was used again
        for (int c = 0; c < 2; c++)
            if (m.flying[s][c] && (!late || (early >> (2 * s + c) & 1))) m.land(s, c);
        if (!late && m.phase[s] != j / stages + 1) return 4;
    }
    if (equal)
        for (int s = 0; s < stages; s++) m.last[0][s] = m.last[1][s] = share[0];
    qrm::drain_pair(mine, peer, stages, m);
    int left = 0, over = 0;
    for (int s = 0; s < stages; s++) {
        left |= m.flying[s][0] | m.flying[s][1];
        over |= m.bytes[s];
    }
    return (m.stuck ? 1 : 0) | (left ? 2 : 0) | (m.wrong ? 4 : 0) | (over ? 8 : 0);
}
"""


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    d = tmp_path_factory.mktemp("drain4")
    src, so = d / "model.cpp", d / "libmodel.so"
    src.write_text(MODEL)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC",
                    "-I", os.path.join(ROOT, "qauntrunner_b200", "csrc"), str(src), "-o", str(so)], check=True)
    return C.CDLL(str(so)).run


def shares(n, first, steps):
    """n stages of tiles of `steps` stages each, every second tile with rows behind it."""
    return (C.c_int * max(n, 1))(*[7 if (j // steps + first) % 2 else 5 for j in range(n)])


@pytest.mark.parametrize("stages", [1, 2, 3])
@pytest.mark.parametrize("steps", [1, 2, 3])
def test_every_copy_has_landed_and_every_wait_ends(model, stages, steps):
    for mine, peer in counts(stages):
        for first in (0, 1):
            s = shares(max(mine, peer), first, steps)
            for early in range(1 << (2 * stages)):
                assert model(mine, peer, stages, early, s, 0) == 0, (mine, peer, first, early)


@pytest.mark.parametrize("stages", [4, 5])
def test_the_rings_of_the_kernel(model, stages):
    for mine, peer in counts(stages):
        for steps in (1, 3, 8):
            s = shares(max(mine, peer), 1, steps)
            for early in (0, 0x3FF, 0x155, 0x2AA, 0x0F3):
                assert model(mine, peer, stages, early, s, 0) == 0, (mine, peer, steps, early)


def test_the_model_sees_what_equal_shares_miss(model):
    s = shares(4, 0, 1)   # 5 7 5 7
    assert model(4, 4, 2, 0, s, 1) == 0
    assert model(4, 3, 2, 0, s, 1) & 1
    assert model(3, 4, 2, 0, s, 1)
