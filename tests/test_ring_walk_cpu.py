"""How the norm's CTAs walk their rows through a ring of copies, and what they do
when a wait for a copy gave up (csrc/ring_walk.h), on the CPU: the header's own steps
against a model of the slots, for every row at which each of three threads can
give up, with every number of copies that land late.  No GPU: the model says
where a row would be read that is not there, a slot loaded too early, or a copy
still in flight at the end."""
import ctypes as C
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

MODEL = r"""
#include <string.h>
#include "ring_walk.h"
constexpr int kThreads = 3, kMost = 8, kNone = -1;
struct Cta {
    int slots, rows;           // rows of this CTA, numbered 0, 1, ...
    int row[kMost];            // what slot holds, or is to hold
    bool issued[kMost], landed[kMost];
    int phase[kMost];          // copies that have landed in the slot
    int passed[kThreads];      // barriers that a thread has passed
    bool flag;
    int wrong, loads, stopped;
    int late_row[kThreads];    // a thread's wait for this row gives up
};
struct Ring {
    Cta* c;
    int thread;
    uint32_t slots, rows, i = 0, parity = 0;
    bool draining = false;
    bool wait(uint32_t slot, uint32_t phase) {
        if ((c->phase[slot] & 1) != (int)phase) return true;   // the phase is over
        if (!c->issued[slot]) {                                // a wait for a copy that nobody issued
            if (!c->flag || draining) c->wrong |= 1;
            return false;
        }
        if (!draining && c->late_row[thread] == c->row[slot]) return false;   // (what the lead waits for at the end lands)
        c->landed[slot] = true;                                // it lands while this thread waits
        c->issued[slot] = false;
        c->phase[slot]++;
        return true;
    }
    void drain(uint32_t slot, uint32_t phase) {
        draining = true;
        wait(slot, phase);
    }
    void load(uint32_t slot, int n) {
        if (n >= (int)rows) return;
        if (c->issued[slot]) c->wrong |= 2;                    // two copies into one slot
        for (int t = 0; t < kThreads; t++)
            if (c->row[slot] != kNone && c->passed[t] <= c->row[slot]) c->wrong |= 4;   // somebody may still read it
        c->row[slot] = n;
        c->issued[slot] = true;
        c->landed[slot] = false;
        c->loads++;
    }
    bool lead() const { return thread == 0; }
    void fail() { c->flag = true; }
    bool failed() const { return c->flag; }
    void stop(int n) {
        if (c->stopped < 0) c->stopped = n < (int)rows ? n : (int)rows;
    }
    bool read(int row) const { return c->row[i] == row && c->landed[i]; }   // what the thread finds in its slot
};
// One walk.  late[t]: the row at which thread t's wait gives up (-1: none).  first: the thread that goes ahead of the
// others behind each barrier, as far as the next one.  Result: 0, or what went wrong.
extern "C" int run(int slots, int rows, const int* late, int first) {
    bool spoilt = false;
    Cta c;
    memset(&c, 0, sizeof c);
    c.slots = slots;
    c.rows = rows;
    c.stopped = -1;
    for (int k = 0; k < kMost; k++) c.row[k] = kNone;
    memcpy(c.late_row, late, sizeof c.late_row);
    Ring r[kThreads];
    for (int t = 0; t < kThreads; t++) {
        r[t].c = &c;
        r[t].thread = t;
        r[t].slots = slots;
        r[t].rows = rows;
    }
    for (int k = 0; k < slots && k < rows; k++) r[0].load(k, k);
    auto take = [&](int t, int row) {
        const bool before = c.flag;
        qrm::ring_wait(r[t]);
        if (!c.flag && !r[t].read(row)) c.wrong |= 8;          // nobody has said that something is wrong
        spoilt |= !before && c.flag;
    };
    for (int t = 0; t < kThreads; t++)
        if (rows) take((first + t) % kThreads, 0);
    for (int row = 0; row < rows; row++) {
        for (int t = 0; t < kThreads; t++) c.passed[t]++;      // the barrier
        bool lead_done = false;
        auto next = [&](int k) {
            if (k || !lead_done) qrm::ring_next(r[k], row + slots);
            lead_done |= k == 0;
        };
        for (int t = 0; t < kThreads; t++) {
            const int k = (first + t) % kThreads;
            next(k);
            // (one slot: the wait lasts until the lead, which has passed the same barrier, has issued the copy)
            if (row + 1 < rows && slots == 1) next(0);
            if (row + 1 < rows) take(k, row + 1);
        }
    }
    if (spoilt != c.flag) c.wrong |= 16;
    if (c.flag) {
        if (c.stopped != c.loads) c.wrong |= 32;               // what the lead drains by
        qrm::ring_drain(r[0], (uint32_t)c.stopped);
    } else if (c.loads != rows) {
        c.wrong |= 32;
    }
    for (int k = 0; k < slots; k++)
        if (c.issued[k]) c.wrong |= 64;                        // still in flight
    return c.wrong;
}
"""


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    d = tmp_path_factory.mktemp("walk")
    src, so = d / "model.cpp", d / "libmodel.so"
    src.write_text(MODEL)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC",
                    "-I", os.path.join(ROOT, "qauntrunner_b200", "csrc"), str(src), "-o", str(so)], check=True)
    return C.CDLL(str(so)).run


@pytest.mark.parametrize("slots", [1, 2, 3, 8])
def test_rows_are_right_or_said_to_be_wrong_and_no_copy_is_left(model, slots):
    for rows in (0, 1, 2, 3, 7, 9, 20):
        at = [-1] + list(range(rows))
        for lead in at:
            for second in at:
                for third in at if rows < 9 else (-1, 0, rows - 1):
                    late = (C.c_int * 3)(lead, second, third)
                    for first in range(3):
                        assert model(slots, rows, late, first) == 0, (rows, lead, second, third, first)


def test_no_wait_of_the_norm_goes_unanswered():
    """Every wait for a copy in norm.cuh is ring_walk.h's, whose answer counts, but for the drain's."""
    with open(os.path.join(ROOT, "qauntrunner_b200", "csrc", "norm.cuh")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    assert [m for m in re.findall(r"[^;}]*[^_]mbar_wait\([^;]*;", text) if "void drain(" not in m] == []
    assert text.count("if (a.slots) ring_wait(ring);") == 2 and text.count("if (a.slots && ring.failed()) spoil") == 2
