"""What a warp that gives up waits for (csrc/kernels/int4_ring.h), on the CPU: rings of copies beside a model of their barriers."""
import os
import shutil
import subprocess

import pytest

from carbon_engine_b200.csrc import build

MODEL = r"""
#include "int4_ring.h"
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>

// A barrier as the hardware has it: a wait for a parity returns when the barrier's present phase is of the other one.
struct Barrier {
    int ended = 0;
    bool wait(unsigned parity) const { return (ended & 1u) != parity; }
};
static int failures = 0;
#define CHECK(what) do { if (!(what)) { std::printf("line %d: %s (seed %u)\n", __LINE__, #what, seed); ++failures; } } while (0)
"""

PASSED_OVER = MODEL + r"""
// Tiles first .. last of ``tiles`` are copied; every copy lands at once but for those behind tile ``late``, which land when they are waited for.
template <int N> void run(unsigned seed) {
    std::srand(seed);
    const int tiles = 1 + std::rand() % 20, first = std::rand() % tiles, last = first + std::rand() % (tiles - first), late = std::rand() % (tiles + 1);
    const bool behind_the_fetch = std::rand() % 2;          // gives up for another reason, with the next tile asked for already
    Barrier bars[N];
    std::set<int> under_way;                                // tiles
    auto asked = [&](int i) { return i >= first && i <= last; };
    auto fetch = [&](int i) {
        if (!asked(i)) return;
        if (i < late) ++bars[i % N].ended;
        else under_way.insert(i);
    };
    I4Ring<N> ring;
    auto wait = [&](int place, unsigned parity) { return bars[place].wait(parity); };
    for (int i = 0; i < N; ++i) fetch(i);
    int next = 0;
    bool ok = true;
    for (int i = 0; i < tiles && ok; ++i) {
        if (asked(i)) ok = ring.landed(i, wait);
        if (!ok) break;
        fetch(i + N);
        next = i + 1;
        if (behind_the_fetch && i >= late) ok = false;
    }
    if (ok) { CHECK(under_way.empty()); return; }
    // each wait is for a copy that has not landed; it lands, and a second wait sees it
    ring.drain(next, asked, [&](int place, unsigned parity) {
        CHECK(!bars[place].wait(parity));
        int tile = -1;
        for (int t : under_way) if (t % N == place) { CHECK(tile < 0); tile = t; }
        CHECK(tile >= 0);
        if (tile >= 0) { under_way.erase(tile); ++bars[place].ended; }
        CHECK(bars[place].wait(parity));
        return true;
    });
    CHECK(under_way.empty());
}
int main() {
    for (unsigned seed = 0; seed < 20000; ++seed) { run<3>(seed); run<1>(seed); run<4>(seed); }
    return failures ? 1 : 0;
}
"""


def check(tmp_path, text):
    cxx = os.environ.get("CXX") or shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    source, program = tmp_path / "model.cpp", tmp_path / "model"
    source.write_text(text)
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-I", build.KERNEL_DIR, str(source), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout[:2000]


def test_a_ring_whose_tiles_may_be_passed_over(tmp_path):
    check(tmp_path, PASSED_OVER)


IN_TURN = MODEL + r"""
// ``issued`` copies, of which each landed or has not, in a ring whose places are taken again once the copy before has landed.
template <int N> void run(unsigned seed) {
    std::srand(seed);
    const int issued = std::rand() % 14, landed_at_least = issued > N ? issued - N : 0;
    Barrier bars[N];
    std::set<int> under_way;
    for (int i = 0; i < issued; ++i) {
        if (i < landed_at_least || std::rand() % 2) ++bars[i % N].ended;
        else under_way.insert(i);
    }
    i4_drain<N>(issued, [&](int place, unsigned parity) {
        int tile = -1;
        for (int t : under_way) if (t % N == place) { CHECK(tile < 0); tile = t; }
        CHECK(bars[place].wait(parity) == (tile < 0));      // at once for what landed, not before for what did not
        if (tile >= 0) { under_way.erase(tile); ++bars[place].ended; }
        CHECK(bars[place].wait(parity));
    });
    CHECK(under_way.empty());
}
int main() {
    for (unsigned seed = 0; seed < 20000; ++seed) { run<3>(seed); run<4>(seed); run<1>(seed); }
    return failures ? 1 : 0;
}
"""


def test_a_ring_that_tiles_take_in_turn(tmp_path):
    check(tmp_path, IN_TURN)
