"""The ring of whole rows in shared memory, followed on the host: what it requests, waits for and gives up, with barriers and copies in the
place of the device's that check every use. Copies land whenever a wait asks for them, late ones a wait later, and one may never be
seen to land within its wait."""
import os
import subprocess

import pytest

from conftest import ROOT

HARNESS = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "rows_ring.cuh"

#define REQUIRE(x) do { if (!(x)) { std::printf("%s: slots %u rows %u lost %d\n", #x, S, mine, lost); std::exit(1); } } while (0)

template <uint32_t S>
void follow(uint32_t mine, int lost) {
    struct Slot { int row = -1; bool flying = false, read = true; uint32_t phase = 0; };  // phase: of the copy that flies, else of the next
    std::vector<Slot> slots(S);
    std::vector<int> asked(mine), reduced(mine), finished(mine);
    int given_up = -1;
    uint32_t at = 0;
    b200::run_ring<S>(
        mine,
        [&](uint32_t n, uint32_t s) {
            REQUIRE(n < mine && s == n % S && !asked[n]++);
            REQUIRE(!slots[s].flying && slots[s].read);   // nothing lands there, and what lay there has been read
            REQUIRE(given_up < 0 && (lost < 0 || static_cast<int>(n) < lost + static_cast<int>(S)));  // nothing is requested once a wait ran out
            slots[s] = {static_cast<int>(n), true, false, slots[s].phase};
        },
        [&](uint32_t s, uint32_t phase) {
            REQUIRE(s < S && slots[s].row >= 0 && phase == (slots[s].row / S & 1));  // a copy that was requested, its own phase
            if (!slots[s].flying) return true;
            if (slots[s].row == lost && at == static_cast<uint32_t>(lost)) {
                at = mine;  // the limit ran out; the copy lands later
                return false;
            }
            slots[s].flying = false;
            return true;
        },
        [&](uint32_t n, uint32_t s, bool there) {
            REQUIRE(slots[s].row == static_cast<int>(n) && there == !slots[s].flying && !reduced[n]++);
            slots[s].read = true;
            at = there ? n + 1 : at;
            return there;
        },
        [&](uint32_t n) { REQUIRE(reduced[n] && !finished[n]++ && static_cast<int>(n) != lost); },
        [&](uint32_t n) {
            REQUIRE(given_up < 0 && static_cast<int>(n) == lost);
            given_up = n;
        });
    for (auto& s : slots) REQUIRE(!s.flying);  // no copy is left when the block ends
    REQUIRE(given_up == (lost < static_cast<int>(mine) ? lost : -1));
    for (uint32_t n = 0; n < mine; ++n) REQUIRE(finished[n] == (lost < 0 || static_cast<int>(n) < lost));
}

int main() {
    for (uint32_t mine = 0; mine < 12; ++mine)
        for (int lost = -1; lost < static_cast<int>(mine); ++lost) follow<1>(mine, lost), follow<2>(mine, lost), follow<3>(mine, lost);
    return 0;
}
"""


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    d = tmp_path_factory.mktemp("ring")
    (d / "ring.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-x", "c++", "-I", os.path.join(ROOT, "llm-infer_b200", "csrc"), str(d / "ring.cpp"),
                    "-o", str(d / "ring")], check=True)
    return str(d / "ring")


def test_a_wait_that_runs_out_ends_the_ring(harness):
    """Nothing is requested behind it, what was requested is waited for, and the row is neither finished nor read again."""
    run = subprocess.run([harness], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


def test_every_wait_of_rows_reports_to_the_callers_word(pkg, built_lib):
    """The status word's place in the arguments, packed and mirrored."""
    from llm_infer_b200 import int8
    a = pkg.binding.AttnRowsI8Args.from_buffer_copy(int8.ROWS_ARGS.pack(*range(1, 12), 13, 1.0, 15, 16, 0x1234560))
    assert a.status == 0x1234560 and a.delta_dtype == 16
