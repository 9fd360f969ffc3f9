"""How a warp waits for the copies it has asked for before its CTA leaves (csrc/paged.cuh, drain_copies), on the host: a ring of barriers whose
copies land late, or never."""
import importlib
import os
import subprocess

import pytest

from conftest import ROOT

build = importlib.import_module("ameva-compute_b200.build")

SOURCE = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "paged.cuh"
// drain ISSUED STAGES LATE LOST: copy i lands LATE polls after the wait has begun (the last one first), copy LOST never
int main(int, char** v) {
    const uint32_t issued = atoi(v[1]), stages = atoi(v[2]), late = atoi(v[3]), lost = atoi(v[4]);
    uint32_t polls = 0;
    std::vector<bool> waited(issued, false);
    auto landed = [&](uint32_t i) { return i + stages < issued || (i != lost && polls > late * (issued - i)); };   // (a stage is asked again once it is empty)
    auto arrived = [&](uint32_t stage, uint32_t parity) {
        ++polls;
        uint32_t phase = 0, last = 0;   // completed phases of the stage's barrier; its last copy
        for (uint32_t i = stage; i < issued; i += stages, ++last)
            if (landed(i)) ++phase;
        const bool done = (phase & 1u) != parity;
        if (done) waited[stage + (last - 1u) * stages] = true;
        return done;
    };
    const bool ok = amv::paged::drain_copies(issued, stages, arrived);
    uint32_t missing = 0;   // copies nobody waited for, or that have not landed
    for (uint32_t i = 0; i < issued; ++i) missing += i + stages >= issued && !(waited[i] && landed(i));
    printf("%d %u %u\n", (int)ok, missing, polls);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    at = tmp_path_factory.mktemp("drain")
    (at / "drain.cu").write_text(SOURCE)
    flags = [f for f in build.NVCC_FLAGS if f != "-O3"]
    subprocess.run([build._nvcc(), *flags, "-I", os.path.join(ROOT, "ameva-compute_b200", "csrc"), "-o", str(at / "drain"),
                    str(at / "drain.cu")], check=True, capture_output=True)

    def run(*args):
        return [int(x) for x in subprocess.run([str(at / "drain"), *map(str, args)], check=True, capture_output=True, text=True).stdout.split()]

    return run


@pytest.mark.parametrize("issued,stages", [(0, 3), (1, 3), (2, 3), (3, 3), (4, 3), (11, 3), (1, 1), (2, 1), (7, 1), (9, 8), (64, 5)])
def test_every_copy_in_flight_is_waited_for(program, issued, stages):
    for late in (0, 1, 40):
        ok, missing, polls = program(issued, stages, late, issued)
        assert (ok, missing) == (1, 0) and polls <= late * (stages + 1) + 2 * stages


def test_a_copy_that_never_lands_ends_the_wait(program):
    ok, missing, polls = program(7, 3, 2, 5)
    assert ok == 0 and missing >= 1 and polls <= (1 << 14) + 20
