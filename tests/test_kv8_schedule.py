"""When the prompt kernel over caches of 8 bits reads and writes LDS (bitnet-rs_amd/csrc/kv8_schedule.hpp): no wave may overwrite, between two barriers, what another wave still reads.  The walk
through the table is compiled for the host; schedules that are wrong have to be found by it.  No GPU."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bitnet-rs_amd", "csrc")

PROGRAM = """
#include "kv8_schedule.hpp"
#include <cstdio>
using bitnet_hip::Kv8Schedule;
int main() {
    const Kv8Schedule kept = bitnet_hip::kKv8Schedule;
    const Kv8Schedule all[] = {
        kept,
        {{2, 2}, 2, 1, 1, 2},  // keys 32 .. 63 of the tile after next, where those of this tile are read
        {{1, 1}, 2, 1, 1, 2},  // keys 0 .. 31 of the next tile, where they are read
        {{2, 1}, 2, 0, 1, 2},  // values of the tile at hand
        {{2, 1}, 2, 2, 1, 2},  // of the tile after next, over those that are read
        {{2, 1}, 2, 1, 0, 2},  // factors where they are read
        {{2, 1}, 2, 1, 2, 2},  // .. and over those that are read
        {{2, 1}, 2, 1, 1, 1},  // scales in one place for tiles two apart
        {{2, 1}, 1, 1, 1, 2},  // scales where they are read
    };
    for (const Kv8Schedule &s : all) std::printf("%d", (int)bitnet_hip::kv8_schedule_holds(s));
}
"""


def test_nothing_is_overwritten_while_it_is_read(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    src, exe = tmp_path / "schedule.cpp", tmp_path / "schedule"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(src), "-o", str(exe)], check=True, timeout=120)
    got = subprocess.run([str(exe)], capture_output=True, text=True, check=True, timeout=30).stdout
    assert got == "1" + "0" * 8
