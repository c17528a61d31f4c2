"""The 4-bit cache's kernels at the largest lengths the library takes, on the CPU execution model (tests/emu/cache_limits.cpp): every count of slots
stays inside its 32 bits (an addition that leaves them ends the program), and the far end is what it has to be."""
import subprocess

import pytest


@pytest.mark.parametrize("what", ["weights", "select", "keep", "columns"])
def test_near_2_to_31_slots(emu_sources, what):
    r = subprocess.run([emu_sources.build_cache_limits(), what], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
