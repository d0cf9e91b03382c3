"""The drain of a ring of copies (csrc/ring.cuh), compiled for the host: after
a wait has run out, every copy in flight is waited for again, that one too."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hexa-lang_b200", "csrc")
MAIN = """
#include <cstdio>
#include <cstdlib>
#include "ring.cuh"
int main(int, char** v) {
    auto wait = [](int slot, int parity) { std::printf("%d %d\\n", slot, parity); };
    if (std::atoi(v[1]) == 2) ring_drain<2>(std::atoi(v[2]), std::atoi(v[3]), wait);
    else ring_drain<5>(std::atoi(v[2]), std::atoi(v[3]), wait);
}
"""


@pytest.fixture(scope="module")
def drain(tmp_path_factory):
    d = tmp_path_factory.mktemp("ring")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(d / "main.cpp"), "-o", str(d / "main")],
                   check=True)

    def run(slots, n_out, n_in):
        out = subprocess.run([str(d / "main"), str(slots), str(n_out), str(n_in)], check=True, capture_output=True)
        return [tuple(map(int, line.split())) for line in out.stdout.decode().splitlines()]

    return run


@pytest.mark.parametrize("slots", [2, 5])
def test_every_copy_in_flight_is_waited_for(drain, slots):
    for n_out in range(0, 4 * slots + 1):
        for in_flight in range(0, slots + 1):
            want = [(n % slots, n // slots % 2) for n in range(n_out, n_out + in_flight)]
            assert drain(slots, n_out, n_out + in_flight) == want
