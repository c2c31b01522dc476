"""Which loads a warp that gives up waits for (csrc/ring.h), on the CPU (tests/cpp/test_ring.cpp): no GPU is made to give up."""
import os

from test_z_cpp_host import CPP, run


def test_loads_in_flight_of_a_warp_that_gives_up():
    run([os.path.join(CPP, "test_ring")])
