"""srhpm_page_free and srhpm_page_compact from several host threads at once (tests/cpp/test_page_threads.cpp): threads of a program
of its own, as Python's take turns at a lock."""
import os

import pytest

from test_z_cpp_host import CPP, run


@pytest.mark.gpu
def test_pools_of_different_sizes():
    run([os.path.join(CPP, "test_page_threads")])
