"""The paged cache in the C++ host API (neural-network-engine_amd/host/nne.hpp) through
its test program tests/cpp/test_paged_api.cpp.  Built by __graft_entry__.build()
(make -C tests/cpp)."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "tests", "cpp", "build", "test_paged_api")


def run(args, timeout, count):
    if not os.path.exists(BIN):
        pytest.fail("C++ host-API tests not built: %s is missing (run __graft_entry__.build())" % BIN)
    res = subprocess.run([BIN] + args, capture_output=True, text=True, timeout=timeout)
    print(res.stdout)
    print(res.stderr)
    assert res.returncode == 0, res.stdout
    assert re.search(r"^0 of %d tests failed$" % count, res.stdout, re.M)


def test_paged_api_cpu_only_parts():
    run(["--cpu"], 60, 1)


@pytest.mark.gpu
def test_paged_api_on_gpu():
    run([], 100, 6)
