"""The paged-attention kernel's plan on the CPU (csrc/paged_plan.cpp), through
tests/cpp/test_paged_plan.cpp: tiles, parts, their order and records of a seeded sweep
of batches, and the divisions the kernels make.  Built by __graft_entry__.build()
(make -C tests/cpp)."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "tests", "cpp", "build", "test_paged_plan")


def test_paged_plan_invariants():
    if not os.path.exists(BIN):
        pytest.fail("planner test not built: %s is missing (run __graft_entry__.build())" % BIN)
    res = subprocess.run([BIN], capture_output=True, text=True, timeout=120)
    print(res.stdout)
    assert res.returncode == 0, res.stdout
    assert re.search(r"^0 of \d+ checks failed$", res.stdout, re.M)
    m = re.search(r"^plans: (\d+) split, (\d+) whole, (\d+) merged by a kernel, (\d+) in 16-row and "
                  r"(\d+) in 32-row tiles, (\d+) places folded$", res.stdout, re.M)
    assert m and all(int(x) > 0 for x in m.groups()), "sweep must reach every outcome"
