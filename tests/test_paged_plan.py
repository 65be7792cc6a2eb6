"""CPU test of the work plans of paged attention (csrc/paged_plan.h), as a
program of its own."""
import os
import subprocess

import pytest

from conftest import ROOT


def test_paged_plans():
    exe = os.path.join(ROOT, "tests", "cpp", "test_paged_plan")
    if not os.path.exists(exe):
        pytest.fail("tests/cpp/test_paged_plan is missing: run __graft_entry__.build()")
    done = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout + done.stderr
