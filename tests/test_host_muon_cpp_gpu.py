"""Runs tests/cpp/muon_tests.cpp (what the Muon optimizer of the C++ host layer takes and refuses) on the GPU."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_host_muon():
    from neuzephyr_b200 import build as B
    B.build()
    exe = B.build_program(os.path.join(ROOT, "tests", "cpp", "muon_tests.cpp"),
                          os.path.join(ROOT, "tests", "cpp", "bin", "muon_tests"), "../../../neuzephyr_b200")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    print(r.stdout[-6000:])
    print(r.stderr[-2000:])
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr[-2000:]
    assert " 0 failures" in r.stdout
